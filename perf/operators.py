"""Cases of the state space block's operators: the causal convolution, the
selective scan, the norms around a block and the clipping of gradients, each in
its plain form (elementary torch operations in 32 bits, rounded once at the
end), through the library's entry points, and in 64 bits from its definition.

Formulas (row t of a sequence; rows past the sequence's length are not read and
come out as zero):
  conv  p_t = bias + sum_j w_j x_{t-W+1+j}, y = silu(p); rows before 0 are the state's
  scan  e = softplus(dt + dt_bias); h_tn = exp(e_t A_n) h_{t-1,n} + e_t x_t B_tn;
        y_t = sum_n C_tn h_tn + D x_t
  norm  r = x + s o (rms(y o silu(z)) o w_post); n = rms(r) o w_pre
  clip  g <- g min(1, max_norm / (|g| + 1e-6)), |g| the 2-norm over all tensors
"""
from __future__ import annotations

import ctypes
import math

import torch

own = False

EPS = 1e-6  # RMSNorm epsilon of the model
CONV_W = 4  # taps of the short convolution


def listed():
    return [
        # The convolution in a training step of the byte model's width: forward, backward.
        dict(name="conv_b16t1024d512", op="conv", B=16, T=1024, D=512, W=4, dtype="f32"),
        # The convolution over ragged bf16 prompts that go on from a state, forward only (serving).
        dict(name="conv_ragged_b8t1000d1000", op="conv_prompt", B=8, T=1000, D=1000, W=4, dtype="bf16"),
        # The scan in a training step of the byte model's width: forward, backward.
        dict(name="ssm_b16t1024d512n16", op="ssm", B=16, T=1024, D=512, N=16, G=1, dtype="f32"),
        # The scan in a training step on long bf16 sequences of a wide block, the largest case.
        dict(name="ssm_b8t4096d2048n16", op="ssm", B=8, T=4096, D=2048, N=16, G=1, dtype="bf16"),
        # Ragged f32 prompts with sizes that fill no tile and two groups of B and C (serving).
        dict(name="ssm_ragged_b4t1000d1000n12", op="ssm_prompt", B=4, T=1000, D=1000, N=12, G=2, dtype="f32"),
        # One long bf16 prompt: few channels, a long time axis (serving).
        dict(name="ssm_b1t16384d1024n16", op="ssm_prompt", B=1, T=16384, D=1024, N=16, G=1, dtype="bf16"),
        # One token of one sequence: convolution and scan on their states, where latency counts.
        dict(name="step_n1d512", op="step", n=1, D=512, N=16, G=1, W=4, dtype="f32"),
        # One token for 512 concurrent sequences of a wide block: the states read and written once.
        dict(name="step_n512d2048", op="step", n=512, D=2048, N=16, G=1, W=4, dtype="bf16"),
        # Norms, gate and residual around a block in a training step: forward, backward.
        dict(name="norm_t16384d512", op="norm", rows=16384, D=512, dtype="f32"),
        # The same for one token of 64 sequences, forward only (serving).
        dict(name="norm_n64d2048", op="norm_fwd", rows=64, D=2048, dtype="bf16"),
        # Clipping the gradients of the 143M-parameter byte model (82 tensors).
        dict(name="clip_model", op="clip", layers=8, D=512, ff=1024, E=16, V=256, dtype="f32"),
        # Clipping the gradients of one narrow block: many small tensors, odd sizes.
        dict(name="clip_block", op="clip", layers=2, D=100, ff=200, E=4, V=256, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["conv", "conv_prompt", "ssm", "ssm", "ssm_prompt", "ssm_prompt", "step", "step", "norm", "norm_fwd",
                     "clip"])
    dtype = rng.choice(["f32", "bf16"])
    if op in ("conv", "conv_prompt"):
        while True:
            c = dict(B=_log(rng, 1, 32), T=_log(rng, 1, 4096), D=_log(rng, 64, 2048), W=rng.choice([2, 3, 4, 4]))
            if c["B"] * c["T"] * c["D"] <= 8 * 4096 * 2048:
                break
    elif op in ("ssm", "ssm_prompt"):
        while True:
            G = rng.choice([1, 1, 1, 2, 4])
            c = dict(B=_log(rng, 1, 32), T=_log(rng, 1, 4096 if op == "ssm" else 16384), D=G * _log(rng, 16, 2048 // G),
                     N=rng.choice([4, 8, 12, 16, 16, 16, 32]), G=G)
            if c["B"] * c["T"] * c["D"] * c["N"] <= 4 * 4096 * 2048 * 16:
                break
    elif op == "step":
        G = rng.choice([1, 1, 2])
        c = dict(n=_log(rng, 1, 512), D=G * _log(rng, 64, 2048 // G), N=rng.choice([8, 12, 16, 16, 32]), G=G,
                 W=rng.choice([2, 3, 4, 4]))
    elif op == "norm":
        c = dict(rows=_log(rng, 64, 16384), D=_log(rng, 64, 2048))
    elif op == "norm_fwd":
        c = dict(rows=_log(rng, 1, 16384), D=_log(rng, 64, 2048))
    else:
        D = _log(rng, 64, 512)
        c = dict(layers=rng.choice([1, 2, 4, 8]), D=D, ff=2 * D, E=rng.choice([1, 4, 8]), V=256)
    return dict(op=op, dtype=dtype, **c)


# ------------------------------------------------------------------- inputs


def _type(case):
    return torch.bfloat16 if case["dtype"] == "bf16" else torch.float32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape, scale=1.0, offset=0.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g, device="cuda") * scale + offset).to(dtype)


def _lens(g, case):
    """Lengths of ragged prompts: from a quarter of T to T, one of them T."""
    if not case["op"].endswith("_prompt"):
        return None
    B, T = case["B"], case["T"]
    lens = torch.randint(max(1, T // 4), T + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    lens[0] = T
    return lens


def _conv_inputs(g, n, T, D, W, ty):
    """x as a projection of normalised rows gives it, taps of about 1/W."""
    return dict(x=_normal(g, n * T, D, dtype=ty), w=_normal(g, W, D, scale=1.0 / math.sqrt(W)),
                bias=_normal(g, D, scale=0.1), state=_normal(g, n, W - 1, D).to(ty).float())


def _ssm_inputs(g, n, T, D, N, G, ty):
    """Steps e of 0.001 to 0.1 around which dt moves, A near -1 .. -N, B and C of unit
    size, as in a trained block; dt, B and C lie in one wider matrix, as one projection
    writes them."""
    u = torch.rand(D, generator=g, device="cuda")
    e = torch.exp(u * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    n_idx = torch.arange(1, N + 1, device="cuda", dtype=torch.float32)[:, None]
    wide = _normal(g, n * T, D + 2 * G * N, dtype=ty)
    return dict(x=_normal(g, n * T, D, dtype=ty), wide=wide, dt=wide[:, :D], Bm=wide[:, D:D + G * N], Cm=wide[:, D + G * N:],
                dt_bias=torch.log(torch.expm1(e)), A=-n_idx * torch.exp(_normal(g, N, D, scale=0.1)),
                Dk=_normal(g, D, scale=0.1, offset=1.0), h=_normal(g, n, N, D, scale=0.1))


def _block_tensors(case):
    """(rows, cols) of the parameters: embedding, head, then per layer the delta block's and the experts'."""
    L, D, ff, E, V = (case[k] for k in ("layers", "D", "ff", "E", "V"))
    H = max(1, D // 64)
    layer = [(D, 3 * D), (1, 3 * D), (D, 2 * H), (1, 2 * H), (D, D), (1, D), (D, E * ff), (1, E * ff), (E * ff, D), (1, D)]
    return [(V, D), (D, V)] + layer * L


def prepare(case, seed):
    g, ty, op = _gen(seed), _type(case), case["op"]
    s = dict(case=case)
    if op in ("conv", "conv_prompt"):
        s.update(_conv_inputs(g, case["B"], case["T"], case["D"], case["W"], ty))
        s["lens"] = _lens(g, case)
        s["dy"] = _normal(g, *s["x"].shape, dtype=ty) if op == "conv" else None
    elif op in ("ssm", "ssm_prompt"):
        s.update(_ssm_inputs(g, case["B"], case["T"], case["D"], case["N"], case["G"], ty))
        s["lens"] = _lens(g, case)
        s["dy"] = _normal(g, *s["x"].shape, dtype=ty) if op == "ssm" else None
    elif op == "step":
        s["conv"] = _conv_inputs(g, case["n"], 1, case["D"], case["W"], ty)
        s["ssm"] = _ssm_inputs(g, case["n"], 1, case["D"], case["N"], case["G"], ty)
    elif op in ("norm", "norm_fwd"):
        rows, D = case["rows"], case["D"]
        for k in ("x", "y", "z"):
            s[k] = _normal(g, rows, D, dtype=ty)
        s["w_post"], s["w_pre"] = _normal(g, D, scale=0.1, offset=1.0), _normal(g, D, scale=0.1, offset=1.0)
        s["scale"] = _normal(g, D, scale=0.05, offset=0.3)
        if op == "norm":
            s["dr"], s["dn"] = _normal(g, rows, D, dtype=ty), _normal(g, rows, D, dtype=ty)
    else:
        # one buffer with every tensor at a multiple of 16 bytes; gradients of different sizes by tensor
        at, where = 0, []
        for r, c in _block_tensors(case):
            where.append((at, r * c))
            at += -(-r * c // 8) * 8
        s["where"], s["src"], s["dst"] = where, torch.zeros(at, device="cuda", dtype=ty), torch.zeros(at, device="cuda", dtype=ty)
        for o, n in where:
            s["src"][o:o + n] = _normal(g, n, scale=0.01 * (1 + (o // 8) % 7), dtype=ty)
        s["max_norm"] = 1.0
    return s


# ------------------------------------------------------------- plain forms


def _valid(lens, B, T):
    """(B, T, 1) truth of the rows that belong to their sequence, or None if all do."""
    if lens is None:
        return None
    return torch.arange(T, device=lens.device)[None, :, None] < lens[:, None, None]


def _last(cat, lens, T, k):
    """Rows len .. len+k-1 of (B, k+T, D): the k inputs that end at each sequence's length."""
    if lens is None:
        return cat[:, T:].contiguous()
    idx = lens.long()[:, None] + torch.arange(k, device=lens.device)[None]
    return torch.gather(cat, 1, idx[:, :, None].expand(-1, -1, cat.shape[2])).contiguous()


def _plain_conv(s, step=False):
    c = s["case"]
    B, T, D, W = (c["n"], 1, c["D"], c["W"]) if step else (c["B"], c["T"], c["D"], c["W"])
    ty, lens, prompt = _type(c), s.get("lens"), step or c["op"] == "conv_prompt"
    x = s["x"].float().view(B, T, D)
    ok = _valid(lens, B, T)
    if ok is not None:
        x = torch.where(ok, x, 0.0)
    before = s["state"] if prompt else torch.zeros(B, W - 1, D, device=x.device)
    cat = torch.cat([before, x], 1)
    p = s["bias"] + sum(s["w"][j] * cat[:, j:j + T] for j in range(W))
    sg = torch.sigmoid(p)
    y = p * sg
    if ok is not None:
        y = torch.where(ok, y, 0.0)
    out = dict(y=y.to(ty).view(B * T, D))
    if prompt:
        out["state"] = _last(cat, lens, T, W - 1)
    if s.get("dy") is not None:
        gr = s["dy"].float().view(B, T, D) * (sg * (1 + p * (1 - sg)))
        tail = torch.cat([gr, torch.zeros(B, W - 1, D, device=x.device)], 1)
        dx = sum(s["w"][j] * tail[:, W - 1 - j:W - 1 - j + T] for j in range(W))
        out.update(dx=dx.to(ty).view(B * T, D), dw=torch.stack([(gr * cat[:, j:j + T]).sum((0, 1)) for j in range(W)]),
                   db=gr.sum((0, 1)))
    return out


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, h_{-1} = 0, by doubling (a and b are overwritten)."""
    T, s = a.shape[1], 1
    while s < T:
        b[:, s:] = b[:, s:] + a[:, s:] * b[:, :-s]
        a[:, s:] = a[:, s:] * a[:, :-s]
        s *= 2
    return b


def _plain_ssm(s, step=False):
    c = s["case"]
    B, T = (c["n"], 1) if step else (c["B"], c["T"])
    D, N, G, ty, lens = c["D"], c["N"], c["G"], _type(c), s.get("lens")
    prompt = step or c["op"] == "ssm_prompt"
    x, dt = s["x"].float().view(B, T, D), s["dt"].float().reshape(B, T, D)
    wide = lambda m: m.float().reshape(B, T, G, N).repeat_interleave(D // G, 2)  # noqa: E731  (B, T, D, N)
    Bm, Cm, A = s["Bm"], s["Cm"], s["A"].t()
    ok = _valid(lens, B, T)
    v = dt + s["dt_bias"]
    e = torch.where(v > 20, v, torch.log1p(torch.exp(v)))
    if ok is not None:
        e, x = torch.where(ok, e, 0.0), torch.where(ok, x, 0.0)
    a = torch.exp(e[..., None] * A)
    b = (e * x)[..., None] * wide(Bm)
    if prompt:
        b[:, 0] = b[:, 0] + a[:, 0] * s["h"].transpose(1, 2)
    train = s.get("dy") is not None
    h = _scan(a.clone() if train else a, b)
    y = (h * wide(Cm)).sum(-1) + s["Dk"] * x
    if ok is not None:
        y = torch.where(ok, y, 0.0)
    out = dict(y=y.to(ty).view(B * T, D))
    if prompt:
        out["h"] = h[:, -1].transpose(1, 2).contiguous()
    if not train:
        return out
    dy = s["dy"].float().view(B, T, D)
    grp = lambda m: m.view(B, T, G, D // G, N).sum(3).to(ty).view(B * T, G * N)  # noqa: E731
    out["dC"] = grp(h * dy[..., None])
    nxt = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    gr = _scan(nxt.flip(1), (dy[..., None] * wide(Cm)).flip(1)).flip(1)
    del nxt
    out["dB"] = grp(gr * (e * x)[..., None])
    gB = (gr * wide(Bm)).sum(-1)
    h[:, 1:] = h[:, :-1].clone()
    h[:, 0] = 0.0
    p = gr * a * h
    del gr, a, h
    de = x * gB + (p * A).sum(-1)
    ddt = de * torch.sigmoid(v)
    out.update(dx=(e * gB + s["Dk"] * dy).to(ty).view(B * T, D), ddt=ddt.to(ty).view(B * T, D), ddt_bias=ddt.sum((0, 1)),
               dA=(p * e[..., None]).sum((0, 1)).t().contiguous(), dD=(dy * x).sum((0, 1)))
    return out


def _plain_norm(s):
    c = s["case"]
    ty = _type(c)
    x, y, z = s["x"].float(), s["y"].float(), s["z"].float()
    sg = torch.sigmoid(z)
    sz = z * sg
    u = y * sz
    i1 = torch.rsqrt((u * u).mean(1, keepdim=True) + EPS)
    uh = u * i1
    p = uh * s["w_post"]
    r = x + s["scale"] * p
    i2 = torch.rsqrt((r * r).mean(1, keepdim=True) + EPS)
    rh = r * i2
    out = dict(r=r.to(ty), n=(rh * s["w_pre"]).to(ty))
    if "dn" not in s:
        return out
    dn = s["dn"].float()
    dnh = dn * s["w_pre"]
    dr = s["dr"].float() + i2 * (dnh - rh * (dnh * rh).mean(1, keepdim=True))
    dp = dr * s["scale"]
    duh = dp * s["w_post"]
    du = i1 * (duh - uh * (duh * uh).mean(1, keepdim=True))
    out.update(dx=dr.to(ty), dy=(du * sz).to(ty), dz=(du * y * (sg * (1 + z * (1 - sg)))).to(ty), dw_post=(dp * uh).sum(0),
               dscale=(dr * p).sum(0), dw_pre=(dn * rh).sum(0))
    return out


def _plain_clip(s):
    g = s["src"].float()
    norm = torch.sqrt((g * g).sum())
    coef = torch.clamp(s["max_norm"] / (norm + 1e-6), max=1.0)
    s["dst"].copy_(g * coef)
    return dict(norm=norm, grads=s["dst"])


def _plain_step(s):
    c = s["case"]
    conv, ssm = dict(s["conv"], case=c), dict(s["ssm"], case=c)
    a = _plain_conv(conv, step=True)
    s["conv"]["state"].copy_(a["state"])
    b = _plain_ssm(ssm, step=True)
    s["ssm"]["h"].copy_(b["h"])
    return dict(c=a["y"], conv_state=s["conv"]["state"], y=b["y"], h=s["ssm"]["h"])


# -------------------------------------------------------- the library's calls


def _ptr(t):
    return None if t is None else t.data_ptr()


def _calls(s):
    """The calls of one pass with their arguments and the outputs that they write, made on a
    state's first pass and kept with it, as a program keeps its buffers."""
    from asca_amd import _lib
    from asca_amd.gpu import gpu

    if gpu() is None:
        raise RuntimeError("no GPU backend")
    c, p = s["case"], _ptr
    op, ty = c["op"], 1 if c["dtype"] == "bf16" else 0
    like, f32 = torch.empty_like, lambda *n: torch.empty(*n, device="cuda")
    calls, out = [], {}

    def add(name, *args):
        calls.append((name, args))

    if op in ("conv", "conv_prompt"):
        B, T, D, W = c["B"], c["T"], c["D"], c["W"]
        prompt = op == "conv_prompt"
        out["y"] = like(s["x"])
        if prompt:
            out["state"] = like(s["state"])
        add("asca_conv_fwd", p(s["x"]), D, p(s["w"]), p(s["bias"]), p(s["state"] if prompt else None), p(s["lens"]), p(out["y"]),
            D, p(out.get("state")), B, T, D, W, 1, ty, None)
        if op == "conv":
            out.update(dx=like(s["x"]), dw=f32(W, D), db=f32(D))
            add("asca_conv_bwd", p(s["x"]), D, p(s["w"]), p(s["bias"]), None, None, p(s["dy"]), D, None, p(out["dx"]), D,
                p(out["dw"]), p(out["db"]), None, B, T, D, W, 1, ty, None)
    elif op in ("ssm", "ssm_prompt"):
        B, T, D, N, G = (c[k] for k in ("B", "T", "D", "N", "G"))
        ld, prompt = s["wide"].stride(0), op == "ssm_prompt"
        out["y"] = like(s["x"])
        ws = None
        if prompt:
            out["h"] = like(s["h"])
        else:
            n = ctypes.c_size_t()
            _lib.call("asca_ssm_ws_bytes", B, T, D, N, ctypes.byref(n))
            ws = s["ws"] = torch.empty(n.value, dtype=torch.uint8, device="cuda")
        ins = (p(s["x"]), D, p(s["dt"]), ld, p(s["dt_bias"]), p(s["A"]), p(s["Bm"]), ld, p(s["Cm"]), ld, p(s["Dk"]))
        add("asca_ssm_fwd", *ins, p(s["h"] if prompt else None), p(s["lens"]), p(out["y"]), D, p(out.get("h")), p(ws), B, T, D, N,
            G, 1, ty, None)
        if op == "ssm":
            wide = out["wide"] = like(s["wide"])
            out.update(dx=like(s["x"]), ddt_bias=f32(D), dA=f32(N, D), dD=f32(D))
            dt, dB, dC = wide[:, :D], wide[:, D:D + G * N], wide[:, D + G * N:]
            add("asca_ssm_bwd", *ins, None, p(s["dy"]), D, None, p(ws), p(out["dx"]), D, p(dt), ld, p(out["ddt_bias"]),
                p(out["dA"]), p(dB), ld, p(dC), ld, p(out["dD"]), None, B, T, D, N, G, 1, ty, None)
            del out["wide"]
            out.update(ddt=dt, dB=dB, dC=dC)
    elif op == "step":
        n, D, N, G, W = (c[k] for k in ("n", "D", "N", "G", "W"))
        a, b = s["conv"], s["ssm"]
        ld = b["wide"].stride(0)
        out.update(c=like(a["x"]), conv_state=a["state"], y=like(b["x"]), h=b["h"])
        add("asca_conv_step", p(a["state"]), p(a["x"]), D, p(a["w"]), p(a["bias"]), p(out["c"]), D, n, D, W, 1, ty, None)
        add("asca_ssm_step", p(b["h"]), p(b["x"]), D, p(b["dt"]), ld, p(b["dt_bias"]), p(b["A"]), p(b["Bm"]), ld, p(b["Cm"]), ld,
            p(b["Dk"]), p(out["y"]), D, n, D, N, G, 1, ty, None)
    elif op in ("norm", "norm_fwd"):
        rows, D = c["rows"], c["D"]
        out.update(r=like(s["x"]), n=like(s["x"]))
        ins = (p(s["x"]), D, p(s["y"]), D, p(s["z"]), D, p(s["w_post"]), p(s["scale"]), p(s["w_pre"]))
        add("asca_block_norm_fwd", *ins, p(out["r"]), D, p(out["n"]), D, rows, D, EPS, ty, None)
        if op == "norm":
            out.update(dx=like(s["x"]), dy=like(s["x"]), dz=like(s["x"]), dw_post=f32(D), dscale=f32(D), dw_pre=f32(D))
            add("asca_block_norm_bwd", *ins, p(s["dr"]), D, p(s["dn"]), D, p(out["dx"]), D, p(out["dy"]), D, p(out["dz"]), D,
                p(out["dw_post"]), p(out["dscale"]), p(out["dw_pre"]), rows, D, EPS, ty, None)
    else:
        k, size = len(s["where"]), s["src"].element_size()
        at = lambda t: (ctypes.c_void_p * k)(*[t.data_ptr() + o * size for o, _ in s["where"]])  # noqa: E731
        plan = ctypes.c_void_p()
        _lib.call("asca_grads_create", at(s["src"]), at(s["dst"]), (ctypes.c_uint64 * k)(*[n for _, n in s["where"]]), k, ty,
                  ctypes.byref(plan))
        s["plan"] = _Plan(plan)
        stat = f32(2)
        out.update(norm=stat[0], grads=s["dst"])
        add("asca_grads_clip", plan, s["max_norm"], p(stat), None)
    return calls, out


class _Plan:
    """A clipping plan, destroyed with the state that holds it."""

    def __init__(self, handle):
        self.handle = handle

    def __del__(self):
        from asca_amd import _lib

        _lib.load().asca_grads_destroy(self.handle)


def run(state):
    if own:
        from asca_amd import _lib

        if "calls" not in state:
            state["calls"] = _calls(state)
        calls, out = state["calls"]
        for name, args in calls:
            _lib.call(name, *args)
        return dict(out)
    op = state["case"]["op"]
    if op in ("conv", "conv_prompt"):
        return _plain_conv(state)
    if op in ("ssm", "ssm_prompt"):
        return _plain_ssm(state)
    if op == "step":
        return _plain_step(state)
    if op in ("norm", "norm_fwd"):
        return _plain_norm(state)
    return _plain_clip(state)


# ------------------------------------------------------------------- work


def work(case):
    op, e = case["op"], 2 if case["dtype"] == "bf16" else 4
    if op in ("conv", "conv_prompt"):
        n = case["B"] * case["T"] * case["D"]
        if op == "conv_prompt":
            return dict(bytes=2 * e * n, flops=n * (2 * case["W"] + 4))
        return dict(bytes=5 * e * n, flops=n * (6 * case["W"] + 12))
    if op in ("ssm", "ssm_prompt"):
        n, bc = case["B"] * case["T"] * case["D"], 2 * case["B"] * case["T"] * case["G"] * case["N"]
        if op == "ssm_prompt":
            return dict(bytes=e * (3 * n + bc), flops=7 * n * case["N"])
        return dict(bytes=e * (8 * n + 3 * bc), flops=23 * n * case["N"])
    if op == "step":
        n = case["n"] * case["D"]
        return dict(bytes=8 * n * (case["N"] + case["W"] - 1) + 5 * e * n, flops=n * (7 * case["N"] + 2 * case["W"]))
    if op in ("norm", "norm_fwd"):
        n = case["rows"] * case["D"]
        return dict(bytes=(13 if op == "norm" else 5) * e * n, flops=(45 if op == "norm" else 15) * n)
    n = sum(r * c for r, c in _block_tensors(case))
    return dict(bytes=2 * e * n, flops=3 * n)


# ------------------------------------------------------------ 64-bit values


def _d(t):
    return t.double()


def _exact_conv(s, B, T, D, W, lens, state, dy):
    x = _d(s["x"]).view(B, T, D)
    n = [T] * B if lens is None else lens.tolist()
    w, bias = _d(s["w"]), _d(s["bias"])
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    last = torch.zeros(B, W - 1, D, dtype=torch.float64, device=x.device)
    dw, db = torch.zeros_like(w), torch.zeros_like(bias)
    for b in range(B):
        rows = torch.cat([_d(state[b]) if state is not None else torch.zeros(W - 1, D, dtype=torch.float64, device=x.device),
                          x[b, :n[b]]])
        p = bias.expand(n[b], D).clone()
        for j in range(W):
            p += rows[j:j + n[b]] * w[j]
        y[b, :n[b]] = p / (1 + torch.exp(-p))
        last[b] = rows[n[b]:]
        if dy is not None:
            q = 1 / (1 + torch.exp(-p))
            gr = _d(dy).view(B, T, D)[b] * (q + p * q * (1 - q))
            db += gr.sum(0)
            for j in range(W):
                dw[j] += (gr * rows[j:j + n[b]]).sum(0)
                k = W - 1 - j  # x_t meets w_j in the output of row t + k
                if k < T:
                    dx[b, :T - k] += w[j] * gr[k:]
    return y.view(B * T, D), last, dx.view(B * T, D), dw, db


def _exact_ssm(s, B, T, D, N, G, lens, h0, dy):
    """The recurrence, row after row; states as (B, N, D)."""
    x, v = _d(s["x"]).view(B, T, D), _d(s["dt"]).reshape(B, T, D) + _d(s["dt_bias"])
    e = torch.logaddexp(v, torch.zeros_like(v))
    Bm, Cm, A, Dk = _d(s["Bm"]).reshape(B, T, G, N), _d(s["Cm"]).reshape(B, T, G, N), _d(s["A"]), _d(s["Dk"])
    spread = lambda m: m.transpose(1, 2).repeat_interleave(D // G, 2)  # noqa: E731  (B, G, N) -> (B, N, D)
    h = torch.zeros(B, N, D, dtype=torch.float64, device=x.device) if h0 is None else _d(h0)
    y, hist = torch.zeros_like(x), []
    for t in range(T):
        new = torch.exp(e[:, t, None] * A) * h + (e[:, t] * x[:, t])[:, None] * spread(Bm[:, t])
        out = (new * spread(Cm[:, t])).sum(1) + Dk * x[:, t]
        if lens is not None:
            ok = (lens > t)[:, None]
            new, out = torch.where(ok[..., None], new, h), torch.where(ok, out, 0.0)
        if dy is not None:
            hist.append(h.float())  # rounded to 32 bits once for room: 3e-8 of its share of a gradient
        h, y[:, t] = new, out
    if dy is None:
        return dict(y=y.view(B * T, D), h=h)
    dy = _d(dy).view(B, T, D)
    dx, ddt, dB, dC = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(Bm), torch.zeros_like(Cm)
    dA, carry = torch.zeros_like(A), torch.zeros_like(h)
    part = lambda m: m.view(B, N, G, D // G).sum(3).transpose(1, 2)  # noqa: E731  (B, N, D) -> (B, G, N)
    for t in reversed(range(T)):
        et, xt, bt = e[:, t, None], x[:, t, None], spread(Bm[:, t])
        prev = hist.pop().double()
        a = torch.exp(et * A)
        dC[:, t] = part((a * prev + et * xt * bt) * dy[:, t, None])
        gr = carry + spread(Cm[:, t]) * dy[:, t, None]
        dB[:, t] = part(gr * et * xt)
        gb = (gr * bt).sum(1)
        carry = gr * a
        p = carry * prev
        dx[:, t] = e[:, t] * gb + Dk * dy[:, t]
        ddt[:, t] = (x[:, t] * gb + (p * A).sum(1)) / (1 + torch.exp(-v[:, t]))
        dA += (p * et).sum(0)
    r = B * T
    return dict(y=y.view(r, D), dx=dx.view(r, D), ddt=ddt.view(r, D), dB=dB.view(r, G * N), dC=dC.view(r, G * N), dA=dA,
                dD=(dy * x).sum((0, 1)), ddt_bias=ddt.sum((0, 1)))


def _exact_norm(s):
    x, y, z, wo, sc, wi = (_d(s[k]) for k in ("x", "y", "z", "w_post", "scale", "w_pre"))
    rows, D = x.shape
    q = 1 / (1 + torch.exp(-z))
    u = y * z * q
    m1 = ((u ** 2).sum(1, keepdim=True) / D + EPS) ** 0.5
    r = x + sc * wo * u / m1
    m2 = ((r ** 2).sum(1, keepdim=True) / D + EPS) ** 0.5
    out = dict(r=r, n=wi * r / m2)
    if "dn" in s:
        dn, dr = _d(s["dn"]), _d(s["dr"])
        k = dn * wi
        dr = dr + k / m2 - r * (k * r).sum(1, keepdim=True) / (D * m2 ** 3)
        k = dr * sc * wo
        du = k / m1 - u * (k * u).sum(1, keepdim=True) / (D * m1 ** 3)
        out.update(dx=dr, dy=du * z * q, dz=du * y * (q + z * q * (1 - q)), dw_post=(dr * sc * u / m1).sum(0),
                   dscale=(dr * wo * u / m1).sum(0), dw_pre=(dn * r / m2).sum(0))
    return out


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op in ("conv", "conv_prompt"):
        prompt = op == "conv_prompt"
        y, last, dx, dw, db = _exact_conv(s, case["B"], case["T"], case["D"], case["W"], s["lens"],
                                          s["state"] if prompt else None, s["dy"])
        return dict(y=y, state=last) if prompt else dict(y=y, dx=dx, dw=dw, db=db)
    if op in ("ssm", "ssm_prompt"):
        return _exact_ssm(s, case["B"], case["T"], case["D"], case["N"], case["G"], s["lens"],
                          s["h"] if op == "ssm_prompt" else None, s["dy"])
    if op == "step":
        n, D, W = case["n"], case["D"], case["W"]
        c, last, *_ = _exact_conv(s["conv"], n, 1, D, W, None, s["conv"]["state"], None)
        o = _exact_ssm(s["ssm"], n, 1, D, case["N"], case["G"], None, s["ssm"]["h"], None)
        return dict(c=c, conv_state=last, y=o["y"], h=o["h"])
    if op in ("norm", "norm_fwd"):
        return _exact_norm(s)
    g = _d(s["src"])
    norm = float((g * g).sum()) ** 0.5
    return dict(norm=torch.tensor(norm, dtype=torch.float64, device=g.device), grads=g * min(1.0, s["max_norm"] / (norm + 1e-6)))
