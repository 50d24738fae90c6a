"""The operators of a gated-recurrence block, case by case: the element-wise gated linear recurrence over time
(`chunk_hgrn`, `fused_recurrent_hgrn`), the root-mean-square norm with the residual's addition and an 8-bit output
(`rms_norm`, `rms_norm_quant`), and the product with bias, activation and residual in its epilogue (`linear`,
`linear_fp8`).

`run` computes a case in plain torch operations where `own` is false, and through the package's entry points where it is
true. `exact` gives the same results from the definitions, in 64 bits."""
import math
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3_MAX = 448.0
LARGEST = 262144 * 2048  # elements of the largest activation


def listed():
    return [
        # one decode step of 256 sequences: one token each, the state kept in 32 bits
        dict(name="hgrn_step", op="hgrn", B=256, T=1, D=2048, dtype="bf16", sequences=0, state=True, train=False),
        # the smallest training step: two short sequences in full precision, a carried state
        dict(name="hgrn_small_fp32", op="hgrn", B=2, T=512, D=256, dtype="fp32", sequences=0, state=True, train=True),
        # an ordinary training step: 8 x 4096 tokens, 2048 channels
        dict(name="hgrn_train", op="hgrn", B=8, T=4096, D=2048, dtype="bf16", sequences=0, state=False, train=True),
        # packed documents of 256 to 8192 tokens, each with a state of its own
        dict(name="hgrn_packed", op="hgrn", B=1, T=0, D=2048, dtype="bf16", sequences=64, shortest=256, longest=8192, lengths_seed=0,
             state=True, train=True),
        # reading one very long document: few channels side by side, a long axis
        dict(name="hgrn_long", op="hgrn", B=1, T=262144, D=2048, dtype="bf16", sequences=0, state=True, train=False),
        # one decode step of 256 tokens in front of an 8-bit product
        dict(name="norm_step_fp8", op="norm", rows=256, N=2048, dtype="bf16", residual="same", quant=True, train=False),
        # the norm of an ordinary training step, with the residual stream handed on
        dict(name="norm_train", op="norm", rows=32768, N=2048, dtype="bf16", residual="same", quant=False, train=True),
        # odd sizes in full precision, no residual
        dict(name="norm_odd_fp32", op="norm", rows=2047, N=1111, dtype="fp32", residual="none", quant=False, train=True),
        # a projection in a decode step of 256 tokens, onto the residual stream
        dict(name="linear_step", op="linear", M=256, K=2048, N=2048, dtype="bf16", activation="none", bias=False, residual=True, train=False),
        # a projection in an ordinary training step, with everything its epilogue can hold
        dict(name="linear_train", op="linear", M=32768, K=2048, N=2048, dtype="bf16", activation="silu", bias=True, residual=True, train=True),
        # ragged sizes in half precision: no side a multiple of a tile, rows that start off a 16-byte boundary
        dict(name="linear_ragged_fp16", op="linear", M=777, K=1001, N=515, dtype="fp16", activation="logsigmoid", bias=True, residual=False,
             train=True),
        # 8-bit tokens times 8-bit weights while reading a prompt
        dict(name="linear_fp8", op="linear_fp8", M=16384, K=2048, N=8192, dtype="bf16", activation="silu", bias=True, residual=False,
             train=False),
    ]


def _between(rng, low, high):
    """A whole number, spread over its logarithm; one in three is rounded to a multiple of 64 where that stays inside."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if n >= 64 and rng.random() < 1 / 3:
        n = n // 64 * 64
    return min(max(n, low), high)


def draw(rng):
    op = rng.choice(["hgrn", "hgrn", "norm", "norm", "linear", "linear", "linear_fp8"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if op == "hgrn":
        D, train, state = _between(rng, 32, 4096), rng.random() < 0.6, rng.random() < 0.5
        if rng.random() < 0.3:
            count = _between(rng, 1, 64)
            return dict(op=op, B=1, T=0, D=min(D, 2048), dtype=dtype, sequences=count, shortest=rng.choice([1, 16, 256]),
                        longest=_between(rng, 256, 4096), lengths_seed=rng.randrange(1 << 30), state=state, train=train)
        B = _between(rng, 1, 256)
        T = _between(rng, 1, max(1, min(65536, LARGEST // 8 // (B * D))))
        return dict(op=op, B=B, T=T, D=D, dtype=dtype, sequences=0, state=state, train=train)
    if op == "norm":
        N = _between(rng, 32, 8192)
        rows = _between(rng, 1, min(65536, (1 << 27) // N))
        quant = rng.random() < 0.4
        residual = rng.choice(["none", "same", "fp32"])
        return dict(op=op, rows=rows, N=N, dtype=dtype, residual=residual, quant=quant, train=not quant and rng.random() < 0.7)
    K, N = _between(rng, 64, 4096), _between(rng, 64, 8192)
    M = _between(rng, 1, min(16384, 32768 * 2048 * 2048 // (K * N)))
    act = rng.choice(["none", "silu", "sigmoid", "logsigmoid", "gelu"])
    half = "fp16" if dtype == "fp16" else "bf16"
    if op == "linear_fp8":
        K = (K + 15) // 16 * 16
    return dict(op=op, M=M, K=K, N=N, dtype=half, activation=act, bias=rng.random() < 0.5, residual=rng.random() < 0.5,
                train=op == "linear" and rng.random() < 0.6)


def _lengths(case):
    rng = random.Random(case["lengths_seed"])
    return [rng.randint(case["shortest"], case["longest"]) for _ in range(case["sequences"])]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    grad = case["train"]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=gen, device="cuda") * std + mean

    s = dict(case)
    if case["op"] == "hgrn":
        B, T, D, offsets, count = case["B"], case["T"], case["D"], None, case["B"]
        if case["sequences"]:
            lengths = _lengths(case)
            T, count = sum(lengths), len(lengths)
            offsets = torch.tensor([sum(lengths[:i]) for i in range(count + 1)], dtype=torch.int32, device="cuda")
        # log forget gates that remember from a few to some hundred tokens, and inputs damped by 1 - gate
        g = torch.nn.functional.logsigmoid(normal(B, T, D, std=2.0, mean=2.0))
        x = torch.nn.functional.silu(normal(B, T, D)) * (1 - g.exp())
        s.update(x=x.to(dtype), g=g.to(dtype), offsets=offsets, h0=normal(count, D) if case["state"] else None)
        del x, g
        if grad:
            s["do"] = normal(B, T, D).to(dtype)
            s["dht"] = normal(count, D) if case["state"] else None
        leaves = ("x", "g", "h0")
    elif case["op"] == "norm":
        rows, N = case["rows"], case["N"]
        s.update(x=normal(rows, N).to(dtype), weight=normal(N, std=0.1, mean=1.0).to(dtype), res=None)
        if case["residual"] != "none":
            s["res"] = normal(rows, N, std=2.0).to(torch.float32 if case["residual"] == "fp32" else dtype)
        if grad:
            s["dy"] = normal(rows, N).to(dtype)
            s["dres"] = None if s["res"] is None else normal(rows, N).to(s["res"].dtype)
        leaves = ("x", "weight", "res")
    else:
        M, K, N = case["M"], case["K"], case["N"]
        x, w = normal(M, K), normal(N, K, std=K ** -0.5)
        s.update(b=normal(N, std=0.5).to(dtype) if case["bias"] else None, res=normal(M, N).to(dtype) if case["residual"] else None)
        if case["op"] == "linear_fp8":
            s["xs"], s["ws"] = x.abs().amax(1) / E4M3_MAX, w.abs().amax(1) / E4M3_MAX
            s.update(x=(x / s["xs"][:, None]).to(torch.float8_e4m3fn), w=(w / s["ws"][:, None]).to(torch.float8_e4m3fn))
            leaves = ()
        else:
            s.update(x=x.to(dtype), w=w.to(dtype))
            if grad:
                s["dy"] = normal(M, N).to(dtype)
            leaves = ("x", "w", "b", "res")
    if grad:
        for name in leaves:
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


# ---- the plain form -------------------------------------------------------------------------------------------------
def _scan(a, x):
    """h_t = a_t h_{t-1} + x_t along dim 1, by doubling the span that each position has taken in."""
    n = 1
    while n < x.shape[1]:
        x = torch.cat([x[:, :n], torch.addcmul(x[:, n:], a[:, n:], x[:, :-n])], 1)
        a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], 1)
        n *= 2
    return x


def _ends(s, T):
    """First and last row of each sequence, as indices into the rows of all batches laid end to end."""
    if s["offsets"] is None:
        first = torch.arange(s["B"], device="cuda") * T
        return first, first + T - 1
    return s["offsets"][:-1].long(), s["offsets"][1:].long() - 1


def _plain_hgrn(s):
    x, g, dtype = s["x"], s["g"], s["x"].dtype
    B, T, D = x.shape
    first, last = _ends(s, T)
    a, u = g.float().exp().reshape(-1, D), x.float().reshape(-1, D)
    if s["h0"] is not None:
        u = u.index_add(0, first, a[first] * s["h0"])
    cut = a.index_fill(0, first, 0.0)
    h = _scan(cut.view(B, T, D), u.view(B, T, D)).view(-1, D)
    del u
    out = [h.to(dtype).view(B, T, D)]
    if s["state"]:
        out.append(h[last])
    if not s["train"]:
        return out
    before = torch.roll(h, 1, 0)  # h_{t-1}
    before = before.index_fill(0, first, 0.0) if s["h0"] is None else before.index_copy(0, first, s["h0"])
    del h
    d = s["do"].float().reshape(-1, D)
    if s["dht"] is not None:
        d = d.index_add(0, last, s["dht"])
    # dh_t = do_t + a_{t+1} dh_{t+1}, the scan from the other end
    nxt = torch.roll(cut, -1, 0).view(B, T, D)
    dh = _scan(nxt.flip(1), d.view(B, T, D).flip(1)).flip(1).reshape(-1, D)
    del nxt, d, cut
    dg = dh * a * before
    out += [dh.to(dtype).view(B, T, D), dg.to(dtype).view(B, T, D)]
    if s["h0"] is not None:
        out.append(dh[first] * a[first])
    return out


EPS = 1e-6


def _plain_norm(s):
    x, w, dtype = s["x"], s["weight"].float(), s["x"].dtype
    t, out = x, []
    if s["res"] is not None:
        t = (x.float() + s["res"].float()).to(s["res"].dtype)  # the residual stream, as it is handed on
        out = [t]
    f = t.float()
    rstd = (f.square().mean(1, keepdim=True) + EPS).rsqrt()
    xhat = f * rstd
    y = xhat * w
    if s["quant"]:
        scale = y.abs().amax(1, keepdim=True) / E4M3_MAX
        q = (y / scale).to(torch.float8_e4m3fn)
        return [(q.float() * scale).to(dtype), scale[:, 0]] + out
    out = [y.to(dtype)] + out
    if s["train"]:
        dy = s["dy"].float()
        wdy = dy * w
        dt = (wdy - xhat * (wdy * xhat).mean(1, keepdim=True)) * rstd
        if s["res"] is not None:
            dt = dt + s["dres"].float()
        out += [dt.to(dtype), (dy * xhat).sum(0).to(dtype)]
        if s["res"] is not None:
            out.append(dt.to(s["res"].dtype))
    return out


def _act(z, name):
    """The activation and its derivative."""
    if name == "silu":
        e = torch.sigmoid(z)
        return z * e, e * (1 + z * (1 - e))
    if name == "sigmoid":
        e = torch.sigmoid(z)
        return e, e * (1 - e)
    if name == "logsigmoid":
        return z.clamp(max=0) - torch.log1p(torch.exp(-z.abs())), torch.sigmoid(-z)
    if name == "gelu":
        p = 0.5 * (1 + torch.erf(z * 0.5 ** 0.5))
        return z * p, p + z * torch.exp(-0.5 * z * z) * (2 * math.pi) ** -0.5
    return z, None


def _plain_linear(s):
    dtype = DTYPES[s["dtype"]]
    x, w = s["x"].float(), s["w"].float()
    z = x @ w.T
    if s["op"] == "linear_fp8":
        z = z * s["xs"][:, None] * s["ws"]
    if s["b"] is not None:
        z = z + s["b"].float()
    y, slope = _act(z, s["activation"])
    if s["res"] is not None:
        y = y + s["res"].float()
    out = [y.to(dtype)]
    if s["train"]:
        dz = s["dy"].float()
        if slope is not None:
            dz = dz * slope
        out += [(dz @ w).to(dtype), (dz.T @ x).to(dtype)]
        if s["b"] is not None:
            out.append(dz.sum(0).to(dtype))
        if s["res"] is not None:
            out.append(s["dy"])
    return out


# ---- the package's entry points --------------------------------------------------------------------------------------
def _package():
    if "flash-linear-attention_b200" not in sys.path:
        sys.path.insert(0, "flash-linear-attention_b200")
    import fla_b200.modules
    import fla_b200.ops
    return fla_b200


def _own_hgrn(s, fla):
    fn = fla.ops.fused_recurrent_hgrn if s["T"] == 1 else fla.ops.chunk_hgrn
    o, ht = fn(s["x"], s["g"], initial_state=s["h0"], output_final_state=s["state"], offsets=s["offsets"])
    out = [o] if ht is None else [o, ht]
    if not s["train"]:
        return out
    leaves = [s["x"], s["g"]] + ([] if s["h0"] is None else [s["h0"]])
    grads = torch.autograd.grad(out, leaves, [s["do"]] + ([] if ht is None else [s["dht"]]))
    return [v.detach() for v in out] + list(grads)


def _own_norm(s, fla):
    wide = s["res"] is not None and s["res"].dtype == torch.float32
    if s["quant"]:
        q, scale, *rest = fla.modules.rms_norm_quant(s["x"], s["weight"], residual=s["res"], eps=EPS, prenorm=s["res"] is not None,
                                                     residual_in_fp32=wide)
        return [(q.float() * scale[:, None]).to(s["x"].dtype), scale] + rest
    out = fla.modules.rms_norm(s["x"], s["weight"], residual=s["res"], eps=EPS, prenorm=s["res"] is not None, residual_in_fp32=wide)
    out = [out] if s["res"] is None else list(out)
    if not s["train"]:
        return out
    leaves = [s["x"], s["weight"]] + ([] if s["res"] is None else [s["res"]])
    grads = torch.autograd.grad(out, leaves, [s["dy"]] + ([] if s["res"] is None else [s["dres"]]))
    return [v.detach() for v in out] + list(grads)


def _own_linear(s, fla):
    act = None if s["activation"] == "none" else s["activation"]
    if s["op"] == "linear_fp8":
        return [fla.modules.linear_fp8(s["x"], s["xs"], s["w"], s["ws"], bias=s["b"], residual=s["res"], activation=act,
                                       out_dtype=DTYPES[s["dtype"]])]
    y = fla.modules.linear(s["x"], s["w"], bias=s["b"], residual=s["res"], activation=act)
    if not s["train"]:
        return [y]
    leaves = [s[n] for n in ("x", "w", "b", "res") if s[n] is not None]
    return [y.detach(), *torch.autograd.grad(y, leaves, s["dy"])]


def run(state):
    if own:
        return {"hgrn": _own_hgrn, "norm": _own_norm}.get(state["op"], _own_linear)(state, _package())
    with torch.no_grad():
        return {"hgrn": _plain_hgrn, "norm": _plain_norm}.get(state["op"], _plain_linear)(state)


# ---- what a pass cannot do without -----------------------------------------------------------------------------------
def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "hgrn":
        tokens, count = case["B"] * case["T"], case["B"]
        if case["sequences"]:
            lengths = _lengths(case)
            tokens, count = sum(lengths), len(lengths)
        D = case["D"]
        # forward: x, g -> o; backward: o, g, do -> dx, dg; states in 32 bits
        moved = tokens * D * e * (8 if case["train"] else 3)
        if case["state"]:
            moved += count * D * 4 * (5 if case["train"] else 2)
        return {"bytes": moved, "flops": tokens * D * (9 if case["train"] else 3)}
    if case["op"] == "norm":
        rows, N = case["rows"], case["N"]
        r = {"none": 0, "same": e, "fp32": 4}[case["residual"]]
        # forward: x, residual -> y, sum; backward: sum, dy, d(sum) -> dx, d(residual)
        per = e + 2 * r + (1 if case["quant"] else e)
        moved = rows * N * per + N * e + (rows * 4 if case["quant"] else 0)
        if case["train"]:
            moved += rows * N * ((3 * r if r else e) + 2 * e) + 2 * N * e
        return {"bytes": moved, "flops": rows * N * (14 if case["train"] else 5)}
    M, K, N = case["M"], case["K"], case["N"]
    i = 1 if case["op"] == "linear_fp8" else e
    extra = N * e * case["bias"] + M * N * e * case["residual"] + (4 * (M + N) if i == 1 else 0)
    moved = (M * K + N * K) * i + M * N * e + extra
    if case["train"]:
        # dy, x, w and (for the activation's slope) the product are read; dx, dw, db are written
        moved += 2 * (M * K + N * K) * e + M * N * e * (1 if case["activation"] == "none" else 2) + N * e * case["bias"]
    return {"bytes": moved, "flops": 2 * M * N * K * (3 if case["train"] else 1)}


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def _recur(a, u):
    """The recurrence along dim 0 of [T, C], row after row: rows are cut into equal runs that are walked side by side, then the
    runs' ends are joined one after the other."""
    T, C = u.shape
    run_len = max(1, math.isqrt(T))
    runs = -(-T // run_len)
    pad = runs * run_len - T
    a = torch.nn.functional.pad(a, (0, 0, 0, pad)).view(runs, run_len, C)
    h = torch.nn.functional.pad(u, (0, 0, 0, pad)).view(runs, run_len, C).clone()
    for t in range(1, run_len):
        h[:, t] += a[:, t] * h[:, t - 1]
    carry = torch.zeros(C, dtype=u.dtype, device=u.device)
    for r in range(runs):
        h[r] += a[r].cumprod(0) * carry
        carry = h[r, -1].clone()
    return h.view(-1, C)[:T]


def _exact_hgrn(s):
    x, g = s["x"].detach(), s["g"].detach()
    B, T, D = x.shape
    first, last = (v.tolist() for v in _ends(s, T))
    h0 = None if s["h0"] is None else s["h0"].detach().double()
    o, ht, dx, dg, dh0 = (torch.zeros(x.shape, dtype=torch.float64, device="cuda") if want else None
                          for want in (True, False, s["train"], s["train"], False))
    ht, dh0 = [], []
    flat = [v if v is None else v.reshape(-1, D) for v in (x, g, s.get("do"), o, dx, dg)]
    fx, fg, fdo, fo, fdx, fdg = flat
    for n, (i, j) in enumerate(zip(first, last)):
        a, u = fg[i:j + 1].double().exp(), fx[i:j + 1].double()
        start = torch.zeros(D, dtype=torch.float64, device="cuda") if h0 is None else h0[n]
        u[0] += a[0] * start
        h = _recur(a, u)
        fo[i:j + 1] = h
        ht.append(h[-1])
        if s["train"]:
            d = fdo[i:j + 1].double().clone()
            if s["dht"] is not None:
                d[-1] += s["dht"][n].double()
            back = torch.cat([a[1:], torch.ones_like(a[:1])]).flip(0)
            dh = _recur(back, d.flip(0)).flip(0)
            fdx[i:j + 1] = dh
            fdg[i:j + 1] = dh * a * torch.cat([start[None], h[:-1]])
            dh0.append(dh[0] * a[0])
    out = [o] + ([torch.stack(ht)] if s["state"] else [])
    if s["train"]:
        out += [dx, dg] + ([torch.stack(dh0)] if h0 is not None else [])
    return out


def _exact_norm(s):
    x, w = s["x"].detach().double(), s["weight"].detach().double()
    total, tail = x, []
    if s["res"] is not None:
        total = (x + s["res"].detach().double()).to(s["res"].dtype).double()
        tail = [total]
    N = x.shape[1]
    r = 1 / torch.sqrt((total * total).sum(1) / N + EPS)
    y = torch.einsum("rn,r,n->rn", total, r, w)
    if s["quant"]:
        scale = y.abs().max(1).values / E4M3_MAX
        held = (y / scale[:, None]).to(torch.float8_e4m3fn).double()
        return [held * scale[:, None], scale] + tail
    out = [y] + tail
    if s["train"]:
        dy = s["dy"].double()
        inner = torch.einsum("rn,n,rn->r", dy, w, total)
        dt = torch.einsum("rn,n,r->rn", dy, w, r) - total * (inner * r ** 3 / N)[:, None]
        if s["res"] is not None:
            dt = dt + s["dres"].double()
        out += [dt, torch.einsum("rn,rn,r->n", dy, total, r)] + ([dt] if s["res"] is not None else [])
    return out


def _exact_linear(s):
    x, w = s["x"].detach().double(), s["w"].detach().double()
    if s["op"] == "linear_fp8":
        x, w = x * s["xs"].double()[:, None], w * s["ws"].double()[:, None]
    z = torch.einsum("mk,nk->mn", x, w)
    if s["b"] is not None:
        z += s["b"].detach().double()
    z.requires_grad_(True)
    with torch.enable_grad():
        f = torch.nn.functional
        y = {"silu": f.silu, "sigmoid": torch.sigmoid, "logsigmoid": f.logsigmoid, "gelu": f.gelu, "none": lambda v: v * 1}[s["activation"]](z)
        dz = torch.autograd.grad(y, z, s["dy"].double())[0] if s["train"] else None
    y = y.detach()
    if s["res"] is not None:
        y = y + s["res"].detach().double()
    out = [y]
    if s["train"]:
        out += [torch.einsum("mn,nk->mk", dz, w), torch.einsum("mn,mk->nk", dz, x)]
        if s["b"] is not None:
            out.append(dz.sum(0))
        if s["res"] is not None:
            out.append(s["dy"].double())
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {"hgrn": _exact_hgrn, "norm": _exact_norm}.get(case["op"], _exact_linear)(s)
