"""Products with bias, activation and residual in the epilogue (`linear`, `linear_fp8`) against the formulas in 64 bits.

Tolerances. A product of K terms is accumulated in fp32, each addition off by at most one unit 2^-23 of the sum of the terms' sizes:
K 2^-23 sum|a b|. The activations' slopes are at most 1.13 and their second derivatives at most 0.8; their fp32 evaluation with the fast
exponential is off by less than 2^-18 (1 + |z|). Backward reads z and dz rounded to the inputs' type (half a step each), and both errors go
through the next product with the sizes of its other operand."""
import pytest
import torch
import torch.nn.functional as F
import torch.utils.checkpoint

from fla_b200 import _lib
from fla_b200.modules import linear, linear_fp8, quantize_rows, rms_norm, rms_norm_quant
from fla_b200.modules import FusedRMSNormSwishGate, RMSNorm
from fla_b200.ops import chunk_hgrn

DEV = "cuda"
BF, FH = torch.bfloat16, torch.float16
ACTS = {None: lambda z: z, "silu": F.silu, "swish": F.silu, "sigmoid": torch.sigmoid, "logsigmoid": F.logsigmoid, "gelu": F.gelu}


def half(v, dtype):
    return v.abs() * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype == FH else 2.0 ** -134)


def within(name, got, want, bound):
    assert got.shape == want.shape, name
    over = ((got.detach().double().cpu() - want).abs() - bound).max().item() if want.numel() else 0
    assert over <= 0, f"{name}: {over:.3e} over its bound"


def make(M, K, N, dtype, seed, bias=True, residual=True):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=gen).to(dtype)
    w = (torch.randn(N, K, generator=gen) * K ** -0.5).to(dtype)
    b = torch.randn(N, generator=gen).to(dtype) if bias else None
    r = torch.randn(M, N, generator=gen).to(dtype) if residual else None
    return x, w, b, r, torch.randn(M, N, generator=gen).to(dtype)


def expected(x, w, b, r, act):
    """z, y in 64 bits and the bound of y in fp32, before its rounding."""
    x, w = x.double(), w.double()
    z = x @ w.T
    size = (x.abs() @ w.abs().T) * x.shape[1] * 2.0 ** -23
    if b is not None:
        z = z + b.double()
    y = ACTS[act](z)
    err = 1.13 * (size + 2.0 ** -23 * z.abs()) + (2.0 ** -18 * (1 + z.abs()) if act else 0)
    if r is not None:
        y = y + r.double()
        err = err + 2.0 ** -23 * (y.abs() + r.double().abs())
    return z, y, size, err


SIZES = [(1, 8, 8), (1, 1, 1), (7, 64, 64), (3, 33, 5), (64, 200, 130), (128, 128, 256), (129, 72, 257), (256, 64, 512), (300, 515, 257), (513, 1000, 96),
         (40, 2048, 640), (2000, 72, 16), (1100, 136, 1032),
         (33, 4096, 40), (5000, 40, 72), (6, 48, 5000), (6, 50, 5001)]  # the last: sums cut into runs, in y, dw and dx


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FH])
@pytest.mark.parametrize("act", [None, "silu", "sigmoid", "logsigmoid", "gelu"])
@pytest.mark.parametrize("M,K,N", SIZES)
def test_forward_and_gradients(M, K, N, act, dtype):
    bias, residual = (M + N) % 3 != 0, (M + K) % 2 == 0
    x, w, b, r, dy = make(M, K, N, dtype, M + K + N, bias, residual)
    z, y, size, err = expected(x, w, b, r, act)
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    xs, ws, bs, rs = next(it), next(it), next(it) if bias else None, next(it) if residual else None
    got = linear(xs, ws, bias=bs, residual=rs, activation=act)
    assert got.dtype == dtype
    within("y", got, y, err + half(y, dtype))
    with torch.no_grad():
        assert torch.equal(linear(xs, ws, bias=bs, residual=rs, activation=act), got)

    names = ["x", "w"] + ["b"] * bias + ["r"] * residual
    grads = dict(zip(names, torch.autograd.grad(got, leaves, dy.to(DEV))))
    zz = z.clone().requires_grad_(True)
    D = dy.double()
    dz = torch.autograd.grad(ACTS[act](zz), zz, D)[0] if act else D
    slope = D.abs() * (0.8 * (half(z, dtype) + size + 2.0 ** -23 * z.abs()) + 2.0 ** -18 * (1 + z.abs())) if act else torch.zeros_like(D)
    edz = slope + (half(dz, dtype) if act else 0)
    X, W = x.double(), w.double()
    dx, dw = dz @ W, dz.T @ X
    within("dx", grads["x"], dx, edz @ W.abs() + (dz.abs() @ W.abs()) * N * 2.0 ** -23 + half(dx, dtype))
    within("dw", grads["w"], dw, edz.T @ X.abs() + (dz.abs().T @ X.abs()) * M * 2.0 ** -23 + half(dw, dtype))
    if bias:
        db = dz.sum(0)
        within("db", grads["b"], db, slope.sum(0) + dz.abs().sum(0) * M * 2.0 ** -24 + half(db, dtype))
    if residual:
        assert torch.equal(grads["r"].cpu(), dy)


@pytest.mark.gpu
@pytest.mark.parametrize("out", [BF, FH])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("M,K,N", [(1, 16, 8), (5, 128, 64), (130, 144, 257), (256, 1024, 512), (600, 272, 96), (1300, 64, 2000), (50, 16384, 40), (17, 8192, 129)])
def test_eight_bits(M, K, N, act, out):
    x, w, b, r, _ = make(M, K, N, out, M * N + K)
    with torch.no_grad():
        (q, qs), (v, vs) = quantize_rows(x.to(DEV)), quantize_rows(w.to(DEV))
        y = linear_fp8(q, qs, v, vs, bias=b.to(DEV), residual=r.to(DEV), activation=act, out_dtype=out)
    X, W = (a.cpu().double() * s.cpu().double()[:, None] for a, s in ((q, qs), (v, vs)))
    _, want, _, err = expected(X, W, b, r, act)
    assert y.dtype == out
    # two products with the scales, each rounded, and the sum of the unscaled terms
    within("y", y, want, 1.01 * err + 2.0 ** -21 * (X @ W.T).abs() + half(want, out))


@pytest.mark.gpu
def test_tiles_in_turn_and_large_rows():
    """More tiles than pairs of SMs (each pair goes through several, both halves of the accumulator in turn), and a long sum."""
    for M, K, N in ((2560, 264, 2304), (256, 20000, 256), (5000, 512, 2056)):
        x, w, b, r, dy = make(M, K, N, BF, 1)
        x, w, b, r, dy = (t.to(DEV) for t in (x, w, b, r, dy))
        z = x.double() @ w.double().T
        y = F.silu(z + b.double()) + r.double()
        got = linear(x, w, bias=b, residual=r, activation="silu")
        size = 1.2 * K * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T) + 2.0 ** -17 * (2 + z.abs())
        assert ((got.double() - y).abs() <= size + half(y, BF)).all()
        xs, ws = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
        dx, dw = torch.autograd.grad(linear(xs, ws), [xs, ws], dy)
        D = dy.double()
        for name, g, want, sz in (("dx", dx, D @ w.double(), N * (D.abs() @ w.double().abs())), ("dw", dw, D.T @ x.double(), M * (D.abs().T @ x.double().abs()))):
            assert ((g.double() - want).abs() <= 2.0 ** -23 * sz + half(want, BF)).all(), name
        again = torch.autograd.grad(linear(xs, ws), [xs, ws], dy)
        assert torch.equal(again[0], dx) and torch.equal(again[1], dw)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [2048, 2047])
def test_offsets_beyond_32_bits(N):
    M, K = 2 ** 31 // N + 900, 16
    x, w, b, _, _ = make(1000, K, N, BF, 4, residual=False)
    x, w, b = x.to(DEV).repeat(M // 1000 + 1, 1)[:M].contiguous(), w.to(DEV), b.to(DEV)
    xs = x.requires_grad_(True)
    y = linear(xs, w, bias=b, activation="silu")
    for rows in (slice(0, 300), slice(M - 300, M)):
        assert torch.equal(y.detach()[rows], linear(x.detach()[rows], w, bias=b, activation="silu"))
    (dx,) = torch.autograd.grad(y, xs, y.detach())
    small = x.detach()[-300:].clone().requires_grad_(True)
    (dx2,) = torch.autograd.grad(linear(small, w, bias=b, activation="silu"), small, y.detach()[-300:])
    # the small call may cut its sums into runs: fp32 in another order, one rounding each
    assert ((dx[-300:].double() - dx2.double()).abs() <= 2 * half(dx2.double(), BF) + 2.0 ** -12).all()


@pytest.mark.gpu
def test_shapes_views_streams_and_graph():
    gen = torch.Generator().manual_seed(2)
    x = torch.randn(3, 5, 80, generator=gen).to(DEV).to(BF)
    w = torch.randn(48, 72, generator=gen).to(DEV).to(BF)
    r = torch.randn(3, 5, 48, generator=gen).to(DEV).to(BF)
    view = x[..., 4:76]
    want = linear(view.contiguous(), w, residual=r, activation="gelu")
    assert want.shape == (3, 5, 48)
    assert torch.equal(linear(view, w, residual=r, activation="gelu"), want)
    off = torch.empty(48 * 72 + 1, device=DEV, dtype=BF)[1:].view(48, 72)  # a weight that begins off a 16-byte boundary
    off.copy_(w)
    assert torch.equal(linear(view, off, residual=r, activation="gelu"), want)
    wt = w.t().contiguous().t()
    assert torch.equal(linear(view, wt, residual=r, activation="swish"), linear(view, w, residual=r, activation="silu"))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = linear(view, w, residual=r, activation="gelu")
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    xs, ws = x.clone().requires_grad_(True), torch.randn(33, 80, generator=gen).to(DEV).to(BF).requires_grad_(True)
    b = torch.zeros(33, device=DEV, dtype=BF, requires_grad=True)

    def step():
        y = linear(xs, ws, bias=b, activation="silu")
        return (y.detach(), *torch.autograd.grad(y, [xs, ws, b], y.detach()))

    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step())
        graphs.append(graph)
    with torch.no_grad():
        xs.copy_(torch.randn(xs.shape, generator=gen))
    torch.cuda.synchronize()
    graphs[0].replay()
    with torch.cuda.stream(side):
        graphs[1].replay()
    torch.cuda.synchronize()
    for out in outs:
        for p, q in zip(out, step()):
            assert torch.equal(p, q)
    assert _lib.load().flab_tc_error_state() == 0


@pytest.mark.gpu
def test_gradient_against_differences():
    gen = torch.Generator().manual_seed(3)
    x, w, b = (torch.randn(s, generator=gen).to(FH) for s in ((6, 24), (10, 24), (10,)))
    a = torch.randn(6, 10, generator=gen).double().to(DEV)
    args = [t.to(DEV) for t in (x, w, b)]

    def f(*t):
        return (linear(t[0], t[1], bias=t[2], activation="sigmoid").double() * a).sum()

    leaves = [t.clone().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(f(*leaves), leaves)
    for i, grad in enumerate(grads):
        way = torch.randint(0, 2, args[i].shape, generator=gen).to(DEV).to(FH) * 2 - 1
        h = 2.0 ** -5
        up, down = ([(t.float() + k * h * way.float()).to(FH) if j == i else t for j, t in enumerate(args)] for k in (1, -1))
        taken = ((up[i].double() - down[i].double()) * grad.double()).sum().item()
        diff = (f(*up) - f(*down)).item()
        # outputs in fp16 (half a step 2^-12 of values below 1, both sides), gradients rounded, and the third-order term
        assert abs(diff - taken) <= a.abs().sum().item() * 2.0 ** -11 + 0.05 * ((up[i].double() - down[i].double()).abs() * grad.double().abs()).sum().item()


@pytest.mark.gpu
def test_a_block_of_them():
    """Norm, projections, recurrence, gated norm and output projection one behind the other, as a layer runs them: training in bf16
    against the same block in fp32 PyTorch with a token loop, and its 8-bit prompt pass against the bf16 one."""
    torch.manual_seed(0)
    B, T, H = 2, 150, 128
    dev = dict(device=DEV, dtype=BF)
    x, res = torch.randn(B, T, H, **dev), torch.randn(B, T, H, **dev)
    wi, wf, wg, wo = (torch.randn(H, H, **dev) * H ** -0.5 for _ in range(4))
    bf = torch.full((H,), 2.0, **dev)
    norm, gate = RMSNorm(H).to(**dev), FusedRMSNormSwishGate(H).to(DEV)
    params = [x, res, wi, wf, wg, wo, bf, norm.weight]
    for t in params:
        t.requires_grad_(True)

    y, stream = norm(x, residual=res, prenorm=True)
    i, f, g = linear(y, wi, activation="silu"), linear(y, wf, bias=bf, activation="logsigmoid"), linear(y, wg)
    h, _ = chunk_hgrn(i, f)
    out = linear(gate(h, g), wo, residual=stream)
    dy = torch.randn_like(out)
    got = torch.autograd.grad(out, params, dy)

    ref = [t.detach().float().requires_grad_(True) for t in params]
    X, R, WI, WF, WG, WO, BFt, NW = ref
    S = X + R
    Y = S * torch.rsqrt(S.square().mean(-1, keepdim=True) + 1e-5) * NW
    I, Fg, Gt = F.silu(Y @ WI.T), F.logsigmoid(Y @ WF.T + BFt), Y @ WG.T
    state, hs = torch.zeros(B, H, device=DEV), []
    for t in range(T):
        state = Fg[:, t].exp() * state + I[:, t]
        hs.append(state)
    Hs = torch.stack(hs, 1)
    N = Hs * torch.rsqrt(Hs.square().mean(-1, keepdim=True) + 1e-5) * F.silu(Gt)
    O = N @ WO.T + S
    want = torch.autograd.grad(O, ref, dy.float())
    # each tensor passes through at most a dozen roundings to bf16 of half a step 2^-9 rms-wise (2^-8 at most); 12 of the largest
    for name, p, q in zip(("out", "x", "res", "wi", "wf", "wg", "wo", "bf", "norm"), (out, *got), (O, *want)):
        err = (p.float() - q).norm() / q.norm()
        assert err < 12 * 2.0 ** -8, (name, err.item())

    with torch.no_grad():
        q, s, stream8 = rms_norm_quant(x, norm.weight, residual=res, eps=norm.eps, prenorm=True)
        assert torch.equal(stream8, stream)
        i8 = linear_fp8(q, s, *quantize_rows(wi), activation="silu")
    # e4m3 rounds each operand by 2^-4 of its size at most: two of them, rms far below that
    assert (i8.float() - i.float()).norm() / i.float().norm() < 2 * 2.0 ** -4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FH])
def test_a_block_under_a_checkpoint(dtype):
    """The block's gradients are the same bits whether its intermediates are kept, worked out again or brought back from the host."""
    gen = torch.Generator().manual_seed(31)
    B, T, D = 2, 70, 96
    x, dy = (torch.randn(B, T, D, generator=gen).to(DEV).to(dtype) for _ in range(2))
    ws = [(torch.randn(D, D, generator=gen) * D ** -0.5).to(DEV).to(dtype) for _ in range(3)]
    leaves = [t.requires_grad_(True) for t in (x, (1 + torch.randn(D, generator=gen)).to(DEV).to(dtype), *ws)]

    def block(x, n, wi, wf, wo):
        y = rms_norm(x, n)
        o, _ = chunk_hgrn(linear(y, wi, activation="silu"), linear(y, wf, activation="logsigmoid"))
        y, s = rms_norm(o, n, residual=x, prenorm=True)
        return linear(y, wo, residual=s)

    want = torch.autograd.grad(block(*leaves), leaves, dy)
    for got, ref in zip(torch.autograd.grad(torch.utils.checkpoint.checkpoint(block, *leaves, use_reentrant=False), leaves, dy), want):
        assert torch.equal(got, ref)
    with torch.autograd.graph.save_on_cpu():
        y = block(*leaves)
    for got, ref in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(got, ref)


@pytest.mark.gpu
def test_only_some_gradients_and_no_rows():
    x, w, b, r, dy = (t.to(DEV) for t in make(70, 40, 24, BF, 0))
    for which in range(4):
        leaves = [t.clone().requires_grad_(i == which) for i, t in enumerate((x, w, b, r))]
        y = linear(leaves[0], leaves[1], bias=leaves[2], residual=leaves[3], activation="gelu")
        (g,) = torch.autograd.grad(y, leaves[which], dy)
        full = [t.clone().requires_grad_(True) for t in (x, w, b, r)]
        y = linear(full[0], full[1], bias=full[2], residual=full[3], activation="gelu")
        assert torch.equal(g, torch.autograd.grad(y, full, dy)[which])
    e = torch.zeros(0, 40, device=DEV, dtype=BF, requires_grad=True)
    ws, bs = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    y = linear(e, ws, bias=bs)
    assert y.shape == (0, 24)
    de, dw, db = torch.autograd.grad(y, [e, ws, bs], torch.empty(0, 24, device=DEV, dtype=BF))
    assert de.shape == (0, 40) and (dw == 0).all() and (db == 0).all()
    with torch.no_grad():
        q = torch.zeros(0, 48, device=DEV).to(torch.float8_e4m3fn)
        assert linear_fp8(q, torch.zeros(0, device=DEV), torch.zeros(24, 48, device=DEV).to(q.dtype), torch.ones(24, device=DEV)).shape == (0, 24)


@pytest.mark.gpu
def test_second_derivatives_are_refused():
    x, w = (torch.randn(n, 32, device=DEV, dtype=BF, requires_grad=True) for n in (6, 8))
    v, one = torch.randn(2, 9, 32, device=DEV, requires_grad=True), torch.ones(32, device=DEV, requires_grad=True)
    for out, leaf in ((linear(x, w, activation="silu"), x), (rms_norm(v, one), v), (chunk_hgrn(v, v)[0], v)):
        dy = torch.ones_like(out).requires_grad_(True)
        (g,) = torch.autograd.grad(out, leaf, dy, create_graph=True)
        with pytest.raises(RuntimeError):  # never a silent zero
            torch.autograd.grad(g.sum(), leaf, retain_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            g.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,N", [(300, 128, 96), (130, 77, 51)])
@pytest.mark.parametrize("bias", [True, False])
def test_operands_that_come_back_elsewhere(M, K, N, bias):
    """A checkpoint works its inputs out again and a hook may keep them on the host: backward reads them where they are then."""
    x, w, b, r, dy = (v if v is None else v.to(DEV) for v in make(M, K, N, BF, 21, bias=bias))
    leaves = [t.requires_grad_(True) for t in (x, w, b, r) if t is not None]

    def step(x, w, b, r):
        return linear(torch.tanh(linear(x * 2, w * 1.5, bias=b, activation="silu")), torch.eye(N, device=DEV, dtype=BF), residual=r)

    want = torch.autograd.grad(step(x, w, b, r), leaves, dy)

    def elsewhere(y):  # what forward freed is given to others before backward
        junk = [torch.full((n,), float("nan"), device=DEV, dtype=BF) for n in (M * K, M * K, N * K, N * K, M * N, N * N)]
        grads = torch.autograd.grad(y, leaves, dy)
        del junk
        return grads

    with torch.autograd.graph.save_on_cpu():
        y = step(x, w, b, r)
    for got, ref in zip(elsewhere(y), want):
        assert torch.equal(got, ref)
    y = torch.utils.checkpoint.checkpoint(step, x, w, b, r, use_reentrant=False)
    for got, ref in zip(elsewhere(y), want):
        assert torch.equal(got, ref)


def test_refusals():
    x, w = torch.zeros(4, 16, dtype=BF), torch.zeros(8, 16, dtype=BF)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        linear(x, w)
    with pytest.raises(ValueError, match="both be bfloat16"):
        linear(x.float(), w.float())
    with pytest.raises(ValueError, match="both be bfloat16"):
        linear(x, w.half())
    with pytest.raises(ValueError, match="not supported"):
        linear(x, w, activation="tanh")
    with pytest.raises(ValueError, match=r"weight \[N, K\]"):
        linear(x, w[:, :8])
    with pytest.raises(ValueError, match="bias must be"):
        linear(x, w, bias=torch.zeros(7, dtype=BF))
    with pytest.raises(ValueError, match="residual must be"):
        linear(x, w, residual=torch.zeros(1, 8, dtype=BF))
    for big in (x[:1].expand(2 ** 31 + 4, 16), x[:1].expand(2 ** 17, 2 ** 15, 16)):
        with pytest.raises(ValueError, match="sides beyond 2"):
            linear(big, w)
    with pytest.raises(ValueError, match="sides beyond 2"):
        linear(x, w[:1].expand(2 ** 32 + 8, 16))
    q, v = x.to(torch.float8_e4m3fn), w.to(torch.float8_e4m3fn)
    with pytest.raises(ValueError, match="float8_e4m3fn"):
        linear_fp8(x, torch.ones(4), w, torch.ones(8))
    with pytest.raises(ValueError, match="x_scale must be"):
        linear_fp8(q, torch.ones(3), v, torch.ones(8))
    with pytest.raises(ValueError, match="weight_scale must be"):
        linear_fp8(q, torch.ones(4), v, torch.ones(8, dtype=BF))
    with pytest.raises(ValueError, match="out_dtype"):
        linear_fp8(q, torch.ones(4), v, torch.ones(8), out_dtype=torch.float32)


@pytest.mark.gpu
def test_refusals_on_the_device():
    q, v = (torch.zeros(n, 24, device=DEV).to(torch.float8_e4m3fn) for n in (4, 8))
    with pytest.raises(ValueError, match="multiple of 16"):
        linear_fp8(q, torch.ones(4, device=DEV), v, torch.ones(8, device=DEV))
    with pytest.raises(NotImplementedError, match="no backward"):
        linear_fp8(q, torch.ones(4, device=DEV), v, torch.ones(8, device=DEV), bias=torch.zeros(8, device=DEV, dtype=BF, requires_grad=True))
    with pytest.raises(RuntimeError, match="expected cuda"):
        linear(torch.zeros(4, 16, dtype=BF, device=DEV), torch.zeros(8, 16, dtype=BF))


def test_abi_refusals():
    lib = _lib.load()
    none = (None, 0, None, 0, None)
    assert lib.flab_linear_fwd(None, None, None, None, None, None, 0, 8, 8, 0, 0, *none) == 0
    assert lib.flab_linear_fwd(16, 16, None, None, 16, None, 8, 8, 8, 5, 0, *none) == -1
    assert b"activation" in lib.flab_last_error()
    assert lib.flab_linear_fwd(16, 16, None, None, 16, None, 8, 8, 8, 0, 2, *none) == -2
    assert lib.flab_linear_fwd(16, 16, None, None, 16, None, (1 << 31) - 1, 8, 8, 0, 0, *none) == -2
    assert b"beyond 2^30" in lib.flab_last_error()
    assert lib.flab_linear_workspace(16, 16, 8, 8, 8) == 0
    assert lib.flab_linear_workspace(16, 18, 8, 8, 8) == 256 and lib.flab_linear_workspace(16, 16, 8, 8, 7) == 512
    assert lib.flab_linear_bwd_scratch(16, 8, 8, 8, 0) == 0 and lib.flab_linear_bwd_scratch(16, 8, 8, 8, 1) == 256
    assert lib.flab_linear_bwd_scratch(18, 8, 8, 8, 0) == 256
    # a long sum of few tiles is cut into runs, the ordinary sizes are not
    assert lib.flab_linear_scratch(64, 64, 1 << 16, 0) > 0 and lib.flab_linear_scratch(32768, 2048, 2048, 0) == 0
    assert lib.flab_linear_bwd_scratch(16, 1 << 16, 64, 64, 0) > 0
    assert lib.flab_linear_fwd(16, 18, None, None, 16, None, 8, 8, 8, 0, 0, *none) == -1
    assert b"workspace" in lib.flab_last_error()
    assert lib.flab_linear_fwd(16, 16, None, None, 16, None, 64, 64, 1 << 16, 0, 0, *none) == -1
    assert b"scratch" in lib.flab_last_error()
    assert lib.flab_linear_bwd(16, 16, None, 16, 16, None, None, None, 8, 8, 8, 1, 0, *none) == -1
    assert lib.flab_linear_bwd(None, 16, None, 16, 16, None, None, None, 8, 8, 8, 0, 0, *none) == -1
    assert lib.flab_linear_bwd(16, 18, None, 16, 16, None, None, None, 8, 8, 8, 0, 0, *none) == -1
    assert b"flab_linear_workspace" in lib.flab_last_error()
    assert lib.flab_linear_bwd(16, 16, 16, 16, 16, None, None, None, 8, 8, 8, 1, 0, *none) == -1
    assert b"scratch" in lib.flab_last_error()
    assert lib.flab_linear_e4m3(16, 16, 16, 16, None, None, 16, 8, 8, 24, 0, 0, None, 0, None) == -2
    assert b"multiple of 16" in lib.flab_last_error()
