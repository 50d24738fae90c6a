"""RMS norm with the residual's addition (`rms_norm`, `RMSNorm`) and its 8-bit output (`rms_norm_quant`, `quantize_rows`) against the
formulas in 64 bits.

Tolerances. The definition rounds s = x + residual to its stored type, so the reference starts from that rounded value (which has to come
back bit for bit). What follows is fp32: a thread adds at most 64 values in turn before a tree of at most 10 levels, so a sum is off by at
most 74 roundings (2^-24) of the sum of its terms' sizes, and a handful of products follow: 96 * 2^-24 of the terms' sizes. dw adds a
row a rounding. Outputs add half a step of their type."""
import pytest
import torch

from fla_b200 import _lib
from fla_b200.modules import RMSNorm, quantize_rows, rms_norm, rms_norm_quant

U = 2.0 ** -24
DEV = "cuda"
BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32


def half_step(value, dtype):
    tiny = {BF: 2.0 ** -134, FH: 2.0 ** -25, F32: 2.0 ** -150}[dtype]
    return value.abs() * torch.finfo(dtype).eps / 2 + tiny


def within(name, got, want, bound):
    got = got.detach().double().cpu()
    over = ((got - want).abs() - bound).max().item() if want.numel() else 0
    assert over <= 0, f"{name}: {over:.3e} over its bound"


def make(rows, n, dtype, res, wdtype, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, n, generator=gen).to(dtype)
    r = None if res is None else (2 * torch.randn(rows, n, generator=gen)).to(res)
    w = None if wdtype is None else (1 + 0.1 * torch.randn(n, generator=gen)).to(wdtype)
    dy = torch.randn(rows, n, generator=gen).to(dtype)
    ds = torch.randn(rows, n, generator=gen)
    return x, r, w, dy, ds


def put(v):
    return None if v is None else v.to(DEV)


def stored(x, r, stream):
    return (x if r is None else x.float() + r.float()).to(stream)


def forward64(s, w, eps):
    s = s.double()
    rstd = 1 / (s.square().mean(1, keepdim=True) + eps).sqrt()
    return s * rstd * (1 if w is None else w.double()), rstd


TYPES = [(BF, None, BF, False), (BF, BF, BF, False), (FH, FH, FH, False), (F32, None, F32, False), (F32, F32, F32, False), (BF, F32, BF, False),
         (BF, BF, F32, True), (FH, F32, FH, True), (BF, None, BF, True), (BF, BF, None, False)]
SIZES = [(1, 1), (3, 8), (5, 33), (130, 64), (2, 1111), (67, 2048), (1, 4096), (300, 520), (2, 8192), (3, 9001), (2, 20000), (1, 33000), (700, 96),
         (9500, 40), (9473, 512), (5000, 264), (1300, 2048), (700, 8192), (2400, 1032),
         (9500, 192), (3, 12288), (600, 6000), (90, 1378), (4, 4100), (2, 66)]  # several rows a group of the ring; the last two ask for 48 KB of shared memory to the byte


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,res,wdtype,wide", TYPES)
@pytest.mark.parametrize("rows,n", SIZES)
def test_forward_and_gradients(rows, n, dtype, res, wdtype, wide):
    eps = 1e-5
    x, r, w, dy, ds = make(rows, n, dtype, res, wdtype, rows * n)
    stream = F32 if wide else (dtype if res is None else res)
    ds = ds.to(stream)
    s = stored(x, r, stream)
    y64, rstd = forward64(s, w, eps)
    leaves = [v.requires_grad_(True) for v in (put(x), put(r), put(w)) if v is not None]
    it = iter(leaves)
    xs, rs, ws = next(it), (next(it) if r is not None else None), (next(it) if w is not None else None)
    y, total = rms_norm(xs, ws, residual=rs, eps=eps, prenorm=True, residual_in_fp32=wide)
    assert y.dtype == dtype and total.dtype == stream
    assert torch.equal(total.detach().cpu(), s)
    within("y", y, y64, 96 * U * y64.abs() + half_step(y64, dtype))
    alone = rms_norm(xs.detach(), put(w), residual=put(r), eps=eps, residual_in_fp32=wide)
    assert torch.equal(alone, y)

    grads = dict(zip("xrw" if r is not None and w is not None else "xw" if w is not None else "xr",
                     torch.autograd.grad([y, total], leaves, [put(dy), put(ds)])))
    D, W = dy.double(), (torch.ones(n).double() if w is None else w.double())
    xhat = s.double() * rstd
    inner = (xhat * W * D).mean(1, keepdim=True)
    d64 = rstd * (W * D - xhat * inner) + ds.double()
    size = rstd * ((W * D).abs() + xhat.abs() * (xhat * W * D).abs().mean(1, keepdim=True)) + ds.double().abs()
    if r is None and not wide:  # the stream is x: the engine adds the two gradients, each rounded to x's type
        own = rstd * (W * D - xhat * inner)
        within("dx", grads["x"], d64, 96 * U * size + half_step(own, dtype) + half_step(d64, dtype))
    else:
        within("dx", grads["x"], d64, 96 * U * size + half_step(d64, dtype))
    if r is not None:
        assert grads["r"].dtype == res
        within("dr", grads["r"], d64, 96 * U * size + half_step(d64, res))
    if w is not None:
        assert grads["w"].dtype == wdtype
        dw = (D * xhat).sum(0)
        within("dw", grads["w"], dw, (96 + rows) * U * (D * xhat).abs().sum(0) + half_step(dw, wdtype))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,res,wdtype,wide", TYPES[:8])
@pytest.mark.parametrize("rows,n", SIZES)
def test_eight_bits(rows, n, dtype, res, wdtype, wide):
    eps = 1e-6
    x, r, w, _, _ = make(rows, n, dtype, res, wdtype, rows + n)
    stream = F32 if wide else (dtype if res is None else res)
    s = stored(x, r, stream)
    y64, _ = forward64(s, w, eps)
    q, scale, total = rms_norm_quant(put(x), put(w), residual=put(r), eps=eps, prenorm=True, residual_in_fp32=wide)
    assert q.dtype == torch.float8_e4m3fn and scale.dtype == F32 and scale.shape == (rows,)
    assert torch.equal(total.cpu(), s)
    held(q, scale, y64)
    held(*quantize_rows(put(x)), x.double())


def held(q, scale, y64):
    top = y64.abs().amax(1)
    within("scale", scale, top / 448, 100 * U * top / 448)
    back = q.cpu().double() * scale.cpu().double()[:, None]
    # half a step of e4m3: 2^-4 of the value, or of the spacing below its normal numbers
    step = torch.maximum(y64.abs() * 2.0 ** -4, top[:, None] / 448 * 2.0 ** -10)
    within("q", back, y64, step * (1 + 200 * U) + 200 * U * y64.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,res,wdtype,wide", [TYPES[1], TYPES[2], TYPES[4], TYPES[5]])
@pytest.mark.parametrize("rows,n", [(1000, 8192), (3700, 2048), (3700, 1032), (14300, 264), (8200, 2048)])
def test_many_rows(rows, n, dtype, res, wdtype, wide):
    """Enough rows for the ring in both directions and in 8 bits, with one to four vectors a thread; the last are 128 MB in 32 bits."""
    test_forward_and_gradients(rows, n, dtype, res, wdtype, wide)
    test_eight_bits(rows, n, dtype, res, wdtype, wide)


@pytest.mark.gpu
def test_rows_without_a_scale():
    x = torch.zeros(4, 512, device=DEV)
    x[1, 3] = float("nan")
    x[2] = 1e-42  # the reciprocal of its scale overflows
    x[3, 0] = -5
    q, scale = quantize_rows(x)
    assert (q[0].float() == 0).all() and scale[0] == 0
    assert torch.isnan(scale[1]) and torch.isnan(q[1].float()).all()
    assert torch.isfinite(q[2].float()).all() and scale[2] < 1e-40
    assert q[3, 0].float() == -448 and scale[3] == torch.tensor(5.0) / 448
    q, scale, s = rms_norm_quant(x[:1], torch.ones(512, device=DEV), residual=x[:1], prenorm=True)
    assert (q.float() == 0).all() and scale[0] == 0


@pytest.mark.gpu
def test_views_streams_module_and_graph():
    gen = torch.Generator().manual_seed(0)
    big = torch.randn(6, 5, 260, generator=gen).to(DEV).bfloat16()
    w = torch.rand(256, generator=gen).to(DEV).bfloat16()
    x = big[:, :, 1:257]  # rows off a 16-byte boundary
    y, s = rms_norm(x, w, residual=x.transpose(0, 1).contiguous().transpose(0, 1), prenorm=True)
    assert y.shape == x.shape and torch.equal(s, (x.float() * 2).bfloat16())
    flat = torch.empty(6 * 5 * 256 + 1, device=DEV, dtype=torch.bfloat16)[1:].view(6, 5, 256)
    flat.copy_(x)
    got, _ = rms_norm(flat, w, residual=flat, prenorm=True)
    y64, _ = forward64(s.reshape(-1, 256).cpu(), w.cpu(), 1e-6)
    for v in (y, got):  # the two paths add in different orders
        within("y", v.reshape(-1, 256), y64, 96 * U * y64.abs() + half_step(y64, BF))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, _ = rms_norm(x, w, residual=x, prenorm=True)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, y)

    mod = RMSNorm(256).to(DEV)
    assert "256" in repr(mod) and mod.weight.dtype == F32
    xs = x.contiguous().requires_grad_(True)

    def step():
        out, tot = mod(xs, residual=xs, prenorm=True, residual_in_fp32=True)
        return (out.detach(), tot.detach(), *torch.autograd.grad([out, tot], [xs, mod.weight], [out.detach(), tot.detach()]))

    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    with torch.no_grad():
        xs.copy_(torch.randn(xs.shape, generator=gen))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(outs, step()):
        assert torch.equal(a, b)  # and bit for bit from run to run


@pytest.mark.gpu
def test_gradient_against_differences():
    gen = torch.Generator().manual_seed(4)
    x, r = (torch.randn(7, 40, generator=gen).to(DEV) for _ in range(2))
    w = torch.rand(40, generator=gen).to(DEV)
    a, b = (torch.randn(7, 40, generator=gen).to(DEV).double() for _ in range(2))

    def f(x, r, w):
        y, s = rms_norm(x, w, residual=r, prenorm=True)
        return (y.double() * a + s.double() ** 2 * b).sum()

    args = [x, r, w]
    leaves = [v.clone().requires_grad_(True) for v in args]
    grads = torch.autograd.grad(f(*leaves), leaves)
    for i, grad in enumerate(grads):
        way, h = torch.randn(args[i].shape, generator=gen).to(DEV), 2.0 ** -8
        up, down = ([v + (k * h * way if j == i else 0) for j, v in enumerate(args)] for k in (1, -1))
        diff, have = (f(*up) - f(*down)).item() / (2 * h), (grad.double() * way.double()).sum().item()
        scale = (grad.double() * way.double()).abs().sum().item()
        assert abs(diff - have) <= 1e-3 * scale + 1e-2, (i, diff, have)


@pytest.mark.gpu
def test_only_some_gradients_and_no_rows():
    x, w = torch.randn(4, 64, device=DEV), torch.ones(64, device=DEV)
    r = torch.randn(4, 64, device=DEV, requires_grad=True)
    y = rms_norm(x, w, residual=r)
    (dr,) = torch.autograd.grad(y, r, torch.ones_like(y))
    assert dr.shape == r.shape and torch.isfinite(dr).all()
    _, s = rms_norm(x, w, residual=r, prenorm=True)
    (dr,) = torch.autograd.grad(s, r, torch.ones_like(s))  # y is not used at all
    assert torch.equal(dr, torch.ones_like(dr))
    ws = w.clone().requires_grad_(True)
    (dw,) = torch.autograd.grad(rms_norm(x, ws), ws, torch.ones_like(x))
    assert torch.isfinite(dw).all()
    for shape in ((0, 64), (2, 0, 64), (3, 0)):
        e = torch.zeros(shape, device=DEV, requires_grad=True)
        ww = torch.ones(shape[-1], device=DEV, requires_grad=True)
        y, s = rms_norm(e, ww, residual=e, prenorm=True)
        assert y.shape == shape and s.shape == shape
        dx, dw = torch.autograd.grad(y, [e, ww], torch.ones_like(y))
        assert dx.shape == shape and (dw == 0).all()
        q, scale = quantize_rows(e.detach())
        assert q.shape == shape and scale.shape == shape[:-1]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2048, 2047])
def test_offsets_beyond_32_bits(n):
    rows = 2 ** 31 // n + 700
    x = torch.empty(rows, n, dtype=BF, device=DEV).normal_()
    w = torch.ones(n, device=DEV, dtype=BF)
    xs = x.requires_grad_(True)
    y = rms_norm(xs, w)
    (dx,) = torch.autograd.grad(y, xs, x.detach())
    small = x.detach()[-300:].clone().requires_grad_(True)
    y2 = rms_norm(small, w)
    (dx2,) = torch.autograd.grad(y2, small, small.detach())
    y64, rstd = forward64(small.detach().cpu(), w.cpu(), 1e-6)
    within("y", y[-300:], y64, 96 * U * y64.abs() + half_step(y64, BF))
    D, xhat = small.detach().double().cpu(), small.detach().double().cpu() * rstd
    inner = (xhat * D).mean(1, keepdim=True)
    d64 = rstd * (D - xhat * inner)
    size = rstd * (D.abs() + xhat.abs() * (xhat * D).abs().mean(1, keepdim=True))
    for d in (dx[-300:], dx2):
        within("dx", d, d64, 96 * U * size + half_step(d64, BF))
    q, scale = quantize_rows(x.detach())
    held(q[-300:], scale[-300:], small.detach().double().cpu())


def test_refusals():
    x, w = torch.zeros(2, 8), torch.ones(8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        rms_norm(x, w)
    with pytest.raises(NotImplementedError, match="bias"):
        rms_norm(x, w, w)
    with pytest.raises(NotImplementedError, match="bias"):
        RMSNorm(8, bias=True)
    with pytest.raises(ValueError, match="weight must be"):
        rms_norm(x, torch.ones(7))
    with pytest.raises(ValueError, match="shape of x"):
        rms_norm(x, w, residual=torch.zeros(1, 8))
    with pytest.raises(ValueError, match="type of x"):
        rms_norm(x, w, residual=x.bfloat16())
    with pytest.raises(ValueError, match="bfloat16, float16 or float32"):
        rms_norm_quant(x.double(), w)
    with pytest.raises(ValueError, match="bfloat16, float16 or float32"):
        quantize_rows(x.int())
    with pytest.raises(ValueError, match="beyond 2"):
        rms_norm(x[:, :1].expand(2, 2 ** 32 + 8), None)


@pytest.mark.gpu
def test_refusals_on_the_device():
    x, w = torch.zeros(2, 8, device=DEV), torch.ones(8, device=DEV, requires_grad=True)
    with pytest.raises(NotImplementedError, match="no backward"):
        rms_norm_quant(x, w)
    with torch.no_grad():
        rms_norm_quant(x, w)
    with pytest.raises(RuntimeError, match="expected cuda"):
        rms_norm(x, torch.ones(8))


def test_abi_refusals():
    lib = _lib.load()
    assert lib.flab_rms_norm_fwd(None, None, None, None, None, None, None, 0, 8, 0, 0, 0, 0, 0, 1e-6, None) == 0
    assert lib.flab_rms_norm_fwd(None, None, None, None, None, None, None, 1, 8, 0, 0, 0, 0, 0, 1e-6, None) == -1
    assert lib.flab_rms_norm_fwd(16, 16, None, 16, None, None, None, 1, 8, 2, 0, 2, 0, 0, 1e-6, None) == -2
    assert b"residual of type" in lib.flab_last_error()
    assert lib.flab_rms_norm_fwd(16, None, None, 16, None, None, None, 1, 8, 0, 0, 0, 0, 1, 1e-6, None) == -1
    assert b"scale" in lib.flab_last_error()
    assert lib.flab_rms_norm_fwd(16, None, 16, 16, None, None, 16, 1, 8, 0, 0, 0, 0, 3, 1e-6, None) == -1
    assert lib.flab_rms_norm_bwd(16, 16, None, None, 16, None, None, None, None, 1, 8, 0, 0, 0, None) == -1
    assert lib.flab_rms_norm_bwd(16, 16, None, 16, 16, 16, None, 16, None, 1, 8, 0, 0, 0, None) == -1
    assert b"dw_partial" in lib.flab_last_error()
    assert lib.flab_rms_norm_partials(0, 8, 0) == 1
