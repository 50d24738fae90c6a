"""The ends of the ranges that the operators of the gated-recurrence block are documented for: values that a type cannot hold, rows of
nothing, derivatives and uses of the results that a program may ask for, waits that ran out. Each test says which value the
definition gives; the tolerances count roundings as in the operators' own test files."""
import os
import subprocess
import sys

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn.functional as F

from fla_b200 import _lib
from fla_b200.modules import RMSNorm, linear, linear_fp8, quantize_rows, rms_norm, rms_norm_quant
from fla_b200.ops import chunk_hgrn, fused_recurrent_hgrn

DEV = "cuda"
BF, FH, F32 = torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def half_step(value, dtype):
    tiny = {BF: 2.0 ** -134, FH: 2.0 ** -25, F32: 2.0 ** -150}[dtype]
    return value.abs() * torch.finfo(dtype).eps / 2 + tiny


def within(name, got, want, bound):
    got = got.detach().double().cpu()
    assert got.shape == want.shape and torch.isfinite(got).all(), name
    over = ((got - want).abs() - bound).max().item()
    assert over <= 0, f"{name}: {over:.3e} over its bound"


ACTIVATIONS = {"silu": F.silu, "sigmoid": torch.sigmoid, "logsigmoid": F.logsigmoid, "gelu": F.gelu}


@pytest.mark.gpu
@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("M,K,N", [(40, 64, 48), (40, 64, 33), (33, 4096, 40)])  # tile stores, other outputs, a sum in runs
def test_gradients_where_fp16_cannot_hold_the_argument(M, K, N, act):
    """z = -131072 and 131072 overflow fp16, in which z is kept for backward; the slopes there are 0 and 1, and so are the gradients'
    parts. The bounds are those of the operator's own tests; beyond |z| = 100 every slope is 0 or 1 to within 2^-20."""
    gen = torch.Generator().manual_seed(M + N)
    x = torch.randn(M, K, generator=gen).to(FH)
    w = (torch.randn(N, K, generator=gen) * K ** -0.5).to(FH)
    w[0] = -64
    x[0], x[1] = 2048.0 / K, -2048.0 / K
    b = torch.randn(N, generator=gen).to(FH)
    dy = torch.randn(M, N, generator=gen).to(FH)
    X, W, D = x.double(), w.double(), dy.double()
    z = (X @ W.T + b.double()).requires_grad_(True)
    assert z[0, 0] < -131000 and z[1, 0] > 131000
    dz = torch.autograd.grad(ACTIVATIONS[act](z), z, D)[0]
    z = z.detach()
    leaves = [t.to(DEV).requires_grad_(True) for t in (x, w, b)]
    y = linear(leaves[0], leaves[1], bias=leaves[2], activation=act)
    dx, dw, db = torch.autograd.grad(y, leaves, dy.to(DEV))
    size = (X.abs() @ W.abs().T) * K * 2.0 ** -23
    near = 0.8 * (half_step(z, FH) + size + 2.0 ** -23 * z.abs()) + 2.0 ** -18 * (1 + z.abs())
    slope = D.abs() * torch.where(z.abs() > 100, 2.0 ** -20, near)
    edz = slope + half_step(dz, FH)
    want = dz @ W
    within("dx", dx, want, edz @ W.abs() + (dz.abs() @ W.abs()) * N * 2.0 ** -23 + half_step(want, FH))
    want = dz.T @ X
    within("dw", dw, want, edz.T @ X.abs() + (dz.abs().T @ X.abs()) * M * 2.0 ** -23 + half_step(want, FH))
    want = dz.sum(0)
    within("db", db, want, slope.sum(0) + dz.abs().sum(0) * M * U + half_step(want, FH))


@pytest.mark.gpu
@pytest.mark.parametrize("N", [48, 33])
def test_an_argument_that_is_not_finite_stays_so(N):
    """What is held in fp16's range are values that fp32 holds: a NaN or an infinity among the inputs still reaches the gradients of its
    row, and no other row's."""
    gen = torch.Generator().manual_seed(7)
    x, w = torch.randn(6, 64, generator=gen).to(FH), (torch.randn(N, 64, generator=gen) / 8).to(FH)
    clean = x.clone()
    x[2, 5], x[4, 5] = float("nan"), float("inf")
    dys = torch.ones(6, N, dtype=FH, device=DEV)
    out = []
    for v in (x, clean):
        v = v.to(DEV).requires_grad_(True)
        out.append(torch.autograd.grad(linear(v, w.to(DEV), activation="silu"), v, dys)[0])
    assert torch.isnan(out[0][2]).all() and not torch.isfinite(out[0][4]).all()
    keep = [0, 1, 3, 5]
    assert torch.equal(out[0][keep], out[1][keep]) and torch.isfinite(out[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(3, 0), (2, 5, 0), (700, 0)])
def test_rows_of_no_elements_have_scale_zero(shape):
    rows = shape[0] if len(shape) == 2 else shape[0] * shape[1]
    for _ in range(4):  # what the allocator hands out next held something else
        junk = torch.full((rows,), float("nan"), device=DEV)
        torch.cuda.synchronize()
        del junk
        x, w = torch.empty(shape, device=DEV, dtype=BF), torch.ones(0, device=DEV, dtype=BF)
        for q, scale in (quantize_rows(x), rms_norm_quant(x, w), rms_norm_quant(x, w, residual=x, prenorm=True)[:2]):
            assert q.shape == shape and scale.shape == shape[:-1] and (scale == 0).all()


@pytest.mark.gpu
def test_a_wait_that_ran_out_stays_with_its_call():
    """A wait for an earlier tile's word, with a short limit, on a word that nothing sets: it hands back NaN, marks its own call's abort
    flag and is recorded. Later calls, whose tiles wait for each other thousands of times, do not look at that record."""
    lib = _lib.load()
    T, D = 120000, 64
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(1, T, D, generator=gen).to(DEV).to(BF)
    odd = torch.randn(1, T // 4, 63, generator=gen).to(DEV)
    g, godd = -x.abs() / 16, -odd.abs() / 16
    want = [chunk_hgrn(x, g, output_final_state=True), chunk_hgrn(odd, godd, output_final_state=True)]
    torch.cuda.synchronize()
    assert lib.flab_tc_check() == 0
    status = torch.zeros(64, dtype=torch.int32, device=DEV)  # [0]: what came back, [32]: the call's abort flag
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.flab_hgrn_wait_selftest(1 << 20, status.data_ptr(), stream) == 0
    torch.cuda.synchronize()
    assert status[0].item() == 700 and status[32].item() == 1  # NaN, and no later wait of that call waits
    assert lib.flab_tc_error_state() == 700
    try:
        for _ in range(5):
            for (v, gate), (o, ht) in zip(((x, g), (odd, godd)), want):
                again, last = chunk_hgrn(v, gate, output_final_state=True)
                assert torch.equal(again, o) and torch.equal(last, ht)
    finally:
        torch.cuda.synchronize()
        assert lib.flab_tc_error_clear() == 0
    # with the flag set the same wait gives up instead of at its limit
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    assert lib.flab_hgrn_wait_selftest(1 << 28, status.data_ptr(), stream) == 0
    end.record()
    torch.cuda.synchronize()
    assert status[0].item() == 700 and begin.elapsed_time(end) < 50  # 2^28 ticks are 130 ms and more
    assert lib.flab_tc_error_clear() == 0 and lib.flab_tc_check() == 0


def test_wait_selftest_refuses():
    lib = _lib.load()
    for limit in (0, -1, (1 << 28) + 1):
        assert lib.flab_hgrn_wait_selftest(limit, 16, None) == -1
    assert lib.flab_hgrn_wait_selftest(1 << 20, None, None) == -1


LONG_ROWS = """
import sys
sys.path.insert(0, sys.argv[1])
from fla_b200 import _lib
lib = _lib.load()
codes = []
for n, dtype, res in ((1 << 30, 2, False), (1 << 29, 2, True), (1 << 30, 0, True), (1 << 30, 2, True), (357913944, 0, True), (1 << 20, 0, True)):
    for flags in (0, 1):
        codes.append(lib.flab_rms_norm_fwd(16, 16 if res else None, 16, 16, 16, 16, 16, 1, n, dtype, dtype, dtype, dtype, flags, 1e-6, None))
    codes.append(lib.flab_rms_norm_bwd(16, 16, 16, 16, 16, 16, None, None, None, 1, n, dtype, dtype, dtype, None))
    codes.append(lib.flab_rms_norm_bwd(16, 16, 16, 16, 16, 16, None, 16, 16, 1, n, dtype, dtype, dtype, None))
print(codes)
assert all(code < 0 for code in codes)  # there is no device to launch on
"""


def test_rows_whose_bytes_pass_32_bits():
    """Rows of up to 2^30 elements are taken; their bytes pass an int. On a machine without a device (none is visible to the process) such a
    call ends with an error's code and not with the process."""
    run = subprocess.run([sys.executable, "-c", LONG_ROWS, os.path.join(ROOT, "flash-linear-attention_b200")], capture_output=True, text=True, timeout=600,
                         env={**os.environ, "CUDA_VISIBLE_DEVICES": ""})
    assert run.returncode == 0, (run.returncode, run.stdout, run.stderr)


@pytest.mark.gpu
@pytest.mark.parametrize("n,dtype", [(64, BF), (512, BF), (256, F32)])
def test_one_warp_rows_with_a_gradient_of_the_stream(n, dtype):
    """Rows of one warp: the stage that holds the stream's gradient is refilled behind all lanes' reads of it. Bit for bit from run to run."""
    rows = 60000
    x, dy, ds = (torch.randn(rows, n, device=DEV, generator=torch.Generator(DEV).manual_seed(i)).to(dtype) for i in range(3))
    r, w = x.flip(0).requires_grad_(True), torch.rand(n, device=DEV, generator=torch.Generator(DEV).manual_seed(4)).to(dtype)
    first = None
    for _ in range(4):
        (dr,) = torch.autograd.grad(rms_norm(x, w, residual=r, prenorm=True), r, (dy, ds))
        first = dr if first is None else first
        assert torch.equal(dr, first)
    s = (x.float() + r.detach().float()).to(dtype).double()
    rstd = 1 / (s.square().mean(1, keepdim=True) + 1e-6).sqrt()
    xhat, wd = s * rstd, w.double() * dy.double()
    d64 = rstd * (wd - xhat * (xhat * wd).mean(1, keepdim=True)) + ds.double()
    size = rstd * (wd.abs() + xhat.abs() * (xhat * wd).abs().mean(1, keepdim=True)) + ds.double().abs()
    within("dr", first, d64.cpu(), (96 * U * size + half_step(d64, dtype)).cpu())


@pytest.mark.gpu
@pytest.mark.parametrize("which", range(10))
@pytest.mark.parametrize("grad", [True, False])
def test_forward_mode_derivatives_are_refused(which, grad):
    """A dual tensor's tangent is never dropped without a word, with and without gradients switched on."""
    gen = torch.Generator().manual_seed(0)
    x = torch.randn(4, 6, 32, generator=gen).to(DEV).to(BF)
    w = torch.randn(32, 32, generator=gen).to(DEV).to(BF)
    h0, v = torch.zeros(4, 32, device=DEV), torch.ones(32, device=DEV, dtype=BF)
    with torch.no_grad():
        (q, qs), (p, ps) = quantize_rows(x), quantize_rows(w)
    calls = [lambda d: chunk_hgrn(d(x), -x.abs()), lambda d: chunk_hgrn(x, d(-x.abs())), lambda d: fused_recurrent_hgrn(x, -x.abs(), initial_state=d(h0)),
             lambda d: rms_norm(d(x), v), lambda d: rms_norm(x, d(v), residual=x), lambda d: rms_norm_quant(x, v, residual=d(x)),
             lambda d: quantize_rows(d(x)), lambda d: linear(x, d(w)), lambda d: linear(x, w, residual=d(x)),
             lambda d: linear_fp8(q, d(qs), p, ps)]
    with torch.set_grad_enabled(grad):
        calls[which](lambda t: t)
        with forward_ad.dual_level():
            calls[which](lambda t: t)  # a level by itself changes nothing
            with pytest.raises(RuntimeError, match="forward"):
                calls[which](lambda t: forward_ad.make_dual(t, torch.ones_like(t)))


INSTALL = """
import sys, types
sys.path.insert(0, sys.argv[1])
def module(name, **names):
    m = sys.modules[name] = types.ModuleType(name)
    m.__dict__.update(names)
    if "." in name:
        setattr(sys.modules[name.rpartition(".")[0]], name.rpartition(".")[2], m)
    return m
for name in ("fla", "fla.modules", "fla.ops"):
    module(name).__path__ = []
module("fla.modules.layernorm", LayerNorm="their LayerNorm", RMSNorm="their RMSNorm")
module("fla.ops.hgrn", chunk_hgrn="their chunk", other="their other").__path__ = ["/nowhere"]
module("fla.ops.hgrn.naive", naive_recurrent_hgrn="their loop")
import fla_b200
for _ in range(2):  # a second call changes nothing
    fla_b200.install_as_fla_modules()
    fla_b200.install_as_fla_ops()
from fla.modules.layernorm import LayerNorm, RMSNorm, rms_norm
assert LayerNorm == "their LayerNorm"
from fla_b200.modules import RMSNorm as ours, rms_norm as own
assert RMSNorm is ours and rms_norm is own
import fla.modules.layernorm as by_path
assert by_path.LayerNorm == LayerNorm and by_path.RMSNorm is ours
from fla.ops.hgrn import chunk_hgrn, other
from fla_b200.ops import chunk_hgrn as own
assert other == "their other" and chunk_hgrn is own
from fla.ops.hgrn.naive import naive_recurrent_hgrn
assert naive_recurrent_hgrn == "their loop"
for bad in ("fla.modules.layernorm", "fla.ops.hgrn"):
    try:
        exec(f"from {bad} import nobody_has_this")
    except ImportError:
        continue
    raise SystemExit(bad)
print("as it should be")
"""


@pytest.mark.parametrize("there", [True, False])
def test_names_of_a_replaced_module_stay(there):
    """Installing the package's modules over a `fla` that was imported before keeps the names that this package has no form of its own
    for; without one, a name that nobody has is an ImportError as ever."""
    code = INSTALL
    if not there:
        code = code[:code.index("def module")] + "import fla_b200\n" + "\n".join(
            ["fla_b200.install_as_fla_modules()", "fla_b200.install_as_fla_ops()", "from fla.modules.layernorm import RMSNorm",
             "from fla.ops.hgrn import chunk_hgrn", code[code.index("for bad in"):]])
    run = subprocess.run([sys.executable, "-c", code, os.path.join(ROOT, "flash-linear-attention_b200")], capture_output=True, text=True, timeout=600)
    assert run.returncode == 0 and "as it should be" in run.stdout, run.stdout + run.stderr


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 64), (64,), (2, 1, 3, 64)])
def test_results_may_be_changed_in_place(shape):
    """As those of nn.Linear may, whatever the number of dimensions."""
    gen = torch.Generator().manual_seed(3)
    x, r = (torch.randn(shape, generator=gen).to(DEV).to(BF).requires_grad_(True) for _ in range(2))
    w = (torch.randn(64, 64, generator=gen) / 8).to(DEV).to(BF).requires_grad_(True)
    n = torch.ones(64, device=DEV, dtype=BF, requires_grad=True)
    for make, leaves in ((lambda: linear(x, w, activation="silu"), (x, w)), (lambda: linear(x, w, residual=r), (x, w, r)),
                         (lambda: rms_norm(x, n), (x, n)), (lambda: rms_norm(x, n, residual=r, prenorm=True)[0], (x, n, r))):
        y = make()
        want = torch.autograd.grad(F.silu(y * 2 + 1), leaves, torch.ones_like(y))
        y = make()
        y.mul_(2).add_(1)
        got = torch.autograd.grad(F.silu(y, inplace=True), leaves, torch.ones_like(y))
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    y, s = rms_norm(x, n, residual=r, prenorm=True)
    assert s.shape == x.shape and y.shape == x.shape
    s += y  # the next block's stream; backward of this norm reads s, so as with any sum that is read again it is not asked for here
    with torch.no_grad():
        y = linear(x, w)
        y += 1
        assert y.shape == shape


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF, FH, F32])
@pytest.mark.parametrize("n", [512, 33])
def test_rows_with_tiny_largest_values(dtype, n):
    """q scale stands for the row down to the smallest numbers: half a step of e4m3, 2^-4 of the value or 2^-10 of the scale, whatever the
    scale is. (Below 448 2^-126 a scale of fp32 has few bits; it may be larger than max|y| / 448, and never smaller by more than a rounding.)"""
    tops = [2.0 ** e * f for e in range(-148, -100, 3) for f in (1.0, 1.3)] + [448 * 2.0 ** -126 * f for f in (0.99, 1.0, 1.01)] + [1e-37, 1e-42, 600 * 2.0 ** -149]
    if dtype == FH:
        tops = [2.0 ** e * f for e in range(-24, -10, 2) for f in (1.0, 1.5)]
    gen = torch.Generator().manual_seed(n)
    y = torch.rand(len(tops), n, generator=gen) * 2 - 1
    y[:, 0] = 1
    y = (y.double() * torch.tensor(tops, dtype=torch.float64)[:, None]).float().to(dtype)
    check_tiny(*quantize_rows(y.to(DEV)), y.double())
    # the norm of ordinary rows with a tiny weight
    x = torch.randn(len(tops), n, generator=gen).to(dtype)
    for top in (tops[2], tops[-1], tops[len(tops) // 2]):
        w = torch.full((n,), top, dtype=F32)
        y = x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
        # the products are rounded to fp32, subnormal ones to 2^-149
        check_tiny(*rms_norm_quant(x.to(DEV), w.to(DEV)), y, 96 * U * y.abs() + 2.0 ** -149)
    # enough rows for the streaming form, which holds rows of 16-byte vectors
    x = torch.randn(16000, 512, generator=gen).to(dtype)
    w = torch.full((512,), 2.0 ** -130, dtype=F32)
    y = x.double() / (x.double().square().mean(1, keepdim=True) + 1e-6).sqrt() * w.double()
    check_tiny(*rms_norm_quant(x.to(DEV), w.to(DEV)), y, 96 * U * y.abs() + 2.0 ** -149)


def check_tiny(q, scale, y, error=0.0):
    q, scale = q.cpu().double(), scale.cpu().double()[:, None]
    top = y.abs().amax(1, keepdim=True)
    assert torch.isfinite(q).all() and ((scale > 0) | (top <= 2.0 ** -149)).all()
    assert (scale * (1 + 4 * U) * 448 >= top * (1 - 100 * U) - 2.0 ** -149).all()
    step = torch.maximum(y.abs() * 2.0 ** -4, scale * 2.0 ** -10)
    over = ((q * scale - y).abs() - (step * (1 + 200 * U) + 200 * U * y.abs() + error)).max().item()
    assert over <= 0, over


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["sigmoid", "logsigmoid", "silu"])
def test_slopes_far_out(act):
    """dz = act'(z) dy where z is exact (a product with one term): the slope to within 2^-18 of itself, or of z's part in it where it is a
    sum, on both sides of zero, and its rounding and that of dx."""
    z = torch.arange(-20, 20.25, 0.25).to(BF)
    x = torch.zeros(len(z), 8, dtype=BF)
    x[:, 0] = z
    w = torch.zeros(8, 8, dtype=BF)
    w[0, 0] = 1
    xs = x.to(DEV).requires_grad_(True)
    y = linear(xs, w.to(DEV), activation=act)
    (dx,) = torch.autograd.grad(y, xs, torch.ones_like(y))
    Z = z.double().requires_grad_(True)
    (want,) = torch.autograd.grad(ACTIVATIONS[act](Z).sum(), Z)
    s = torch.sigmoid(-Z.detach().abs())
    own = want.abs() if act != "silu" else want.abs() + (1 + Z.detach().abs()) * torch.sigmoid(Z.detach())
    bound = 2.0 ** -18 * own + 2.02 * half_step(want, BF)
    assert (s > 0).all()
    within("dz", dx[:, 0], want, bound)


class Elsewhere(torch.autograd.graph.saved_tensors_hooks):
    """Saved tensors that come back with other strides, or at an address of two bytes behind a 16-byte boundary."""

    def __init__(self, strided):
        def pack(t):
            return t.detach().clone()

        def unpack(t):
            if strided and t.dim() > 1:
                return t.transpose(-1, -2).contiguous().transpose(-1, -2)
            flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)[1:]
            return flat.view(t.shape).copy_(t)

        super().__init__(pack, unpack)


@pytest.mark.gpu
@pytest.mark.parametrize("strided", [True, False])
@pytest.mark.parametrize("D", [64, 33])
def test_saved_tensors_that_come_back_otherwise(D, strided):
    """A hook may bring saved tensors back in any layout: the gradients are those without it, up to the order of fp32 sums."""
    gen = torch.Generator().manual_seed(D)
    x, r, dy = (torch.randn(3, 50, D, generator=gen).to(DEV).to(BF) for _ in range(3))
    w = (torch.randn(D, D, generator=gen) * D ** -0.5).to(DEV).to(BF)
    n, h0 = torch.rand(D, generator=gen).to(DEV).to(BF), torch.randn(3, D, generator=gen).to(DEV)
    for t in (x, r, w, n, h0):
        t.requires_grad_(True)
    cases = [(lambda: linear(x, w, activation="silu"), (x, w)), (lambda: linear(x, w, residual=r), (x, w, r)),
             (lambda: rms_norm(x, n, residual=r), (x, n, r)), (lambda: rms_norm(x, n, residual=r, residual_in_fp32=True), (x, n, r)),
             (lambda: chunk_hgrn(x, -r.abs(), initial_state=h0)[0], (x, r, h0)), (lambda: fused_recurrent_hgrn(x[:, :9], -r[:, :9].abs())[0], (x, r))]
    for make, of in cases:
        y = make()
        g = dy[:, :y.shape[1]]
        want = torch.autograd.grad(y, of, g)
        with Elsewhere(strided):
            y = make()
        for a, b in zip(torch.autograd.grad(y, of, g), want):
            a, b = a.double(), b.double()
            assert ((a - b).abs() <= 2.02 * half_step(b, BF) + 2.0 ** -14 * b.abs().max()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["x", "weight"])
def test_eight_bit_operands_that_ask_for_a_gradient(which):
    q, v = (torch.zeros(n, 32, device=DEV).to(torch.float8_e4m3fn) for n in (4, 8))
    one = [torch.ones(n, device=DEV) for n in (4, 8)]
    (q if which == "x" else v).requires_grad_(True)
    with pytest.raises(NotImplementedError, match="no backward"):
        linear_fp8(q, one[0], v, one[1])
    with torch.no_grad():
        assert linear_fp8(q, one[0], v, one[1]).shape == (4, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 63])
def test_products_of_gates_that_overflow_behind_an_edge(D):
    """A sequence that holds nothing stays at nothing, although the products of its gates overflow and the sequence before it ended in
    something; in backward the same in front of a sequence's end."""
    lengths = [1500, 1700, 90]
    T = sum(lengths)
    off = torch.tensor([0, 1500, 3200, T], device=DEV)
    gen = torch.Generator().manual_seed(0)
    x, g = torch.randn(T, D, generator=gen), -torch.rand(T, D, generator=gen)
    x[1500:3200] = 0
    g[1500:3200] = 60
    do = torch.randn(T, D, generator=gen)
    do[1500:3200] = 0
    xs, gs = (v.to(DEV).view(1, T, D).requires_grad_(True) for v in (x, g))
    o, ht = chunk_hgrn(xs, gs, output_final_state=True, offsets=off)
    dht = torch.ones(3, D, device=DEV)
    dht[1] = 0
    dx, dg = torch.autograd.grad([o, ht], [xs, gs], [do.to(DEV).view_as(o), dht])
    for v in (o, dx, dg):
        assert torch.isfinite(v).all() and (v[0, 1500:3200] == 0).all() and (v[0, :1500] != 0).any() and (v[0, 3200:] != 0).any()
    assert torch.isfinite(ht).all() and (ht[1] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(1, 57856), (3, 57856), (300, 57856), (1, 57857), (3, 57857), (300, 57857), (300, 70000), (1, 300001), (3, 300001)])
def test_the_weight_gradient_of_long_rows(rows, n):
    """Sums over the rows that shared memory holds (57856 columns), and longer ones, with rows for more than one turn of every block."""
    gen = torch.Generator().manual_seed(n)
    x, dy = torch.randn(rows, n, generator=gen), torch.randn(rows, n, generator=gen)
    for dtype, wdtype in ((BF, F32), (F32, F32), (FH, FH)):
        w = (1 + 0.1 * torch.randn(n, generator=gen)).to(wdtype)
        xs, ws = x.to(dtype).to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
        dx, dw = torch.autograd.grad(rms_norm(xs, ws), (xs, ws), dy.to(dtype).to(DEV))
        X, D, W = x.to(dtype).double(), dy.to(dtype).double(), w.double()
        rstd = 1 / (X.square().mean(1, keepdim=True) + 1e-6).sqrt()
        xhat = X * rstd
        # a thread adds n / 1024 values in turn, then the tree: 293 + 10 + a handful
        adds = (n / 1024 + 30) * U
        want = (D * xhat).sum(0)
        within("dw", dw, want, (adds + rows * U) * (D * xhat).abs().sum(0) + half_step(want, wdtype))
        want = rstd * (W * D - xhat * (xhat * W * D).mean(1, keepdim=True))
        size = rstd * ((W * D).abs() + xhat.abs() * (xhat * W * D).abs().mean(1, keepdim=True))
        within("dx", dx, want, adds * size + half_step(want, dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [8, 9])
@pytest.mark.parametrize("tokens,empty", [(300, 1 << 22), (1, 1 << 22), (40000, 70000), (300, 0)])
def test_more_empty_sequences_than_tokens(tokens, empty, D):
    """A table of one-token sequences with a run of empty ones in its middle: states pass through, outputs are those without the run, and
    the call's time does not go by the run's length one sequence after the other (a third of a second, of which a wait bears one)."""
    gen = torch.Generator().manual_seed(5)
    x, g = (torch.randn(1, tokens, D, generator=gen).to(DEV) for _ in range(2))
    g = -g.abs()
    head = tokens // 2
    off = torch.cat([torch.arange(head + 1), torch.full((empty,), head), torch.arange(head + 1, tokens + 1)]).to(torch.int32).to(DEV)
    N = tokens + empty
    h0, dht = (torch.randn(N, D, device=DEV, generator=torch.Generator(DEV).manual_seed(i)) for i in range(2))
    full = torch.ones(N, dtype=torch.bool, device=DEV)
    full[head:head + empty] = False
    xs, gs, hs = (v.requires_grad_(True) for v in (x, g, h0))
    o, ht = chunk_hgrn(xs, gs, initial_state=hs, output_final_state=True, offsets=off)
    grads = torch.autograd.grad([o, ht], [xs, gs, hs], [torch.ones_like(o), dht])
    few = h0.detach()[full].requires_grad_(True)
    dense = torch.arange(tokens + 1, dtype=torch.int32, device=DEV)
    o2, ht2 = chunk_hgrn(xs, gs, initial_state=few, output_final_state=True, offsets=dense)
    want = torch.autograd.grad([o2, ht2], [xs, gs, few], [torch.ones_like(o2), dht[full]])
    assert torch.equal(o, o2) and torch.equal(ht[full], ht2) and torch.equal(ht[~full], h0[~full])
    assert torch.equal(grads[0], want[0]) and torch.equal(grads[1], want[1])
    assert torch.equal(grads[2][full], want[2]) and torch.equal(grads[2][~full], dht[~full])
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    chunk_hgrn(x.detach(), g.detach(), initial_state=h0.detach(), output_final_state=True, offsets=off)
    end.record()
    torch.cuda.synchronize()
    assert begin.elapsed_time(end) < 100
    assert _lib.load().flab_tc_error_state() == 0
