"""Element-wise gated recurrence (`chunk_hgrn`, `fused_recurrent_hgrn`) against a token loop in 64 bits.

Tolerances. The loop gets the very inputs. Every state of the kernel is fp32, where a value that has gone through n steps of a
contracting recurrence carries at most a few n roundings of 2^-24 of the terms it sums; n is bounded by the memory of the gates used
here (below 200 tokens), so 400 * 2^-24 = 2.4e-5 of the largest value bounds what is not a rounding to the output's type. Outputs in
16 bits add half a step of their own value; dg is a product with the stored (rounded) state, so it has two half steps."""
import math

import pytest
import torch

from fla_b200 import _lib
from fla_b200.ops import chunk_hgrn, fused_recurrent_hgrn

STATE = 400 * 2.0 ** -24
DEV = "cuda"


def loop(x, g, h0, lengths):
    """h_t = e^{g_t} h_{t-1} + x_t over the packed rows of `lengths`; x, g [T, D] float64, h0 [N, D] or None."""
    out, last, at = [], [], 0
    for n, length in enumerate(lengths):
        h = torch.zeros(x.shape[1], dtype=torch.float64) if h0 is None else h0[n]
        for t in range(at, at + length):
            h = g[t].exp() * h + x[t]
            out.append(h)
        at += length
        last.append(h)
    rest = [torch.zeros(x.shape[1], dtype=torch.float64)] * (x.shape[0] - at)
    return torch.stack(out + rest) if out or rest else x, torch.stack(last)


def inputs(rows, D, N, dtype, seed, state):
    gen = torch.Generator().manual_seed(seed)
    g = torch.nn.functional.logsigmoid(2 * torch.randn(rows, D, generator=gen) + 2).to(dtype)
    x = torch.randn(rows, D, generator=gen).to(dtype)
    do = torch.randn(rows, D, generator=gen).to(dtype)
    h0 = torch.randn(N, D, generator=gen) if state else None
    dht = torch.randn(N, D, generator=gen) if state else None
    return x, g, do, h0, dht


def near(name, got, want, dtype, halves=1):
    want = want.double()
    got = got.detach().double().cpu()
    eps = torch.finfo(dtype).eps / 2
    bound = halves * eps * want.abs() + (STATE if dtype != torch.float32 else 2 * STATE) * max(1.0, want.abs().max().item())
    if dtype == torch.float16:
        bound += 2.0 ** -24  # subnormal steps
    worst = ((got - want).abs() - bound).max().item()
    assert worst <= 0, f"{name}: {worst:.3e} over its bound"


def check(x, g, do, h0, dht, lengths, dtype, shape, offsets, fn=chunk_hgrn, final=True):
    X, G = x.double().requires_grad_(True), g.double().requires_grad_(True)
    H = None if h0 is None else h0.double().requires_grad_(True)
    o, ht = loop(X, G, H, lengths)
    loss = (o * do.double()).sum() + (0 if dht is None else (ht * dht.double()).sum())
    leaves = [v for v in (X, G, H) if v is not None]
    want = torch.autograd.grad(loss, leaves, allow_unused=True)
    want = [torch.zeros_like(v) if w is None else w for v, w in zip(leaves, want)]

    xs, gs = (v.to(DEV).view(shape).requires_grad_(True) for v in (x, g))
    hs = None if h0 is None else h0.to(DEV).requires_grad_(True)
    oc, hc = fn(xs, gs, initial_state=hs, output_final_state=final, offsets=offsets)
    assert oc.dtype == dtype and (hc is None) == (not final)
    outs, grads = [oc], [do.to(DEV).view(shape)]
    if dht is not None and final:
        outs.append(hc), grads.append(dht.to(DEV))
    got = torch.autograd.grad(outs, [v for v in (xs, gs, hs) if v is not None], grads)
    near("o", oc.reshape(o.shape), o.detach(), dtype)
    if hc is not None:
        assert hc.dtype == torch.float32
        near("ht", hc, ht.detach(), torch.float32)
    near("dx", got[0].reshape(want[0].shape), want[0], dtype)
    near("dg", got[1].reshape(want[1].shape), want[1], dtype, halves=2.1)
    if h0 is not None:
        near("dh0", got[2], want[2], torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("B,T,D,state", [(1, 1, 1, True), (2, 1, 64, True), (3, 2, 33, False), (1, 7, 2, True), (2, 127, 66, True), (1, 128, 64, False),
                                         (2, 129, 31, True), (1, 700, 130, True), (1, 1500, 8, False), (5, 260, 96, True), (2, 9, 24, True),
                                         (2, 1300, 72, True), (3, 1024, 136, False), (1, 129, 8, True), (1, 8300, 72, True), (2, 8192, 8, False),
                                         (2, 15, 77, True), (3, 32, 34, True), (2, 33, 64, True), (1, 32, 16, False), (160, 40, 512, True)])
def test_fixed_length(B, T, D, state, dtype):
    x, g, do, h0, dht = inputs(B * T, D, B, dtype, B * T + D, state)
    check(x, g, do, h0, dht, [T] * B, dtype, (B, T, D), None)
    check(x, g, do, h0, dht, [T] * B, dtype, (B, T, D), None, fn=fused_recurrent_hgrn)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("lengths,behind,D,state", [([1], 0, 64, True), ([5, 1, 130], 0, 34, True), ([0, 3, 0, 0, 300, 1, 0], 0, 70, True),
                                                    ([128, 128, 256], 0, 64, False), ([1] * 150, 0, 65, True), ([600, 90], 17, 32, True),
                                                    ([0, 0], 5, 32, True), ([127, 1, 129], 140, 64, False),
                                                    ([1] * 300, 0, 64, True), ([0, 3, 0, 0, 300, 1, 0], 0, 72, True),
                                                    ([700, 513, 1, 0, 900], 0, 136, True), ([0, 1100], 1200, 8, True)])
def test_packed(lengths, behind, D, state, index, dtype):
    """Sequences of no and of one token, edges on and next to a tile's edge, rows behind the last sequence (zeros)."""
    N, rows = len(lengths), sum(lengths) + behind
    x, g, do, h0, dht = inputs(rows, D, N, dtype, rows, state)
    if behind:  # nothing of those rows may come through, whatever they hold
        x[-behind:] = float("nan")
        g[-behind:] = float("inf")
        X, G = x.clone(), g.clone()
        X[-behind:] = 0
        G[-behind:] = 0
    off = torch.tensor([sum(lengths[:i]) for i in range(N + 1)], dtype=index, device=DEV)
    if not behind:
        return check(x, g, do, h0, dht, lengths, dtype, (1, rows, D), off)
    outs = []
    for xx, gg in ((x, g), (X, G)):
        xs, gs = (v.to(DEV).view(1, rows, D).requires_grad_(True) for v in (xx, gg))
        o, ht = chunk_hgrn(xs, gs, initial_state=None if h0 is None else h0.to(DEV), output_final_state=True, cu_seqlens=off)
        dx, dg = torch.autograd.grad([o, ht], [xs, gs], [do.to(DEV).view_as(o), torch.ones_like(ht)])
        for v in (o, dx, dg):
            assert (v[0, -behind:] == 0).all()
        outs.append((o, ht, dx, dg))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    used = rows - behind
    if used:
        check(x[:used], g[:used], do[:used], h0, dht, lengths, dtype, (1, used, D), off)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_long_axis(dtype):
    """Hundreds of tiles along time and few channels: the look-back path. Against the same loop over halves with the state handed on
    (bitwise in the state's type is not required: the maps compose in another order)."""
    T, D = 40000, 20
    x, g, do, _, _ = inputs(T, D, 1, dtype, 5, False)
    xs, gs = x.to(DEV).view(1, T, D), g.to(DEV).view(1, T, D)
    o, ht = chunk_hgrn(xs, gs, output_final_state=True)
    want, last = loop(x.double(), g.double(), None, [T])
    near("o", o[0], want, dtype)
    near("ht", ht, last, torch.float32)
    o1, h1 = chunk_hgrn(xs[:, :12345], gs[:, :12345], output_final_state=True)
    o2, h2 = chunk_hgrn(xs[:, 12345:], gs[:, 12345:], initial_state=h1, output_final_state=True)
    near("handed on", torch.cat([o1, o2], 1)[0], want, dtype)
    near("handed on ht", h2, last, torch.float32)
    for _ in range(3):  # bit for bit, whatever block runs when
        again, ht2 = chunk_hgrn(xs, gs, output_final_state=True)
        assert torch.equal(again, o) and torch.equal(ht2, ht)


@pytest.mark.gpu
def test_gates_at_their_limits():
    """A gate of 0 (log -inf) forgets, a gate of 1 sums, gates above 1 grow; channels that hold nothing stay at nothing."""
    T, D = 300, 8
    g = torch.zeros(1, T, D)
    g[..., 0] = float("-inf")
    g[..., 1] = 0.0
    g[..., 2] = 0.1
    g[..., 3] = 60.0  # its products overflow
    g[..., 4] = -200.0
    x = torch.ones(1, T, D)
    x[..., 3] = 0.0
    h0 = torch.tensor([[9.0, 1.0, 0.0, 0.0, 5.0, 0.0, 0.0, 0.0]])
    o, ht = chunk_hgrn(x.to(DEV), g.to(DEV), initial_state=h0.to(DEV), output_final_state=True)
    want, last = loop(x[0].double(), g[0].double(), h0.double(), [T])
    assert torch.isfinite(o).all()
    # the same factor T times: its own error (2^-23) and a rounding a step add up the same way
    bound = 4 * T * 2.0 ** -24
    assert ((o[0].cpu().double() - want).abs() <= bound * want.abs()).all()
    assert ((ht.cpu().double() - last).abs() <= bound * last.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_sequences_do_not_touch_each_other(bad):
    """What is not finite stays inside its sequence, and stays there to the sequence's end even where the gates underflow."""
    T, D, cuts = 900, 40, [0, 130, 500, 700, 900]
    x, g, do, h0, dht = inputs(T, D, 4, torch.float32, 3, True)
    g[200:400] = -5.0  # e^-1000 in a tile
    off = torch.tensor(cuts, device=DEV)

    def run(x, do, h0):
        leaves = [v.to(DEV).requires_grad_(True) for v in (x.view(1, T, D), g.view(1, T, D), h0)]
        o, ht = chunk_hgrn(*leaves[:2], initial_state=leaves[2], output_final_state=True, offsets=off)
        return (o, ht, *torch.autograd.grad([o, ht], leaves, [do.to(DEV).view_as(o), dht.to(DEV)]))

    clean = run(x, do, h0)
    x2, do2, h2 = x.clone(), do.clone(), h0.clone()
    x2[150] = bad
    do2[499] = bad
    h2[3] = bad
    dirty = run(x2, do2, h2)
    for k, (a, b) in enumerate(zip(clean, dirty)):
        a, b = a.detach().reshape(-1, D), b.detach().reshape(-1, D)
        if len(a) == T:
            keep = [slice(0, 130), slice(500, 700)]
        else:
            keep = [slice(0, 1), slice(2, 3)]
        for s in keep:
            assert torch.equal(a[s], b[s]), k
    o, ht = dirty[0][0], dirty[1]
    assert not torch.isfinite(o[150:500]).any() and not torch.isfinite(o[700:]).any()
    assert not torch.isfinite(ht[1]).any() and not torch.isfinite(dirty[2][0, 130:500]).any()
    assert torch.equal(clean[0][0, :150], o[:150])


@pytest.mark.gpu
def test_gradient_against_differences():
    T, D = 150, 3
    x, g, do, h0, dht = inputs(T, D, 1, torch.float32, 3, True)
    off = torch.tensor([0, 40, T], device=DEV)
    h0 = torch.randn(2, D, generator=torch.Generator().manual_seed(1))
    args = [v.to(DEV) for v in (x.view(1, T, D), g.view(1, T, D), h0)]

    def f(*a):
        o, ht = chunk_hgrn(*a[:2], initial_state=a[2], output_final_state=True, offsets=off)
        return (o.double() * do.to(DEV).view_as(o).double()).sum() + (ht.double() ** 2).sum()

    leaves = [a.clone().requires_grad_(True) for a in args]
    grads = torch.autograd.grad(f(*leaves), leaves)
    gen = torch.Generator().manual_seed(2)
    for i, grad in enumerate(grads):
        way = torch.randn(args[i].shape, generator=gen).to(DEV)
        step = 2.0 ** -8
        up, down = ([a + (k * step * way if j == i else 0) for j, a in enumerate(args)] for k in (1, -1))
        diff = ((f(*up) - f(*down)) / (2 * step)).item()
        have = (grad.double() * way.double()).sum().item()
        # third-order term of the difference (step^2 of sums of the size of the value) and fp32 values divided by the step
        scale = (grad.double().abs() * way.double().abs()).sum().item()
        assert abs(diff - have) <= 2e-3 * scale + 1e-2, (i, diff, have, scale)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 31])
def test_tables_that_leave_the_tensor(D):
    """Offsets beyond the tensor are taken as its ends, and leading tokens of no sequence get zeros; nothing outside is touched."""
    T = 400
    x, g, do, h0, dht = inputs(T, D, 3, torch.float32, 3, True)
    bad = torch.tensor([-5, 150, 10 ** 6, 10 ** 6 + 3], dtype=torch.int32, device=DEV)
    good = torch.tensor([0, 150, T, T], dtype=torch.int64, device=DEV)
    late = torch.tensor([20, 150, 390, 390], dtype=torch.int32, device=DEV)

    def run(off):
        leaves = [v.to(DEV).requires_grad_(True) for v in (x.view(1, T, D), g.view(1, T, D), h0)]
        o, ht = chunk_hgrn(*leaves[:2], initial_state=leaves[2], output_final_state=True, offsets=off)
        return [o, ht, *torch.autograd.grad([o, ht], leaves, [do.to(DEV).view_as(o), dht.to(DEV)])]

    for a, b in zip(run(bad), run(good)):
        assert torch.equal(a, b)
    o, ht, dx, dg, dh0 = run(late)
    for v in (o, dx, dg):
        assert (v[0, :20] == 0).all() and (v[0, 390:] == 0).all() and (v[0, 20:390] != 0).any()
    want, last = loop(x[20:390].double(), g[20:390].double(), h0.double(), [130, 240, 0])
    near("o", o[0, 20:390], want, torch.float32)
    near("ht", ht, last, torch.float32)
    assert torch.equal(ht[2], h0[2].to(DEV)) and torch.equal(dh0[2], dht[2].to(DEV))


@pytest.mark.gpu
def test_strided_inputs_other_stream_and_graph():
    B, T, D = 2, 333, 48
    gen = torch.Generator().manual_seed(0)
    both = torch.randn(B, T, 2 * D, generator=gen).to(DEV)
    x, g = both[..., :D], -both[..., D:].abs()  # a slice of a joint projection
    want, hw = chunk_hgrn(x.contiguous(), g.contiguous(), output_final_state=True)
    got, hg = chunk_hgrn(x, g, output_final_state=True)
    assert torch.equal(got, want) and torch.equal(hg, hw)
    t = both.transpose(0, 1).contiguous().transpose(0, 1)
    got, _ = chunk_hgrn(t[..., :D], -t[..., D:].abs())
    assert torch.equal(got, want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got, _ = chunk_hgrn(x, g)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    # captured forward and backward of packed sequences, replayed on other values and other lengths; two graphs at once
    xs, gs = (v.reshape(1, B * T, D).clone().requires_grad_(True) for v in (x.contiguous(), g.contiguous()))
    off = torch.tensor([0, 100, B * T], dtype=torch.int32, device=DEV)
    w = torch.randn(1, B * T, D, generator=gen).to(DEV)

    def step():
        o, ht = chunk_hgrn(xs, gs, output_final_state=True, offsets=off)
        return (o.detach(), ht.detach(), *torch.autograd.grad([o, ht], [xs, gs], [w, ht.detach()]))

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
        off.copy_(torch.tensor([0, 511, B * T]))
    torch.cuda.synchronize()
    s2 = torch.cuda.Stream()
    graphs[0].replay()
    with torch.cuda.stream(s2):
        graphs[1].replay()
    torch.cuda.synchronize()
    want = step()
    for out in outs:
        for a, b in zip(out, want):
            assert (a.double() - b.double()).abs().max() <= STATE * max(1.0, b.abs().max().item())
    assert _lib.load().flab_tc_error_state() == 0


@pytest.mark.gpu
def test_decode_matches_one_pass():
    B, T, D = 4, 40, 96
    x, g, _, h0, _ = inputs(B * T, D, B, torch.bfloat16, 9, True)
    x, g, h0 = x.to(DEV).view(B, T, D), g.to(DEV).view(B, T, D), h0.to(DEV)
    want, last = chunk_hgrn(x, g, initial_state=h0, output_final_state=True)
    h, outs = h0, []
    for t in range(T):
        o, h = fused_recurrent_hgrn(x[:, t:t + 1], g[:, t:t + 1], initial_state=h, output_final_state=True)
        outs.append(o)
    near("ht", h, last.cpu(), torch.float32)
    near("o", torch.cat(outs, 1), want.cpu(), torch.bfloat16, halves=2.1)


@pytest.mark.gpu
def test_no_tokens():
    for shape, N in (((2, 0, 8), 2), ((0, 5, 8), 0), ((2, 5, 0), 2)):
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        h0 = torch.ones(N, shape[2], device=DEV, requires_grad=True)
        o, ht = chunk_hgrn(x, x, initial_state=h0, output_final_state=True)
        assert o.shape == shape and ht.shape == h0.shape
        if shape[1] == 0:
            assert torch.equal(ht, h0)
        dx, dh0 = torch.autograd.grad([o, ht], [x, h0], [torch.ones_like(o), torch.ones_like(ht)])
        assert dx.shape == shape and dh0.shape == h0.shape


@pytest.mark.gpu
@pytest.mark.parametrize("D", [2048, 2047])
def test_offsets_beyond_32_bits(D):
    """More than 2^31 elements (aligned rows, and rows that TMA cannot address): the ends against calls on the ends alone."""
    T, tail = 2 ** 31 // D + 5000, 3000
    x = torch.empty(1, T, D, dtype=torch.bfloat16, device=DEV).normal_()
    g = torch.empty_like(x).uniform_(-2, -0.1)
    off = torch.tensor([0, T - tail - 10, T], device=DEV)
    xs, gs = x.requires_grad_(True), g.requires_grad_(True)
    o, ht = chunk_hgrn(xs, gs, output_final_state=True, offsets=off)
    dx, dg = torch.autograd.grad(o, [xs, gs], x.detach())
    part = [v.detach()[:, -tail - 10:].clone().requires_grad_(True) for v in (x, g)]
    o2, h2 = chunk_hgrn(*part, output_final_state=True)
    dx2, dg2 = torch.autograd.grad(o2, part, part[0].detach())
    # the same rows in tiles that begin elsewhere: fp32 sums in another order, one rounding each
    near("o", o[0, -tail - 10:], o2[0].cpu(), torch.bfloat16, halves=2.1)
    near("ht", ht[1], h2[0].cpu(), torch.float32)
    near("dx", dx[0, -tail - 10:], dx2[0].cpu(), torch.bfloat16, halves=2.1)
    near("dg", dg[0, -tail - 10:], dg2[0].cpu(), torch.bfloat16, halves=4.2)
    head, _ = chunk_hgrn(x.detach()[:, :500], g.detach()[:, :500])
    near("head", o[0, :500], head[0].cpu(), torch.bfloat16, halves=2.1)


def test_refusals():
    x = torch.zeros(2, 4, 8)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        chunk_hgrn(x, x)
    with pytest.raises(ValueError, match=r"\[B, T, D\]"):
        chunk_hgrn(x, x[:, :3])
    with pytest.raises(ValueError, match="share one of the types"):
        chunk_hgrn(x, x.bfloat16())
    with pytest.raises(ValueError, match="share one of the types"):
        fused_recurrent_hgrn(x.double(), x.double())
    for big in (x[:1].expand(2 ** 32 + 1, 4, 8), x[:, :, :1].expand(2, 4, 2 ** 32 + 8)):
        with pytest.raises(ValueError, match="more than 2"):
            chunk_hgrn(big, big)
    with pytest.raises(ValueError, match="either"):
        chunk_hgrn(x, x, offsets=torch.tensor([0, 4]), cu_seqlens=torch.tensor([0, 4]))


def test_abi_refusals():
    lib = _lib.load()
    assert lib.flab_hgrn_fwd(None, None, None, None, None, None, 0, 1, 1, 1, 1, 0, None, 0, None) == -1
    assert b"positive" in lib.flab_last_error()
    assert lib.flab_hgrn_fwd(16, 16, None, 16, None, 16, 0, 2, 8, 8, 2, 0, None, 0, None) == -1
    assert b"B = 1" in lib.flab_last_error()
    # more than one tile along time needs the workspace
    assert lib.flab_hgrn_workspace(2, 32, 8) == 0 and lib.flab_hgrn_workspace(1, 1 << 14, 8) > 0
    assert lib.flab_hgrn_bwd(16, 16, None, 16, None, 16, 16, None, None, 0, 1, 1 << 14, 8, 1, 0, None, 0, None) == -1
    assert b"workspace" in lib.flab_last_error()
    assert lib.flab_hgrn_fwd(16, 16, None, 16, None, None, 0, 1, 8, 8, 1, 7, None, 0, None) == -1
    assert b"dtype" in lib.flab_last_error()
    assert math.isclose(STATE, 2.4e-5, rel_tol=0.01)


@pytest.mark.gpu
def test_refusals_on_the_device():
    x = torch.zeros(2, 4, 8, device=DEV)
    off = torch.tensor([0, 4], device=DEV)
    with pytest.raises(ValueError, match="batch size is expected to be 1"):
        chunk_hgrn(x, x, offsets=off)
    with pytest.raises(ValueError, match="number of initial states"):
        chunk_hgrn(x[:1], x[:1], offsets=off, initial_state=torch.zeros(2, 8, device=DEV))
    with pytest.raises(ValueError, match="int32 or int64"):
        chunk_hgrn(x[:1], x[:1], offsets=off.float())
    with pytest.raises(RuntimeError, match="expected cuda"):
        chunk_hgrn(x, x, initial_state=torch.zeros(2, 8))
