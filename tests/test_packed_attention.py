"""Attention inside the sequences of a packed batch, forward and backward: against the formulas in 64 bits at the sizes
and masks where it can go wrong, against differences, its refusals, graphs, and together with the cache."""
import ctypes
import math
import os

import pytest
import torch

from conftest import PKG

HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}        # largest relative error of one rounding


# ------------------------------------------------------------------------------------------------ CPU: refusals
def test_packed_validation_codes():
    path = os.path.join(PKG, "libbsa_b200.so")
    if not os.path.exists(path):
        pytest.skip("kernel library not built")
    lib = ctypes.CDLL(path)
    i, p, z = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t
    f = lib.bsa_packed_forward
    f.argtypes = [ctypes.c_int] + [p, i, i] * 3 + [p, p, p, p] + [i] * 5 + [ctypes.c_float, ctypes.c_int, p, z, p]

    def call(dtype=1, q=32, strides=(1024, 128), o=32, offsets=16, rows=10, batch=1, heads=8, kv=4, dim=128, ws=16, ws_bytes=256, low=32):
        return f(dtype, q, *strides, 32, *strides, 32, *strides, o, low, 32, offsets, rows, batch, heads, kv, dim, 1.0, 1, ws, ws_bytes, None)

    assert call(dtype=0) == 3 and call(dim=96) == 4 and call(heads=6) == 4 and call(kv=0) == 4 and call(rows=-1) == 4
    assert call(batch=-1) == 4 and call(rows=2 ** 31) == 10 and call(rows=2 ** 30, heads=65532, kv=4) == 10
    assert call(low=None) == 1 and call(low=48) == 6             # lse without the rest of o
    assert call(q=None) == 1 and call(o=None) == 1 and call(offsets=None) == 1
    assert call(q=24) == 6 and call(o=16) == 6 and call(strides=(1023, 128)) == 6 and call(strides=(0, 128)) == 4
    assert call(ws=None) == 7 and call(ws_bytes=0) == 7
    assert call(rows=0) == 0

    g = lib.bsa_packed_backward
    g.argtypes = [ctypes.c_int] + [p, i, i] * 3 + [p, p, p, i, i] + [p] * 5 + [i] * 5 + [ctypes.c_float, ctypes.c_int, p, z, p, z, p]

    def back(dtype=1, dout=32, dk=32, lse=32, rows=10, heads=8, stats=32, stats_bytes=1 << 20, low=32):
        return g(dtype, 32, 1024, 128, 32, 512, 128, 32, 512, 128, 32, low, dout, 1024, 128, lse, 32, dk, 32, 32, rows, 1, heads, 4, 128,
                 1.0, 1, stats, stats_bytes, 16, 256, None)

    assert back(dtype=0) == 3 and back(heads=9) == 4 and back(dout=None) == 1 and back(lse=None) == 1 and back(low=None) == 1 and back(stats=None) == 1
    assert back(dk=48) == 6 and back(stats_bytes=10 * 8 * 8 - 1) == 7 and back(rows=0) == 0


def test_packed_number_of_sequences():
    """Finding the work takes time that grows with the square of the number of sequences: one that would hold the device
    for minutes is refused."""
    path = os.path.join(PKG, "libbsa_b200.so")
    if not os.path.exists(path):
        pytest.skip("kernel library not built")
    lib = ctypes.CDLL(path)
    i, p, z = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t
    lib.bsa_packed_forward.argtypes = [ctypes.c_int] + [p, i, i] * 3 + [p, p, p, p] + [i] * 5 + [ctypes.c_float, ctypes.c_int, p, z, p]
    lib.bsa_packed_backward.argtypes = [ctypes.c_int] + [p, i, i] * 3 + [p, p, p, i, i] + [p] * 5 + [i] * 5 + [ctypes.c_float, ctypes.c_int, p, z, p, z, p]
    for batch, code in ((65537, 10), (2 ** 24, 10), (65536, 1)):       # (without queries: the sizes are looked at first)
        assert lib.bsa_packed_forward(1, None, 1024, 128, 32, 512, 128, 32, 512, 128, 32, None, None, 32, 10, batch, 8, 4, 128, 1.0, 1,
                                      16, 256, None) == code
        assert lib.bsa_packed_backward(1, None, 1024, 128, 32, 512, 128, 32, 512, 128, 32, 32, 32, 1024, 128, 32, 32, 32, 32, 32, 10,
                                       batch, 8, 4, 128, 1.0, 1, 32, 1 << 20, 16, 256, None) == code


def test_python_refusals_without_a_gpu():
    from sparse import packed_attention
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        packed_attention(x, x, x, torch.tensor([0, 4], dtype=torch.int32))


def test_forward_mode_derivatives_are_refused():
    """A dual tensor does not require grad: its derivative would be dropped without a word."""
    import torch.autograd.forward_ad as fwd
    from sparse import packed_attention
    x = torch.zeros(4, 2, 64, dtype=torch.float16)
    offsets = torch.tensor([0, 4], dtype=torch.int32)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        for args in ((dual, x, x), (x, dual, x), (x, x, dual), (dual, x.clone().requires_grad_(), x)):
            with pytest.raises(RuntimeError, match="forward-mode"):
                packed_attention(*args, offsets)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                packed_attention(*args, offsets)


# ------------------------------------------------------------------------------------------------ GPU
def _status():
    from sparse.kernel import sparse_ops
    torch.cuda.synchronize()
    sparse_ops.check_device_status(0)


def _inputs(lengths, tail, hq, hk, dim, dtype, seed, spread=1.0):
    gen = torch.Generator().manual_seed(seed)
    rows = sum(lengths) + tail
    q, do = (torch.randn(rows, hq, dim, generator=gen).mul(spread).to(dtype) for _ in range(2))
    k, v = (torch.randn(rows, hk, dim, generator=gen).mul(spread).to(dtype) for _ in range(2))
    offsets = torch.tensor([0] + lengths).cumsum(0).to(torch.int32)
    return q, k, v, do, offsets


def _reference(q, k, v, do, lengths, scale, causal):
    """(o, dq, dk, dv) in 64 bits, and bounds on the kernels' errors."""
    u = HALF[q.dtype]
    g = q.size(1) // k.size(1)
    q, k, v, do = (t.double().cuda() for t in (q, k, v, do))
    out = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
    bound = [torch.zeros_like(t) for t in out]
    start = 0
    d = q.size(2)
    # below 2^-14 fp16 rounds in steps of 2^-24, whatever the value
    tiny = 2.0 ** -25 if u == 2.0 ** -11 else 0.0
    for n in lengths:
        r = slice(start, start + n)
        start += n
        if n == 0:
            continue
        seen = torch.ones(n, n, dtype=torch.bool, device="cuda")
        if causal:
            seen = seen.tril()
        for h in range(q.size(1)):
            qh, kh, vh, doh = q[r, h], k[r, h // g], v[r, h // g], do[r, h]
            p = torch.softmax((qh @ kh.T * scale).masked_fill(~seen, -math.inf), -1)
            o = p @ vh
            # fp32: a score is off by (d + 8) steps of its sum of magnitudes, relative in the weight and again in the row's
            # sum; 2^-20 for the exponential; P rounded once to 16 bits (relative u; in fp16 also 2^-25 of 2^8 at most,
            # the running maximum being kept within 2^8)
            off = 2 * (d + 8) * 2.0 ** -24 * ((qh.abs() @ kh.abs().T) * abs(scale) * seen).amax(-1, keepdim=True) + 2.0 ** -20
            p_max = p.amax(-1, keepdim=True)
            floor = tiny * p_max                            # an unnormalised weight 1 stands for at least p_max / 2^8 .. p_max
            e_p = (u + off) * p + floor * seen              # error of the weights that multiply V, per element
            sums = n * 2.0 ** -24                           # fp32 accumulation over n terms
            out[0][r, h] = o
            w = p @ vh.abs()
            bound[0][r, h] = u * o.abs() + (1 + u) * (e_p @ vh.abs() + (off + sums) * w) + tiny
            # gradients
            dp = doh @ vh.T
            delta = (doh * o).sum(-1, keepdim=True)
            ds = p * (dp - delta) * seen
            # P of the backward is fp32 (error off), lse's error is in off; delta is made from the rounded output
            e_delta = (doh.abs() * bound[0][r, h]).sum(-1, keepdim=True) + d * 2.0 ** -24 * (doh.abs() @ vh.abs().T * seen).amax(-1, keepdim=True)
            e_dp = d * 2.0 ** -24 * (doh.abs() @ vh.abs().T)
            e_ds = (off * 2 + u) * ds.abs() + p * (e_delta + e_dp) * (1 + u) + tiny * seen
            dq = ds @ kh * scale
            out[1][r, h] = dq
            bound[1][r, h] = u * dq.abs() + abs(scale) * (1 + u) * (e_ds @ kh.abs() + sums * (ds.abs() @ kh.abs())) + tiny
            out[2][r, h // g] += ds.T @ qh * scale
            bound[2][r, h // g] += abs(scale) * (1 + u) * (e_ds.T @ qh.abs() + g * sums * (ds.abs().T @ qh.abs()))
            # the backward's weights are normalised: fp16 rounds them in steps of 2^-24 from 2^-14 down
            e_pb = (u + 2 * off) * p + tiny * seen
            out[3][r, h // g] += p.T @ doh
            bound[3][r, h // g] += (1 + u) * (e_pb.T @ doh.abs() + g * sums * (p.T @ doh.abs()))
    for i in (2, 3):
        bound[i] += u * out[i].abs() + tiny
    return out, bound


def _check(got, reference):
    for name, x, ref, bound in zip(("out", "dq", "dk", "dv"), got, *reference):
        x = x.double()
        assert x.isfinite().all(), name
        over = (x - ref).abs() - bound
        assert (over <= 0).all(), "%s: off by %.3e more than the bound at %s" % (
            name, over.max(), [int(i) for i in torch.unravel_index(over.argmax(), over.shape)])


def _run(q, k, v, do, offsets, scale, causal):
    from sparse import packed_attention
    q, k, v = (t.cuda().requires_grad_() for t in (q, k, v))
    out = packed_attention(q, k, v, offsets.cuda(), scale, causal)
    return (out.detach(),) + torch.autograd.grad(out, (q, k, v), do.cuda())


CASES = [
    # lengths, rows behind, q heads, kv heads, dim, causal
    ([1], 0, 1, 1, 64, True),
    ([1, 2, 1, 0, 3], 0, 2, 2, 128, True),
    ([127, 128, 129], 0, 2, 1, 64, True),
    ([127, 128, 129], 3, 2, 1, 128, False),
    ([255, 256, 257, 5], 0, 3, 3, 128, True),
    ([300, 0, 0, 77, 513], 200, 6, 2, 64, True),
    ([300, 0, 0, 77, 513], 130, 8, 2, 128, True),
    ([40] * 70, 1, 5, 1, 64, False),
    ([1000, 31], 0, 4, 4, 64, True),
    ([1000, 31], 0, 4, 1, 128, True),
    ([640, 641], 7, 1, 1, 128, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths,tail,hq,hk,dim,causal", CASES)
def test_packed_attention_and_gradients(dtype, lengths, tail, hq, hk, dim, causal):
    q, k, v, do, offsets = _inputs(lengths, tail, hq, hk, dim, dtype, len(lengths))
    got = _run(q, k, v, do, offsets, dim ** -0.5, causal)
    _status()
    _check(got, _reference(q, k, v, do, lengths, dim ** -0.5, causal))
    if tail:
        for t in got:
            assert (t[sum(lengths):] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.3, 0.0, 1.5])
def test_other_scales(scale):
    """A negative scale (the largest score is the smallest product), none, and one that makes rows peaked."""
    lengths = [200, 131]
    q, k, v, do, offsets = _inputs(lengths, 0, 4, 2, 64, torch.bfloat16, 3, spread=0.7)
    got = _run(q, k, v, do, offsets, scale, True)
    _status()
    _check(got, _reference(q, k, v, do, lengths, scale, True))


@pytest.mark.gpu
def test_rising_scores_rescale_the_output():
    """Keys that grow along the sequence: the running maximum rises by far more than the lazy threshold, many times."""
    lengths = [700]
    q, k, v, do, offsets = _inputs(lengths, 0, 2, 2, 128, torch.bfloat16, 4)
    k = (k.double() * torch.linspace(0.1, 12.0, 700)[:, None, None]).to(k.dtype)
    got = _run(q, k, v, do, offsets, 128 ** -0.5, True)
    _status()
    _check(got, _reference(q, k, v, do, lengths, 128 ** -0.5, True))


@pytest.mark.gpu
def test_gradients_against_differences():
    """The gradient of sum(o * do) along random directions, by central differences of the 64-bit formula."""
    lengths, scale = [150, 40], 0.125
    q, k, v, do, offsets = _inputs(lengths, 0, 4, 2, 64, torch.float16, 6)
    _, dq, dk, dv = (t.double().cpu() for t in _run(q, k, v, do, offsets, scale, True))

    def loss(q, k, v):
        total, start = 0.0, 0
        for n in lengths:
            r = slice(start, start + n)
            start += n
            seen = torch.ones(n, n, dtype=torch.bool).tril()
            s = torch.einsum("ihd,jhd->hij", q[r], k[r].repeat_interleave(2, 1)) * scale
            p = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
            total = total + (torch.einsum("hij,jhd->ihd", p, v[r].repeat_interleave(2, 1)) * do[r].double()).sum()
        return total

    x = [t.double() for t in (q, k, v)]
    gen = torch.Generator().manual_seed(1)
    for i, grad in enumerate((dq, dk, dv)):
        direction = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
        step = 1e-4
        up, down = list(x), list(x)
        up[i], down[i] = x[i] + step * direction, x[i] - step * direction
        slope = (loss(*up) - loss(*down)) / (2 * step)
        # roundings of the gradient are independent: their sum along the direction has at most a few times the size of
        # (4 roundings of relative 2^-11) x |grad| x |direction| / sqrt(n) x sqrt(n)
        assert abs((grad * direction).sum() - slope) <= 4 * 2.0 ** -11 * 6 * grad.norm() + 1e-4, i


@pytest.mark.gpu
def test_gradients_of_views_and_of_broadcast_heads():
    """q, k, v as views of one projection; k and v broadcast over heads; a gradient that is a broadcast; transposed rows."""
    from sparse import packed_attention
    lengths = [130, 70, 9]
    q, k, v, do, offsets = _inputs(lengths, 2, 4, 2, 64, torch.bfloat16, 7)
    want = _run(q, k, v, do, offsets, 0.125, True)
    fused = torch.cat([q, k, v], 1).cuda().requires_grad_()
    out = packed_attention(*fused.split([4, 2, 2], 1), offsets.cuda(), 0.125)
    (grad,) = torch.autograd.grad(out, fused, do.cuda())
    assert torch.equal(out, want[0]) and torch.equal(grad, torch.cat(want[1:], 1))
    # heads first in memory, rows on odd places
    for make in (lambda t: t.transpose(0, 1).contiguous().transpose(0, 1),
                 lambda t: torch.cat([t[..., :1], t, t[..., :2]], -1)[..., 1:65]):
        laid = [make(t.cuda()).detach().requires_grad_() for t in (q, k, v)]
        out = packed_attention(*laid, offsets.cuda(), 0.125)
        got = torch.autograd.grad(out, laid, make(do.cuda()))
        assert torch.equal(out, want[0]) and all(torch.equal(a, b) for a, b in zip(got, want[1:]))
    # one key head seen by all query heads through expand
    one_k, one_v = (t[:, :1].cuda().requires_grad_() for t in (k, v))
    out = packed_attention(q.cuda(), one_k.expand(-1, 2, -1), one_v.expand(-1, 2, -1), offsets.cuda(), 0.125)
    dk, dv = torch.autograd.grad(out, (one_k, one_v), do.cuda())
    plain = _run(q, k[:, :1].expand(-1, 2, -1).contiguous(), v[:, :1].expand(-1, 2, -1).contiguous(), do, offsets, 0.125, True)
    assert torch.equal(out, plain[0]) and torch.equal(dk, plain[2].sum(1, keepdim=True)) and torch.equal(dv, plain[3].sum(1, keepdim=True))
    # sum().backward(): the gradient of the output is one element, broadcast
    a = [t.cuda().requires_grad_() for t in (q, k, v)]
    packed_attention(*a, offsets.cuda(), 0.125).sum().backward()
    ones = _run(q, k, v, torch.ones_like(do), offsets, 0.125, True)
    assert all(torch.equal(t.grad, w) for t, w in zip(a, ones[1:]))
    _status()


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_a_sequence_of_no_numbers_stays_alone(dim):
    """NaN and infinities in one sequence leave its neighbours as they were, forward and backward."""
    lengths = [100, 131, 0, 1, 60]
    q, k, v, do, offsets = _inputs(lengths, 3, 4, 2, dim, torch.float16, 8)
    want = _run(q, k, v, do, offsets, 0.1, True)
    bad = slice(100, 231)
    for t in (q, k, v, do):
        t[bad] = math.nan
        t[bad][::3] = math.inf
        t[-3:] = math.nan                                  # rows that belong to nobody
    got = _run(q, k, v, do, offsets, 0.1, True)
    for a, b in zip(got, want):
        assert torch.equal(a[:100], b[:100]) and torch.equal(a[231:], b[231:])
    assert got[0][bad].isnan().all()
    _status()


@pytest.mark.gpu
def test_repeats_streams_and_small_calls():
    from sparse import packed_attention
    lengths = [513, 200, 3]
    q, k, v, do, offsets = _inputs(lengths, 0, 8, 2, 128, torch.bfloat16, 9)
    want = _run(q, k, v, do, offsets, 0.1, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, do, offsets, 0.1, True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    empty = torch.zeros(0, 8, 128, dtype=torch.bfloat16, device="cuda")
    none = torch.zeros(1, dtype=torch.int32, device="cuda")
    assert packed_attention(empty, empty[:, :2], empty[:, :2], none).shape == (0, 8, 128)
    x = torch.ones(5, 8, 128, dtype=torch.bfloat16, device="cuda")
    assert (packed_attention(x, x, x, none) == 0).all()    # no sequences: every row is behind the last one
    _status()


@pytest.mark.gpu
def test_offsets_that_are_none_are_reported():
    from sparse import packed_attention
    from sparse.kernel import sparse_ops
    x = torch.ones(300, 2, 64, dtype=torch.float16, device="cuda", requires_grad=True)
    for bad in ([0, 301], [0, 200, 100, 300], [5, 300], [0, -7, 300], [0, 2 ** 31 - 1]):
        out = packed_attention(x, x, x, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        with pytest.raises(RuntimeError):
            sparse_ops.check_device_status(0)
        out.backward(torch.ones_like(out))
        with pytest.raises(RuntimeError):
            sparse_ops.check_device_status(0)
    _status()


@pytest.mark.gpu
def test_gpu_refusals():
    from sparse import packed_attention
    x = torch.ones(8, 4, 64, dtype=torch.float16, device="cuda")
    offsets = torch.tensor([0, 8], dtype=torch.int32, device="cuda")
    for q, k, v, o in ((x.float(), x.float(), x.float(), offsets), (x, x.bfloat16(), x, offsets), (x, x[:, :3], x[:, :3], offsets),
                       (x, x, x[:, :2], offsets), (x, x[:7], x[:7], offsets), (x[..., :32], x[..., :32], x[..., :32], offsets),
                       (x, x, x, offsets.long()), (x, x, x, offsets.cpu()), (x, x, x, offsets[:0]), (x[0], x[0], x[0], offsets),
                       (x, x[:, :0], x[:, :0], offsets)):
        with pytest.raises(RuntimeError):
            packed_attention(q, k, v, o)
    a = x.clone().requires_grad_()
    out = packed_attention(a, a, a, offsets)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.sum(), a, create_graph=True)
    _status()


@pytest.mark.gpu
def test_which_inputs_learn_and_debug_checks():
    from sparse import kernel, packed_attention
    lengths = [90, 41]
    q, k, v, do, offsets = _inputs(lengths, 0, 4, 2, 64, torch.bfloat16, 13)
    want = _run(q, k, v, do, offsets, 0.125, True)
    q, k, v, do, offsets = (t.cuda() for t in (q, k, v, do, offsets))
    with torch.no_grad():
        assert not packed_attention(q.requires_grad_(), k, v, offsets, 0.125).requires_grad
    q.requires_grad_(False)
    assert not packed_attention(q, k, v, offsets, 0.125).requires_grad
    for learns in range(3):
        x = [t.detach().requires_grad_(i == learns) for i, t in enumerate((q, k, v))]
        out = packed_attention(*x, offsets, 0.125)
        out.backward(do)
        assert torch.equal(out, want[0])
        for i in range(3):
            assert torch.equal(x[i].grad, want[1 + i]) if i == learns else x[i].grad is None
    kernel.debug_checks = True
    try:
        x = [t.detach().requires_grad_() for t in (q, k, v)]
        packed_attention(*x, offsets, 0.125).backward(do)
        with pytest.raises(RuntimeError):
            packed_attention(*x, torch.tensor([0, 200], dtype=torch.int32, device="cuda"))
    finally:
        kernel.debug_checks = False
    _status()


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore:The AccumulateGrad node's stream does not match")
def test_training_step_in_a_graph_follows_its_offsets():
    from sparse import packed_attention
    q, k, v, do, _ = _inputs([400], 0, 4, 2, 128, torch.bfloat16, 11)
    q, k, v = (t.cuda().requires_grad_() for t in (q, k, v))
    do = do.cuda()
    offsets = torch.tensor([0, 100, 390, 400], dtype=torch.int32, device="cuda")

    def step():
        out = packed_attention(q, k, v, offsets, 0.1)
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), do)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for lengths in ([0, 100, 390, 400], [0, 0, 129, 300], [0, 398, 399, 400]):
        offsets.copy_(torch.tensor(lengths, dtype=torch.int32))
        want = [t.clone() for t in step()]
        for t in captured:
            t.fill_(7)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(captured, want))
    _status()


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore:The AccumulateGrad node's stream does not match")
@pytest.mark.parametrize("through", ["grad", "backward", "a layer before"])
def test_capture_beside_a_living_eager_graph_is_refused(through):
    """The accumulation nodes of the leaves belong to the default stream as long as the eager graph lives."""
    from sparse import packed_attention
    q, k, v, do, offsets = _inputs([100, 28], 0, 4, 2, 64, torch.bfloat16, 21)
    q, k, v = (t.cuda().requires_grad_() for t in (q, k, v))
    do, offsets = do.cuda(), offsets.cuda()

    def forward():
        return packed_attention(*((t * 2 for t in (q, k, v)) if through == "a layer before" else (q, k, v)), offsets, 0.1)

    def backward(out):
        if through == "grad":
            return torch.autograd.grad(out, (q, k, v), do)
        for t in (q, k, v):
            t.grad = None
        out.backward(do)
        return q.grad, k.grad, v.grad

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = [t.clone() for t in backward(forward())]
    torch.cuda.current_stream().wait_stream(side)
    eager = forward()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = forward()
        with pytest.raises(RuntimeError, match="recorded on the default"):
            backward(out)
    del out, eager
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = backward(forward())
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, want))
    _status()


@pytest.mark.gpu
def test_prompt_then_tokens_matches_the_whole():
    """Prompts attended to at once and written to a 16-bit cache, then three tokens each one by one: the rows equal those
    of the whole sequences attended to at once, within the roundings of both."""
    from sparse import cache_slots, cache_write, cached_attention, make_cache, packed_attention
    prompts, more, hq, hk, dim, page, dtype = [70, 1, 200], 3, 4, 2, 64, 16, torch.float16
    full = [n + more for n in prompts]
    q, k, v, _, offsets = _inputs(full, 0, hq, hk, dim, dtype, 12)
    reference, bound = _reference(q, k, v, torch.zeros_like(q), full, 0.125, True)
    q, k, v = q.cuda(), k.cuda(), v.cuda()
    cache = make_cache(40, page, hk, dim, dtype)
    table = torch.randperm(40)[:39].view(3, 13).to(torch.int32).cuda()
    seq = torch.cat([torch.full((n,), i) for i, n in enumerate(full)]).cuda()
    at = torch.cat([torch.arange(n) for n in full]).cuda()
    prompt = at < torch.tensor(prompts, device="cuda")[seq]
    got = torch.empty_like(q)
    with torch.no_grad():
        starts = torch.tensor([0] + prompts).cumsum(0).to(torch.int32).cuda()
        got[prompt] = packed_attention(q[prompt], k[prompt], v[prompt], starts, 0.125)
        cache_write(k[prompt], v[prompt], cache_slots(table, seq[prompt], at[prompt], page), *cache)
        for t in range(more):
            rows = offsets[:-1].long().cuda() + torch.tensor(prompts, device="cuda") + t
            cache_write(k[rows], v[rows], cache_slots(table, seq[rows], at[rows], page), *cache)
            lengths = (at[rows] + 1).to(torch.int32)
            got[rows] = cached_attention(q[rows][:, None], *cache, table, lengths, scale=0.125)[:, 0]
    _status()
    over = (got.double() - reference[0]).abs() - bound[0]
    assert (over <= 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,tail,hq,hk,dim", [([0] * 3000 + [5, 0, 300] + [0] * 2000 + [129], 0, 2, 1, 64),
                                                    ([0] * 700 + [257] + [0] * 300, 140, 12, 12, 128)])
def test_many_places_behind_the_end_of_the_list(lengths, tail, hq, hk, dim):
    """The grid is an upper bound of the tiles: with thousands of empty sequences a CTA meets the list's end again and
    again, and every tile that it is handed before or after is still made."""
    q, k, v, do, offsets = _inputs(lengths, tail, hq, hk, dim, torch.bfloat16, 17)
    got = _run(q, k, v, do, offsets, dim ** -0.5, True)
    _status()
    _check(got, _reference(q, k, v, do, lengths, dim ** -0.5, True))
    for t in got:
        assert (t[sum(lengths):] == 0).all()


@pytest.mark.gpu
def test_as_many_sequences_as_there_may_be():
    """65536 sequences of one row: a row's only weight is 1, so its output is its value and dV is dO, bit for bit."""
    n, dim, scale = 65536, 64, 0.125
    q, k, v, do, offsets = _inputs([1] * n, 0, 1, 1, dim, torch.float16, 19)
    out, dq, dk, dv = _run(q, k, v, do, offsets, scale, True)
    _status()
    assert torch.equal(out.cpu(), v) and torch.equal(dv.cpu(), do)
    # dP and delta are the same sum in another order: 2 dim steps of its magnitudes, and once rounded to fp16
    off = 2 * dim * 2.0 ** -24 * (do.double().abs() * v.double().abs()).sum(-1, keepdim=True) + 2.0 ** -25
    assert (dq.double().cpu().abs() <= scale * 1.01 * off * k.double().abs() + 2.0 ** -25).all()
    assert (dk.double().cpu().abs() <= scale * 1.01 * off * q.double().abs() + 2.0 ** -25).all()
