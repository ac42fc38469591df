"""Out-of-bounds write check without a sanitizer: every output buffer of the C-ABI entry points sits
between two guard regions filled with a sentinel; after the call the guards must be untouched and
the output must equal the one computed into a plain buffer.  Covers the three matmul engines (tcgen05
block 64 and block 32, CUDA cores), every mode, the softmax forward / backward and the fused
attention forward and backward, on a layout with an empty block row and an empty block column; packed
attention forward and backward with odd lengths, empty sequences and rows behind the last; the paged
cache written and read up to its first and last place; and attention over it, with whole and split
sequences and a scratch of just the bytes asked for."""
import ctypes
import os

import pytest
import torch

from conftest import PKG, load_golden_layout

pytestmark = pytest.mark.gpu

GUARD = 4096          # elements on either side
MATMUL_ARGS = [ctypes.c_int] * 4 + [ctypes.c_void_p] * 5 + [ctypes.c_int64] * 6 + \
    [ctypes.c_int, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.c_void_p]


def _library():
    lib = ctypes.CDLL(os.path.join(PKG, "libbsa_b200.so"))
    lib.bsa_matmul.argtypes = MATMUL_ARGS
    lib.bsa_softmax_forward.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                        ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_int64,
                                        ctypes.c_int, ctypes.c_float, ctypes.c_int, ctypes.c_void_p,
                                        ctypes.c_int64, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p]
    lib.bsa_softmax_backward.argtypes = [ctypes.c_int, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p,
                                         ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64,
                                         ctypes.c_int64, ctypes.c_int, ctypes.c_float, ctypes.c_int64, ctypes.c_void_p]
    lib.bsa_attention_forward.argtypes = [ctypes.c_int] + [ctypes.c_void_p] * 7 + [ctypes.c_int64] * 5 + \
        [ctypes.c_int, ctypes.c_float, ctypes.c_int, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_int,
         ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    lib.bsa_attention_backward.argtypes = [ctypes.c_int] + [ctypes.c_void_p] * 13 + [ctypes.c_int64] * 5 + \
        [ctypes.c_int, ctypes.c_float, ctypes.c_int, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_int,
         ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_void_p]
    lib.bsa_workspace_status.argtypes = [ctypes.c_void_p, ctypes.c_void_p]
    return lib


class Guarded:
    """An output tensor of `shape` inside a larger allocation whose margins hold a sentinel."""

    def __init__(self, shape, dtype):
        n = 1
        for s in shape:
            n *= s
        self.sentinel = 123.0 if dtype != torch.float32 else 12345.0
        self.raw = torch.full((n + 2 * GUARD,), self.sentinel, device="cuda", dtype=dtype)
        self.view = self.raw[GUARD:GUARD + n].view(shape)
        self.view.fill_(float("nan"))

    def check(self, what):
        torch.cuda.synchronize()
        assert bool((self.raw[:GUARD] == self.sentinel).all()), "%s wrote below its output" % what
        assert bool((self.raw[-GUARD:] == self.sentinel).all()), "%s wrote above its output" % what
        assert not bool(torch.isnan(self.view.float()).any()), "%s left part of its output unwritten" % what


@pytest.mark.parametrize("block,dtype,engine", [(64, torch.float16, 2), (32, torch.float32, 2), (32, torch.float16, 2),
                                                (64, torch.float32, 1), (128, torch.float16, 1)])
@pytest.mark.parametrize("mode", ["sdd", "dsd", "dds"])
def test_matmul_writes_only_its_output(block, dtype, engine, mode):
    from sparse import SparseLayout
    lib = _library()
    pattern = torch.tensor(load_golden_layout("empty_row_col_5x4")["pattern"])
    layout = SparseLayout(pattern, block=block)
    rows, cols = pattern.shape[0] * block, pattern.shape[1] * block
    nnz, z, d = layout.num_blocks, 3, 64
    code = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}[dtype]
    gen = torch.Generator(device="cuda").manual_seed(3)
    rnd = lambda *shape: torch.randn(*shape, device="cuda", generator=gen).to(dtype)
    ws = torch.zeros(256, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    if mode == "sdd":       # blocks = A[rows, d] . B[cols, d]^T
        a, b, out_shape = rnd(z, rows, d), rnd(z, cols, d), (z, nnz, block, block)
        m, n, k, flags, (blk, tab) = rows, cols, d, (0, 0, 1), layout.row_layout
    elif mode == "dsd":     # C[rows, d] = blocks . B[cols, d]
        a, b, out_shape = rnd(z, nnz, block, block), rnd(z, cols, d), (z, rows, d)
        m, n, k, flags, (blk, tab) = rows, d, cols, (1, 0, 0), layout.row_layout
    else:                   # C[d, cols] = A[rows, d]^T . blocks
        a, b, out_shape = rnd(z, rows, d), rnd(z, nnz, block, block), (z, d, cols)
        m, n, k, flags, (blk, tab) = d, cols, rows, (2, 1, 0), layout.col_layout
    out = Guarded(out_shape, dtype)
    st = lib.bsa_matmul(flags[0], code, flags[1], flags[2], a.data_ptr(), b.data_ptr(), out.view.data_ptr(),
                        blk.data_ptr(), tab.data_ptr(), nnz, tab.numel() - 1, z, m, n, k, block,
                        ws.data_ptr(), 256, engine, stream)
    assert st == 0, st
    out.check("%s block %d %s engine %d" % (mode, block, dtype, engine))
    assert lib.bsa_workspace_status(ws.data_ptr(), stream) == 0
    from sparse.kernel import sparse_ops
    names = {1: "simt", 2: "tcgen05"}
    ref = sparse_ops.sparse_matmul(a, b, mode, layout.row_layout, layout.col_layout, bool(flags[1]), bool(flags[2]),
                                   block, names[engine])
    assert torch.equal(out.view, ref)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_softmax_and_attention_write_only_their_outputs(dtype):
    from sparse import SparseLayout
    from sparse.kernel import sparse_ops
    lib = _library()
    pattern = torch.tensor(load_golden_layout("empty_row_col_5x4")["pattern"])
    block = 64
    layout = SparseLayout(pattern, block=block)
    nnz, z = layout.num_blocks, 4
    code = {torch.float32: 0, torch.float16: 1}[dtype]
    blk, tab = layout.row_layout
    stream = torch.cuda.current_stream().cuda_stream
    gen = torch.Generator(device="cuda").manual_seed(4)
    x = torch.randn(z, nnz, block, block, device="cuda", generator=gen).to(dtype)
    dy = torch.randn(z, nnz, block, block, device="cuda", generator=gen).to(dtype)
    y = Guarded((z, nnz, block, block), dtype)
    st = lib.bsa_softmax_forward(code, x.data_ptr(), y.view.data_ptr(), blk.data_ptr(), tab.data_ptr(), nnz,
                                 pattern.shape[0], z, block, 0.5, 0, None, 0, 0, layout.max_row_blocks, stream)
    assert st == 0, st
    y.check("softmax forward")
    assert torch.equal(y.view, sparse_ops.sparse_softmax_forward(x, blk, tab, 0.5, False, None, layout.max_row_blocks))
    dx = Guarded((z, nnz, block, block), dtype)
    st = lib.bsa_softmax_backward(code, y.view.data_ptr(), dy.data_ptr(), dx.view.data_ptr(), blk.data_ptr(),
                                  tab.data_ptr(), nnz, pattern.shape[0], z, block, 0.5, layout.max_row_blocks, stream)
    assert st == 0, st
    dx.check("softmax backward")
    if dtype != torch.float16:
        return
    d = 128
    q = torch.randn(z, pattern.shape[0] * block, d, device="cuda", generator=gen).half()
    k = torch.randn(z, pattern.shape[1] * block, d, device="cuda", generator=gen).half()
    v = torch.randn(z, pattern.shape[1] * block, d, device="cuda", generator=gen).half()
    o = Guarded((z, pattern.shape[0] * block, d), torch.float16)
    lse = Guarded((z, pattern.shape[0] * block), torch.float32)
    lse.view.fill_(0.0)            # (-inf is a legal value of this output)
    ws = torch.zeros(256, dtype=torch.uint8, device="cuda")
    st = lib.bsa_attention_forward(1, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.view.data_ptr(), lse.view.data_ptr(),
                                   blk.data_ptr(), tab.data_ptr(), nnz, pattern.shape[0], pattern.shape[1], z, d, block,
                                   0.1, 0, None, 0, 0, 0, ws.data_ptr(), 256, stream)
    assert st == 0, st
    o.check("attention forward output")
    torch.cuda.synchronize()
    assert bool((lse.raw[:GUARD] == lse.sentinel).all()) and bool((lse.raw[-GUARD:] == lse.sentinel).all())
    assert lib.bsa_workspace_status(ws.data_ptr(), stream) == 0
    # fused backward: three gradient outputs and the statistics scratch
    do = torch.randn(z, pattern.shape[0] * block, d, device="cuda", generator=gen).half()
    cblk, ctab = layout.col_layout
    dq = Guarded((z, pattern.shape[0] * block, d), torch.float16)
    dk = Guarded((z, pattern.shape[1] * block, d), torch.float16)
    dv = Guarded((z, pattern.shape[1] * block, d), torch.float16)
    stats = Guarded((z, pattern.shape[0] * block, 2), torch.float32)
    st = lib.bsa_attention_backward(1, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.view.data_ptr(), do.data_ptr(),
                                    lse.view.data_ptr(), dq.view.data_ptr(), dk.view.data_ptr(), dv.view.data_ptr(),
                                    blk.data_ptr(), tab.data_ptr(), cblk.data_ptr(), ctab.data_ptr(),
                                    nnz, pattern.shape[0], pattern.shape[1], z, d, block, 0.1, 0, None, 0, 0, 0,
                                    stats.view.data_ptr(), stats.view.numel() * 4, ws.data_ptr(), 256, stream)
    assert st == 0, st
    dq.check("attention backward dQ")
    dk.check("attention backward dK")
    dv.check("attention backward dV")
    torch.cuda.synchronize()
    assert bool((stats.raw[:GUARD] == stats.sentinel).all()) and bool((stats.raw[-GUARD:] == stats.sentinel).all())
    assert lib.bsa_workspace_status(ws.data_ptr(), stream) == 0
    got = sparse_ops.sparse_attention_backward(q, k, v, o.view, do, lse.view, blk, tab, cblk, ctab, block, 0.1, False, None)
    assert torch.equal(dq.view, got[0]) and torch.equal(dk.view, got[1]) and torch.equal(dv.view, got[2])


# ------------------------------------------------------------------------------------------------ packed batches and the cache
def _filled(shape, dtype, value):
    """A guarded buffer that starts from `value` (a cache, a scratch, or an output that may hold NaN or infinities)."""
    buffer = Guarded(shape, torch.float16 if dtype == torch.uint8 else dtype)
    if dtype == torch.uint8:                               # (Guarded starts from NaN)
        n = buffer.view.numel()
        buffer.raw, buffer.sentinel = torch.full((n + 2 * GUARD,), 123, device="cuda", dtype=dtype), 123
        buffer.view = buffer.raw[GUARD:GUARD + n].view(shape)
    buffer.view.fill_(value)
    return buffer


def _guards_hold(buffer, what):
    torch.cuda.synchronize()
    assert bool((buffer.raw[:GUARD] == buffer.sentinel).all()), "%s wrote below its buffer" % what
    assert bool((buffer.raw[-GUARD:] == buffer.sentinel).all()), "%s wrote above its buffer" % what


@pytest.mark.parametrize("causal", [0, 1])
@pytest.mark.parametrize("dim,hq,hk,lengths,tail", [(64, 2, 2, [1, 127, 129, 0, 300], 3), (128, 4, 2, [130, 5, 128], 0),
                                                    (128, 3, 1, [257], 133)])
def test_packed_attention_writes_only_its_outputs(dim, hq, hk, lengths, tail, causal):
    from sparse.kernel import sparse_ops
    lib = _library()
    i, p, z = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t
    lib.bsa_packed_forward.argtypes = [ctypes.c_int] + [p, i, i] * 3 + [p, p, p, p] + [i] * 5 + [ctypes.c_float, ctypes.c_int, p, z, p]
    lib.bsa_packed_backward.argtypes = [ctypes.c_int] + [p, i, i] * 3 + [p, p, p, i, i] + [p] * 5 + [i] * 5 + \
        [ctypes.c_float, ctypes.c_int, p, z, p, z, p]
    rows, stream = sum(lengths) + tail, torch.cuda.current_stream().cuda_stream
    gen = torch.Generator(device="cuda").manual_seed(5)
    q, do = (torch.randn(rows, hq, dim, device="cuda", generator=gen).half() for _ in range(2))
    k, v = (torch.randn(rows, hk, dim, device="cuda", generator=gen).half() for _ in range(2))
    offsets = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
    ws = torch.zeros(256, dtype=torch.uint8, device="cuda")
    wide, narrow = (hq * dim, dim), (hk * dim, dim)
    o, low = Guarded((rows, hq, dim), torch.float16), Guarded((rows, hq, dim), torch.float16)
    lse = _filled((hq, rows), torch.float32, float("nan"))
    st = lib.bsa_packed_forward(1, q.data_ptr(), *wide, k.data_ptr(), *narrow, v.data_ptr(), *narrow, o.view.data_ptr(),
                                low.view.data_ptr(), lse.view.data_ptr(), offsets.data_ptr(), rows, len(lengths), hq, hk, dim,
                                0.1, causal, ws.data_ptr(), 256, stream)
    assert st == 0, st
    o.check("packed forward")
    low.check("packed forward, the rest of the output")
    lse.check("packed forward, log-sum-exp")
    assert bool((lse.view[:, rows - tail:] == float("-inf")).all()) and bool(lse.view[:, :rows - tail].isfinite().all())
    dq, dk, dv = Guarded((rows, hq, dim), torch.float16), Guarded((rows, hk, dim), torch.float16), Guarded((rows, hk, dim), torch.float16)
    stats = _filled((hq, rows, 2), torch.float32, 0.0)
    st = lib.bsa_packed_backward(1, q.data_ptr(), *wide, k.data_ptr(), *narrow, v.data_ptr(), *narrow, o.view.data_ptr(),
                                 low.view.data_ptr(), do.data_ptr(), *wide, lse.view.data_ptr(), dq.view.data_ptr(),
                                 dk.view.data_ptr(), dv.view.data_ptr(), offsets.data_ptr(), rows, len(lengths), hq, hk, dim, 0.1,
                                 causal, stats.view.data_ptr(), stats.view.numel() * 4, ws.data_ptr(), 256, stream)
    assert st == 0, st
    for name, buffer in (("dQ", dq), ("dK", dk), ("dV", dv)):
        buffer.check("packed backward " + name)
    _guards_hold(stats, "packed backward, statistics")
    for buffer in (o, low, lse):
        _guards_hold(buffer, "packed backward")
    assert lib.bsa_workspace_status(ws.data_ptr(), stream) == 0
    want = sparse_ops.packed_attention_forward(q, k, v, offsets, 0.1, bool(causal))
    assert torch.equal(o.view, want[0]) and torch.equal(lse.view, want[1]) and torch.equal(low.view, want[2])
    back = sparse_ops.packed_attention_backward(q, k, v, want[0], want[2], do, want[1], offsets, 0.1, bool(causal))
    assert torch.equal(dq.view, back[0]) and torch.equal(dk.view, back[1]) and torch.equal(dv.view, back[2])


@pytest.mark.parametrize("store", ["same", "e4m3"])
@pytest.mark.parametrize("tokens,heads,dim,page", [(45, 3, 64, 16), (16384 // 5 + 7, 5, 128, 128)])
def test_cache_writes_and_reads_only_its_places(store, tokens, heads, dim, page):
    from sparse.kernel import sparse_ops
    lib = _library()
    i, p, z = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t
    lib.bsa_cache_write.argtypes = [ctypes.c_int] * 2 + [p, p, i, i, i, i, p, i, p, p, p, p, i, i, i, i, p, z, p]
    lib.bsa_cache_read.argtypes = [ctypes.c_int] * 2 + [p, i, p, p, p, p, p, p, i, i, i, i, p, z, p]
    stream = torch.cuda.current_stream().cuda_stream
    pages = -(-tokens // page) + 1
    gen = torch.Generator(device="cuda").manual_seed(6)
    k, v = (torch.randn(tokens, heads, dim, device="cuda", generator=gen).half() for _ in range(2))
    slots = torch.randperm(pages * page, generator=torch.Generator().manual_seed(7))[:tokens].cuda()
    slots[0], slots[1] = pages * page - 1, 0               # the last place and the first
    slots[2:] = torch.where((slots[2:] == 0) | (slots[2:] == pages * page - 1), -1, slots[2:])
    ws = torch.zeros(256, dtype=torch.uint8, device="cuda")
    coded = store == "e4m3"
    cache = [_filled((pages, heads, page, dim), torch.uint8 if coded else torch.float16, 3) for _ in range(2)]
    scales = [_filled((pages, heads, page), torch.float32, 3.0) for _ in range(2 if coded else 0)]
    at = [t.view.data_ptr() for t in scales] if coded else [None, None]
    st = lib.bsa_cache_write(1, int(coded), k.data_ptr(), v.data_ptr(), heads * dim, dim, heads * dim, dim, slots.data_ptr(), tokens,
                             cache[0].view.data_ptr(), cache[1].view.data_ptr(), *at, pages, heads, page, dim, ws.data_ptr(), 256, stream)
    assert st == 0, st
    for buffer in cache + scales:
        _guards_hold(buffer, "cache write")
    want = [t.view.clone().fill_(3) for t in cache + scales]
    if coded:
        want[:2] = [t.view(torch.float8_e4m3fn) for t in want[:2]]
    sparse_ops.cache_write(k, v, slots, *want)
    for a, b in zip(cache + scales, want):
        assert torch.equal(a.view, b.view(torch.uint8) if b.dtype == torch.float8_e4m3fn else b)
    out = [Guarded((tokens, heads, dim), torch.float16) for _ in range(2)]
    st = lib.bsa_cache_read(1, int(coded), slots.data_ptr(), tokens, cache[0].view.data_ptr(), cache[1].view.data_ptr(), *at,
                            out[0].view.data_ptr(), out[1].view.data_ptr(), pages, heads, page, dim, ws.data_ptr(), 256, stream)
    assert st == 0, st
    for buffer in out:
        buffer.check("cache read")
    for buffer in cache + scales:
        _guards_hold(buffer, "cache read")
    assert lib.bsa_workspace_status(ws.data_ptr(), stream) == 0
    if not coded:
        kept = slots >= 0
        assert torch.equal(out[0].view[kept], k[kept]) and torch.equal(out[1].view[kept], v[kept])


@pytest.mark.parametrize("store", ["same", "e4m3"])
@pytest.mark.parametrize("dim,kv,group,drafts,lengths", [(128, 2, 2, 1, [700, 3, 0, 64]), (64, 1, 3, 11, [5000, 40]),
                                                         (128, 2, 5, 13, [129, 9000, 20]), (64, 2, 4, 40, [64])])
def test_cached_attention_writes_only_its_output_and_scratch(store, dim, kv, group, drafts, lengths):
    """A scratch of just the bytes that the library asks for; shares that hold a whole sequence and sequences split over many."""
    from sparse.kernel import sparse_ops
    lib = _library()
    i, p, z = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t
    lib.bsa_cached_attention.argtypes = [ctypes.c_int] * 2 + [p, i, i, i] + [p] * 10 + [i] * 11 + [ctypes.c_float, p, z, p, z, p]
    lib.bsa_cached_attention_scratch.argtypes, lib.bsa_cached_attention_scratch.restype = [i] * 4, z
    stream = torch.cuda.current_stream().cuda_stream
    page, heads, batch, coded = 32, kv * group, len(lengths), store == "e4m3"
    width = -(-max(lengths) // page)
    pages = batch * width
    gen = torch.Generator(device="cuda").manual_seed(8)
    q = torch.randn(batch, drafts, heads, dim, device="cuda", generator=gen).half()
    keys, values = (torch.randn(pages, kv, page, dim, device="cuda", generator=gen).to(torch.float8_e4m3fn if coded else torch.half) for _ in range(2))
    scales = [torch.rand(pages, kv, page, device="cuda", generator=gen) + 0.5 for _ in range(2)] if coded else [None, None]
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(9)).view(batch, width).to(torch.int32).cuda()
    count = torch.tensor([min(n, drafts) for n in lengths], dtype=torch.int32).cuda()
    length = torch.tensor(lengths, dtype=torch.int32).cuda()
    ws = torch.zeros(256, dtype=torch.uint8, device="cuda")
    o = Guarded((batch, drafts, heads, dim), torch.float16)
    size = lib.bsa_cached_attention_scratch(drafts, heads, kv, dim)
    scratch = _filled((size // 4,), torch.float32, float("nan"))
    st = lib.bsa_cached_attention(1, int(coded), q.data_ptr(), drafts * heads * dim, heads * dim, dim, keys.data_ptr(), values.data_ptr(),
                                  *(None if t is None else t.data_ptr() for t in scales), o.view.data_ptr(), table.data_ptr(),
                                  length.data_ptr(), count.data_ptr(), None, None, 0, 0, 0, batch, drafts, heads, kv, dim, pages,
                                  page, width, 0.1, scratch.view.data_ptr(), size, ws.data_ptr(), 256, stream)
    assert st == 0 and size % 4 == 0, (st, size)
    o.check("cached attention")
    _guards_hold(scratch, "cached attention, scratch")
    assert lib.bsa_workspace_status(ws.data_ptr(), stream) == 0
    assert torch.equal(o.view, sparse_ops.cached_attention(q, keys, values, *scales, table, length, count, None, 0.1))
