"""The paged key / value cache and the attention that reads it: against the definitions in 64 bits, at the sizes,
types and masks where they can go wrong, their refusals, and a run of them together."""
import ctypes
import math
import os
import subprocess
import sys
import textwrap

import pytest
import torch

from conftest import PKG

E4M3 = torch.float8_e4m3fn
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}        # largest relative error of one rounding


# ------------------------------------------------------------------------------------------------ CPU: refusals
@pytest.fixture(scope="module")
def lib():
    path = os.path.join(PKG, "libbsa_b200.so")
    if not os.path.exists(path):
        pytest.skip("kernel library not built")
    return ctypes.CDLL(path)


def test_cache_validation_codes(lib):
    f = lib.bsa_cache_write
    i, p = ctypes.c_int64, ctypes.c_void_p
    f.argtypes = [ctypes.c_int] * 2 + [p, p, i, i, i, i, p, i, p, p, p, p, i, i, i, i, p, ctypes.c_size_t, p]

    def call(dtype=1, store=0, k=16, strides=(1024, 128, 1024, 128), slots=16, tokens=1, keys=32, scales=None, pages=4,
             heads=8, page=64, dim=128, ws=16, ws_bytes=256):
        return f(dtype, store, k, 16, *strides, slots, tokens, keys, 32, scales, scales, pages, heads, page, dim, ws,
                 ws_bytes, None)

    assert call(dtype=0) == 3                                   # float32 tokens
    assert call(store=2) == 2
    assert call(store=1) == 1                                   # e4m3 without scales
    assert call(page=48) == 5 and call(page=0) == 5 and call(page=256) == 5
    assert call(dim=80) == 4 and call(pages=0) == 4 and call(heads=0) == 4 and call(tokens=-1) == 4
    assert call(strides=(-1024, 128, 1024, 128)) == 4
    assert call(strides=(1020, 128, 1024, 128)) == 6 and call(k=24) == 6 and call(keys=16) == 6
    assert call(k=None) == 1 and call(slots=None) == 1
    assert call(ws=None) == 7 and call(ws_bytes=255) == 7
    assert call(pages=2 ** 31) == 10 and call(tokens=2 ** 31) == 10
    assert call(tokens=0) == 0                                  # nothing to do: nothing is launched

    r = lib.bsa_cache_read
    r.argtypes = [ctypes.c_int] * 2 + [p, i, p, p, p, p, p, p, i, i, i, i, p, ctypes.c_size_t, p]
    assert r(1, 0, 16, 1, 16, 16, None, None, None, 16, 4, 8, 64, 128, 16, 256, None) == 1
    assert r(2, 1, 16, 1, 16, 16, None, None, 16, 16, 4, 8, 64, 128, 16, 256, None) == 1
    assert r(2, 0, 16, 1, 16, 16, None, None, 16, 16, 4, 8, 65, 128, 16, 256, None) == 5


def test_cached_attention_validation_codes(lib):
    f = lib.bsa_cached_attention
    i, p, z = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t
    f.argtypes = [ctypes.c_int] * 2 + [p, i, i, i] + [p] * 10 + [i] * 11 + [ctypes.c_float, p, z, p, z, p]

    def call(dtype=1, store=0, q=16, stride=1024, table=16, pattern=None, block=64, batch=1, drafts=1, heads=8, kv=4,
             dim=128, pages=4, page=64, width=4, scratch=16, scratch_bytes=1 << 40, ws_bytes=256):
        return f(dtype, store, q, stride, stride, 128, 16, 16, None, None, 16, table, 16, None, None, pattern, 4, 4, block,
                 batch, drafts, heads, kv, dim, pages, page, width, 1.0, scratch, scratch_bytes, 16, ws_bytes, None)

    assert call(dtype=0) == 3 and call(store=1) == 1 and call(page=24) == 5 and call(dim=96) == 4
    assert call(batch=-1) == 4 and call(drafts=0) == 4 and call(heads=6) == 4 and call(width=0) == 4 and call(kv=0) == 4
    assert call(drafts=65) == 10 and call(width=2 ** 30) == 10
    assert call(q=None) == 1 and call(table=None) == 1 and call(scratch=None) == 1
    assert call(q=8) == 6 and call(stride=1021) == 6 and call(scratch=8) == 6
    assert call(ws_bytes=0) == 7
    assert call(pattern=16, block=48) == 5
    assert call(batch=0) == 0


def test_cached_attention_number_of_sequences(lib):
    """The join's time grows with the square of the number of sequences: one that would hold the device is refused."""
    f = lib.bsa_cached_attention
    i, p, z = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t
    f.argtypes = [ctypes.c_int] * 2 + [p, i, i, i] + [p] * 10 + [i] * 11 + [ctypes.c_float, p, z, p, z, p]

    def call(batch):                                       # (without queries: the sizes are looked at first)
        return f(1, 0, None, 1024, 1024, 128, 16, 16, None, None, 32, 16, 16, None, None, None, 0, 0, 0, batch, 1, 8, 4, 128, 4, 64, 4,
                 1.0, 16, 1 << 40, 16, 256, None)
    assert call(65537) == 10 and call(2 ** 24) == 10 and call(65536) == 1


def test_tree_words_and_their_refusals():
    from sparse import tree_words
    assert tree_words([[-1, 0, 0, 2, -1]]).tolist() == [[0b1, 0b11, 0b101, 0b1101, 0b10000]]
    chain = tree_words([list(range(-1, 63))])
    assert chain[0, 62].item() == 2 ** 63 - 1 and chain[0, 63].item() == -1      # bit 63 is the sign
    for bad in ([[0]], [[-1, 1]], [[-2]], [[-1] * 65], [[-1], [-1, 0]]):
        with pytest.raises(ValueError):
            tree_words(bad)


def test_cache_slots():
    from sparse import cache_slots
    table = torch.tensor([[5, 2, -1], [7, -1, -1]], dtype=torch.int32)
    got = cache_slots(table, torch.tensor([0, 0, 0, 0, 1, 1, 0]), torch.tensor([0, 17, 32, 48, 15, 16, -1]), 16)
    assert got.tolist() == [80, 33, -1, -1, 127, -1, -1]
    assert cache_slots(table, torch.tensor([[0], [1]]), torch.tensor([0, 1]), 16).tolist() == [80, 81, 112, 113]


def test_python_refusals_without_a_gpu():
    from sparse import cache_read, cache_write, cached_attention, make_cache
    with pytest.raises(ValueError):
        make_cache(4, 64, 2, 128, torch.float32, device="cpu")
    with pytest.raises(ValueError):
        make_cache(4, 48, 2, 128, torch.float16, device="cpu")
    with pytest.raises(ValueError):
        make_cache(4, 64, 2, 96, torch.float16, device="cpu")
    cache = make_cache(4, 64, 2, 128, E4M3, device="cpu")
    assert cache.keys.dtype == E4M3 and cache.key_scales.shape == (4, 2, 64)
    k = torch.zeros(3, 2, 128, dtype=torch.float16)
    slots = torch.arange(3)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache_write(k, k, slots, *cache)
    with pytest.raises(RuntimeError, match="CUDA"):
        cache_read(slots, *cache)
    q = torch.zeros(1, 1, 2, 128, dtype=torch.float16, requires_grad=True)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no gradient"):
        cached_attention(q, *cache, table, lengths)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
        cached_attention(q, *cache, table, lengths)


def test_cached_attention_output_on_32_bytes(lib):
    """The kernel for many rows stores 32 bytes at a time; every output of this entry point is on 32, as the others'."""
    f = lib.bsa_cached_attention
    i, p, z = ctypes.c_int64, ctypes.c_void_p, ctypes.c_size_t
    f.argtypes = [ctypes.c_int] * 2 + [p, i, i, i] + [p] * 10 + [i] * 11 + [ctypes.c_float, p, z, p, z, p]
    for drafts in (1, 24):
        for o in (16, 48, 40):
            assert f(1, 0, 16, 1024, 1024, 128, 16, 16, None, None, o, 16, 16, None, None, None, 0, 0, 0, 1, drafts, 16, 4, 128, 4,
                     64, 4, 1.0, 16, 1 << 40, 16, 256, None) == 6


def test_cache_slots_of_sequences_that_are_none():
    """A sequence outside the table has no slots: a negative number does not count from the table's end."""
    from sparse import cache_slots
    table = torch.tensor([[5, 2], [7, 3]], dtype=torch.int32)
    got = cache_slots(table, torch.tensor([-1, 0, 1, 2, 2 ** 40, -3]), torch.tensor([0, 1, 17, 0, 5, 1]), 16)
    assert got.tolist() == [-1, 81, 49, -1, -1, -1]
    assert cache_slots(table[:, :0], torch.tensor([0, 1]), torch.tensor([0, 1]), 16).tolist() == [-1, -1]
    assert cache_slots(table[:0], torch.tensor([0, 1]), torch.tensor([0, 1]), 16).tolist() == [-1, -1]


def test_derivatives_that_the_cache_has_not_are_refused():
    """Forward-mode derivatives (whose tensors do not require grad) and a cache that requires grad: refused, not dropped."""
    import torch.autograd.forward_ad as fwd
    from sparse import cache_read, cache_write, cached_attention, make_cache
    k = torch.zeros(3, 2, 128, dtype=torch.float16)
    slots = torch.arange(3)
    q = torch.zeros(1, 1, 2, 128, dtype=torch.float16)
    table, lengths = torch.zeros(1, 1, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    plain, coded = make_cache(4, 64, 2, 128, torch.float16, device="cpu"), make_cache(4, 64, 2, 128, E4M3, device="cpu")
    with fwd.dual_level(), torch.no_grad():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))
        for a, b in ((dual(k), k), (k, dual(k))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                cache_write(a, b, slots, *plain)
        for cache, side in ((plain, 0), (plain, 1), (coded, 2), (coded, 3)):
            held = list(cache)
            held[side] = dual(held[side])
            with pytest.raises(RuntimeError, match="forward-mode"):
                cache_read(slots, *held, dtype=torch.float16)
            with pytest.raises(RuntimeError, match="forward-mode"):
                cached_attention(q, *held, table, lengths)
            with pytest.raises(RuntimeError, match="forward-mode"):
                cache_write(k, k, slots, *held)
        with pytest.raises(RuntimeError, match="forward-mode"):
            cached_attention(dual(q), *plain, table, lengths)
    for cache, side in ((plain, 0), (plain, 1), (coded, 2), (coded, 3)):
        held = list(cache)
        held[side] = held[side].clone().requires_grad_()
        with pytest.raises(RuntimeError, match="no gradient"):
            cache_read(slots, *held, dtype=torch.float16)
        with pytest.raises(RuntimeError, match="no gradient"):
            cached_attention(q, *held, table, lengths)
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            cache_read(slots, *held, dtype=torch.float16)


# ------------------------------------------------------------------------------------------------ GPU: write and read
def _quantised(x):
    """e4m3 codes and fp32 scales by the definition, in the same order of fp32 operations (codes are compared exactly)."""
    amax = x.float().abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
    most = torch.full_like(amax, 448.0)                    # (a Python number would be multiplied by the rounded reciprocal)
    return (x.float() * (most / amax)).to(E4M3), (amax / most).squeeze(-1)


def _same(a, b):
    """Equal values, NaN where NaN (fp16 rows of this spread hold infinities, whose codes are NaN of either sign)."""
    if a.dtype == torch.uint8:
        a, b = a.view(E4M3), b.view(E4M3)
    a, b = a.float().cpu(), b.float().cpu()
    wrong = ~((a == b) | (a.isnan() & b.isnan()))
    return a.shape == b.shape and not wrong.any()


def _status():
    from sparse.kernel import sparse_ops
    torch.cuda.synchronize()
    sparse_ops.check_device_status(0)


def _normal(shape, seed, dtype, spread=0.0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=gen)
    if spread:                                             # rows of very different size
        x = x * torch.exp(torch.randn(shape[:-1] + (1,), generator=gen) * spread)
    return x.to(dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("store", ["same", "e4m3"])
@pytest.mark.parametrize("tokens,heads,dim,page", [(1, 1, 64, 16), (1, 8, 128, 64), (37, 5, 64, 32), (333, 3, 128, 128),
                                                   (6000, 8, 128, 64)])
def test_write_then_read(dtype, store, tokens, heads, dim, page):
    from sparse import Cache, cache_read, cache_write, make_cache
    pages = -(-tokens // page) + 3
    gen = torch.Generator().manual_seed(tokens)
    slots = torch.randperm(pages * page, generator=gen)[:tokens]
    if tokens > 4:
        slots[::7] = -1
    cache = make_cache(pages, page, heads, dim, E4M3 if store == "e4m3" else dtype)
    # what is not written must stay: start from something recognisable
    for t in cache:
        if t is not None:
            (t.view(torch.uint8) if t.dtype == E4M3 else t).fill_(3)
    before = Cache(*(None if t is None else t.clone() for t in cache))
    both = _normal((2, tokens, heads, dim), tokens + 1, dtype, spread=3.0)
    both[:, tokens // 2, 0] = 0.0                          # a row of zeros
    k, v = both[0].cuda(), both[1].cuda()
    cache_write(k, v, slots.cuda(), *cache)
    _status()
    real = slots >= 0
    at = slots[real]

    def want(old, new):
        raw = old.view(torch.uint8) if old.dtype == E4M3 else old
        raw = raw.cpu().clone()
        new = new.view(torch.uint8) if new.dtype == E4M3 else new
        raw[at // page, :, at % page] = new[real]
        return raw

    for side, x in enumerate((both[0], both[1])):
        got = cache[side].view(torch.uint8) if store == "e4m3" else cache[side]
        if store == "same":
            assert _same(got, want(before[side], x))
        else:
            codes, scales = _quantised(x)
            assert _same(got, want(before[side], codes))
            assert _same(cache[2 + side], want(before[2 + side], scales))
    back = cache_read(slots.cuda(), *cache, dtype=dtype)
    _status()
    for x, got in zip((both[0], both[1]), back):
        assert got.dtype == dtype and got.shape == x.shape
        held = x.float()
        if store == "e4m3":
            codes, scales = _quantised(x)
            held = codes.float() * scales[..., None]
        expected = torch.where(real[:, None, None], held, 0.0).to(dtype)
        assert _same(got, expected)


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["same", "e4m3"])
@pytest.mark.parametrize("heads,dim", [(1, 64), (5, 64), (3, 128)])
def test_many_rows_and_odd_heads(store, heads, dim):
    """The same rows at once (two heads of both sides per lane group) and in small calls (one row): the same bits."""
    from sparse import cache_read, cache_write, make_cache
    tokens, page, dtype = 16384 // heads + 77, 64, torch.float16
    pages = -(-tokens // page) + 1
    slots = torch.randperm(pages * page)[:tokens].cuda()
    slots[5::11] = -1
    k, v = (_normal((tokens, heads, dim), 8 + i, dtype, spread=3.0).cuda() for i in range(2))
    caches = [make_cache(pages, page, heads, dim, E4M3 if store == "e4m3" else dtype) for _ in range(2)]
    for cache in caches:
        for t in cache:
            if t is not None:
                (t.view(torch.uint8) if t.dtype == E4M3 else t).fill_(3)
    cache_write(k, v, slots, *caches[0])
    for i in range(0, tokens, 1000):
        cache_write(k[i:i + 1000], v[i:i + 1000], slots[i:i + 1000], *caches[1])
    for a, b in zip(*caches):
        if a is not None:
            assert _same(*((x.view(torch.uint8) if x.dtype == E4M3 else x) for x in (a, b)))
    whole = cache_read(slots, *caches[0], dtype=dtype)
    parts = [cache_read(slots[i:i + 1000], *caches[0], dtype=dtype) for i in range(0, tokens, 1000)]
    for side in range(2):
        assert _same(whole[side], torch.cat([p[side] for p in parts]))
        assert (whole[side][slots < 0] == 0).all()
    _status()


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["same", "e4m3"])
def test_write_takes_strided_and_misaligned_tokens(store):
    from sparse import cache_read, cache_write, make_cache
    dtype, tokens, heads, dim = torch.bfloat16, 21, 4, 64
    fused = _normal((tokens, 3 * heads, dim), 3, dtype).cuda()
    _, k, v = fused.split(heads, dim=1)                    # views of one projection
    odd = _normal((tokens, heads, dim + 3), 4, dtype).cuda()[:, :, 1:dim + 1]      # rows start on odd places
    transposed = _normal((heads, tokens, dim), 5, dtype).cuda().transpose(0, 1)
    expanded = _normal((tokens, 1, dim), 6, dtype).cuda().expand(tokens, heads, dim)
    slots = torch.randperm(64)[:tokens].cuda()
    for a, b in ((k, v), (odd, transposed), (transposed, expanded), (expanded, odd)):
        cache, plain = (make_cache(4, 16, heads, dim, E4M3 if store == "e4m3" else dtype) for _ in range(2))
        cache_write(a, b, slots, *cache)
        cache_write(a.contiguous(), b.contiguous(), slots, *plain)
        for x, y in zip(cache_read(slots, *cache), cache_read(slots, *plain)):
            assert torch.equal(x, y)
    _status()


@pytest.mark.gpu
def test_rows_that_are_no_numbers_read_back_as_none():
    from sparse import cache_read, cache_write, make_cache
    k = _normal((4, 2, 64), 1, torch.bfloat16)
    k[0, 0, 5], k[1, 1, 63], k[2, 0, 0] = math.inf, math.nan, -math.inf
    k[3, 0] = 2.0 ** -126                                  # below the floor of amax: zeros, not infinities
    k[3, 1] = torch.finfo(torch.bfloat16).max
    cache = make_cache(1, 16, 2, 64, E4M3)
    slots = torch.arange(4).cuda()
    cache_write(k.cuda(), k.cuda(), slots, *cache)
    for got in cache_read(slots, *cache):
        got = got.cpu()
        for t, h in ((0, 0), (1, 1), (2, 0)):
            assert got[t, h].isnan().all()
        assert got[0, 1].isfinite().all() and got[1, 0].isfinite().all()
        assert (got[3, 0] == 0).all()
        assert torch.equal(got[3, 1], k[3, 1])
    _status()


@pytest.mark.gpu
def test_slots_behind_the_end_are_skipped_and_reported():
    from sparse import cache_read, cache_write, make_cache
    from sparse.kernel import sparse_ops
    cache = make_cache(2, 16, 1, 64, torch.float16)
    x = torch.ones(3, 1, 64, dtype=torch.float16, device="cuda")
    slots = torch.tensor([31, 32, 2 ** 40], device="cuda")
    cache_write(x, x, slots, *cache)
    with pytest.raises(RuntimeError):
        sparse_ops.check_device_status(0)
    assert cache.keys.sum().item() == 64 and (cache.keys[1, 0, 15] == 1).all()
    k, _ = cache_read(slots, *cache)
    with pytest.raises(RuntimeError):
        sparse_ops.check_device_status(0)
    assert (k[0] == 1).all() and (k[1:] == 0).all()
    _status()


@pytest.mark.gpu
def test_gpu_refusals():
    from sparse import cache_read, cache_write, cached_attention, kernel, make_cache
    cache = make_cache(2, 16, 2, 64, torch.float16)
    coded = make_cache(2, 16, 2, 64, E4M3)
    x = torch.ones(3, 2, 64, dtype=torch.float16, device="cuda")
    slots = torch.arange(3, device="cuda")
    for args in ((x, x, slots[:2], *cache), (x[:, :1], x[:, :1], slots, *cache), (x.float(), x.float(), slots, *cache),
                 (x.bfloat16(), x.bfloat16(), slots, *cache), (x, x, slots.int(), *cache), (x, x, slots, coded.keys, coded.values),
                 (x, x, slots, coded.keys, coded.values, coded.key_scales), (x, x, slots, *cache[:2], *coded[2:]),
                 (x, x[:, :, ::2], slots, *cache), (x, x, slots.cpu(), *cache),
                 (x, x, slots, cache.keys.transpose(1, 2), cache.values.transpose(1, 2))):
        with pytest.raises(RuntimeError):
            cache_write(*args)
    with pytest.raises(RuntimeError):
        cache_read(slots, *cache, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        cache_read(slots, *coded, dtype=torch.float32)
    q = torch.ones(1, 2, 4, 64, dtype=torch.float16, device="cuda")
    table = torch.zeros(1, 2, dtype=torch.int32, device="cuda")
    lengths = torch.full((1,), 20, dtype=torch.int32, device="cuda")
    for kw in ({"table": table.long()}, {"table": table[:, :0]}, {"lengths": lengths.long()}, {"counts": lengths.long()},
               {"tree": torch.zeros(1, 3, dtype=torch.int64, device="cuda")}, {"q": q[:, :, :3]}, {"q": q.bfloat16()},
               {"q": q.expand(1, 2, 4, 64).repeat(1, 33, 1, 1)}, {"q": q[..., :32]}, {"lengths": lengths.cpu()},
               {"q": q.repeat(2, 1, 1, 1)}):
        args = {"q": q, "table": table, "lengths": lengths, **kw}
        with pytest.raises(RuntimeError):
            cached_attention(args["q"], *cache, args["table"], args["lengths"], counts=args.get("counts"), tree=args.get("tree"))
    kernel.debug_checks = True
    try:
        with pytest.raises(ValueError):
            cache_write(x, x, torch.tensor([3, -1, 3], device="cuda"), *cache)
        cache_write(x, x, torch.tensor([3, -1, -1], device="cuda"), *cache)
    finally:
        kernel.debug_checks = False
    _status()


# ------------------------------------------------------------------------------------------------ GPU: attention
class _Case:
    def __init__(self, dtype, store, dim, page, kv_heads, group, drafts, lengths, counts=None, tree=False, seed=0, spread=0.0):
        gen = torch.Generator().manual_seed(seed + 17)
        self.dtype, self.store, self.dim, self.page = dtype, store, dim, page
        self.kv_heads, self.group, self.drafts, self.lengths = kv_heads, group, drafts, lengths
        self.counts = counts
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + 3
        order = torch.randperm(pages, generator=gen).to(torch.int32)
        self.table = torch.full((len(lengths), max(need + [1])), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (pages, kv_heads, page, dim)
        k, v = _normal(shape, seed, dtype, spread), _normal(shape, seed + 1, dtype, spread)
        # places that belong to no token hold NaN
        used = torch.zeros(pages, page, dtype=torch.bool)
        for i, n in enumerate(lengths):
            for j in range(need[i]):
                used[self.table[i, j], :max(0, min(page, n - j * page))] = True
        k[~used[:, None, :].expand(-1, kv_heads, -1)] = math.nan
        v[~used[:, None, :].expand(-1, kv_heads, -1)] = math.nan
        if store == "e4m3":
            (self.keys, self.key_scales), (self.values, self.value_scales) = _quantised(k), _quantised(v)
            self.k, self.v = (c.double() * s.double()[..., None] for c, s in ((self.keys, self.key_scales), (self.values, self.value_scales)))
        else:
            self.keys, self.values, self.key_scales, self.value_scales = k, v, None, None
            self.k, self.v = k.double(), v.double()
        self.q = _normal((len(lengths), drafts, kv_heads * group, dim), seed + 2, dtype, spread)
        self.tree = None
        if tree:
            from sparse import tree_words
            self.tree = tree_words([[int(torch.randint(-1, i, (1,), generator=gen)) if i else -1 for i in range(drafts)]
                                    for _ in lengths])
        self.scale = dim ** -0.5

    def seen(self, b, pattern=None, block=1):
        n, c = self.lengths[b], self.drafts if self.counts is None else self.counts[b]
        words = [(1 << (i + 1)) - 1 if self.tree is None else self.tree[b, i].item() for i in range(self.drafts)]
        depth = [bin(w & (1 << 64) - 1).count("1") - 1 for w in words]
        seen = torch.zeros(self.drafts, n, dtype=torch.bool)
        for i in range(min(c, self.drafts)):
            for j in range(n):
                d = j - (n - c)
                seen[i, j] = d < 0 or bool(words[i] >> d & 1)
                if pattern is not None:
                    base = max(n - c, 0)
                    row, col = base + max(depth[i], 0), j if d < 0 else base + max(depth[d], 0)
                    row, col = row // block, col // block
                    seen[i, j] &= row < pattern.size(0) and col < pattern.size(1) and bool(pattern[row, col])
        return seen

    def reference(self, pattern=None, block=1):
        """(output, bound on the kernel's error) in 64 bits."""
        out = torch.zeros(self.q.shape, dtype=torch.float64)
        bound = torch.zeros_like(out)
        u = HALF[self.dtype]
        u_p = 2.0 ** -11 if self.store == "e4m3" else u              # the weights are rounded once, to the products' type
        for b, n in enumerate(self.lengths):
            if n == 0:
                continue
            pages = self.table[b, :-(-n // self.page)].long()
            k = self.k[pages].transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(self.group, 0)      # [heads, n, d]
            v = self.v[pages].transpose(0, 1).flatten(1, 2)[:, :n].repeat_interleave(self.group, 0)
            q = self.q[b].double().transpose(0, 1)
            seen = self.seen(b, pattern, block)
            s = (q @ k.transpose(1, 2) * self.scale).masked_fill(~seen, -math.inf)
            p = torch.softmax(s, -1).nan_to_num(0.0)
            o = p @ v
            # products and sums in fp32: each score is off by at most (dim + 8) steps of its sum of magnitudes, a weight
            # by that much relative to itself, and once more through the row's sum; the exponential adds 2^-20
            off = ((q.abs() @ k.abs().transpose(1, 2)) * abs(self.scale)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
            rel = u_p + 2 * (self.dim + 8) * 2.0 ** -24 * off + 2.0 ** -20
            # (fp32 sums over n keys: n 2^-24 relative to the sum of magnitudes)
            weight = p @ v.abs() * (1 + u)
            out[b] = o.transpose(0, 1)
            tiny = 2.0 ** -25 if self.dtype == torch.float16 else 0.0                   # fp16 rounds below 2^-14 to 2^-24
            # weights below 2^-14 of the row's largest are rounded to steps of 2^-24 of it in fp16
            floor = 0.0
            if u_p == 2.0 ** -11:
                scale_v = (p.amax(-1, keepdim=True) * v.abs().amax(1, keepdim=True)).clamp_min(0)
                floor = n * 2.0 ** -25 * scale_v * (2.0 if self.store == "e4m3" else 1.0)
            bound[b] = (u * o.abs() + (rel + n * 2.0 ** -24) * weight + floor + tiny).transpose(0, 1)
        return out, bound

    def call(self, layout=None, q=None, **kw):
        from sparse import cached_attention
        dev = [None if t is None else t.cuda() for t in (self.keys, self.values, self.key_scales, self.value_scales)]
        return cached_attention(self.q.cuda() if q is None else q, *dev, self.table.cuda(),
                                torch.tensor(self.lengths, dtype=torch.int32).cuda(),
                                counts=None if self.counts is None else torch.tensor(self.counts, dtype=torch.int32).cuda(),
                                tree=None if self.tree is None else self.tree.cuda(), scale=self.scale, layout=layout, **kw)


def _check(got, reference):
    out, bound = reference
    got = got.double().cpu()
    assert got.isfinite().all()
    over = (got - out).abs() - bound
    assert (over <= 0).all(), "off by %.3e more than the bound" % over.max()


ATTENTION = [
    # dim, page, kv_heads, group, drafts, lengths, counts, tree
    (128, 64, 4, 4, 1, [391], None, False),
    (64, 16, 1, 1, 1, [1], None, False),
    (128, 128, 2, 8, 1, [1, 64, 65, 127, 128, 129, 0, 700], None, False),
    (64, 32, 3, 5, 3, [3, 40, 63, 66, 200], None, False),
    (128, 16, 2, 3, 8, [300, 8, 9, 71, 0, 5], [8, 8, 3, 0, 0, 5], True),
    (128, 64, 1, 8, 24, [1000, 24, 90], [24, 24, 1], True),
    (64, 64, 2, 1, 64, [64, 130, 500], None, True),
    (128, 32, 5, 2, 33, [33, 100], [33, 7], False),
    (64, 128, 1, 16, 13, [2500, 13], None, True),
    # many query rows per key head: lengths around a tile of 128 keys, one and several tiles per share, empty sequences
    (128, 16, 1, 16, 3, [1, 2, 3, 127, 128, 129, 255, 256, 257, 0, 700], None, False),
    (64, 64, 8, 8, 8, [50, 3000, 8, 0, 131] * 9, [8, 3, 8, 0, 1] * 9, True),
    (128, 128, 4, 5, 60, [60, 61, 9000], None, True),
    # many tiles per share: every stage of the ring is used again and again, by both streams of tiles
    (128, 64, 4, 8, 1, [4000] * 8, None, False),
    (64, 16, 2, 4, 2, [20000, 5, 9000], None, False),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("store", ["same", "e4m3"])
@pytest.mark.parametrize("dim,page,kv_heads,group,drafts,lengths,counts,tree", ATTENTION)
def test_cached_attention(dtype, store, dim, page, kv_heads, group, drafts, lengths, counts, tree):
    case = _Case(dtype, store, dim, page, kv_heads, group, drafts, lengths, counts, tree, seed=drafts)
    got = case.call()
    _status()
    _check(got, case.reference())


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["same", "e4m3"])
def test_cached_attention_scales_of_all_sizes(store):
    """Tokens whose values differ by many orders of magnitude (the scale of a value goes into its weight)."""
    case = _Case(torch.bfloat16, store, 128, 64, 2, 4, 2, [500, 77], seed=5, spread=2.0)
    case.q = (case.q.double() * 0.05).to(case.dtype)
    _check(case.call(), case.reference())
    _status()


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [-0.2, 0.0])
@pytest.mark.parametrize("store,group,drafts", [("same", 2, 2), ("e4m3", 2, 2), ("same", 8, 12)])
def test_cached_attention_negative_and_zero_scale(store, group, drafts, scale):
    """The largest score is the smallest product, or all are equal; what is masked stays out (0 times an infinity)."""
    case = _Case(torch.bfloat16, store, 64, 32, 2, group, drafts, [300, 40, 1], counts=[drafts, 1, 1], seed=31)
    case.scale = scale
    _check(case.call(), case.reference())
    _status()


@pytest.mark.gpu
def test_cached_attention_tiny_and_huge_queries():
    """bf16 queries outside fp16's range over an 8-bit cache."""
    case = _Case(torch.bfloat16, "e4m3", 64, 16, 1, 4, 1, [90], seed=8)
    q = case.q.clone()
    q[:, :, 0] *= 2.0 ** -60
    q[:, :, 1] = 0.0
    case.q = q
    _check(case.call(), case.reference())
    case.q = (q.double() * 2.0 ** 20).to(torch.bfloat16)
    case.scale = 2.0 ** -23
    _check(case.call(), case.reference())
    _status()


@pytest.mark.gpu
@pytest.mark.parametrize("block,drafts,tree", [(16, 1, False), (64, 5, False), (128, 9, True)])
def test_cached_attention_with_a_layout(block, drafts, tree):
    from sparse import SparseLayout
    lengths = [700, 129, 64, 9]
    gen = torch.Generator().manual_seed(block)
    pattern = (torch.rand(6 * 128 // block, 6 * 128 // block, generator=gen) < 0.4).to(torch.uint8)
    pattern[3] = 0                                         # a block row without blocks: its rows see nothing
    case = _Case(torch.bfloat16, "same", 64, 32, 2, 2, drafts, lengths, tree=tree, seed=block)
    got = case.call(layout=SparseLayout(pattern, block=block))
    _status()
    _check(got, case.reference(pattern, block))


@pytest.mark.gpu
@pytest.mark.parametrize("store,group,drafts", [("same", 2, 1), ("same", 8, 8), ("e4m3", 4, 2)])
def test_cached_attention_pages_that_are_none(store, group, drafts):
    """A page id outside the cache leaves its keys out and is reported; other sequences are not touched."""
    from sparse.kernel import sparse_ops
    case = _Case(torch.float16, store, 64, 16, 2, group, drafts, [100, 70], seed=2)
    good = case.call()
    for bad in (-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
        table = case.table.clone()
        case.table[0, 2] = bad
        got = case.call()
        with pytest.raises(RuntimeError):
            sparse_ops.check_device_status(0)
        assert got.isfinite().all() and torch.equal(got[1], good[1]) and not torch.equal(got[0], good[0])
        case.table = table
    too_long = case.lengths
    case.lengths = [100, 10 ** 9]                          # a length behind the table's end is cut off
    case.table[1, 5:] = 0
    got = case.call()
    with pytest.raises(RuntimeError):
        sparse_ops.check_device_status(0)
    assert torch.equal(got[0], good[0])
    case.lengths = too_long
    _status()


@pytest.mark.gpu
def test_cached_attention_strided_queries_streams_and_repeats():
    case = _Case(torch.bfloat16, "e4m3", 128, 64, 2, 4, 3, [600, 90, 3000], seed=4)
    want = case.call()
    fused = torch.zeros(3, 3, 12, 128, dtype=torch.bfloat16, device="cuda")
    fused[:, :, :8] = case.q.cuda()
    assert torch.equal(case.call(q=fused[:, :, :8]), want)                     # a view of a projection's output
    odd = torch.zeros(3, 3, 8, 131, dtype=torch.bfloat16, device="cuda")[..., 2:130]
    odd.copy_(case.q)
    assert torch.equal(case.call(q=odd), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = case.call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want) and torch.equal(case.call(), want)
    _status()


@pytest.mark.gpu
def test_serving_step_in_a_graph_follows_its_buffers():
    """Write, read and attend captured once; replayed with other tokens, lengths and pages in the same buffers."""
    from sparse import cache_read, cache_slots, cache_write, cached_attention, make_cache
    dtype, heads, group, dim, page = torch.bfloat16, 2, 4, 128, 16
    cache = make_cache(40, page, heads, dim, E4M3)
    table = torch.randperm(40)[:36].view(3, 12).to(torch.int32).cuda()
    lengths = torch.tensor([1, 40, 100], dtype=torch.int32, device="cuda")
    k, v = (_normal((3, heads, dim), i, dtype).cuda() for i in (1, 2))
    q = _normal((3, 1, heads * group, dim), 3, dtype).cuda()
    fill = _normal((40 * page, heads, dim), 4, dtype).cuda()
    cache_write(fill, fill, torch.arange(40 * page, device="cuda"), *cache)

    def step():
        slots = cache_slots(table, torch.arange(3, device="cuda"), lengths - 1, page)
        cache_write(k, v, slots, *cache)
        return cached_attention(q, *cache, table, lengths, scale=0.1), *cache_read(slots, *cache)

    with torch.no_grad():
        step()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graphs = []
        for _ in range(2):                                 # two graphs of the same step, replayed in turn
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                captured = step()
            graphs.append((graph, captured))
        for turn in range(4):
            k.copy_(_normal(k.shape, 10 + turn, dtype))
            q.copy_(_normal(q.shape, 20 + turn, dtype))
            lengths.copy_(torch.tensor([turn + 2, 41 + 30 * turn, 101], dtype=torch.int32))
            want = [t.clone() for t in step()]
            graph, captured = graphs[turn % 2]
            for t in captured:
                t.zero_()
            graph.replay()
            for a, b in zip(captured, want):
                assert torch.equal(a, b)
    _status()


@pytest.mark.gpu
def test_offsets_behind_32_bits():
    """A cache side of more than 4 GB: the last pages are written, read and attended to."""
    from sparse import cache_read, cache_write, cached_attention, make_cache
    heads, dim, page = 8, 128, 64
    pages = 2 ** 32 // (heads * dim * page) + 40           # more than 2^32 elements, 8.6 GB a side
    cache = make_cache(pages, page, heads, dim, torch.float16)
    n = 100
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    at = torch.arange(n, device="cuda")
    slots = table[0].long()[at // page] * page + at % page
    k, v = (_normal((n, heads, dim), i, torch.float16).cuda() for i in (1, 2))
    cache_write(k, v, slots, *cache)
    back = cache_read(slots, *cache)
    assert torch.equal(back[0], k) and torch.equal(back[1], v)
    q = _normal((1, 1, heads, dim), 3, torch.float16).cuda()
    got = cached_attention(q, *cache, table, torch.tensor([n], dtype=torch.int32, device="cuda"), scale=0.1)
    _status()
    p = torch.softmax(torch.einsum("hd,nhd->hn", q[0, 0].double(), k.double()) * 0.1, -1)
    want = torch.einsum("hn,nhd->hd", p, v.double())
    # two roundings to fp16 of values up to max |v|
    assert ((got[0, 0].double() - want).abs() <= 3 * 2.0 ** -11 * v.abs().max()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("restricted", [False, True])
def test_first_call_of_a_process_under_capture(restricted):
    """What a first call sets up (the workspace, the layout's flags) does not depend on a replay."""
    script = textwrap.dedent("""
        import torch
        from sparse import SparseLayout, cache_slots, cache_write, cached_attention, make_cache
        from sparse.kernel import sparse_ops
        torch.manual_seed(0)
        layout = SparseLayout(torch.tensor([[1, 0], [1, 1]], device="cuda"), block=64) if RESTRICTED else None
        k, v = (torch.randn(100, 2, 64, device="cuda", dtype=torch.float16) for _ in range(2))
        q = torch.randn(1, 1, 4, 64, device="cuda", dtype=torch.float16)
        cache = make_cache(8, 16, 2, 64, torch.float16, "cuda")
        table = torch.arange(8, device="cuda", dtype=torch.int32)[None]
        lengths = torch.full((1,), 100, device="cuda", dtype=torch.int32)
        slots = cache_slots(table, torch.zeros(100, dtype=torch.int64, device="cuda"), torch.arange(100, device="cuda"), 16)
        # blocks of memory to be handed out again, holding anything but zeros
        dirt = [torch.full((n,), 255, dtype=torch.uint8, device="cuda") for n in (4, 64, 512, 4096) * 8]
        del dirt
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache_write(k, v, slots, *cache)
            captured = cached_attention(q, *cache, table, lengths, scale=0.125, layout=layout)
        sparse_ops.check_device_status(0)              # nothing has run
        cache_write(k, v, slots, *cache)
        eager = cached_attention(q, *cache, table, lengths, scale=0.125, layout=layout)
        sparse_ops.check_device_status(0)
        captured.zero_()
        graph.replay()
        assert torch.equal(captured, eager)
        table.fill_(8)                                 # pages that are not the cache's: reported by a replay
        graph.replay()
        try:
            sparse_ops.check_device_status(0)
        except RuntimeError:
            print("first call under capture: ok")
    """).replace("RESTRICTED", str(restricted))
    done = subprocess.run([sys.executable, "-c", script], env=dict(os.environ, PYTHONPATH=PKG), capture_output=True,
                          text=True, timeout=300)
    assert done.returncode == 0 and "first call under capture: ok" in done.stdout, done.stderr[-2000:]


# ------------------------------------------------------------------------------------------------ scales of every kind
def _check_any_scale(case, pattern=None, block=1, **kw):
    """As `_check`.  The weights P sv / r are rounded to fp16, r a power of two of at most the largest |sv| of a sequence
    and head: below 2^-14 in steps of 2^-24, so that each of n keys is off by at most 2^-25 r 448, relative to a row sum
    that is at least 1 / p_max.  (The bound of `_Case.reference` has the largest value of the column in place of 448 r,
    which only holds where the scales are of one size.)"""
    out, bound = case.reference(pattern, block)
    for b, n in enumerate(case.lengths):
        if n:
            pages = case.table[b, :-(-n // case.page)].long()
            top = case.value_scales[pages].double().abs().transpose(0, 1).flatten(1)[:, :n].amax(1).repeat_interleave(case.group)
            bound[b] += n * 2.0 ** -25 * 448 * top[None, :, None]
    _check(case.call(**kw), (out, bound))
    _status()


@pytest.mark.gpu
@pytest.mark.parametrize("drafts,tree", [(1, False), (6, True), (22, True)])
@pytest.mark.parametrize("kind", ["zero", "negative", "zeros beside huge ones", "all zero", "tiny"])
def test_cached_attention_value_scales_of_any_kind(kind, drafts, tree):
    """A stored value is code * scale whatever the scale is, and a key's weight does not depend on it: the softmax of a
    place that was never written (scale 0) counts, that of a row of zeros (scale 2^-100 / 448) too."""
    case = _Case(torch.bfloat16, "e4m3", 64, 16, 2, 3, drafts, [200, 50, 23], tree=tree, seed=41)
    some = torch.rand(case.value_scales.shape, generator=torch.Generator().manual_seed(1)) < 0.4
    if kind == "zero":
        case.value_scales[some] = 0.0
    elif kind == "negative":
        case.value_scales[some] *= -1.0
        case.key_scales[~some] *= -1.0
    elif kind == "all zero":
        case.value_scales[:] = 0.0
    elif kind == "tiny":
        case.value_scales *= 2.0 ** -90
    else:
        case.value_scales *= 2.0 ** 100
        case.value_scales[some] = 2.0 ** -100 / 448
        case.values.view(torch.uint8)[some] = 0
    # (places that belong to no token keep a NaN scale)
    case.value_scales[case.keys.float().isnan().any(-1)] = math.nan
    case.k, case.v = (c.double() * s.double()[..., None] for c, s in ((case.keys, case.key_scales), (case.values, case.value_scales)))
    _check_any_scale(case)


@pytest.mark.gpu
@pytest.mark.parametrize("drafts", [1, 4])
def test_places_that_were_never_written_count_as_zeros(drafts):
    """A length that covers skipped places and a padding sequence, over caches as `make_cache` gives them: the same weights
    over 8 bits as over 16."""
    from sparse import cache_slots, cache_write, cached_attention, make_cache
    heads, group, dim, page, dtype = 2, 2, 64, 16, torch.float16
    table = torch.arange(8, dtype=torch.int32).view(2, 4).cuda()
    k, v = (_normal((50, heads, dim), i, dtype).cuda() for i in (1, 2))
    q = _normal((2, drafts, heads * group, dim), 3, dtype).cuda()
    slots = cache_slots(table, torch.zeros(50, dtype=torch.int64, device="cuda"), torch.arange(50, device="cuda"), page)
    slots[3::7] = -1
    lengths = torch.tensor([60, 20], dtype=torch.int32, device="cuda")      # 10 places behind the last token, and a sequence of none
    for store in (dtype, E4M3):
        cache = make_cache(8, page, heads, dim, store)
        cache_write(k, v, slots, *cache)
        got = cached_attention(q, *cache, table, lengths, scale=0.125).double()
        every = cache_slots(table, torch.arange(2, device="cuda")[:, None], torch.arange(60, device="cuda"), page)
        held = []
        for side in range(2):
            x = cache[side].double() if store == dtype else cache[side].double() * cache[2 + side].double()[..., None]
            held.append(x[every // page, :, every % page].view(2, 60, heads, dim).repeat_interleave(group, 2))
        s = torch.einsum("bihd,bjhd->bhij", q.double(), held[0]) * 0.125
        at, n = torch.arange(60, device="cuda"), lengths[:, None, None]
        seen = at <= n - drafts + torch.arange(drafts, device="cuda")[:, None]
        want = torch.einsum("bhij,bjhd->bihd", torch.softmax(s.masked_fill(~seen[:, None], -math.inf), -1), held[1])
        assert got.isfinite().all()
        # the weights are rounded once (2^-11, or 2^-25 for each of 60 keys), so is the result; scores in fp32 (64 + 8 steps of
        # their magnitudes, at most 64 * 4.5^2 / 8), twice, and 2^-20 for the exponential
        off = 2 * 2.0 ** -11 + 60 * 2.0 ** -25 + 2 * 72 * 2.0 ** -24 * 162 + 2.0 ** -20
        assert ((got - want).abs() <= off * held[1].abs().amax()).all()
        assert (got[1] == 0).all()
    _status()


# ------------------------------------------------------------------------------------------------ layouts
@pytest.mark.gpu
@pytest.mark.parametrize("store", ["same", "e4m3"])
@pytest.mark.parametrize("block,page,dim,group,drafts,tree", [(32, 64, 64, 2, 1, False), (128, 16, 128, 4, 9, True),
                                                              (64, 32, 64, 3, 11, False), (64, 128, 64, 5, 15, True),
                                                              (16, 16, 128, 2, 64, True)])
def test_cached_attention_with_a_layout_over_both_caches_and_many_rows(store, block, page, dim, group, drafts, tree):
    """One row group to several row tiles (drafts x group of 2 to 128), drafts on both sides of a block's border."""
    from sparse import SparseLayout
    lengths = [700, 129, 64, 9, 0, 2 * block + 5]
    counts = [min(n, drafts) for n in lengths]
    pattern = (torch.rand(6 * 128 // block, 6 * 128 // block, generator=torch.Generator().manual_seed(block)) < 0.4).to(torch.uint8)
    pattern[2] = 0                                         # a block row without blocks: its rows see nothing
    case = _Case(torch.float16, store, dim, page, 2, group, drafts, lengths, counts, tree=tree, seed=block)
    got = case.call(layout=SparseLayout(pattern, block=block))
    _status()
    _check(got, case.reference(pattern, block))


@pytest.mark.gpu
@pytest.mark.parametrize("store", ["same", "e4m3"])
@pytest.mark.parametrize("group,drafts", [(2, 1), (4, 5), (3, 22)])
def test_numbers_of_blocks_outside_the_layout_are_not_used(store, group, drafts):
    """Keys and values of places that no draft of a sequence sees under the layout may be NaN."""
    from sparse import SparseLayout
    block, page = 32, 16
    lengths = [500, 90, 33]
    gen = torch.Generator().manual_seed(5)
    pattern = (torch.rand(16, 16, generator=gen) < 0.4).to(torch.uint8) | torch.eye(16, dtype=torch.uint8)
    case = _Case(torch.bfloat16, store, 64, page, 2, group, drafts, lengths, tree=drafts > 5, seed=6)
    reference = case.reference(pattern, block)
    hidden = 0
    for b, n in enumerate(lengths):
        for j in (~case.seen(b, pattern, block).any(0)).nonzero()[:, 0].tolist():
            at = (int(case.table[b, j // page]), slice(None), j % page)
            hidden += 1
            for t in (case.keys, case.values):
                if store == "e4m3":
                    t.view(torch.uint8)[at] = 0x7f
                else:
                    t[at] = math.nan
            if store == "e4m3":
                case.key_scales[at] = math.nan
                case.value_scales[at] = math.inf
    assert hidden > 100
    got = case.call(layout=SparseLayout(pattern, block=block))
    _status()
    _check(got, reference)


class _Blind(_Case):
    """Drafts that do not see themselves (bit i of word i is not set): their ancestors are all that they see."""

    def seen(self, b, pattern=None, block=1):
        n, c = self.lengths[b], self.drafts if self.counts is None else self.counts[b]
        words = [w & (1 << 64) - 1 for w in self.tree[b].tolist()]
        place = [max(n - c, 0) + bin(w & ~(1 << i)).count("1") for i, w in enumerate(words)]
        seen = torch.zeros(self.drafts, n, dtype=torch.bool)
        for i in range(min(c, self.drafts)):
            for j in range(n):
                d = j - (n - c)
                row, col = place[i] // block, (j if d < 0 else place[d]) // block
                seen[i, j] = (d < 0 or bool(words[i] >> d & 1)) and (pattern is None or bool(pattern[row, col]))
        return seen


@pytest.mark.gpu
@pytest.mark.parametrize("drafts,group", [(5, 2), (20, 3)])
def test_position_of_a_draft_that_does_not_see_itself(drafts, group):
    """It stands behind its ancestors as any other does: on the borders of small blocks one place decides."""
    from sparse import SparseLayout
    block = 16
    lengths = [16 * 7 + 3, 16 * 3 + drafts, 16 * 5 + drafts - 1, 16 * 4 + drafts - 2]
    pattern = (torch.rand(12, 12, generator=torch.Generator().manual_seed(3)) < 0.5).to(torch.uint8)
    case = _Blind(torch.float16, "same", 64, 16, 2, group, drafts, lengths, tree=True, seed=9)
    for i in range(0, drafts, 2):
        case.tree[:, i] &= ~(1 << i)
    got = case.call(layout=SparseLayout(pattern, block=block))
    _status()
    _check(got, case.reference(pattern, block))


@pytest.mark.gpu
@pytest.mark.parametrize("group,drafts", [(1, 1), (40, 1)])
def test_as_many_sequences_as_there_may_be(group, drafts):
    """65536 sequences of one token: every row is its value, bit for bit."""
    from sparse import cached_attention
    n, dim, page = 65536, 64, 16
    k, v = (_normal((n, 1, page, dim), i, torch.float16).cuda() for i in (1, 2))
    q = _normal((n, drafts, group, dim), 3, torch.float16).cuda()
    table = torch.randperm(n, generator=torch.Generator().manual_seed(4)).to(torch.int32)[:, None].cuda()
    lengths = torch.ones(n, dtype=torch.int32, device="cuda")
    got = cached_attention(q, k, v, None, None, table, lengths, scale=0.125)
    _status()
    assert torch.equal(got, v[table[:, 0].long(), :, :1].expand(-1, -1, group, -1))
