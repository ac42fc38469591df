"""A causal block-sparse self-attention module served over a paged cache: whole sequences written by ``forward``, tokens
by ``decode``, against ``forward`` over the whole sequence."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _module(block, seq, dtype, heads=4, head_dim=64):
    from sparse import BlockSparseSelfAttention, SparseLayout
    from sparse.patterns import local_global_causal
    torch.manual_seed(block)
    layout = SparseLayout(local_global_causal(seq // block, 2, 1), block=block)
    return BlockSparseSelfAttention(heads * head_dim, heads, layout, causal=True, device="cuda", dtype=dtype)


def _bound(module, x, whole):
    """Both ways make the same projections (bit for bit but for the order of fp32 sums, then one rounding) and round P and
    the context once each: the contexts differ by at most 2 (2 u) max|v| and what the projections' roundings (u of q, k
    and v, each side) move: the scores by 2 u |q| |k| scale each, twice.  Through the output projection: sum of |W|."""
    u = 2.0 ** -11 if x.dtype == torch.float16 else 2.0 ** -8
    qkv = module.qkv(x).double().view(x.size(0), x.size(1), 3, module.num_heads, module.head_dim)
    q, k, v = qkv.unbind(2)
    score = (q.norm(dim=-1).amax() * k.norm(dim=-1).amax() * module.scale)
    ctx = (4 * u + 2 * u + 2 * 4 * u * score) * v.abs().amax()
    return ctx * module.out.weight.double().abs().sum(1).max() + 2 * u * whole.double().abs().max()


@pytest.mark.parametrize("block,dtype", [(32, torch.float16), (64, torch.bfloat16)])
def test_decode_continues_forward(block, dtype):
    from sparse import cache_slots, make_cache
    from sparse.kernel import sparse_ops
    batch, seq, page = 2, 256, 32
    module = _module(block, seq, dtype)
    x = torch.randn(batch, seq, module.embed_dim, device="cuda", dtype=dtype)
    with torch.no_grad():
        whole = module(x)
        cache = make_cache(20, page, module.num_heads, module.head_dim, dtype)
        table = torch.randperm(20)[:16].view(batch, 8).to(torch.int32).cuda()
        sequences = torch.arange(batch, device="cuda")[:, None]
        prompt = torch.tensor([[150], [37]], device="cuda")            # tokens of each sequence that forward keeps
        at = torch.arange(seq, device="cuda")[None].expand(batch, seq)
        slots = cache_slots(table, sequences, torch.where(at < prompt, at, -1), page)
        assert torch.equal(module(x, cache=cache, slots=slots), whole)
        got = torch.zeros_like(whole)
        bound = _bound(module, x, whole)
        # one token, a chain of three, one token ..
        place = prompt.clone()
        for drafts in (1, 3, 1, 30, 2):
            new = place + torch.arange(drafts, device="cuda")
            out = module.decode(x.gather(1, new[..., None].expand(-1, -1, x.size(2))), cache,
                                cache_slots(table, sequences, new, page), table, (place + drafts)[:, 0].to(torch.int32))
            want = whole.gather(1, new[..., None].expand(-1, -1, x.size(2)))
            assert ((out.double() - want.double()).abs() <= bound).all()
            place = place + drafts
    torch.cuda.synchronize()
    sparse_ops.check_device_status(0)


def test_forward_with_a_cache_still_trains():
    from sparse import cache_slots, make_cache
    module = _module(64, 256, torch.float16)
    x = torch.randn(1, 256, module.embed_dim, device="cuda", dtype=torch.float16)
    cache = make_cache(8, 32, module.num_heads, module.head_dim, torch.float8_e4m3fn)
    table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    slots = cache_slots(table, torch.tensor([0], device="cuda"), torch.arange(256, device="cuda"), 32)
    module(x, cache=cache, slots=slots).sum().backward()
    with_cache = module.qkv.weight.grad.clone()
    module.zero_grad()
    module(x).sum().backward()
    assert torch.equal(with_cache, module.qkv.weight.grad)


def test_serving_refusals():
    from sparse import BlockSparseSelfAttention, make_cache
    module = _module(64, 256, torch.float16)
    plain = BlockSparseSelfAttention(module.embed_dim, module.num_heads, module.layout, causal=False, device="cuda", dtype=torch.float16)
    cache = make_cache(8, 32, module.num_heads, module.head_dim, torch.float16)
    x = torch.randn(1, 1, module.embed_dim, device="cuda", dtype=torch.float16)
    table = torch.zeros(1, 8, dtype=torch.int32, device="cuda")
    one = torch.ones(1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        plain.decode(x, cache, torch.zeros(1, dtype=torch.int64, device="cuda"), table, one)
    with pytest.raises(ValueError):
        module(x.expand(1, 256, -1), cache=cache)
    with pytest.raises(RuntimeError):
        module.decode(x, make_cache(8, 32, 2, module.head_dim, torch.float16), torch.zeros(1, dtype=torch.int64, device="cuda"), table, one)
