"""Cases, plain forms and 64-bit values of the packed, cached and cache-writing attention operators.

Four operators are covered, the ones a model with these attention layers needs for training on packed
documents and for answering with a key / value cache:

* ``packed``: attention inside every sequence of a packed batch, grouped heads, with its gradient;
* ``write``:  keys and values of new tokens into a paged cache, 16-bit or e4m3 with a scale per token and head;
* ``read``:   keys and values of given places of that cache, as 16-bit values;
* ``cached``: attention of one or more drafted tokens per sequence over the paged cache (a chain or a tree).
"""
import math

import torch

own = False

E4M3_MAX = 448.0
AMAX_FLOOR = 2.0 ** -100         # smallest amax a scale is made from: keeps 448 / amax finite


# ------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # Serving: prompts of one scheduler step, grouped heads.
        {"name": "packed_prompts_bf16_d128", "op": "packed", "dtype": "bfloat16", "grad": False, "causal": True,
         "q_heads": 16, "kv_heads": 4, "dim": 128, "fused": True, "tail": 0,
         "lengths": "4096,4001,2987,2500,1777,700,65,1"},
        # Many short requests of odd lengths, one key head per query head, rows behind the last sequence.
        {"name": "packed_short_fp16_d64", "op": "packed", "dtype": "float16", "grad": False, "causal": True,
         "q_heads": 12, "kv_heads": 12, "dim": 64, "fused": False, "tail": 5,
         "lengths": "1024,33,517,1,250,128,129,90,600,17,2,311,64,777,405,63"},
        # Training on packed documents: forward and backward of one layer.
        {"name": "packed_train_bf16_d128", "op": "packed", "dtype": "bfloat16", "grad": True, "causal": True,
         "q_heads": 16, "kv_heads": 4, "dim": 128, "fused": True, "tail": 0,
         "lengths": "4096,2049,1000,801,200,45,1"},
        {"name": "packed_train_fp16_d64", "op": "packed", "dtype": "float16", "grad": True, "causal": True,
         "q_heads": 16, "kv_heads": 16, "dim": 64, "fused": False, "tail": 0,
         "lengths": "2048,1500,333,129,86"},
        # One new token of one request: the smallest write.
        {"name": "write_token_e4m3", "op": "write", "dtype": "bfloat16", "store": "e4m3", "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 1, "start": 300, "tokens": 1, "skipped": 0},
        # Prompts into the 8-bit cache.
        {"name": "write_prompts_e4m3", "op": "write", "dtype": "bfloat16", "store": "e4m3", "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 4, "start": 0, "tokens": 4001, "skipped": 3},
        # A decoding step's drafts into a 16-bit cache with small pages.
        {"name": "write_drafts_fp16", "op": "write", "dtype": "float16", "store": "same", "kv_heads": 12, "dim": 64,
         "page": 16, "sequences": 96, "start": 701, "tokens": 9, "skipped": 20},
        # A long prefix read back from the 8-bit cache (moved to another pool, or attended to as a prompt).
        {"name": "read_prefix_e4m3", "op": "read", "dtype": "bfloat16", "store": "e4m3", "kv_heads": 8, "dim": 128,
         "page": 64, "sequences": 2, "start": 0, "tokens": 8191, "skipped": 0},
        {"name": "read_blocks_fp16", "op": "read", "dtype": "float16", "store": "same", "kv_heads": 12, "dim": 64,
         "page": 16, "sequences": 7, "start": 5, "tokens": 150, "skipped": 4},
        # One token of one request over a short cache: latency.
        {"name": "cached_one_token_bf16", "op": "cached", "dtype": "bfloat16", "store": "same", "q_heads": 16,
         "kv_heads": 4, "dim": 128, "page": 64, "drafts": 1, "ragged": False, "tree": False, "lengths": "391"},
        # One token of each of many requests, 8-bit cache: the ordinary decoding step.
        {"name": "cached_batch_e4m3", "op": "cached", "dtype": "bfloat16", "store": "e4m3", "q_heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "drafts": 1, "ragged": False, "tree": False,
         "lengths": "8192,5000,4097,3500,3001,2800,2222,2048,1999,1500,1203,1024,1000,900,800,777,"
                    "650,600,513,512,400,333,300,256,200,129,100,65,64,33,7,1"},
        # Trees of drafted tokens over a long cache.
        {"name": "cached_tree_bf16", "op": "cached", "dtype": "bfloat16", "store": "same", "q_heads": 16,
         "kv_heads": 4, "dim": 128, "page": 32, "drafts": 24, "ragged": True, "tree": True,
         "lengths": "32768,9001,4000,150"},
    ]


def _spread(rng, low, high):
    """A whole number, its logarithm uniform between those of `low` and `high`."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["packed", "packed", "write", "read", "cached", "cached"])
    dtype = rng.choice(["float16", "bfloat16"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 5, 8])
    group = rng.choice([1, 2, 3, 4, 8])
    page = rng.choice([16, 32, 64, 128])
    if op == "packed":
        group = min(group, 16 // kv_heads) or 1
        longest = _spread(rng, 16, 4096)
        count = max(1, min(_spread(rng, 1, 64), 2 ** 26 // longest ** 2))
        lengths = [longest] + [_spread(rng, 1, longest) for _ in range(count - 1)]
        rng.shuffle(lengths)
        case = {"op": op, "dtype": dtype, "grad": rng.random() < 0.5, "causal": rng.random() < 0.8,
                "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim, "fused": rng.random() < 0.5,
                "tail": rng.choice([0, 0, 3, 130]), "lengths": ",".join(str(n) for n in lengths)}
        while work(case)["flops"] > 2.0e11:                   # within the cost of the largest listed case
            lengths = [-(-n * 2 // 3) for n in lengths]
            case["lengths"] = ",".join(str(n) for n in lengths)
        return case
    store = rng.choice(["same", "e4m3"])
    if op in ("write", "read"):
        sequences = _spread(rng, 1, 64)
        return {"op": op, "dtype": dtype, "store": store, "kv_heads": kv_heads, "dim": dim, "page": page,
                "sequences": sequences, "start": rng.randrange(0, 300),
                "tokens": _spread(rng, 1, 16000 // sequences), "skipped": rng.choice([0, 0, 1, 5])}
    batch = _spread(rng, 1, 32)
    longest = _spread(rng, 16, 32768 // batch)
    lengths = [longest] + [_spread(rng, 1, longest) for _ in range(batch - 1)]
    drafts = rng.choice([1, 1, 1, 2, 5, 8, 13, 24])
    return {"op": op, "dtype": dtype, "store": store, "q_heads": kv_heads * group, "kv_heads": kv_heads, "dim": dim,
            "page": page, "drafts": drafts, "ragged": rng.random() < 0.5, "tree": drafts > 1 and rng.random() < 0.6,
            "lengths": ",".join(str(n) for n in lengths)}


def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def _counts(case):
    """Drafted tokens of every sequence of a `cached` case (never more than the sequence has tokens)."""
    return [min(n, case["drafts"] - i % case["drafts"] if case["ragged"] else case["drafts"])
            for i, n in enumerate(_lengths(case))]


def work(case):
    d, hk = case["dim"], case["kv_heads"]
    if case["op"] == "packed":
        lengths = _lengths(case)
        total, hq = sum(lengths) + case["tail"], case["q_heads"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lengths)
        forward = 2 * total * d * (2 * hq + 2 * hk)                       # q, o; k, v
        backward = 2 * total * d * (2 * hq + 2 * hk)                      # dout, dq; dk, dv
        return {"bytes": forward + (backward if case["grad"] else 0),
                "flops": (14 if case["grad"] else 4) * d * hq * pairs}
    held = d + 4 if case["store"] == "e4m3" else 2 * d                    # bytes of one stored head of one token
    if case["op"] in ("write", "read"):
        given = case["sequences"] * case["tokens"]
        used = given - min(case["skipped"], given)
        moved = (given if case["op"] == "read" else used) * 2 * d + used * held
        return {"bytes": 2 * hk * moved + 8 * given, "flops": 2 * hk * used * d * (2 if case["store"] == "e4m3" else 0)}
    lengths, counts, hq = _lengths(case), _counts(case), case["q_heads"]
    pages = sum(-(-n // case["page"]) for n in lengths)
    return {"bytes": 2 * hk * held * sum(lengths) + 4 * len(lengths) * case["drafts"] * hq * d + 4 * pages,
            "flops": 4 * d * hq * sum(n * c for n, c in zip(lengths, counts))}


# ------------------------------------------------------------------------------------------------- the inputs
def _ancestors(parents):
    """Bit j of word i: draft i is draft j or a descendant of it (as signed 64-bit words)."""
    words = []
    for i, p in enumerate(parents):
        words.append((words[p] if p >= 0 else 0) | 1 << i)
    return [w - (1 << 64) if w >> 63 else w for w in words]


def _pages(gen, lengths, page, spare):
    """A page table (-1 behind a sequence's last page) over pages in random order, and the number of pages."""
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need) + spare, generator=gen, dtype=torch.int64)
    table = torch.full((len(lengths), max(need)), -1, dtype=torch.int64)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, sum(need) + spare


def _cache(case, pages, dev_gen, dtype):
    """Keys, values and their scales (None in a 16-bit cache) of a cache that is in use."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    x = torch.randn((2,) + shape, generator=dev_gen, device="cuda", dtype=torch.float32)
    if case["store"] == "same":
        return x[0].to(dtype), x[1].to(dtype), None, None
    (keys, key_scales), (values, value_scales) = _quantised(x[0]), _quantised(x[1])
    return keys, values, key_scales, value_scales


def prepare(case, seed):
    gen = torch.Generator().manual_seed(seed)
    dev_gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = getattr(torch, case["dtype"])
    d, hk = case["dim"], case["kv_heads"]

    def normal(*shape):
        return torch.randn(shape, generator=dev_gen, device="cuda", dtype=torch.float32).to(dtype)

    if case["op"] == "packed":
        lengths, hq = _lengths(case), case["q_heads"]
        rows = sum(lengths) + case["tail"]
        if case["fused"]:                                     # views of one projection's output
            q, k, v = normal(rows, hq + 2 * hk, d).split([hq, hk, hk], dim=1)
        else:
            q, k, v = normal(rows, hq, d), normal(rows, hk, d), normal(rows, hk, d)
        offsets = torch.tensor([0] + lengths).cumsum(0).to(torch.int32).cuda()
        return {"op": "packed", "q": q, "k": k, "v": v, "dout": normal(rows, hq, d) if case["grad"] else None,
                "offsets": offsets, "longest": max(lengths), "scale": d ** -0.5, "causal": case["causal"]}
    if case["op"] in ("write", "read"):
        sequences, tokens, page = case["sequences"], case["tokens"], case["page"]
        table, pages = _pages(gen, [case["start"] + tokens] * sequences, page, 3)
        at = torch.arange(case["start"], case["start"] + tokens)
        slots = (table[:, at // page] * page + at % page).reshape(-1)
        skip = torch.randperm(slots.numel(), generator=gen)[:case["skipped"]]
        slots[skip] = -1                                      # padding of the batch: not written, read as zero
        keys, values, key_scales, value_scales = _cache(case, pages, dev_gen, dtype)
        state = {"op": case["op"], "slots": slots.cuda(), "keys": keys, "values": values, "key_scales": key_scales,
                 "value_scales": value_scales, "dtype": dtype}
        if case["op"] == "write":
            state["k"], state["v"] = normal(slots.numel(), hk, d), normal(slots.numel(), hk, d)
        return state
    lengths, counts, drafts = _lengths(case), _counts(case), case["drafts"]
    table, pages = _pages(gen, lengths, case["page"], 2)
    keys, values, key_scales, value_scales = _cache(case, pages, dev_gen, dtype)
    tree = None
    if case["tree"]:
        parents = [[int(torch.randint(-1, i, (1,), generator=gen)) if i else -1 for i in range(drafts)] for _ in lengths]
        tree = torch.tensor([_ancestors(p) for p in parents], dtype=torch.int64).cuda()
    return {"op": "cached", "q": normal(len(lengths), drafts, case["q_heads"], d), "keys": keys, "values": values,
            "key_scales": key_scales, "value_scales": value_scales, "table": table.to(torch.int32).cuda(),
            "lengths": torch.tensor(lengths, dtype=torch.int32).cuda(),
            "counts": torch.tensor(counts, dtype=torch.int32).cuda(), "tree": tree, "scale": d ** -0.5}


# ------------------------------------------------------------------------------------------------- plain forms
def _quantised(x):
    """e4m3 codes of fp32 `x` and the fp32 scale of every row of its last axis."""
    amax = x.abs().amax(dim=-1, keepdim=True).clamp_min(AMAX_FLOOR)
    return (x * (E4M3_MAX / amax)).to(torch.float8_e4m3fn), (amax / E4M3_MAX).squeeze(-1)


def _softmax(scores, visible):
    """Row softmax over the visible places; a row that sees nothing is zero."""
    scores = scores.masked_fill(~visible, -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    return p / p.sum(dim=-1, keepdim=True).clamp_min(1e-30)


def _plain_packed(state):
    """The sequences padded to the longest one, attention in fp32, and the rows gathered back."""
    q, k, v, offsets, longest = state["q"], state["k"], state["v"], state["offsets"].long(), state["longest"]
    rows, hq, d = q.shape
    hk, batch = k.size(1), offsets.numel() - 1
    g, dtype, scale = hq // hk, q.dtype, state["scale"]
    at = torch.arange(longest, device=q.device)
    inside = at < (offsets[1:] - offsets[:-1])[:, None]                             # [batch, longest]
    take = (offsets[:-1, None] + at).clamp_max(rows - 1)
    token = torch.arange(rows, device=q.device)
    seq = torch.searchsorted(offsets, token, right=True) - 1
    real = (seq < batch)[:, None, None]
    seq = seq.clamp_max(batch - 1)
    place = (token - offsets[seq]).clamp_max(longest - 1)

    def padded(x, heads, share):                                                    # [batch, hk, share, longest, d]
        return x[take].float().view(batch, longest, heads // share, share, d).permute(0, 2, 3, 1, 4)

    def gathered(x, heads):
        x = x.permute(0, 3, 1, 2, 4).reshape(batch, longest, heads, d)[seq, place]
        return torch.where(real, x, 0.0).to(dtype)

    qp, kp, vp = padded(q, hq, g), padded(k, hk, 1), padded(v, hk, 1)
    visible = inside[:, None, :] & inside[:, :, None]
    if state["causal"]:
        visible = visible & (at <= at[:, None])
    p = _softmax(qp @ kp.transpose(-1, -2) * scale, visible[:, None, None])
    out = gathered(p @ vp, hq)
    if state["dout"] is None:
        return out
    do = padded(state["dout"], hq, g) * inside[:, None, None, :, None]
    dv = (p.transpose(-1, -2) @ do).sum(dim=2, keepdim=True)
    dp = do @ vp.transpose(-1, -2)
    ds = p * (dp - (p * dp).sum(dim=-1, keepdim=True)) * scale
    dk = (ds.transpose(-1, -2) @ qp).sum(dim=2, keepdim=True)
    return out, gathered(ds @ kp, hq), gathered(dk, hk), gathered(dv, hk)


def _plain_write(state):
    keys, values, slots = state["keys"], state["values"], state["slots"]
    pages, hk, page, d = keys.shape
    # a skipped token writes to a place behind the cache's end, which is cut off again
    to = torch.where(slots < 0, pages * page, slots)

    def put(buffer, new):
        raw = buffer.view(torch.uint8) if buffer.dtype == torch.float8_e4m3fn else buffer
        flat = raw.transpose(1, 2).reshape((pages * page, hk) + raw.shape[3:])
        flat = torch.cat([flat, flat[:1]]).index_copy_(0, to, new)[:-1]
        raw.copy_(flat.view((pages, page, hk) + raw.shape[3:]).transpose(1, 2))

    for buffer, scales, new in ((keys, state["key_scales"], state["k"]), (values, state["value_scales"], state["v"])):
        if scales is None:
            put(buffer, new)
        else:
            codes, made = _quantised(new.float())
            put(buffer, codes.view(torch.uint8))
            put(scales, made)
    return _cache_of(state)


def _cache_of(state):
    return [t for t in (state["keys"], state["values"], state["key_scales"], state["value_scales"]) if t is not None]


def _plain_read(state):
    slots, page = state["slots"], state["keys"].size(2)
    real = (slots >= 0)[:, None, None]
    at = slots.clamp_min(0)

    def get(buffer, scales):
        x = buffer.float() if scales is None else buffer.float() * scales[..., None]
        return torch.where(real, x[at // page, :, at % page], 0.0).to(state["dtype"])

    return get(state["keys"], state["key_scales"]), get(state["values"], state["value_scales"])


def _plain_cached(state):
    q, table, lengths, counts = state["q"], state["table"].long().clamp_min(0), state["lengths"], state["counts"]
    batch, drafts, hq, d = q.shape
    hk = state["keys"].size(1)

    def gathered(buffer, scales):                                                   # [batch, hk, 1, keys, d]
        x = buffer[table] if scales is None else buffer.view(torch.uint8)[table].view(buffer.dtype)
        x = x.float() if scales is None else x.float() * scales[table][..., None]
        return x.transpose(1, 2).reshape(batch, hk, 1, -1, d)

    k, v = gathered(state["keys"], state["key_scales"]), gathered(state["values"], state["value_scales"])
    at = torch.arange(k.size(3), device=q.device)
    place = at - (lengths - counts)[:, None]                                        # number of a key among the drafts
    row = torch.arange(drafts, device=q.device)
    if state["tree"] is None:
        seen = place[:, None, :] <= row[:, None]
    else:
        seen = (place[:, None, :] < 0) | ((state["tree"][:, :, None] >> place[:, None, :].clamp(0, 63)) & 1).bool()
    seen = seen & (place < counts[:, None])[:, None, :] & (row < counts[:, None])[:, :, None]
    q = q.float().view(batch, drafts, hk, hq // hk, d).permute(0, 2, 3, 1, 4)
    p = _softmax(q @ k.transpose(-1, -2) * state["scale"], seen[:, None, None])
    return (p @ v).permute(0, 3, 1, 2, 4).reshape(batch, drafts, hq, d).to(state["q"].dtype)


# ------------------------------------------------------------------------------------------------- one pass
def _own(state):
    import sys
    folder = "experiments-pytorch-cuda-extension-for-sparse-matmul_b200"
    if folder not in sys.path:
        sys.path.insert(0, folder)
    import sparse
    op = state["op"]
    if op == "packed":
        if state["dout"] is None:
            return sparse.packed_attention(state["q"], state["k"], state["v"], state["offsets"], state["scale"],
                                           state["causal"])
        q, k, v = (state[name].detach().requires_grad_() for name in ("q", "k", "v"))
        out = sparse.packed_attention(q, k, v, state["offsets"], state["scale"], state["causal"])
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), state["dout"])
    cache = (state["keys"], state["values"], state["key_scales"], state["value_scales"])
    if op == "write":
        sparse.cache_write(state["k"], state["v"], state["slots"], *cache)
        return _cache_of(state)
    if op == "read":
        return sparse.cache_read(state["slots"], *cache, dtype=state["dtype"])
    return sparse.cached_attention(state["q"], *cache, state["table"], state["lengths"], counts=state["counts"],
                                   tree=state["tree"], scale=state["scale"])


def run(state):
    if own:
        return _own(state)
    return {"packed": _plain_packed, "write": _plain_write, "read": _plain_read, "cached": _plain_cached}[state["op"]](state)


# ------------------------------------------------------------------------------------------------- 64-bit values
def exact(case, seed):
    state = prepare(case, seed)
    return {"packed": _exact_packed, "write": _exact_write, "read": _exact_read, "cached": _exact_cached}[case["op"]](state, case)


def _exact_rows(q, k, v, scale, visible):
    """Probabilities and output of one head of one sequence in 64 bits."""
    s = torch.where(visible, (q @ k.T) * scale, -math.inf)
    p = torch.softmax(s, dim=-1).nan_to_num(0.0)
    return p, p @ v


def _exact_packed(state, case):
    q, k, v = (state[n].double() for n in ("q", "k", "v"))
    dout = None if state["dout"] is None else state["dout"].double()
    g, scale = q.size(1) // k.size(1), state["scale"]
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    start = 0
    for n in _lengths(case):
        rows = slice(start, start + n)
        visible = torch.ones(n, n, dtype=torch.bool, device=q.device)
        visible = visible.tril() if case["causal"] else visible
        for h in range(q.size(1)):
            c = h // g
            p, out[rows, h] = _exact_rows(q[rows, h], k[rows, c], v[rows, c], scale, visible)
            if dout is not None:
                do = dout[rows, h]
                dv[rows, c] += p.T @ do
                ds = p * (do @ v[rows, c].T - (do * out[rows, h]).sum(-1, keepdim=True)) * scale
                dq[rows, h] = ds @ k[rows, c]
                dk[rows, c] += ds.T @ q[rows, h]
        start += n
    return out if dout is None else (out, dq, dk, dv)


def _exact_write(state, case):
    """The cache after the write. Codes are e4m3 values of x / (amax / 448); a code that is rounded is no number of
    64 bits, so the codes stand for themselves and only the scales are given."""
    if case["store"] == "same":
        keys, values = state["keys"].double(), state["values"].double()
        for token, slot in enumerate(state["slots"].tolist()):
            if slot >= 0:
                keys[slot // case["page"], :, slot % case["page"]] = state["k"][token].double()
                values[slot // case["page"], :, slot % case["page"]] = state["v"][token].double()
        return [keys, values]
    held = []
    real = state["slots"] >= 0
    at = state["slots"][real]
    for scales, new in ((state["key_scales"], state["k"]), (state["value_scales"], state["v"])):
        made = scales.double()
        made[at // case["page"], :, at % case["page"]] = new[real].double().abs().amax(-1).clamp_min(AMAX_FLOOR) / E4M3_MAX
        held.append(made)
    return [None, None] + held


def _exact_read(state, case):
    slots = state["slots"]
    out = []
    for buffer, scales in ((state["keys"], state["key_scales"]), (state["values"], state["value_scales"])):
        flat = buffer.double().transpose(1, 2).flatten(0, 1)
        if scales is not None:
            flat = flat * scales.double().transpose(1, 2).flatten(0, 1).unsqueeze(-1)
        got = flat[slots.clamp_min(0)]
        got[slots < 0] = 0.0
        out.append(got)
    return tuple(out)


def _exact_cached(state, case):
    lengths, counts, page = _lengths(case), _counts(case), case["page"]
    q = state["q"].double()
    out = torch.zeros_like(q)
    g = q.size(2) // case["kv_heads"]
    for b, (n, c) in enumerate(zip(lengths, counts)):
        pages = state["table"][b, :-(-n // page)].long()
        held = []
        for buffer, scales in ((state["keys"], state["key_scales"]), (state["values"], state["value_scales"])):
            raw = buffer if scales is None else buffer.view(torch.uint8)
            x = raw[pages].view(buffer.dtype).double()
            if scales is not None:
                x = x * scales[pages].double().unsqueeze(-1)
            held.append(x.transpose(0, 1).flatten(1, 2)[:, :n])
        words = None if state["tree"] is None else state["tree"][b].tolist()
        visible = torch.ones(c, n, dtype=torch.bool)
        for i in range(c):
            for j in range(c):
                visible[i, n - c + j] = j <= i if words is None else words[i] >> j & 1
        visible = visible.to(q.device)
        for h in range(q.size(2)):
            out[b, :c, h] = _exact_rows(q[b, :c, h], held[0][h // g], held[1][h // g], state["scale"], visible)[1]
    return out
