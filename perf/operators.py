"""What the operators over a paged key/value cache in 8 bits are measured on, and their plain forms.

The cache: ``key_cache`` and ``value_cache`` hold float8_e4m3fn codes ``[num_blocks, num_kv_heads,
block_size, head_dim]``; ``kv_scale`` holds float32 ``[num_blocks, num_kv_heads, 2]``, one scale for the
keys and one for the values of each block and head.  An element stands for code * scale.

Three operators:

* ``append``: the rotary embedding of a step's queries and keys and the write of the rotated keys and the
  values into the cache (``rope_cache_write_fp8``).  A block's scale is the smallest power of two with
  which its largest value fits 448; it grows as rows come in, and the rows already there are rounded anew
  to it.  Writing a block's first slot starts the block anew.
* ``decode``: attention of one query token per sequence over its blocks (``paged_decode_attention_fp8``).
* ``prefill``: causal attention of chunks of query tokens over their sequences' blocks, the chunk's own
  positions among them (``paged_prefill_attention_fp8``).
"""

import math

import numpy as np
import torch

own = False

E4M3 = torch.float8_e4m3fn
FP8_MAX = 448.0
MIN_EXP = -100  # the smallest scale is 2**MIN_EXP (a block of zeros)
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    small = dict(heads=14, kv_heads=2, head_dim=64, block_size=16)
    large = dict(heads=32, kv_heads=8, head_dim=128, block_size=16)
    return [
        # one sequence's next token: nothing but latency
        dict(name="append 1", op="append", seqs=1, lo=700, hi=700, query=1, dtype="bf16", table="f32", pad=0, **small),
        # the decode step of 256 sequences (contexts of 128 to 2048)
        dict(name="append 256", op="append", seqs=256, lo=128, hi=2048, query=1, dtype="bf16", table="same", pad=0,
             **small),
        # the decode step of 1024 sequences of a larger model, in a batch padded to a graph's size
        dict(name="append 1024 wide", op="append", seqs=1024, lo=16, hi=1500, query=1, dtype="f16", table="same",
             pad=24, **large),
        # prefill chunks: ragged pieces of 12 sequences, each after a cached prefix of its own
        dict(name="append chunks wide", op="append", seqs=12, lo=0, hi=3000, query=1200, dtype="bf16", table="f32",
             pad=0, **large),
        # one sequence answered alone
        dict(name="decode 1x1000", op="decode", seqs=1, lo=1000, hi=1000, dtype="bf16", **small),
        # the serving step: 256 sequences of 128 to 2048 tokens
        dict(name="decode 256x2048", op="decode", seqs=256, lo=128, hi=2048, dtype="bf16", **small),
        # long contexts, few sequences
        dict(name="decode 32x32768", op="decode", seqs=32, lo=32768, hi=32768, dtype="f16", **small),
        # one GPU's share of a larger model's batch: many short contexts, a few long ones
        dict(name="decode 256 wide", op="decode", seqs=256, lo=16, hi=8192, dtype="bf16", skew=1, **large),
        # the last short chunk of a prompt whose prefix is cached
        dict(name="prefill 37+1003", op="prefill", seqs=1, lo=1003, hi=1003, query=37, dtype="bf16", **small),
        # a step's chunks of eight prompts, ragged, some with a prefix
        dict(name="prefill 8x512", op="prefill", seqs=8, lo=0, hi=2000, query=512, dtype="bf16", **small),
        # one long prompt at once
        dict(name="prefill 1x8192", op="prefill", seqs=1, lo=0, hi=0, query=8192, dtype="bf16", **small),
        # long chunks after long prefixes, a larger model
        dict(name="prefill 4x2048 wide", op="prefill", seqs=4, lo=3000, hi=6144, query=2048, dtype="f16", **large),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kv_heads, group, head_dim = rng.choice([(2, 7, 64), (8, 4, 128), (8, 1, 128), (1, 16, 64), (4, 3, 64), (4, 8, 128),
                                            (2, 5, 128), (1, 12, 128), (12, 1, 64), (2, 20, 64)])
    case = dict(op=rng.choice(["append", "decode", "prefill"]), heads=kv_heads * group, kv_heads=kv_heads,
                head_dim=head_dim, block_size=rng.choice([16, 16, 16, 32, 64, 128]), dtype=rng.choice(["bf16", "f16"]))
    width = kv_heads * head_dim
    if case["op"] == "append":
        case["query"] = rng.choice([1, 1, _log(rng, 2, 4000)])
        case["seqs"] = _log(rng, 1, 1024 if case["query"] == 1 else max(1, 9000 // case["query"]))
        case["hi"] = _log(rng, 1, 3000)
        case["lo"] = rng.randint(0, case["hi"])
        case["pad"] = rng.choice([0, 0, rng.randint(1, 40)])
        case["table"] = rng.choice(["f32", "same"])
    elif case["op"] == "decode":
        tokens = _log(rng, 1, 64 * 1024 * 1024 // width)  # of all sequences, as many as the large listed case has
        case["hi"] = max(1, min(_log(rng, 1, 65536), tokens))
        case["seqs"] = max(1, min(1024, tokens // case["hi"]))
        case["lo"] = max(1, int(case["hi"] * rng.random()))
    else:
        case["query"] = _log(rng, 1, 2048)
        case["hi"] = _log(rng, 1, 6000) - 1
        case["lo"] = rng.randint(0, case["hi"])
        most = (1 << 31) // (case["heads"] * case["query"] * (case["hi"] + case["query"]))
        case["seqs"] = max(1, min(_log(rng, 1, 64), most))
    return case


def _lengths(case):
    """Cached tokens and query tokens of each sequence: a function of the case alone."""
    r = np.random.RandomState(case["seqs"] * 131 + case["hi"] * 7 + case.get("query", 0))
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    if case.get("skew"):
        cached = np.clip(np.rint(r.lognormal(7.0, 0.8, n)), lo, hi).astype(np.int64)
    else:
        cached = r.randint(lo, hi + 1, n).astype(np.int64)
    q = case.get("query", 0)
    if case["op"] == "decode" or n == 1:
        query = np.full(n, q, dtype=np.int64)
    else:
        query = r.randint(max(1, q // 4), q + 1, n).astype(np.int64)
        query[0] = q
    return cached, query


def work(case):
    cached, query = _lengths(case)
    H, KH, D, BS = case["heads"], case["kv_heads"], case["head_dim"], case["block_size"]
    total, T = int((cached + query).sum()), int(query.sum())
    blocks = int((-(-(cached + query) // BS)).sum())
    if case["op"] == "append":
        touched = int(((cached + query - 1) // BS - cached // BS + 1).sum())
        table = 4 if case["table"] == "f32" else 2
        moved = T * D * (2 * H * 2 + 2 * KH * 2 + 2 * KH + 2 * table) + 16 * T + 16 * touched * KH
        return {"bytes": moved, "flops": T * D * (3 * H + 5 * KH)}
    if case["op"] == "decode":
        return {"bytes": total * 2 * KH * D + blocks * (8 * KH + 8) + case["seqs"] * (4 * H * D + 4),
                "flops": 4 * total * H * D}
    pairs = int((query * cached + query * (query + 1) // 2).sum())
    return {"bytes": total * 2 * KH * D + blocks * (8 * KH + 8) + T * H * D * 4, "flops": 4 * pairs * H * D}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _power_of_two_scale(amax):
    """The smallest power of two s >= 2**MIN_EXP with amax <= 448 s (448 = 0.875 * 2**9)."""
    f, e = torch.frexp(amax)
    e = torch.where(f > 0.875, e - 8, e - 9)
    return torch.ldexp(torch.ones_like(amax), torch.where(amax > 0, e.clamp_min(MIN_EXP), torch.full_like(e, MIN_EXP)))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    r = np.random.RandomState(seed % (1 << 31))
    H, KH, D, BS = case["heads"], case["kv_heads"], case["head_dim"], case["block_size"]
    dtype = DTYPES[case["dtype"]]
    cached, query = _lengths(case)
    n, T = case["seqs"], int(query.sum())
    need = -(-(cached + query) // BS)
    num_blocks = int(need.sum() * 1.1) + 16
    perm = r.permutation(num_blocks)
    table = np.full((n, int(need.max())), -1, dtype=np.int64)
    start = np.concatenate([[0], np.cumsum(need)])
    for i in range(n):
        table[i, :need[i]] = perm[start[i]:start[i + 1]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    spread = torch.exp(0.5 * normal(1, KH, 1, D))  # some channels of the keys are larger than others
    caches, scales = [], []
    for which in range(2):
        x = normal(num_blocks, KH, BS, D)
        x = x * spread if which == 0 else x
        s = _power_of_two_scale(x.abs().amax((2, 3)))
        caches.append((x / s[..., None, None]).to(E4M3))
        scales.append(s)
        del x
    state = {"case": case, "key_cache": caches[0], "value_cache": caches[1], "kv_scale": torch.stack(scales, -1),
             "block_table": torch.from_numpy(table).to(dev)}
    if case["op"] == "decode":
        kv_len = torch.from_numpy(cached.astype(np.int32)).to(dev)
        # what lies behind a sequence's last token is what the memory held: codes of NaN among it
        at = torch.arange(table.shape[1] * BS, device=dev).view(1, -1, BS) >= kv_len[:, None, None]
        at &= (state["block_table"] >= 0)[..., None]
        seq, blk, off = at.nonzero(as_tuple=True)
        for c in caches:
            c.view(torch.uint8)[state["block_table"][seq, blk], :, off] = 0x7F
        state["kv_len"] = kv_len
        state["query"] = (normal(n, H, D) / spread.view(1, KH, 1, D).expand(1, KH, H // KH, D).reshape(1, H, D)).to(dtype)
        return state
    seq = np.repeat(np.arange(n), query)
    pos = np.concatenate([np.arange(c, c + q) for c, q in zip(cached, query)])
    if case["op"] == "prefill":
        state["query"] = (0.7 * normal(T, H, D)).to(dtype)
        for name, v in (("seq_rows", np.arange(n)), ("cached_len", cached), ("query_len", query)):
            state[name] = torch.from_numpy(v.astype(np.int64)).to(dev)
        state["max_query"] = int(query.max())
        return state
    slots = table[seq, pos // BS] * BS + pos % BS
    pad = case["pad"]
    slots = np.concatenate([slots, np.full(pad, -1, dtype=np.int64)])  # rows of a padded batch write nothing
    pos = np.concatenate([pos, np.zeros(pad, dtype=np.int64)])
    rows = int(pos.max()) + 1
    angle = torch.arange(rows, device=dev, dtype=torch.float64)[:, None] * 1e6 ** (
        -torch.arange(0, D, 2, device=dev, dtype=torch.float64) / D)
    angle = torch.cat([angle, angle], -1)
    tables = torch.float32 if case["table"] == "f32" else dtype
    qkv = normal(T + pad, H + 2 * KH, D)  # the fused projection's output: query, key and value are views of it
    qkv[:, H:H + KH] *= spread[:, :, 0] * torch.exp(0.7 * normal(T + pad, KH, 1))
    qkv = qkv.to(dtype)
    state.update(query=qkv[:, :H], key=qkv[:, H:H + KH], value=qkv[:, H + KH:], cos=angle.cos().to(tables),
                 sin=angle.sin().to(tables), positions=torch.from_numpy(pos).to(dev),
                 slot_mapping=torch.from_numpy(slots).to(dev))
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return {"append": _append, "decode": _decode, "prefill": _prefill}[state["case"]["op"]](state)


def _append(s):
    BS = s["case"]["block_size"]
    if own:
        import mini_vllm_b200 as M

        query, _ = M.rope_cache_write_fp8(s["query"], s["key"], s["value"], s["positions"], s["cos"], s["sin"],
                                          s["key_cache"], s["value_cache"], s["kv_scale"], s["slot_mapping"], BS,
                                          strict=False)
        return {"query": query, "key_cache": s["key_cache"], "value_cache": s["value_cache"], "kv_scale": s["kv_scale"]}
    cos, sin = (s[k][s["positions"]].double()[:, None] for k in ("cos", "sin"))

    def rotated(x):  # in 64 bits: the largest value of a block may lie next to a power of two of its scale
        x = x.double()
        lo, hi = x.chunk(2, -1)
        return (x * cos + torch.cat([-hi, lo], -1) * sin).float()

    live = (s["slot_mapping"] >= 0).nonzero()[:, 0]
    slot = s["slot_mapping"][live]
    block, offset = slot // BS, slot % BS
    fresh = torch.zeros(s["kv_scale"].shape[0], dtype=torch.bool, device=slot.device)
    fresh[block[offset == 0]] = True
    scale = s["kv_scale"].clone()
    for which, (x, cache) in enumerate(((rotated(s["key"]), s["key_cache"]), (s["value"].float(), s["value_cache"]))):
        x = x[live]
        base = torch.where(fresh[:, None], 0.0, s["kv_scale"][..., which])
        amax = torch.zeros_like(base).index_reduce_(0, block, x.abs().amax(-1), "amax")
        new = torch.maximum(base, _power_of_two_scale(amax))[block]  # of each row's block
        codes = cache.view(torch.uint8)
        held = codes[block]  # [rows, KH, BS, D]: the whole block of every row
        grown = (base[block] > 0) & (new > base[block])
        ratio = torch.where(grown, base[block] / new, 1.0)[..., None, None]
        again = (held.view(E4M3).float() * ratio).to(E4M3).view(torch.uint8)
        codes[block] = torch.where(grown[..., None, None], again, held)
        codes[block, :, offset] = (x / new[..., None]).to(E4M3).view(torch.uint8)
        scale[..., which][block] = new
    s["kv_scale"].copy_(scale)
    return {"query": rotated(s["query"]).to(s["query"].dtype), "key_cache": s["key_cache"],
            "value_cache": s["value_cache"], "kv_scale": s["kv_scale"]}


def _rows(s, cache, which):
    """[sequences, KH, tokens, D] float32 of every block in the table."""
    at = s["block_table"].clamp_min(0)
    x = s[cache].view(torch.uint8)[at].view(E4M3).float() * s["kv_scale"][at][..., which][..., None, None]
    n, blocks, KH, BS, D = x.shape
    return x.transpose(1, 2).reshape(n, KH, blocks * BS, D)


def _decode(s):
    c = s["case"]
    if own:
        import mini_vllm_b200 as M

        return M.paged_decode_attention_fp8(s["query"], s["key_cache"], s["value_cache"], s["kv_scale"],
                                            s["block_table"], s["kv_len"], c["block_size"], strict=False)
    n, H, D = s["query"].shape
    KH = c["kv_heads"]
    k, v = _rows(s, "key_cache", 0), _rows(s, "value_cache", 1)
    live = torch.arange(k.shape[2], device=k.device) < s["kv_len"][:, None]
    v = torch.where(live[:, None, :, None], v, 0.0)
    q = s["query"].float().view(n, KH, H // KH, D)
    x = torch.matmul(q, k.transpose(2, 3)) * D ** -0.5
    x = torch.where(live[:, None, None], x, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    return (torch.matmul(p, v) / p.sum(-1, keepdim=True)).reshape(n, H, D).to(s["query"].dtype)


def _prefill(s):
    c = s["case"]
    if own:
        import mini_vllm_b200 as M

        return M.paged_prefill_attention_fp8(s["query"], s["key_cache"], s["value_cache"], s["kv_scale"],
                                             s["block_table"], s["seq_rows"], s["cached_len"], s["query_len"],
                                             c["block_size"], strict=False)
    T, H, D = s["query"].shape
    KH, most, n = c["kv_heads"], s["max_query"], c["seqs"]
    end = torch.cumsum(s["query_len"], 0)
    first = end - s["query_len"]
    step = torch.arange(most, device=end.device)
    at = (first[:, None] + step).clamp_max(T - 1)  # [n, most]: chunks padded to the longest
    q = s["query"].float()[at].view(n, most, KH, H // KH, D).permute(0, 2, 3, 1, 4).reshape(n, KH, -1, D)
    k, v = _rows(s, "key_cache", 0), _rows(s, "value_cache", 1)
    seen = torch.arange(k.shape[2], device=k.device) <= (s["cached_len"][:, None] + step)[..., None]  # [n, most, L]
    x = (torch.matmul(q, k.transpose(2, 3)) * D ** -0.5).view(n, KH, H // KH, most, -1)
    x = torch.where(seen[:, None, None], x, -math.inf)
    x -= x.amax(-1, keepdim=True)
    p = torch.exp_(x)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(n, KH, (H // KH) * most, -1), v).view(n, KH, H // KH, most, D) / total
    chunk = torch.searchsorted(end, torch.arange(T, device=end.device), right=True)
    row = torch.arange(T, device=end.device) - first[chunk]
    return o.permute(0, 3, 1, 2, 4)[chunk, row].reshape(T, H, D).to(s["query"].dtype)


# ---------------------------------------------------------------------------
# the same in 64 bits
# ---------------------------------------------------------------------------
def _e4m3_grid(x):
    """x rounded to the nearest value of 4 exponent and 3 mantissa bits, ties to the even one (|x| <= 448)."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    BS, H, KH, D = case["block_size"], case["heads"], case["kv_heads"], case["head_dim"]
    if case["op"] == "append":
        return _exact_append(s, BS, D)
    cached, query = _lengths(case)
    group, outs, row = H // KH, [], 0
    for i in range(case["seqs"]):
        length = int(cached[i] + query[i])
        blocks = s["block_table"][i, :-(-length // BS)]
        kv = []
        for which, name in enumerate(("key_cache", "value_cache")):
            x = s[name].view(torch.uint8)[blocks].view(E4M3).double() * s["kv_scale"][blocks, :, which].double()[..., None, None]
            kv.append(x.permute(1, 0, 2, 3).reshape(KH, -1, D)[:, :length])
        rows = 1 if case["op"] == "decode" else int(query[i])
        q = s["query"][row:row + rows].double().permute(1, 0, 2)  # [H, rows, D]
        o = torch.empty_like(q)
        last = torch.arange(length - rows, length, device=q.device)
        hide = torch.arange(length, device=q.device) > last[:, None]
        for h in range(H):
            x = (q[h] @ kv[0][h // group].T) / math.sqrt(D)
            x.masked_fill_(hide, -math.inf)
            o[h] = torch.softmax(x, -1) @ kv[1][h // group]
        outs.append(o.permute(1, 0, 2))
        row += rows
    return torch.cat(outs)


def _exact_append(s, BS, D):
    half = D // 2
    pos = s["positions"]
    cos, sin = s["cos"].double()[pos].unsqueeze(1), s["sin"].double()[pos].unsqueeze(1)

    def turn(x):
        x = x.double()
        out = torch.empty_like(x)
        out[..., :half] = x[..., :half] * cos[..., :half] - x[..., half:] * sin[..., :half]
        out[..., half:] = x[..., half:] * cos[..., half:] + x[..., :half] * sin[..., half:]
        return out

    num_blocks, KH = s["kv_scale"].shape[:2]
    # which token writes a slot (-1: none), block by block
    writer = torch.full((num_blocks * BS + 1,), -1, dtype=torch.long, device=pos.device)
    writer[s["slot_mapping"]] = torch.arange(len(pos), device=pos.device)  # slot -1 falls on the spare place
    writer = writer[:-1].view(num_blocks, BS)
    hit = (writer >= 0).any(1).nonzero()[:, 0]
    w = writer[hit]
    out = {"query": turn(s["query"])}
    scale = s["kv_scale"].double()
    for which, (name, x) in enumerate((("key_cache", turn(s["key"]).float().double()), ("value_cache", s["value"].double()))):
        rows = x[w.clamp_min(0)].permute(0, 2, 1, 3)  # [blocks hit, KH, BS, D]
        new = (w >= 0)[:, None, :, None]
        rows = torch.where(new, rows, 0.0)
        base = torch.where((w[:, 0] >= 0)[:, None], 0.0, scale[hit, :, which])
        amax = rows.abs().flatten(2).amax(2)
        least = torch.exp2(torch.ceil(torch.log2((amax / FP8_MAX).clamp_min(2.0 ** MIN_EXP))))
        now = torch.maximum(base, least)
        cache = s[name].double()
        held = cache[hit]
        factor = torch.where(base > 0, base / now, 1.0)[..., None, None]
        held = torch.where(factor < 1, _e4m3_grid(held * factor), held)
        cache[hit] = torch.where(new, _e4m3_grid(rows / now[..., None, None]), held)
        scale[hit, :, which] = now
        out[name] = cache
    out["kv_scale"] = scale
    return out
