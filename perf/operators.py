"""Cases that measure the operators of a serving step over an 8-bit KV cache: writing K and V rows into the
cache, reading cached rows back, decode attention over the cache, and sampling the next token.

`own = False` computes each operator in its plain form (elementary torch operations in 32 bits, in 64 where
sums or borders need it); `own = True` calls this package's operators (include/qwen_b200_ops.h) on the same
buffers. The cache holds blocks of 64 tokens: int8 codes [block][kv head][64][128] and one fp32 scale per
block and kv head, for K and for V; a table lists each sequence's blocks.
"""
import math

import numpy as np
import torch

own = False

BLOCK = 64
HEAD = 128
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
CODES = {"f32": 0, "f16": 1, "bf16": 2}
TINY = 2.0 ** -126
SCALE = 0.08838834764831845  # 1 / sqrt(128)


# ---------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------
def listed():
    def write(name, **kw):
        return dict({"name": name, "op": "write", "kv_heads": 2, "fused": False, "pad": 0}, **kw)

    def read(name, **kw):
        return dict({"name": name, "op": "read", "kv_heads": 2, "pad": 0}, **kw)

    def attend(name, **kw):
        return dict({"name": name, "op": "attend", "q_heads": 12, "kv_heads": 2, "drafts": 1, "pad": 0}, **kw)

    def sample(name, **kw):
        return dict({"name": name, "op": "sample", "vocab": 151936, "extra_stride": 0}, **kw)

    return [
        # one decode step of 64 running sequences: a row each, taken out of a fused q|k|v row
        write("write_decode_64", seqs=64, count=1, ragged=False, history=2048, dtype="f32", fused=True),
        # a whole prompt of one sequence
        write("write_prompt_4096", seqs=1, count=4096, ragged=False, history=0, dtype="f32"),
        # chunks of several prompts in one call, cut anywhere, after odd histories, in a padded row buffer
        write("write_chunks_bf16", seqs=24, count=1500, ragged=True, history=777, dtype="bf16", pad=9),
        # the cached rows that a chunk of a long prompt attends to
        read("read_8x4096", seqs=8, count=4096, ragged=False, history=0, dtype="f32"),
        # odd windows of several sequences
        read("read_ragged_bf16", seqs=13, count=1111, ragged=True, history=300, dtype="bf16", pad=5),
        # the bench line's history: one sequence, latency
        attend("attend_1x517", seqs=1, length=517, ragged=False, dtype="f32"),
        # the batched decode configuration
        attend("attend_64x2048", seqs=64, length=2048, ragged=False, dtype="f32"),
        # one very long context
        attend("attend_1x131072", seqs=1, length=131072, ragged=False, dtype="bf16"),
        # a ragged batch, each sequence checking four drafted tokens at once, with padded rows behind
        attend("attend_drafts_f16", seqs=24, length=6000, ragged=True, dtype="f16", drafts=4, pad=3),
        # one sequence's logits, the usual filters
        sample("sample_1_filtered", rows=1, dtype="f32", filters="all", peak=6.0),
        # a batch whose requests bring their own settings, greedy ones among them
        sample("sample_64_mixed", rows=64, dtype="f32", filters="mixed", peak=6.0),
        # a large batch of plain sampling over flat distributions; 16-bit logits tie often
        sample("sample_256_bf16", rows=256, dtype="bf16", filters="none", peak=2.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "sample"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if op in ("write", "read"):
        seqs = _log_int(rng, 1, 64)
        case = {"op": op, "seqs": seqs, "count": _log_int(rng, 1, max(1, 32768 // seqs)), "ragged": rng.random() < 0.6,
                "history": rng.choice([0, 1, 63, 64, _log_int(rng, 1, 4000)]), "dtype": dtype,
                "kv_heads": rng.choice([1, 2, 2, 2, 8]), "pad": rng.choice([0, 0, rng.randint(1, 70)])}
        if case["kv_heads"] == 8:
            case["count"] = max(1, case["count"] // 4)
        if op == "write":
            case["fused"] = rng.random() < 0.5
        return case
    if op == "attend":
        q_heads, kv_heads = rng.choice([(12, 2), (12, 2), (12, 2), (8, 8), (32, 8), (16, 2), (14, 2), (12, 1), (1, 1)])
        drafts = rng.choice([1, 1, 1, 2, 5])
        seqs = _log_int(rng, 1, 128)
        longest = min(100000, max(1, 131072 * 2 // (seqs * drafts * kv_heads)))
        return {"op": op, "seqs": seqs, "length": _log_int(rng, 1, longest), "ragged": rng.random() < 0.6, "dtype": dtype,
                "q_heads": q_heads, "kv_heads": kv_heads, "drafts": drafts, "pad": rng.choice([0, 0, rng.randint(1, 9)])}
    vocab = rng.choice([151936, 151936, _log_int(rng, 2, 200000)])
    return {"op": op, "rows": _log_int(rng, 1, 200), "vocab": vocab, "dtype": dtype,
            "filters": rng.choice(["all", "mixed", "none", "top_k", "top_p", "min_p"]), "peak": rng.uniform(0.5, 10.0),
            "extra_stride": rng.choice([0, 0, rng.randint(1, 40)])}


# ---------------------------------------------------------------------------------------------------
# sizes: everything about a case that does not need the GPU
# ---------------------------------------------------------------------------------------------------
def _counts(case, seed):
    """Tokens that each sequence brings (or reads), and the tokens before them; ragged: anything down to none."""
    r = np.random.RandomState(seed % (1 << 31))
    n, count, history = case["seqs"], case["count"], case["history"]
    if not case["ragged"]:
        starts = np.full(n, history) - (r.randint(0, BLOCK, n) if n > 1 and history >= BLOCK else 0)
        return np.full(n, count), starts
    counts = r.randint(0, count + 1, n)
    counts[r.randint(n)] = count  # the longest is there with every seed
    return counts, r.randint(0, history + 1, n)


def _lengths(case, seed):
    """Tokens in the cache of each sequence of an attention case (drafted ones included)."""
    n, length, drafts = case["seqs"], case["length"], case["drafts"]
    if not case["ragged"]:
        return np.full(n, max(length, drafts))
    r = np.random.RandomState(seed % (1 << 31))
    lens = r.randint(drafts, max(length, drafts) + 1, n)
    lens[r.randint(n)] = max(length, drafts)
    return lens


def _size(dtype):
    return 4 if dtype == "f32" else 2


def work(case):
    """Bytes and operations that one pass cannot do without (a ragged case by its mean)."""
    if case["op"] in ("write", "read"):
        rows = case["seqs"] * case["count"] * (0.5 if case["ragged"] else 1.0)
        values = 2 * rows * case["kv_heads"] * HEAD  # K and V
        if case["op"] == "read":
            return {"bytes": values * (1 + _size(case["dtype"])), "flops": values}
        old = 2 * case["seqs"] * case["kv_heads"] * HEAD * (0 if case["history"] == 0 else BLOCK / 2)  # open blocks
        out = (values + old) * (1 + _size(case["dtype"]))  # the touched blocks read back
        return {"bytes": values * (_size(case["dtype"]) + 1) + out, "flops": 4 * values + old}
    if case["op"] == "attend":
        tokens = case["seqs"] * case["length"] * (0.5 if case["ragged"] else 1.0)
        rows = case["seqs"] * case["drafts"]
        moved = tokens * 2 * case["kv_heads"] * (HEAD + 4 / BLOCK) + 2 * rows * case["q_heads"] * HEAD * _size(case["dtype"])
        return {"bytes": moved, "flops": tokens * case["drafts"] * case["q_heads"] * HEAD * 4}
    return {"bytes": case["rows"] * case["vocab"] * _size(case["dtype"]), "flops": case["rows"] * case["vocab"] * 4}


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(values):
    return torch.as_tensor(np.asarray(values), dtype=torch.int32, device="cuda")


def _cache(g, tokens, kv_heads, longest):
    """A filled cache: random blocks for `tokens[i]` (at most `longest`) tokens of each sequence, and spare blocks."""
    need = np.maximum(1, -(-np.asarray(tokens) // BLOCK))
    width = int(need.max())
    total = int(need.sum())
    n_blocks = len(need) * -(-max(1, longest) // BLOCK) + 3
    order = torch.randperm(n_blocks, generator=g, device="cuda", dtype=torch.int64)[:total].to(torch.int32)
    first = np.concatenate([[0], np.cumsum(need)[:-1]])
    at = np.minimum(first[:, None] + np.arange(width)[None, :], total - 1)
    table = order[torch.as_tensor(at, device="cuda")]
    table = torch.where(torch.as_tensor(np.arange(width)[None, :] < need[:, None], device="cuda"), table, torch.full_like(table, -1))
    shape = (n_blocks, kv_heads, BLOCK, HEAD)
    c = {"table": table.contiguous(), "n_blocks": n_blocks, "kv_heads": kv_heads}
    for w in "kv":
        # what such a cache holds: values near a normal distribution, one scale near (largest / 127) a block
        spread = torch.randn(shape, generator=g, device="cuda").mul_(31.0).round_().clamp_(-127, 127)
        c[w + "_codes"] = spread.to(torch.int8)
        c[w + "_scales"] = torch.rand((n_blocks, kv_heads), generator=g, device="cuda") * 0.02 + 0.02
    return c


def _rows(g, case, rows, seed):
    """K and V rows as a layer's projections leave them: some channels larger, tokens of different sizes."""
    heads, dtype = case["kv_heads"], DTYPES[case["dtype"]]
    size = torch.exp(0.4 * torch.randn((rows, 1, 1), generator=g, device="cuda"))
    chan = torch.exp(0.5 * torch.randn((1, heads, HEAD), generator=g, device="cuda"))
    k = torch.randn((rows, heads, HEAD), generator=g, device="cuda") * size * chan
    v = torch.randn((rows, heads, HEAD), generator=g, device="cuda") * size
    if case.get("fused"):  # [q | k | v] rows of one projection: k and v are strided views
        q = torch.zeros((rows, 6 * heads, HEAD), device="cuda")
        both = torch.cat([q, k, v], 1).to(dtype).contiguous()
        return both[:, 6 * heads : 7 * heads], both[:, 7 * heads :]
    return k.to(dtype).contiguous(), v.to(dtype).contiguous()


def _cache_handle(state):
    from work_llm_accelerator_b200 import host

    c = state["cache"]
    return host.Kv8Cache(c["k_codes"].data_ptr(), c["v_codes"].data_ptr(), c["k_scales"].data_ptr(), c["v_scales"].data_ptr(),
                         c["n_blocks"], c["kv_heads"], c["table"].data_ptr(), c["table"].shape[0], c["table"].shape[1])


def prepare(case, seed):
    g = _generator(seed)
    op, dtype = case["op"], DTYPES[case["dtype"]]
    s = {"case": case, "op": op, "dtype": CODES[case["dtype"]]}
    if op in ("write", "read"):
        counts, starts = _counts(case, seed)
        s["cache"] = _cache(g, counts + starts, case["kv_heads"], case["count"] + case["history"])
        s["seqs"] = torch.randperm(case["seqs"], generator=g, device="cuda").to(torch.int32)
        perm = s["seqs"].cpu().numpy()
        counts, starts = counts[perm], starts[perm]
        s["total"], s["starts"] = int(counts.sum()), _ints(starts)
        s["offsets"] = _ints(np.concatenate([[0], np.cumsum(counts)]))
        out_starts, out_counts = starts, counts
        if op == "write":
            # read back from the start of the first block that a sequence's new rows touch
            out_starts = np.where(counts > 0, starts // BLOCK * BLOCK, starts)
            out_counts = counts + starts - out_starts
            s["k"], s["v"] = _rows(g, case, s["total"] + case["pad"], seed)
        s["out_total"], s["out_starts"] = int(out_counts.sum()), _ints(out_starts)
        s["out_offsets"] = _ints(np.concatenate([[0], np.cumsum(out_counts)]))
        # a buffer for the most rows that such a call can ask for: those behind the last one stay as they are
        most = case["seqs"] * (case["count"] + (BLOCK - 1 if op == "write" else 0)) + case["pad"]
        for w in "kv":
            s["out_" + w] = torch.zeros((most, case["kv_heads"], HEAD), dtype=dtype, device="cuda")
    elif op == "attend":
        lens = _lengths(case, seed)
        drafts, rows = case["drafts"], case["seqs"] * case["drafts"] + case["pad"]
        s["cache"] = _cache(g, lens, case["kv_heads"], max(case["length"], drafts))
        row_seq, row_len = np.full(rows, -1), np.zeros(rows, dtype=np.int64)
        row_seq[: rows - case["pad"]] = np.repeat(np.arange(case["seqs"]), drafts)
        row_len[: rows - case["pad"]] = (lens[:, None] - drafts + 1 + np.arange(drafts)[None, :]).reshape(-1)
        if case["ragged"] and case["seqs"] > 1:
            row_len[0] = 0  # a sequence that has nothing yet
        s["row_seq"], s["row_len"], s["longest"] = _ints(row_seq), _ints(row_len), int(row_len.max())
        s["q"] = (2.0 * torch.randn((rows, case["q_heads"], HEAD), generator=g, device="cuda")).to(dtype)
        s["out"] = torch.zeros((rows, case["q_heads"], HEAD), dtype=dtype, device="cuda")
        s["lse"] = torch.zeros((rows, case["q_heads"]), dtype=torch.float32, device="cuda")
        if own:
            from work_llm_accelerator_b200 import host

            s["work"] = torch.empty(host.kv8_attention_workspace(rows, case["q_heads"], case["kv_heads"]), dtype=torch.uint8, device="cuda")
    else:
        rows, vocab = case["rows"], case["vocab"]
        logits = torch.randn((rows, vocab + case["extra_stride"]), generator=g, device="cuda") * 1.7
        few = min(vocab, 40)
        logits[:, torch.randperm(vocab, generator=g, device="cuda")[:few]] += case["peak"] * torch.rand((rows, few), generator=g, device="cuda")
        s["logits"] = logits.to(dtype)[:, :vocab]
        u = lambda: torch.rand(rows, generator=g, device="cuda")  # noqa: E731
        on = lambda x, off: x if case["filters"] != "mixed" else torch.where(u() < 0.6, x, torch.full_like(x, off))  # noqa: E731
        s["temperature"] = 0.4 + 0.9 * u()
        if case["filters"] == "mixed":
            s["temperature"] = torch.where(u() < 0.15, torch.zeros_like(s["temperature"]), s["temperature"])
        ks = torch.exp(u() * math.log(200.0)).floor().to(torch.int32)
        s["top_k"] = on(ks, 0) if case["filters"] in ("all", "mixed", "top_k") else None
        s["top_p"] = on(0.6 + 0.39 * u(), 1) if case["filters"] in ("all", "mixed", "top_p") else None
        s["min_p"] = on(0.1 * u(), 0) if case["filters"] in ("all", "mixed", "min_p") else None
        s["uniform"] = u()
        s["tokens"] = torch.zeros(rows, dtype=torch.int32, device="cuda")
        s["probs"] = torch.zeros(rows, dtype=torch.float32, device="cuda")
    if own and "cache" in s:
        s["handle"] = _cache_handle(s)
    return s


# ---------------------------------------------------------------------------------------------------
# the operators in their plain form
# ---------------------------------------------------------------------------------------------------
def _places(s, starts, offsets, total):
    """(block, slot) in the cache of rows 0 .. total - 1 of the segments."""
    r = torch.arange(total, device="cuda")
    seg = torch.searchsorted(offsets[1:].long(), r, right=True)
    pos = starts.long()[seg] + r - offsets.long()[seg]
    return s["cache"]["table"][s["seqs"].long()[seg], pos // BLOCK].long(), pos % BLOCK


def _plain_write_one(s, codes, scales, x, block, slot):
    """The scale of a block opened by this call is (largest value / 127); one that held tokens already keeps its
    scale, doubled as often as the new values need, and its codes are halved as often. Codes round to even."""
    x = x[: s["total"]].float()
    n_blocks, heads = scales.shape
    at = block[:, None].expand(-1, heads)
    amax = torch.zeros_like(scales).scatter_reduce(0, at, x.abs().amax(-1), "amax")
    first = torch.full((n_blocks,), BLOCK, device="cuda").scatter_reduce(0, block, slot, "amin")
    need = torch.where(amax > 0, (amax / 127).clamp_min(TINY), torch.zeros_like(amax))
    (m1, e1), (m2, e2) = torch.frexp(need), torch.frexp(scales)
    kept = ((first > 0) & (first < BLOCK))[:, None] & (scales > 0)
    twice = torch.where(kept & (need > 0), (e1 - e2 + (m1 > m2)).clamp_min(0), 0)
    grown = torch.where(kept, torch.ldexp(scales, twice), need)
    scales.copy_(torch.where((first < BLOCK)[:, None], grown, scales))
    # only the first block of a segment can hold earlier tokens; a sequence's own first block stands in where there is none
    table = s["cache"]["table"][s["seqs"].long()].long()
    open_block = table.gather(1, (s["starts"] // BLOCK).long().clamp_max(table.shape[1] - 1)[:, None])[:, 0]
    open_block = torch.where(open_block >= 0, open_block, table[:, 0])
    keep = torch.arange(BLOCK, device="cuda")[None, :] < (s["starts"] % BLOCK)[:, None]
    old = codes[open_block]
    halved = torch.round(torch.ldexp(old.float(), -twice[open_block][:, :, None, None])).to(torch.int8)
    codes.index_copy_(0, open_block, torch.where(keep[:, None, :, None], halved, old))
    div = scales[block][:, :, None]
    new = torch.where(div > 0, torch.round(x / div).clamp(-127, 127), torch.zeros_like(x)).to(torch.int8)
    codes[block, :, slot] = new


def _plain_read_one(codes, scales, out, block, slot):
    out[: block.shape[0]] = (codes[block, :, slot].float() * scales[block][:, :, None]).to(out.dtype)


def _plain_read(s):
    c = s["cache"]
    block, slot = _places(s, s["out_starts"], s["out_offsets"], s["out_total"])
    _plain_read_one(c["k_codes"], c["k_scales"], s["out_k"], block, slot)
    _plain_read_one(c["v_codes"], c["v_scales"], s["out_v"], block, slot)


def _plain_write(s):
    c = s["cache"]
    block, slot = _places(s, s["starts"], s["offsets"], s["total"])
    _plain_write_one(s, c["k_codes"], c["k_scales"], s["k"], block, slot)
    _plain_write_one(s, c["v_codes"], c["v_scales"], s["v"], block, slot)
    _plain_read(s)


def _plain_attend(s):
    c = s["cache"]
    rows, q_heads, _ = s["q"].shape
    heads = c["kv_heads"]
    width = -(-max(1, s["longest"]) // BLOCK)
    blocks = c["table"][s["row_seq"].long().clamp_min(0), :width].long().clamp_min(0)  # [rows, width]
    live = torch.arange(width * BLOCK, device="cuda")[None, :] < s["row_len"][:, None]

    def values(w):
        x = c[w + "_codes"][blocks].float() * c[w + "_scales"][blocks][..., None, None]  # [rows, width, heads, 64, 128]
        return x.permute(0, 2, 1, 3, 4).reshape(rows, heads, width * BLOCK, HEAD)

    q = s["q"].float().reshape(rows, heads, q_heads // heads, HEAD)
    scores = torch.matmul(q, values("k").transpose(2, 3)) * SCALE
    scores = scores.masked_fill(~live[:, None, None, :], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    out = torch.matmul(e, values("v").masked_fill(~live[:, None, :, None], 0.0)) / torch.where(total > 0, total, torch.ones_like(total))
    lse = (top + torch.log(total)).reshape(rows, q_heads)
    real = (s["row_seq"] >= 0)
    s["out"].copy_(torch.where(real[:, None, None], out.reshape(rows, q_heads, HEAD).to(s["out"].dtype), s["out"]))
    s["lse"].copy_(torch.where(real[:, None], lse, s["lse"]))


def _plain_sample(s):
    """Sorted by logit (ties: lowest index first), a row keeps a prefix: at most top_k tokens, then the fewest whose
    sum reaches top_p of those, then those of at least min_p times the likeliest; the uniform number picks by the sum."""
    logits = s["logits"].double()
    rows, vocab = logits.shape
    order = torch.sort(logits, dim=-1, descending=True, stable=True)
    t = s["temperature"].double()
    greedy = t <= 0
    top = order.values[:, :1]
    z = (order.values - top) / torch.where(greedy, torch.ones_like(t), t)[:, None]
    w = torch.exp(z)
    rank = torch.arange(vocab, device="cuda")[None, :]
    if s["top_k"] is not None:
        k = torch.where(s["top_k"] > 0, s["top_k"], vocab)[:, None]
        w = torch.where(rank < k, w, torch.zeros_like(w))
    if s["top_p"] is not None:
        p = s["top_p"].double()[:, None]
        cum = torch.cumsum(w, -1)
        w = torch.where((p >= 1) | (rank == 0) | (cum - w < p * cum[:, -1:]), w, torch.zeros_like(w))
    if s["min_p"] is not None:
        w = torch.where((rank == 0) | (torch.exp(z) >= s["min_p"].double()[:, None]), w, torch.zeros_like(w))
    cum = torch.cumsum(w, -1)
    total = cum[:, -1:]
    at = (cum <= s["uniform"].double()[:, None] * total).sum(-1)
    at = torch.minimum(at, (w > 0).sum(-1) - 1)
    at = torch.where(greedy, torch.zeros_like(at), at)[:, None]
    s["tokens"].copy_(order.indices.gather(1, at)[:, 0])
    prob = (w.gather(1, at) / total)[:, 0]
    s["probs"].copy_(torch.where(greedy, torch.ones_like(prob), prob))


# ---------------------------------------------------------------------------------------------------
# the framework's operators
# ---------------------------------------------------------------------------------------------------
def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _own(s):
    from work_llm_accelerator_b200 import host

    stream = torch.cuda.current_stream().cuda_stream
    if s["op"] == "write":
        k, v = s["k"], s["v"]
        host.kv8_append(s["handle"], k.data_ptr(), v.data_ptr(), s["dtype"], k.stride(0), k.shape[0], s["seqs"].data_ptr(),
                        s["starts"].data_ptr(), s["offsets"].data_ptr(), s["seqs"].shape[0], stream)
    if s["op"] in ("write", "read"):
        k, v = s["out_k"], s["out_v"]
        host.kv8_read(s["handle"], k.data_ptr(), v.data_ptr(), s["dtype"], k.stride(0), k.shape[0], s["seqs"].data_ptr(),
                      s["out_starts"].data_ptr(), s["out_offsets"].data_ptr(), s["seqs"].shape[0], stream)
    elif s["op"] == "attend":
        q, out = s["q"], s["out"]
        host.kv8_attention(s["handle"], q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), s["dtype"], q.shape[0], q.shape[1],
                           s["row_seq"].data_ptr(), s["row_len"].data_ptr(), SCALE, s["work"].data_ptr(), s["work"].shape[0],
                           s["lse"].data_ptr(), stream)
    else:
        x = s["logits"]
        host.sample(x.data_ptr(), s["dtype"], x.shape[0], x.shape[1], x.stride(0), s["temperature"].data_ptr(), _ptr(s["top_k"]),
                    _ptr(s["top_p"]), _ptr(s["min_p"]), s["uniform"].data_ptr(), s["tokens"].data_ptr(), s["probs"].data_ptr(), stream)


def run(s):
    op = s["op"]
    if own:
        _own(s)
    elif op == "write":
        _plain_write(s)
    elif op == "read":
        _plain_read(s)
    elif op == "attend":
        _plain_attend(s)
    else:
        _plain_sample(s)
    if op == "write":
        # 8-bit codes come back as the values that they stand for (the touched blocks), and the cache's scales
        return {"k": s["out_k"], "v": s["out_v"], "k_scales": s["cache"]["k_scales"], "v_scales": s["cache"]["v_scales"]}
    if op == "read":
        return {"k": s["out_k"], "v": s["out_v"]}
    if op == "attend":
        return {"out": s["out"], "lse": s["lse"]}
    return {"tokens": s["tokens"], "probs": s["probs"]}


# ---------------------------------------------------------------------------------------------------
# the definitions in 64 bits, on the host side sequence by sequence
# ---------------------------------------------------------------------------------------------------
def _round32(x):
    return x.float().double()


def _exact_block(codes, scale, x, slot):
    """One block of one kv head after rows x [n][128] were written at `slot`: (codes, scale) in float64."""
    a = float(x.abs().max())
    need = float(np.float32(max(np.float64(np.float32(a / 127.0)), TINY))) if a > 0 else 0.0
    if slot > 0 and scale > 0:
        new = scale
        while new < need:
            new = new * 2
        codes = torch.round(codes * (scale / new)) if new > scale else codes
    else:
        new = need
    codes = codes.clone()
    q = _round32(x / new) if new > 0 else torch.zeros_like(x)  # the quotient is a 32-bit one by definition
    codes[slot : slot + x.shape[0]] = torch.clamp(torch.round(q), -127, 127)
    return codes, new


def _exact_cache(s, case):
    """The cache after the write as {w: (codes [block][head][64][128], scales)} in float64 on the CPU."""
    c = s["cache"]
    got = {w: (c[w + "_codes"].cpu().double(), c[w + "_scales"].cpu().double()) for w in "kv"}
    if case["op"] == "read":
        return got
    table, seqs, starts, offsets = (t.cpu().tolist() for t in (c["table"], s["seqs"], s["starts"], s["offsets"]))
    for w in "kv":
        x = s[w].cpu().double()
        codes, scales = got[w]
        for i, q in enumerate(seqs):
            row, pos = offsets[i], starts[i]
            while row < offsets[i + 1]:
                slot = pos % BLOCK
                n = min(BLOCK - slot, offsets[i + 1] - row)
                b = table[q][pos // BLOCK]
                for h in range(case["kv_heads"]):
                    codes[b, h], scales[b, h] = _exact_block(codes[b, h], float(scales[b, h]), x[row : row + n, h], slot)
                row, pos = row + n, pos + n
    return got


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("write", "read"):
        blocks = case["seqs"] * (case["count"] / BLOCK + 1) * case["kv_heads"]
        if blocks > 8000:
            return None
        cache = _exact_cache(s, case)
        table, seqs, starts, offsets = (t.cpu().tolist() for t in (s["cache"]["table"], s["seqs"], s["out_starts"], s["out_offsets"]))
        out = {}
        for w in "kv":
            codes, scales = cache[w]
            rows = torch.zeros(s["out_" + w].shape, dtype=torch.float64)
            for i, q in enumerate(seqs):
                pos = torch.arange(starts[i], starts[i] + offsets[i + 1] - offsets[i])
                b = torch.tensor(table[q])[pos // BLOCK].long()
                rows[offsets[i] : offsets[i + 1]] = codes[b, :, pos % BLOCK] * scales[b][:, :, None]
            out[w] = rows
        if case["op"] == "write":
            out |= {w + "_scales": cache[w][1] for w in "kv"}
        return out
    if case["op"] == "attend":
        c = s["cache"]
        rows, q_heads, _ = s["q"].shape
        group = q_heads // case["kv_heads"]
        out = torch.zeros((rows, q_heads, HEAD), dtype=torch.float64, device="cuda")
        lse = torch.zeros((rows, q_heads), dtype=torch.float64, device="cuda")
        seqs, lens = s["row_seq"].tolist(), s["row_len"].tolist()
        for r in range(rows):
            if seqs[r] < 0:
                continue
            if lens[r] == 0:
                lse[r] = float("-inf")
                continue
            b = c["table"][seqs[r], : -(-lens[r] // BLOCK)].long()
            k, v = ((c[w + "_codes"][b].double() * c[w + "_scales"][b].double()[:, :, None, None]).transpose(0, 1).flatten(1, 2)[:, : lens[r]] for w in "kv")
            k, v = k.repeat_interleave(group, 0), v.repeat_interleave(group, 0)  # [q head, token, 128]
            sc = (k * s["q"][r].double()[:, None, :]).sum(-1) * SCALE
            lse[r] = torch.logsumexp(sc, -1)
            out[r] = (torch.exp(sc - lse[r][:, None])[:, :, None] * v).sum(1)
        return {"out": out, "lse": lse}
    # the probability of the token that the sampler takes, by sorted sums on the CPU
    x = s["logits"].cpu().double().numpy()
    rows, vocab = x.shape
    if rows * vocab > 45_000_000:
        return None
    get = lambda k, off: s[k].cpu().double().numpy() if s[k] is not None else np.full(rows, off)  # noqa: E731
    t, u, top_k, top_p, min_p = get("temperature", 0), get("uniform", 0), get("top_k", 0), get("top_p", 1), get("min_p", 0)
    probs = np.ones(rows)
    for r in range(rows):
        if t[r] <= 0:
            continue
        w = -np.sort(-np.exp((x[r] - x[r].max()) / t[r]))
        if 0 < top_k[r] < vocab:
            w = w[: int(top_k[r])]
        if top_p[r] < 1:
            w = w[: 1 + int(np.searchsorted(np.cumsum(w), top_p[r] * w.sum()))]
        w = w[: max(1, int((w >= min_p[r]).sum()))]
        at = np.searchsorted(np.cumsum(w), u[r] * w.sum(), side="right")
        probs[r] = w[min(at, len(w) - 1)] / w.sum()
    return {"tokens": None, "probs": probs}
