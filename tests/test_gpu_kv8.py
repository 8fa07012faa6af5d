"""GPU tests of the 8-bit KV cache operators (include/qwen_b200_ops.h) against the plain model in kv8_model.py:
writing and reading back bit for bit, decode attention in float64 at a bound that its roundings give."""
from __future__ import annotations

import numpy as np
import pytest

import kv8_model as km

pytestmark = pytest.mark.gpu

SCALE = 1.0 / np.sqrt(128.0)
TYPES = {"f32": 0, "f16": 1, "bf16": 2}
HALF_STEP = {"f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}


@pytest.fixture(autouse=True)
def _device(built_libs, gpu_available):
    if not gpu_available:
        pytest.fail("no CUDA device: the -m gpu suite must run on a B200")
    from work_llm_accelerator_b200 import host

    host.kernel_error(reset=True)
    yield
    import torch

    torch.cuda.synchronize()


def dt(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def ints(v):
    import torch

    return torch.as_tensor(np.asarray(v), dtype=torch.int32).cuda()


class Cache:
    """A cache on the GPU full of leftovers, and its models."""

    def __init__(self, lens, heads, seed, spare=2, width=None):
        import torch
        from work_llm_accelerator_b200 import host

        r = np.random.RandomState(seed)
        need = [max(1, -(-n // km.BLOCK)) for n in lens]
        width = max(need) if width is None else width
        self.n_blocks = sum(need) + spare
        ids = r.permutation(self.n_blocks)[: sum(need)]
        self.table = np.full((len(lens), width), -1, np.int64)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = ids[at : at + n]
            at += n
        shape = (self.n_blocks, heads, km.BLOCK, km.HEAD)
        self.model = {}
        for w in "kv":
            codes = r.randint(-127, 128, shape).astype(np.float64)
            scales = (0.004 + 0.02 * r.rand(self.n_blocks, heads)).astype(np.float32)
            scales[r.rand(self.n_blocks, heads) < 0.2] = np.nan  # left by an earlier user of the block
            self.model[w] = km.Model(codes, scales, self.table)
        self.codes = {w: torch.as_tensor(self.model[w].codes.astype(np.int8)).cuda() for w in "kv"}
        self.scales = {w: torch.as_tensor(self.model[w].scales).cuda() for w in "kv"}
        self.d_table = ints(self.table)
        self.heads = heads
        self.handle = host.Kv8Cache(self.codes["k"].data_ptr(), self.codes["v"].data_ptr(), self.scales["k"].data_ptr(),
                                    self.scales["v"].data_ptr(), self.n_blocks, heads, self.d_table.data_ptr(), len(lens), width)

    def append(self, x, dtype, seqs, starts, counts, pad=0, fused=False):
        """x {"k", "v"} fp32 arrays [rows][heads][128], given as `dtype`; the models get the rounded values."""
        import torch
        from work_llm_accelerator_b200 import host

        t = {w: torch.as_tensor(x[w]).to(dt(dtype)) for w in "kv"}
        if pad:
            t = {w: torch.cat([t[w], torch.full((pad, self.heads, km.HEAD), float("nan"), dtype=dt(dtype))]) for w in "kv"}
        if fused:
            both = torch.cat([torch.zeros_like(t["k"]), t["k"], t["v"]], 1).cuda()
            d = {"k": both[:, self.heads : 2 * self.heads], "v": both[:, 2 * self.heads :]}
        else:
            d = {w: t[w].cuda() for w in "kv"}
        off = np.concatenate([[0], np.cumsum(counts)]).astype(int)
        a = [ints(seqs), ints(starts), ints(off)]
        host.kv8_append(self.handle, d["k"].data_ptr(), d["v"].data_ptr(), TYPES[dtype], d["k"].stride(0), d["k"].shape[0],
                        *(v.data_ptr() for v in a), len(seqs), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        for w in "kv":
            for i, q in enumerate(seqs):
                if counts[i]:
                    self.model[w].append(t[w].float().numpy()[off[i] : off[i + 1]], q, starts[i])

    def read(self, dtype, seqs, starts, counts, pad=0):
        import torch
        from work_llm_accelerator_b200 import host

        off = np.concatenate([[0], np.cumsum(counts)]).astype(int)
        a = [ints(seqs), ints(starts), ints(off)]
        out = {w: torch.full((off[-1] + pad, self.heads, km.HEAD), 7.0, dtype=dt(dtype)).cuda() for w in "kv"}
        host.kv8_read(self.handle, out["k"].data_ptr(), out["v"].data_ptr(), TYPES[dtype], out["k"].stride(0), out["k"].shape[0],
                      *(v.data_ptr() for v in a), len(seqs), torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        return out, off

    def check(self, lens):
        """Codes and scales of every live block equal the models', bit for bit."""
        for w in "kv":
            codes, scales = self.codes[w].cpu().numpy(), self.scales[w].cpu().numpy()
            for q, n in enumerate(lens):
                for j in range(-(-n // km.BLOCK)):
                    b, live = self.table[q, j], min(km.BLOCK, n - j * km.BLOCK)
                    np.testing.assert_array_equal(scales[b], self.model[w].scales[b])
                    np.testing.assert_array_equal(codes[b, :, :live], self.model[w].codes[b, :, :live])


def rows(r, n, heads, size=1.0):
    return {w: (size * r.randn(n, heads, km.HEAD) * np.exp(0.7 * r.randn(n, 1, 1))).astype(np.float32) for w in "kv"}


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,counts", [(2, [1]), (2, [64]), (2, [63, 0, 65, 1]), (1, [200, 7, 129]), (8, [70, 64])])
def test_append_then_append_equals_model(dtype, heads, counts):
    """A first write from position 0, then a ragged one behind it (open blocks grow), in a padded row buffer."""
    r = np.random.RandomState(len(counts) + heads)
    more = [(7 * c + 3) % 150 for c in counts]
    lens = [a + b for a, b in zip(counts, more)]
    c = Cache(lens, heads, seed=sum(counts))
    seqs = list(r.permutation(len(counts)))
    c.append(rows(r, sum(counts), heads), dtype, seqs, [0] * len(counts), [counts[q] for q in seqs], pad=3)
    c.check(counts)
    seqs = seqs[::-1]
    c.append(rows(r, sum(more), heads, 3.0), dtype, seqs, [counts[q] for q in seqs], [more[q] for q in seqs], fused=True)
    c.check(lens)
    from work_llm_accelerator_b200 import host

    assert host.kernel_error() == 0


def test_append_token_by_token_and_dropped_drafts():
    """Single tokens that grow an open block several times, then a draft that is written, dropped and rewritten."""
    r = np.random.RandomState(5)
    c = Cache([130, 10], 2, seed=3)
    for t in range(130):
        c.append(rows(r, 1, 2, 1.0 + 0.2 * t), "f32", [0], [t], [1])
    c.check([130])
    c.append(rows(r, 4, 2, 50.0), "f32", [0], [124], [4])
    c.append(rows(r, 2, 2, 0.1), "f32", [0], [125], [2])
    c.check([127])


@pytest.mark.parametrize("size", [0.0, 1e-44, 1e-39, 1e30, 3e37])
def test_append_extreme_sizes(size):
    """Zeros, subnormals (the scale stops at 2^-126) and values near the largest finite one."""
    r = np.random.RandomState(9)
    c = Cache([100], 2, seed=4)
    x = {w: np.clip(r.randn(40, 2, 128), -3, 3).astype(np.float32) * np.float32(size) for w in "kv"}
    c.append(x, "f32", [0], [0], [40])
    c.append({w: r.randn(60, 2, 128).astype(np.float32) for w in "kv"}, "f32", [0], [40], [60])
    c.check([100])


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_append_non_finite_poisons_its_block_alone(bad):
    r = np.random.RandomState(2)
    c = Cache([200], 2, seed=6)
    x = rows(r, 200, 2)
    x["k"][70, 1, 5] = bad
    c.append(x, "f32", [0], [0], [200])
    c.check([200])
    out, _ = c.read("f32", [0], [0], [200])
    k = out["k"].cpu().numpy()
    assert np.isnan(k[64:128, 1]).all() and np.isfinite(k[64:128, 0]).all() and np.isfinite(k[:64]).all()
    assert np.isfinite(k[128:]).all() and np.isfinite(out["v"].cpu().numpy()).all()
    c.append(rows(r, 10, 2), "f32", [0], [64], [10])  # opened again: sound again
    c.check([74])
    assert np.isfinite(c.scales["k"].cpu().numpy()[c.table[0, 1]]).all()


def test_halved_values_stay_within_one_step():
    """The documented bound: a value is off by less than its block's final scale, whatever it grew through."""
    r = np.random.RandomState(8)
    c = Cache([64], 2, seed=1)
    x = {w: (r.randn(64, 2, 128) * np.exp(np.linspace(-4, 4, 64))[:, None, None]).astype(np.float32) for w in "kv"}
    for t in range(64):
        c.append({w: x[w][t : t + 1] for w in "kv"}, "f32", [0], [t], [1])
    out, _ = c.read("f32", [0], [0], [64])
    for w in "kv":
        s = c.scales[w].cpu().numpy()[c.table[0, 0]]
        # the reading back rounds code * scale once more: 2^-24 of a value of at most 127 steps
        assert (np.abs(out[w].cpu().numpy().astype(np.float64) - x[w]) < s[None, :, None] * (1 + 127 * 2.0**-23)).all()


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("starts,counts", [([0], [1]), ([63, 5, 0], [2, 0, 200]), ([100, 64, 1, 1], [28, 64, 127, 127])])
def test_read_equals_model(dtype, starts, counts):
    import torch

    c = Cache([200] * len(starts), 2, seed=len(starts))
    out, off = c.read(dtype, list(range(len(starts))), starts, counts, pad=5)
    for w in "kv":
        for i in range(len(starts)):
            want = torch.as_tensor(c.model[w].values(i, counts[i], starts[i])).to(dt(dtype))
            torch.testing.assert_close(out[w][off[i] : off[i + 1]].cpu(), want, rtol=0, atol=0, equal_nan=True)
        assert (out[w][off[-1] :] == 7.0).all()  # rows behind the last: as they were


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_read_into_wider_rows_and_nothing_to_read(dtype):
    """Rows that lie inside wider ones: what is beside them stays; segments without a token write nothing."""
    import torch
    from work_llm_accelerator_b200 import host

    c = Cache([90, 70], 2, seed=4)
    for counts in ([33, 70], [0, 0]):
        wide = torch.full((110, 7, km.HEAD), 7.0, dtype=dt(dtype)).cuda()
        k, v = wide[:, 1:3], wide[:, 4:6]
        a = [ints([1, 0]), ints([20, 5]), ints([0, counts[0], sum(counts)])]
        host.kv8_read(c.handle, k.data_ptr(), v.data_ptr(), TYPES[dtype], wide.stride(0), 110, *(x.data_ptr() for x in a), 2,
                      torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        want = torch.full((110, 7, km.HEAD), 7.0, dtype=dt(dtype))
        for at, w in ((1, "k"), (4, "v")):
            rows_ = np.concatenate([c.model[w].values(1, counts[0], 20), c.model[w].values(0, counts[1], 5)])
            want[: sum(counts), at : at + 2] = torch.as_tensor(rows_).to(dt(dtype))
        torch.testing.assert_close(wide.cpu(), want, rtol=0, atol=0, equal_nan=True)
    assert host.kernel_error() == 0


def test_more_segments_than_threads():
    """600 sequences of a token each, some of them empty: the segment search takes several passes."""
    r = np.random.RandomState(1)
    counts = (r.rand(600) < 0.8).astype(int)
    c = Cache([1] * 600, 1, seed=2)
    c.append(rows(r, counts.sum(), 1), "f32", list(range(600)), [0] * 600, list(counts))
    c.check(list(counts))
    counts = r.randint(0, 3, 600)
    out, off = c.read("f32", [5] * 600, [0] * 600, list(np.minimum(counts, 1)))
    assert out["k"].shape[0] == np.minimum(counts, 1).sum()
    np.testing.assert_array_equal(out["k"].cpu().numpy(), np.repeat(c.model["k"].values(5, 1), out["k"].shape[0], 0))


def test_bad_indexes_are_skipped_and_flagged():
    """Device-side indexes outside of the buffers: no access, the flag, NaN where values were asked for."""
    import torch
    from work_llm_accelerator_b200 import host

    r = np.random.RandomState(0)
    for what in ("block", "negative block", "seq", "start", "offset"):
        c = Cache([128, 128], 2, seed=7)
        if what == "block":
            c.d_table[1, 1] = c.n_blocks
        if what == "negative block":
            c.d_table[1, 1] = -7
        before = {w: c.codes[w].clone() for w in "kv"}
        seqs = [0, 2] if what == "seq" else [0, 1]
        starts = [0, 100 if what == "start" else 64]
        t = {w: torch.as_tensor(rows(r, 80, 2)[w]).cuda() for w in "kv"}
        a = [ints(seqs), ints(starts), ints([0, 16, 81 if what == "offset" else 80])]
        args = (TYPES["f32"], 256, 80, *(v.data_ptr() for v in a), 2, torch.cuda.current_stream().cuda_stream)
        host.kv8_append(c.handle, t["k"].data_ptr(), t["v"].data_ptr(), *args)
        torch.cuda.synchronize()
        assert host.kernel_error(reset=True) == 2, what
        untouched = [b for b in range(c.n_blocks) if b != c.table[0, 0]]
        for w in "kv":
            assert torch.equal(c.codes[w][untouched], before[w][untouched]), what
        host.kv8_read(c.handle, t["k"].data_ptr(), t["v"].data_ptr(), *args)
        torch.cuda.synchronize()
        assert host.kernel_error(reset=True) == 2, what
        if "block" in what:
            assert torch.isnan(t["k"][16:]).all() and torch.isnan(t["v"][16:]).all()


# ---------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------
def attend(c, q, dtype, seqs, lens, out=None, lse=None, scale=SCALE, stream=None, work=None):
    import torch
    from work_llm_accelerator_b200 import host

    n, heads, _ = q.shape
    out = torch.full_like(q, 7.0, memory_format=torch.contiguous_format) if out is None else out
    lse = torch.full((n, heads), 7.0, device="cuda") if lse is None else lse
    size = host.kv8_attention_workspace(n, heads, c.heads)
    # any contents: here every byte 0xff (NaN, -1)
    work = torch.full((size,), 255, dtype=torch.uint8, device="cuda") if work is None else work
    s = stream or torch.cuda.current_stream()
    host.kv8_attention(c.handle, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), TYPES[dtype], n, heads,
                       seqs.data_ptr(), lens.data_ptr(), scale, work.data_ptr(), work.numel(), lse.data_ptr(), s.cuda_stream)
    return out, lse, work


def check_rows(c, q, dtype, seqs, lens, out, lse, scale=SCALE):
    """Bound, from the roundings (u = 2^-24, first order, factor 2 for the rest): a score is a sum of 128 products of an
    operand that keeps 22 bits, so it is off by d = (128 + 8) u A with A = sum |scale q k|; the softmax weights by
    2 d + 4 u (exponentials), their sums by (64 + tiles + splits) u; the result by the type's half step."""
    u = 2.0**-24
    got, got_lse = out.float().cpu().numpy(), lse.cpu().numpy()
    num = den = 0.0
    for r in range(len(seqs)):
        if seqs[r] < 0:
            assert (got[r] == 7.0).all() and (got_lse[r] == 7.0).all()
            continue
        k, v = (c.model[w].values(seqs[r], lens[r]) for w in "kv")
        want, want_lse, mag = km.attention(q[r].float().cpu().numpy(), k, v, scale)
        if lens[r] == 0:
            assert (got[r] == 0).all() and (got_lse[r] == -np.inf).all()
            continue
        d = 136 * u * mag
        eps = 2 * (2 * d + 4 * u + (64 + lens[r] / 32 + 160) * u)
        tol = eps * np.abs(v).max() + HALF_STEP[dtype] * np.abs(want) + 2.0**-25
        assert (np.abs(got[r] - want) <= tol).all(), (r, lens[r], np.abs(got[r] - want).max())
        assert (np.abs(got_lse[r] - want_lse) <= eps + 2 * u * np.abs(want_lse)).all(), r
        num += ((got[r] - want) ** 2).sum()
        den += (want**2).sum()
    if den:  # and the framework's bound for an fp32 attention, in the mean
        assert np.sqrt(num / den) <= 1e-5 + HALF_STEP[dtype]


def filled(lens, heads, seed, **kw):
    """A cache whose every live block has finite scales, NaN scales left in the others."""
    import torch

    c = Cache(lens, heads, seed, **kw)
    for w in "kv":
        for i, n in enumerate(lens):
            for b in c.table[i, : -(-n // km.BLOCK)]:
                s = c.model[w].scales[b]
                s[np.isnan(s)] = 0.01
        c.scales[w].copy_(torch.as_tensor(c.model[w].scales))
    return c


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("lens", [[1], [2], [31, 32, 33], [63, 64, 65], [127, 0, 129, 1], [517], [1000, 64, 3], [2048] * 5])
def test_attention_matches_model(dtype, lens):
    import torch

    c = filled(lens, 2, seed=len(lens) + lens[0])
    g = torch.Generator().manual_seed(lens[0])
    q = (1.5 * torch.randn(len(lens), 12, 128, generator=g)).to(dt(dtype)).cuda()
    out, lse, _ = attend(c, q, dtype, ints(range(len(lens))), ints(lens))
    check_rows(c, q, dtype, list(range(len(lens))), lens, out, lse)


@pytest.mark.parametrize("q_heads,heads", [(1, 1), (8, 8), (32, 8), (16, 2), (14, 2), (12, 1), (24, 2), (17, 1)])
def test_attention_head_layouts(q_heads, heads):
    import torch

    lens = [150, 20, 700]
    c = filled(lens, heads, seed=q_heads)
    q = torch.randn(3, q_heads, 128, generator=torch.Generator().manual_seed(q_heads)).cuda()
    out, lse, _ = attend(c, q, "f32", ints([2, 0, 1]), ints([700, 150, 20]))
    check_rows(c, q, "f32", [2, 0, 1], [700, 150, 20], out, lse)


@pytest.mark.parametrize("n,length", [(1, 20011), (3, 9000), (300, 130)])
def test_attention_long_and_many(n, length):
    """Histories that are split over the GPU, and more rows than it has SMs."""
    import torch

    r = np.random.RandomState(n)
    lens = [length] + list(r.randint(0, length, n - 1))
    c = filled(lens, 2, seed=n)
    q = torch.randn(n, 12, 128, generator=torch.Generator().manual_seed(n)).cuda()
    out, lse, _ = attend(c, q, "f32", ints(range(n)), ints(lens))
    check_rows(c, q, "f32", list(range(n)), lens, out, lse)


@pytest.mark.parametrize("n,length", [(60, 1100), (70, 700), (148, 64)])
def test_attention_equal_lengths(n, length):
    """Batches whose sequences are alike: each fits a CTA's share of the work or nearly does."""
    import torch

    lens = [length] * n
    c = filled(lens, 2, seed=n)
    q = torch.randn(n, 12, 128, generator=torch.Generator().manual_seed(n)).cuda()
    out, lse, _ = attend(c, q, "f32", ints(range(n)), ints(lens))
    check_rows(c, q, "f32", list(range(n)), lens, out, lse)


def test_attention_workspace_is_used_again():
    """Calls of other shapes, one after the other in one workspace, leave nothing behind that a later one takes up."""
    import torch

    lens = [9000, 700, 2500]
    c = filled(lens, 2, seed=71)
    q = torch.randn(3, 12, 128, generator=torch.Generator().manual_seed(9)).cuda()
    work = None
    for rows in ([0], [1, 2], [0, 1, 2], [2], [0], [0, 1, 2]):
        ns = [lens[r] - 3 for r in rows]
        out, lse, work = attend(c, q[rows], "f32", ints(rows), ints(ns), work=work)
        torch.cuda.synchronize()
        check_rows(c, q[rows], "f32", rows, ns, out, lse)


def test_attention_two_graphs_share_a_workspace():
    """Two captured calls with one workspace, replayed in turn: each finds what the other left."""
    import torch

    lens = [9000, 4000]
    c = filled(lens, 2, seed=72)
    shapes = [([0, 1], [9000, 4000]), ([0], [8000])]
    qs = [torch.randn(len(s), 12, 128, generator=torch.Generator().manual_seed(i)).cuda() for i, (s, _) in enumerate(shapes)]
    idx = [(ints(s), ints(n)) for s, n in shapes]
    outs, lses, graphs = [torch.full_like(q, 7.0) for q in qs], [torch.full(q.shape[:2], 7.0, device="cuda") for q in qs], []
    _, _, work = attend(c, qs[0], "f32", *idx[0])
    torch.cuda.synchronize()
    for i, q in enumerate(qs):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            attend(c, q, "f32", *idx[i], out=outs[i], lse=lses[i], work=work)
    for turn in (0, 1, 0, 0, 1, 1, 0):
        outs[turn].fill_(7.0)
        graphs[turn].replay()
        torch.cuda.synchronize()
        check_rows(c, qs[turn], "f32", *shapes[turn], outs[turn], lses[turn])


def test_attention_drafts_padded_rows_and_strides():
    """Several rows of one sequence with rising lengths, rows without a sequence, q inside a wider row, out too."""
    import torch

    lens = [90, 65]
    c = filled(lens, 2, seed=11)
    seqs, ns = [0, 0, 0, -1, 1, 1, -5, 0], [88, 89, 90, 3, 64, 65, 1 << 30, 0]
    wide = torch.randn(8, 16, 128, generator=torch.Generator().manual_seed(1)).cuda()
    q = wide[:, 2:14]
    big = torch.full((8, 20, 128), 7.0, device="cuda")
    out, lse, _ = attend(c, q, "f32", ints(seqs), ints(ns), out=big[:, 4:16])
    check_rows(c, q, "f32", seqs, ns, out, lse)
    assert (big[:, :4] == 7.0).all() and (big[:, 16:] == 7.0).all()


@pytest.mark.parametrize("size,scale", [(0.0, SCALE), (300.0, SCALE), (1e-30, 1e30), (1e20, 1e-20), (1.0, -SCALE), (1.0, 0.0)])
def test_attention_query_sizes(size, scale):
    """Queries far from 1 (the kernel must not lose them to a narrow type), a negative and a zero scale."""
    import torch

    lens = [300, 64]
    c = filled(lens, 2, seed=21)
    q = (size * torch.randn(2, 12, 128, generator=torch.Generator().manual_seed(2))).cuda()
    out, lse, _ = attend(c, q, "f32", ints([0, 1]), ints(lens), scale=scale)
    check_rows(c, q, "f32", [0, 1], lens, out, lse, scale=scale)


def test_attention_keeps_many_small_weights():
    """One token far above 20000 others whose sum still counts: none of them may vanish in a narrow type."""
    import torch

    n = 20000
    c = filled([n], 1, seed=2)
    for w in "kv":
        c.model[w].codes[:] = 0.0 if w == "k" else 100.0
        c.model[w].scales[:] = 0.01
    b = c.table[0, 0]
    c.model["k"].codes[b, 0, 0, :] = 100  # score 128 * q * 1.0 * SCALE
    c.model["v"].codes[b, 0, 0, :] = -100
    for w in "kv":
        c.codes[w].copy_(torch.as_tensor(c.model[w].codes.astype(np.int8)))
        c.scales[w].copy_(torch.as_tensor(c.model[w].scales))
    q = torch.full((1, 1, 128), float(16.0 / (128 * SCALE))).cuda()  # e^-16 = 1.1e-7 each
    out, lse, _ = attend(c, q, "f32", ints([0]), ints([n]))
    check_rows(c, q, "f32", [0], [n], out, lse)


def test_attention_poisoned_block_and_bad_indexes():
    """A block whose scale is NaN, a block id, a sequence or a length outside of the cache: NaN in the rows that reach
    it, no other row, and the flag for the bad indexes."""
    import torch
    from work_llm_accelerator_b200 import host

    lens = [200, 200, 200, 200]
    c = filled(lens, 2, seed=5)
    c.scales["k"][c.table[0, 1]] = float("nan")
    q = torch.randn(6, 12, 128, generator=torch.Generator().manual_seed(3)).cuda()
    out, _, _ = attend(c, q[:2], "f32", ints([0, 1]), ints([64, 200]))
    torch.cuda.synchronize()
    assert torch.isfinite(out).all() and host.kernel_error(reset=True) == 0
    c.d_table[2, 3] = c.n_blocks
    seqs, ns = [0, 1, 2, 3, 4, 3], [65, 200, 193, 200, 10, 64 * 4 + 1]
    out, lse, _ = attend(c, q, "f32", ints(seqs), ints(ns))
    torch.cuda.synchronize()
    assert host.kernel_error(reset=True) == 2
    for r in (0, 2, 4, 5):
        assert torch.isnan(out[r]).all() and torch.isnan(lse[r]).all(), r
    good = [1, 3]
    check_rows(c, q[good], "f32", [1, 3], [200, 200], out[good], lse[good])


def test_attention_is_deterministic_and_independent_of_the_batch_order():
    import torch

    lens = [3000, 17, 900, 0, 2222]
    c = filled(lens, 2, seed=31)
    q = torch.randn(5, 12, 128, generator=torch.Generator().manual_seed(7)).cuda()
    first, lse, _ = attend(c, q, "f32", ints(range(5)), ints(lens))
    for _ in range(3):
        again, lse2, _ = attend(c, q, "f32", ints(range(5)), ints(lens))
        torch.cuda.synchronize()
        assert torch.equal(first, again) and torch.equal(lse, lse2)


def test_attention_two_streams_at_once():
    """Two calls that overlap, each with a workspace of its own."""
    import torch

    lens = [8000, 5000]
    c = filled(lens, 2, seed=41)
    q = [torch.randn(2, 12, 128, generator=torch.Generator().manual_seed(i)).cuda() for i in range(2)]
    alone = [attend(c, x, "f32", ints([0, 1]), ints(lens))[0] for x in q]
    seqs, ns = ints([0, 1]), ints(lens)
    streams = [torch.cuda.Stream() for _ in q]
    works = [attend(c, x, "f32", seqs, ns)[2] for x in q]
    torch.cuda.synchronize()
    outs = [torch.empty_like(x) for x in q]
    lses = [torch.empty(2, 12, device="cuda") for _ in q]
    torch.cuda.synchronize()
    for _ in range(5):
        for i, s in enumerate(streams):
            attend(c, q[i], "f32", seqs, ns, out=outs[i], lse=lses[i], stream=s, work=works[i])
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(outs[i], alone[i])


def test_calls_on_a_stream_of_their_own_follow_it():
    """Append, attention, read and sampling enqueued on a side stream behind work that is still running there."""
    import torch
    from work_llm_accelerator_b200 import host

    c = filled([200], 2, seed=81)
    r = np.random.RandomState(3)
    x = rows(r, 8, 2)
    side = torch.cuda.Stream()
    src = {w: torch.as_tensor(x[w]).cuda() for w in "kv"}
    late = {w: torch.zeros_like(src[w]) for w in "kv"}
    a = [ints([0]), ints([150]), ints([0, 8])]
    q = torch.randn(1, 12, 128, generator=torch.Generator().manual_seed(4)).cuda()
    seqs, ns = ints([0]), ints([158])
    out, lse = torch.zeros_like(q), torch.zeros(1, 12, device="cuda")
    work = torch.empty(host.kv8_attention_workspace(1, 12, 2), dtype=torch.uint8, device="cuda")
    back = {w: torch.zeros_like(src[w]) for w in "kv"}
    busy = torch.randn(4096, 4096, device="cuda")
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(5):
            busy = busy @ busy * 1e-3
        for w in "kv":
            late[w].copy_(src[w])  # not there yet when the calls below are made
        s = side.cuda_stream
        host.kv8_append(c.handle, late["k"].data_ptr(), late["v"].data_ptr(), host.F32, 256, 8, *(v.data_ptr() for v in a), 1, s)
        attend(c, q, "f32", seqs, ns, out=out, lse=lse, stream=side, work=work)
        host.kv8_read(c.handle, back["k"].data_ptr(), back["v"].data_ptr(), host.F32, 256, 8, *(v.data_ptr() for v in a), 1, s)
    torch.cuda.synchronize()
    for w in "kv":
        c.model[w].append(x[w], 0, 150)
        np.testing.assert_array_equal(back[w].cpu().numpy(), c.model[w].values(0, 8, 150))
    check_rows(c, q, "f32", [0], [158], out, lse)


def test_attention_block_offsets_past_31_bits():
    """A pool of more than 2^31 codes: blocks at its end."""
    import torch

    heads, n_blocks = 8, 33000  # 2.16e9 codes
    c = filled([130], heads, seed=51)
    big = {w: torch.empty((n_blocks, heads, 64, 128), dtype=torch.int8, device="cuda") for w in "kv"}
    scales = {w: torch.full((n_blocks, heads), float("nan"), device="cuda") for w in "kv"}
    from work_llm_accelerator_b200 import host

    moved = n_blocks - 1 - c.table[0, :3]
    for w in "kv":
        for j in range(3):
            big[w][moved[j]] = c.codes[w][c.table[0, j]]
            scales[w][moved[j]] = c.scales[w][c.table[0, j]]
    table = ints(moved[None, :])
    c.handle = host.Kv8Cache(big["k"].data_ptr(), big["v"].data_ptr(), scales["k"].data_ptr(), scales["v"].data_ptr(), n_blocks,
                             heads, table.data_ptr(), 1, 3)
    q = torch.randn(1, 16, 128, generator=torch.Generator().manual_seed(1)).cuda()
    out, lse, _ = attend(c, q, "f32", ints([0]), ints([130]))
    check_rows(c, q, "f32", [0], [130], out, lse)
    got, _ = c.read("f32", [0], [0], [130])
    np.testing.assert_array_equal(got["k"].cpu().numpy(), c.model["k"].values(0, 130))


# ---------------------------------------------------------------------------------------------------
# a serving step
# ---------------------------------------------------------------------------------------------------
def test_decode_loop_in_a_graph():
    """Prompt, then 70 captured-and-replayed decode steps of three sequences (append, attention, sampling from logits
    made of the context); positions advance on the device. Checked step by step against the models."""
    import torch
    from work_llm_accelerator_b200 import host

    heads, q_heads, vocab, steps = 2, 12, 999, 70
    prompt = [5, 64, 130]
    lens = [n + steps for n in prompt]
    c = Cache(lens, heads, seed=61)
    r = np.random.RandomState(3)
    c.append(rows(r, sum(prompt), heads), "f32", [0, 1, 2], [0, 0, 0], prompt)
    g = torch.Generator().manual_seed(5)
    qkv = torch.zeros(3, q_heads + 2 * heads, 128, device="cuda")
    head = (0.3 * torch.randn(vocab, q_heads * 128, generator=g)).cuda()
    ctx, lse = torch.zeros(3, q_heads, 128, device="cuda"), torch.zeros(3, q_heads, device="cuda")
    logits = torch.zeros(3, vocab, device="cuda")
    seqs, pos, off = ints([0, 1, 2]), ints(prompt), ints([0, 1, 2, 3])
    n_now = ints([p + 1 for p in prompt])
    temp, top_k = torch.full((3,), 0.8, device="cuda"), ints([0, 20, 5])
    top_p = torch.tensor([0.9, 0.8, 1.0], device="cuda")
    u, tokens, probs = torch.zeros(3, device="cuda"), ints([0, 0, 0]), torch.zeros(3, device="cuda")
    work = torch.empty(host.kv8_attention_workspace(3, q_heads, heads), dtype=torch.uint8, device="cuda")

    def step():
        s = torch.cuda.current_stream().cuda_stream
        stride = qkv.stride(0)
        host.kv8_append(c.handle, qkv[:, q_heads].data_ptr(), qkv[:, q_heads + heads].data_ptr(), host.F32, stride, 3,
                        seqs.data_ptr(), pos.data_ptr(), off.data_ptr(), 3, s)
        host.kv8_attention(c.handle, qkv.data_ptr(), stride, ctx.data_ptr(), ctx.stride(0), host.F32, 3, q_heads,
                           seqs.data_ptr(), n_now.data_ptr(), SCALE, work.data_ptr(), work.numel(), lse.data_ptr(), s)
        torch.matmul(ctx.view(3, -1), head.t(), out=logits)
        host.sample(logits.data_ptr(), host.F32, 3, vocab, vocab, temp.data_ptr(), top_k.data_ptr(), top_p.data_ptr(), 0,
                    u.data_ptr(), tokens.data_ptr(), probs.data_ptr(), s)
        pos.add_(1)
        n_now.add_(1)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.matmul(ctx.view(3, -1), head.t(), out=logits)  # library set-up before the capture
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for t in range(steps):
        x = torch.randn(3, q_heads + 2 * heads, 128, generator=g)
        qkv.copy_(x)
        u.copy_(torch.rand(3, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        for i in range(3):
            c.model["k"].append(x[i : i + 1, q_heads : q_heads + heads].numpy(), i, prompt[i] + t)
            c.model["v"].append(x[i : i + 1, q_heads + heads :].numpy(), i, prompt[i] + t)
        if t % 9 == 0 or t == steps - 1:
            check_rows(c, x[:, :q_heads], "f32", [0, 1, 2], [p + t + 1 for p in prompt], ctx, lse)
            lg = logits.cpu().numpy()
            for i in range(3):
                ids, w = km.kept(lg[i], float(temp[i]), int(top_k[i]), float(top_p[i]))
                tok, ui = int(tokens[i]), float(u[i])
                assert tok in ids
                j = int(np.nonzero(ids == tok)[0][0])
                cum = np.concatenate([[0.0], np.cumsum(w)]) / w.sum()
                # the weights are within 2^-20 of exact ones, a cut at the border of top-p within one token
                assert cum[j] - 1e-5 - w[-1] / w.sum() <= ui <= cum[j + 1] + 1e-5 + w[-1] / w.sum()
    c.check(lens)
    assert host.kernel_error() == 0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_queries_near_the_largest_number(dtype):
    """Queries on both sides of 2^127, up to the largest finite value of the type, with a scale that brings them back to 1."""
    import torch

    lens = [300, 64, 1]
    c = filled(lens, 2, seed=22)
    g = torch.Generator().manual_seed(6)
    q = (2 * torch.rand(3, 12, 128, generator=g) - 1) * torch.tensor([3.3e38, 1.7e38, 2.5e38])[:, None, None]
    q[0, 0, 0], q[1, 0, 0] = torch.finfo(dt(dtype)).max, 2.0**127
    q = q.to(dt(dtype)).cuda()
    assert torch.isfinite(q).all()
    scale = 2.0**-128
    out, lse, _ = attend(c, q, dtype, ints([0, 1, 2]), ints(lens), scale=scale)
    check_rows(c, q, dtype, [0, 1, 2], lens, out, lse, scale=scale)


def values64(c, w, seq, n):
    """code * scale in 64 bits, where the model rounds it to fp32 as the reading back does (2^-24 of a value, which is more
    than the bounds below leave)."""
    pos = np.arange(n)
    b = c.table[seq, pos // km.BLOCK]
    return c.model[w].codes[b, :, pos % km.BLOCK] * c.model[w].scales[b].astype(np.float64)[:, :, None]


def score_bound(q, k, scale, s):
    """How far a score may be off: q is held to 2^-30 of its row's largest channel (half a step of 31-bit integers; the
    2^-6 covers the digits' joining), the exact digit products are joined, scaled and carried to lse in at most 12
    roundings of 2^-24."""
    q, k = np.abs(np.asarray(q, np.float64)), np.abs(np.asarray(k, np.float64))
    return abs(scale) * 2.0**-30 * (1 + 2.0**-6) * q.max(-1) * k.sum(-1) + 12 * 2.0**-24 * np.abs(s)


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("ratio,code", [(1.0, 1.0), (50.0, 1.0), (200.0, 0.02), (1000.0, 0.0), (30000.0, 0.0), (1000.0, 0.01)])
def test_attention_one_large_channel(dtype, ratio, code):
    """A channel far larger than the others, whose keys are small or zero: the others must not lose their bits to it. With one
    token, lse is its score."""
    import torch

    n = 40
    c = filled([1] * n, 2, seed=23)
    for b in c.table[:, 0]:
        c.model["k"].codes[b, :, 0, 17] = np.rint(code * c.model["k"].codes[b, :, 0, 17])
    c.codes["k"].copy_(torch.as_tensor(c.model["k"].codes.astype(np.int8)))
    q = torch.randn(n, 12, 128, generator=torch.Generator().manual_seed(int(ratio)))
    q[:, :, 17] *= ratio / q[:, :, 17].abs()
    q = q.to(dt(dtype)).cuda()
    out, lse, _ = attend(c, q, dtype, ints(range(n)), ints([1] * n))
    q, lse = q.float().cpu().numpy().astype(np.float64), lse.cpu().numpy()
    for r in range(n):
        k = values64(c, "k", r, 1)[0]
        for h in range(12):
            want = float(k[h // 6] @ q[r, h] * np.float32(SCALE))
            assert abs(lse[r, h] - want) <= score_bound(q[r, h], k[h // 6], SCALE, want), (r, h, lse[r, h] - want)
    check_rows(c, torch.as_tensor(q), dtype, list(range(n)), [1] * n, out, torch.as_tensor(lse))


@pytest.mark.parametrize("below", [2.0, 5.0, 8.0, 11.0, 14.0])
def test_attention_small_weights_beside_a_large_one(below):
    """A first token that takes almost all of the weight and whose values are zero: the result is that of the others in its
    tile. Their weights are held to 2^-30 of the largest."""
    import torch

    u, n = 2.0**-24, 32
    c = filled([n], 1, seed=24)
    b = c.table[0, 0]
    for w in "kv":
        c.model[w].codes[b, 0, 0] = 0.0
        c.model[w].scales[b] = 0.01
    c.model["k"].codes[b, 0, 1:] = np.rint(c.model["k"].codes[b, 0, 1:] / 16) - 100
    for w in "kv":
        c.codes[w].copy_(torch.as_tensor(c.model[w].codes.astype(np.int8)))
        c.scales[w].copy_(torch.as_tensor(c.model[w].scales))
    q = (below / (128 * SCALE) * (0.5 + torch.rand(1, 6, 128, generator=torch.Generator().manual_seed(3)))).cuda()
    out, lse, _ = attend(c, q, "f32", ints([0]), ints([n]))
    k, v = (values64(c, w, 0, n)[:, 0] for w in "kv")
    got, qs = out[0].cpu().numpy(), q[0].cpu().numpy().astype(np.float64)
    for h in range(6):
        s = k @ qs[h] * np.float32(SCALE)
        p = np.exp(s - s.max())
        d = score_bound(qs[h], k, SCALE, s).max()
        want = p @ v / p.sum()
        # weights: 2^-30 each, 2 d from the scores, 4 u from the exponential; sums of 32 and the last steps: 48 u
        tol = 2.0**-30 * (1 + 2.0**-6) * np.abs(v).sum(0) / p.sum() + (2 * d + 52 * u) * (p @ np.abs(v)) / p.sum() + 2.0**-149
        assert (np.abs(got[h] - want) <= tol).all(), (h, np.abs(got[h] - want).max(), tol.min())
        assert abs(float(lse[0, h]) - (s.max() + np.log(p.sum()))) <= 2 * d + 52 * u


@pytest.mark.parametrize("size", [1e-37, 1e-30, 1e-20, 1e20, 1e34])
def test_attention_sizes_of_values(size):
    """Values of V far from 1, down to scales of a few smallest normal numbers: the result keeps all of their bits."""
    import torch

    u, n = 2.0**-24, 150
    c = filled([n], 2, seed=25)
    c.model["v"].scales[:] = np.float32(size)
    c.scales["v"].copy_(torch.as_tensor(c.model["v"].scales))
    q = torch.randn(1, 12, 128, generator=torch.Generator().manual_seed(5)).cuda()
    out, lse, _ = attend(c, q, "f32", ints([0]), ints([n]))
    k, v = (values64(c, w, 0, n) for w in "kv")
    want, _, mag = km.attention(q[0].cpu().numpy(), k, v, float(np.float32(SCALE)))
    # scores: 12 roundings of a sum of absolute products; 2 d of them, weights and sums of 5 tiles
    eps = 2 * 12 * u * mag + 2.0**-29 + 100 * u
    assert (np.abs(out[0].cpu().numpy() - want) <= eps * np.abs(v).max() + 2.0**-149).all()


def test_attention_rows_in_another_order_or_batch():
    """The same rows permuted, and a few of them alone: other splits of the work, so equal up to the bound of check_rows, and
    each order repeats bit for bit."""
    import torch

    lens = [3000, 17, 900, 0, 2222, 64, 5000]
    n = len(lens)
    c = filled(lens, 2, seed=32)
    q = torch.randn(n, 12, 128, generator=torch.Generator().manual_seed(8)).cuda()
    r = np.random.RandomState(4)
    for order in [list(range(n)), list(range(n))[::-1], list(r.permutation(n)), [4], [6, 2], [2, 6]]:
        ns = [lens[i] for i in order]
        out, lse, _ = attend(c, q[order], "f32", ints(order), ints(ns))
        again, lse2, _ = attend(c, q[order], "f32", ints(order), ints(ns))
        torch.cuda.synchronize()
        check_rows(c, q[order], "f32", order, ns, out, lse)
        assert torch.equal(out, again) and torch.equal(lse, lse2)


def test_read_next_to_the_largest_number():
    """65504 in a block whose scale was doubled is a number of steps rounded up: documented to read as infinity in fp16;
    within a step in fp32."""
    c = Cache([2], 1, seed=26)
    c.append({w: np.full((1, 1, 128), 35000.0, np.float32) for w in "kv"}, "f32", [0], [0], [1])
    c.append({w: np.full((1, 1, 128), 65504.0, np.float32) for w in "kv"}, "f16", [0], [1], [1])
    c.check([2])
    for dtype in ("f16", "f32"):
        out, _ = c.read(dtype, [0], [0], [2])
        for w in "kv":
            want = c.model[w].values(0, 2)
            with np.errstate(over="ignore"):
                want = want.astype(np.float16).astype(np.float32) if dtype == "f16" else want
            np.testing.assert_array_equal(out[w].float().cpu().numpy(), want)
            if dtype == "f32":
                step = c.model[w].scales[c.table[0, 0]][0]
                assert (np.abs(want[:, 0] - [[35000.0], [65504.0]]) < step).all()
