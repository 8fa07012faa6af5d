"""GPU tests of token sampling (include/qwen_b200_ops.h) against the plain float64 model in kv8_model.py. Uniform
numbers and top_p values are put in the middle between two borders, at least 1e-6 of the whole from either, where the
kernel's weights (each within 2^-20 of the exact one, so their sums too) cannot change the answer."""
from __future__ import annotations

import numpy as np
import pytest

import kv8_model as km

pytestmark = pytest.mark.gpu

TYPES = {"f32": 0, "f16": 1, "bf16": 2}


@pytest.fixture(autouse=True)
def _device(built_libs, gpu_available):
    if not gpu_available:
        pytest.fail("no CUDA device: the -m gpu suite must run on a B200")


def run(logits, u, dtype="f32", temperature=None, top_k=None, top_p=None, min_p=None, vocab=None, probs=True):
    """logits [rows][>= vocab] torch tensor of its type on the CPU; the settings lists or None."""
    import torch
    from work_llm_accelerator_b200 import host

    x = logits.cuda()
    n = x.shape[0]
    vocab = x.shape[1] if vocab is None else vocab
    f = lambda v, t: None if v is None else torch.tensor(v, dtype=t).cuda()  # noqa: E731
    t, k, p, m = f(temperature, torch.float32), f(top_k, torch.int32), f(top_p, torch.float32), f(min_p, torch.float32)
    u = f(u, torch.float32)
    tokens = torch.full((n,), -9, dtype=torch.int32).cuda()
    out = torch.full((n,), -9.0).cuda()
    ptr = lambda v: 0 if v is None else v.data_ptr()  # noqa: E731
    host.sample(x.data_ptr(), TYPES[dtype], n, vocab, x.stride(0), ptr(t), ptr(k), ptr(p), ptr(m), u.data_ptr(),
                tokens.data_ptr(), out.data_ptr() if probs else 0, torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    return tokens.cpu().numpy(), out.cpu().numpy()


def middle(w, r):
    """A uniform number in the middle of the interval of one of the larger weights, and that weight's place."""
    p = w / w.sum()
    at = int(r.choice(np.nonzero(p >= min(1e-5, p.max()))[0]))
    return float((np.cumsum(p)[at] - p[at] / 2)), at


def check(rows, dtype, seed, **settings):
    """Every row: filters on, u in the middle of a kept token's interval."""
    import torch

    r = np.random.RandomState(seed)
    x = rows.float().numpy()
    n = len(x)
    us, want, want_p = [], [], []
    for i in range(n):
        f = {k: v[i] for k, v in settings.items() if v is not None}
        if "temperature" in f:
            f["temperature"] = np.float32(f["temperature"])
        ids, w = km.kept(x[i], **{k: (float(np.float32(v)) if k != "top_k" else v) for k, v in f.items()})
        if len(ids) == 0:
            us.append(0.5), want.append(-1), want_p.append(0.0)
            continue
        u, at = middle(w, r)
        us.append(u), want.append(ids[at]), want_p.append(w[at] / w.sum())
    got, p = run(rows, us, dtype, **settings)
    np.testing.assert_array_equal(got, want)
    np.testing.assert_allclose(p, want_p, rtol=2.0**-18, atol=0)  # 2^-20 of a weight and of their sum, rounding


def gaussian(rows, vocab, dtype, seed, size=1.7, peak=6.0):
    import torch

    g = torch.Generator().manual_seed(seed)
    x = size * torch.randn(rows, vocab, generator=g)
    x[:, torch.randperm(vocab, generator=g)[: min(vocab, 30)]] += peak * torch.rand(rows, min(vocab, 30), generator=g)
    return x.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype])


def safe_top_p(x, temperature, top_k, near):
    """Per row a top_p near `near` that lies in the middle of a token's share."""
    out = []
    for i in range(len(x)):
        _, w = km.kept(x[i].float().numpy(), float(np.float32(temperature[i])) if temperature else 1.0, top_k[i] if top_k else 0)
        c = np.cumsum(w) / w.sum()
        p = w / w.sum()
        ok = np.nonzero(p >= min(4e-6, p.max()))[0]
        at = ok[np.argmin(np.abs(c[ok] - near))]
        out.append(float(c[at] - p[at] / 2))
    return out


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 50257, 151936, 262144])
def test_plain_sampling(dtype, vocab):
    check(gaussian(3, vocab, dtype, vocab), dtype, vocab, temperature=[0.7, 1.0, 1.3])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [7, 1000, 151936])
@pytest.mark.parametrize("k", [1, 2, 50, 900, 70000])
def test_top_k(dtype, vocab, k):
    check(gaussian(2, vocab, dtype, k), dtype, k, temperature=[0.8, 1.5], top_k=[k, max(1, k // 2)])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("near", [0.01, 0.5, 0.9, 0.97])
@pytest.mark.parametrize("vocab,size,peak", [(1000, 1.7, 6.0), (151936, 1.7, 6.0), (151936, 1.7, 12.0)])
def test_top_p_alone_and_after_top_k(dtype, near, vocab, size, peak):
    x = gaussian(4, vocab, dtype, int(near * 100), size, peak)
    t, k = [0.6, 1.0, 1.0, 0.9], [0, 0, 40, 300]
    check(x, dtype, 1, temperature=t, top_k=k, top_p=safe_top_p(x, t, k, near))


@pytest.mark.parametrize("min_p", [1e-6, 0.013, 0.3, 1.0, 2.0])
def test_min_p(min_p):
    """The border is compared in 64 bits; rows where a weight lies within 2^-40 of it do not occur here."""
    x = gaussian(3, 20000, "f32", 5)
    check(x, "f32", 2, temperature=[0.9, 1.0, 1.1], min_p=[min_p] * 3)


@pytest.mark.parametrize("temperature", [1.0, 0.7, 1.3])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_min_p_at_weights_of_its_own_size(dtype, temperature):
    """Logits in steps of 1/64 of the temperature, min_p the weight of one of them rounded to fp32: whether it reaches is
    decided in the last bits, and the weights lie on the borders of a coarse view."""
    import torch

    t = np.float32(temperature)
    steps = (3, 64, 100, 128, 192, 321)
    for k in steps:
        x = torch.tensor(np.float32(8.0) - (np.arange(400) / 64 * t).astype(np.float32))[torch.randperm(400, generator=torch.Generator().manual_seed(k))]
        x = x[None].to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype])
        # the weight of a token that is there, as the definition has it, rounded once
        z = (x.double().max() - x.double().sort(descending=True).values[0, k]) / float(t)
        check(x, dtype, k, temperature=[float(t)], min_p=[float(np.float32(np.exp(-float(z))))])


def test_all_filters_with_rows_of_their_own():
    x = gaussian(24, 151936, "bf16", 8)
    r = np.random.RandomState(1)
    t = [0.0 if i % 7 == 3 else float(0.4 + r.rand()) for i in range(24)]
    k = [int(v) for v in r.randint(0, 80, 24)]
    p = safe_top_p(x, [v or 1.0 for v in t], k, 0.9)
    p = [1.0 if i % 5 == 0 else v for i, v in enumerate(p)]
    check(x, "bf16", 3, temperature=t, top_k=k, top_p=p, min_p=[0.0 if i % 3 else 0.02 for i in range(24)])


@pytest.mark.parametrize("vocab", [1, 5, 8193, 151936])
@pytest.mark.parametrize("k", [0, 3, 2000, 100000])
def test_ties_go_to_the_lowest_index(vocab, k):
    """Every logit equal: token j's interval is the j-th. Zeros of both signs tie."""
    import torch

    x = torch.zeros(2, vocab)
    x[1, ::2] = -0.0
    n = min(k, vocab) if k else vocab
    js = [0, n - 1]
    got, p = run(x, [(j + 0.5) / n for j in js], top_k=[k, k])
    assert list(got) == js
    np.testing.assert_allclose(p, 1.0 / n, rtol=2.0**-18)
    # half of the mass: top_p in the middle of the share of token m
    m = n // 2
    got, p = run(x, [(m + 0.5) / (m + 1)] * 2, top_k=[k, k], top_p=[(m + 0.5) / n] * 2)
    assert list(got) == [m, m]
    np.testing.assert_allclose(p, 1.0 / (m + 1), rtol=2.0**-18)


def test_two_levels_of_ties():
    """70000 tokens tie at the border of the kept set."""
    import torch

    x = torch.full((1, 151936), -1.0)
    x[0, 50000:120000] = 0.25
    x[0, [149000, 3]] = 0.5
    ids, w = km.kept(x[0].numpy(), 1.0, 30002)
    for at in (0, 1, 2, 3, 15000, 30001):
        p = w / w.sum()
        got, _ = run(x, [float(np.cumsum(p)[at] - p[at] / 2)], top_k=[30002])
        assert got[0] == ids[at], at


@pytest.mark.parametrize("rows", [18, 19, 40, 75, 150])
def test_row_counts_that_share_the_gpu_differently(rows):
    """Ties by the thousand and ordinary rows, at numbers of rows that give a row 8, 4, 2 CTAs and one."""
    import torch

    x = gaussian(rows, 20000, "f32", rows)
    x[::2] = 0.5  # every second row: all equal
    k = [[0, 12000, 700][i % 3] for i in range(rows)]
    check(x, "f32", rows, temperature=[0.9] * rows, top_k=k)
    js = [i * 7 % 600 for i in range(rows)]
    got, _ = run(x[::2], [(j + 0.5) / 12000 for j in js][: len(x[::2])], top_k=[12000] * len(x[::2]))
    assert list(got) == js[: len(got)]


@pytest.mark.parametrize("rows", [1, 40, 150])
def test_the_largest_vocabulary_with_one_value(rows):
    """262143 tokens of one value just below the best: the sums at their largest, on 8, 4 and 1 CTAs per row."""
    import torch

    x = torch.zeros(rows, 262144)
    x[:, 200000] = 0.0156
    _, w = km.kept(x[0].numpy())
    p = w / w.sum()
    places = [0, 1, 2, 100000, 262142, 262143]
    us = [float(np.cumsum(p)[at] - p[at] / 2) for at in places]
    ids = [200000] + [i for i in range(262144) if i != 200000]
    got, prob = run(x, [us[i % 6] for i in range(rows)])
    assert list(got) == [ids[places[i % 6]] for i in range(rows)]
    np.testing.assert_allclose(prob, [p[places[i % 6]] for i in range(rows)], rtol=2.0**-18)


@pytest.mark.parametrize("spread", [1e-6, 1e-3, 0.05])
def test_crowded_logits(spread):
    """All logits within a narrow band: thousands share what a coarse view would call one value."""
    x = gaussian(2, 151936, "f32", 4, size=spread, peak=0.0)
    check(x, "f32", 5, top_k=[100, 77777])
    check(x, "f32", 6, temperature=[1.0, 30.0], top_p=safe_top_p(x, [1.0, 30.0], None, 0.4))


def test_masked_rows_and_infinities():
    import torch

    inf, nan = float("inf"), float("nan")
    x = torch.tensor([[-inf, -inf, -inf, -inf], [nan, nan, -inf, nan], [-inf, 2.0, nan, 2.0], [1.0, inf, 3.0, inf],
                      [-inf, -3e38, 3e38, 3e38], [3.0, 1.0, -inf, 3.0]])
    for t in (0.0, 0.5, 1.0):
        got, p = run(x, [0.6] * 6, temperature=[t] * 6, top_k=[3] * 6, top_p=[0.99] * 6, min_p=[0.1] * 6)
        assert list(got) == ([-1, -1, 1, 1, 2, 0] if t == 0 else [-1, -1, 3, 3, 3, 3])
        # the last row keeps its third token where e^(-2 / t) is at least 0.1
        last = 0.5 if t == 0.5 else 1 / (2 + np.exp(-2.0))
        np.testing.assert_allclose(p, [0, 0, 1, 1, 1, 1] if t == 0 else [0, 0, 0.5, 0.5, 0.5, last], rtol=2.0**-18)


def test_a_mask_of_the_lowest_value():
    """Banned tokens as the type's lowest value instead of -infinity: weight 0 next to any other, equal among themselves."""
    import torch

    low = torch.finfo(torch.float32).min
    x = torch.full((2, 5000), low)
    x[0, 4321] = 1.0
    got, p = run(x, [0.9999, (1234 + 0.5) / 5000])
    assert list(got) == [4321, 1234] and p[0] == 1.0


@pytest.mark.parametrize("t", [float("nan"), -1.0, 1e-40, 2.0**-126, 1e-3, 1e30, float("inf")])
def test_extreme_temperatures(t):
    import torch

    x = torch.tensor([[0.5, 2.0, 1.0, 2.0]])
    if not t >= 2.0**-126:
        want = [(0.7, 1, 1.0)]
    elif t < 1:
        want = [(0.25, 1, 0.5), (0.75, 3, 0.5)]
    else:
        want = [(0.125, 1, 0.25), (0.375, 3, 0.25), (0.625, 2, 0.25), (0.875, 0, 0.25)]
    for u, token, prob in want:
        got, p = run(x, [u], temperature=[t])
        assert got[0] == token
        np.testing.assert_allclose(p, prob, rtol=2.0**-18)


def test_settings_at_their_borders():
    import torch

    x = torch.tensor([[1.0, 3.0, 2.0]])
    for kw in ({"top_p": [0.0]}, {"top_p": [-1.0]}, {"top_k": [1]}, {"min_p": [1.0]}, {"min_p": [5.0]}):
        for u in (0.0, 0.999):
            assert run(x, [u], **kw)[0][0] == 1, kw
    for kw in ({"top_p": [1.0]}, {"top_p": [2.0]}, {"top_p": [float("nan")]}, {"top_k": [0]}, {"top_k": [-3]}, {"top_k": [99]},
               {"min_p": [0.0]}, {"min_p": [-1.0]}, {"min_p": [float("nan")]}):
        assert run(x, [0.0], **kw)[0][0] == 1 and run(x, [0.999], **kw)[0][0] == 0, kw
    # uniform numbers outside of [0, 1): the first and the last kept token
    for u, token in ((-1.0, 1), (float("nan"), 1), (1.0, 0), (7.0, 0)):
        assert run(x, [u])[0][0] == token


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab,stride", [(1001, 1001), (1000, 1003), (151935, 151936), (50257, 50300)])
def test_strides_and_alignment(dtype, vocab, stride):
    """Rows that start at any element; what lies between them must not be read as logits."""
    import torch

    x = gaussian(3, vocab, dtype, 9)
    wide = torch.full((3, stride), 60000.0).to(x.dtype)
    wide[:, :vocab] = x
    us = [0.1, 0.5, 0.8]
    want, wp = run(x, us, dtype, top_k=[50] * 3)
    got, p = run(wide, us, dtype, top_k=[50] * 3, vocab=vocab)
    np.testing.assert_array_equal(got, want)
    np.testing.assert_array_equal(p, wp)


def test_many_rows_repeat_exactly_and_without_probs():
    x = gaussian(400, 5000, "f32", 12)
    us = list(np.linspace(0, 0.999, 400))
    a, p = run(x, us, top_p=[0.9] * 400)
    b, q = run(x, us, top_p=[0.9] * 400)
    c, none = run(x, us, top_p=[0.9] * 400, probs=False)
    assert (a == b).all() and (p == q).all() and (a == c).all() and (none == -9).all()


def test_engine_samples_from_its_own_logits():
    """A generation loop: prompt, then batched steps whose tokens are sampled on the device from the engine's logits."""
    from work_llm_accelerator_b200 import host

    eng = host.Engine(0, 8, max_seqs=3, max_len=256)
    try:
        eng.init_synthetic(5)
        with pytest.raises(host.EngineError):
            eng.sample([0.5])  # no call yet
        eng.set_option("logits", 1)
        r = np.random.RandomState(0)
        nxt = []
        for slot in range(3):
            greedy = eng.prefill(slot, r.randint(0, host.VOCAB, 5 + slot))
            x = eng.read_logits(1)[0]
            tokens, probs = eng.sample([0.7], temperature=[0.0])
            assert tokens[0] == greedy == int(x.argmax()) and probs[0] == 1.0
            nxt.append(int(tokens[0]))
        for step in range(4):
            eng.decode([0, 1, 2], nxt)
            x = eng.read_logits(3)
            kw = dict(temperature=[0.7, 1.0, 1.2], top_k=[50, 0, 7], min_p=[0.0, 0.01, 0.0])
            us, want = [], []
            for i in range(3):
                f = {k: (float(np.float32(v[i])) if k != "top_k" else v[i]) for k, v in kw.items()}
                ids, w = km.kept(x[i], **f)
                u, at = middle(w, r)
                us.append(u)
                want.append((int(ids[at]), w[at] / w.sum()))
            tokens, probs = eng.sample(us, **kw)
            assert [int(t) for t in tokens] == [t for t, _ in want]
            np.testing.assert_allclose(probs, [p for _, p in want], rtol=2.0**-18)
            nxt = [int(t) for t in tokens]
        with pytest.raises(host.EngineError):
            eng.sample([0.5, 0.5])  # the last call had three rows
        with pytest.raises(ValueError):
            eng.sample([0.5] * 3, top_k=[1, 2])
        eng.set_option("logits", 0)
        eng.decode([0, 1, 2], nxt)
        with pytest.raises(host.EngineError):
            eng.sample([0.5] * 3)  # kept no logits
    finally:
        eng.close()


@pytest.mark.parametrize("rows", [1, 18, 19, 74, 75, 148])
@pytest.mark.parametrize("vocab", [8193, 20000])
def test_short_rows_on_several_ctas_started_one_by_one(rows, vocab):
    """A row's CTAs exchange their largest logits after a first pass of a microsecond. Launches behind work that frees its
    SMs one at a time start them apart: every row still has the argmax of all its parts."""
    import torch
    from work_llm_accelerator_b200 import host

    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, vocab, generator=g).cuda()
    want = x.argmax(1).to(torch.int32)
    zero, t = torch.zeros(rows, device="cuda"), torch.zeros(rows, device="cuda")
    tokens = torch.full((40, rows), -9, dtype=torch.int32, device="cuda")
    other = torch.cuda.Stream()
    busy = torch.randn(3000, 700, device="cuda")
    torch.cuda.synchronize()
    for i in range(40):
        with torch.cuda.stream(other):
            busy = (busy * 1.0001).sin()
        host.sample(x.data_ptr(), host.F32, rows, vocab, vocab, t.data_ptr(), 0, 0, 0, zero.data_ptr(), tokens[i].data_ptr(), 0,
                    torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert (tokens == want[None]).all()


@pytest.mark.parametrize("rows", [1, 18, 40, 75, 150])
@pytest.mark.parametrize("u", [1.0, 7.0, 3e38, float("inf")])
def test_uniform_numbers_from_one_on_take_the_last_kept_token(rows, u):
    """Thousands of ties around the border of what is kept and thousands of tokens behind it, none of which may be counted
    with the draw: [0, 1) is asked for, but the numbers lie on the device, where nothing else checks them."""
    import torch

    x = torch.full((rows, 60000), -9.0)
    r = np.random.RandomState(rows)
    places = r.permutation(60000)
    x[:, np.sort(places[:20000])] = 1.0
    x[:, np.sort(places[20000:39000])] = 0.5
    x[:, places[39000]] = -3.0
    one = np.sort(places[:20000])
    second = np.sort(places[20000:39000])
    rest = np.setdiff1d(np.arange(60000), places[:39001])
    got, p = run(x, [u] * rows, top_k=[10000] * rows)
    assert (got == one[9999]).all()
    np.testing.assert_allclose(p, 1e-4, rtol=2.0**-18)
    got, _ = run(x, [u] * rows, top_k=[20000] * rows)  # the border is the bucket's
    assert (got == one[19999]).all()
    got, _ = run(x, [u] * rows, top_k=[25000] * rows)
    assert (got == second[4999]).all()
    # half of the first 20000: top_p in the middle of a share
    got, _ = run(x, [u] * rows, top_k=[20000] * rows, top_p=[(9999 + 0.5) / 20000] * rows)
    assert (got == one[9999]).all()
    got, _ = run(x, [u] * rows, min_p=[0.5] * rows)  # exp(-1 / 2) = 0.607, exp(-4) = 0.018
    assert (got == second[-1]).all()
    got, _ = run(x, [u] * rows, min_p=[0.01] * rows)
    assert (got == places[39000]).all()
    got, _ = run(x, [u] * rows)
    assert (got == rest[-1]).all()
    # few tokens in every bucket, all filters: what is listed and sorted at once
    x = gaussian(rows, 20000, "f32", rows)
    k, t = [50] * rows, [0.9] * rows
    top_p = safe_top_p(x, t, k, 0.9)
    got, _ = run(x, [u] * rows, temperature=t, top_k=k, top_p=top_p)
    want = [km.kept(x[i].numpy(), float(np.float32(0.9)), 50, float(np.float32(top_p[i])))[0][-1] for i in range(rows)]
    np.testing.assert_array_equal(got, want)


def step_borders(dtype, n):
    """(temperature, distance) pairs, fp32 and of the type: 64 * distance / temperature lies below a whole number but rounds
    to it in fp32."""
    r = np.random.RandomState(7)
    found = []
    while len(found) < n:
        t = (0.5 + r.rand(1000)).astype(np.float32)
        c = np.float32(64) * (np.float32(1) / t)
        bits = {"f32": 24, "f16": 11, "bf16": 8}[dtype]
        d = np.ldexp(r.randint(1 << (bits - 1), 1 << bits, 1000), 2 - bits).astype(np.float32)  # 2 to 4
        exact = c[:, None].astype(np.float64) * d[None, :]  # 48 bits at most
        near = exact.astype(np.float32)
        i, j = np.nonzero((near == np.rint(near)) & (near > exact) & (near >= 128) & (near < 256))
        found = list(dict.fromkeys(found + [(float(t[a]), float(d[b])) for a, b in zip(i, j)]))
    return found[:n]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [6, 24, 78, 156])
def test_logits_that_round_to_a_border(dtype, rows):
    """Distances whose steps round up to a border between two coarse views, thousands of tokens at each: the sums and the
    search for a token must put them on the same side. On 8, 4, 2 CTAs per row and one, in every type."""
    import torch

    pairs = step_borders(dtype, 6)
    x = torch.full((rows, 9000), float("-inf"))
    for i in range(rows):
        many = [3000, 300][i % 2]
        places = np.random.RandomState(i).permutation(9000)
        x[i, places[0]] = 0.0
        x[i, places[1 : 1 + many]] = -pairs[i % 6][1]
    x = x.to({"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype])
    t = [pairs[i % 6][0] for i in range(rows)]
    check(x, dtype, rows, temperature=t)
    check(x, dtype, rows + 1, temperature=t, top_k=[[1500, 150][i % 2] for i in range(rows)])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows", [16, 64, 148, 200])
def test_numbers_on_the_borders_between_tokens(dtype, rows):
    """A uniform number and a top_p that round to the sum at a token's end, with wide gaps between the logits: either
    neighbour may be drawn (the sums are those of other roundings), never a token that is not there."""
    import torch

    r = np.random.RandomState(rows)
    vocab = 9000
    x = torch.full((rows, vocab), float("-inf"))
    for i in range(rows):
        n = [40, 3000][i % 2]  # every second row: levels of a hundred ties each, more than are sorted at once
        level = np.sort(r.randint(0, 600, 30))[r.randint(0, 30, n)] / 40.0
        x[i, r.permutation(vocab)[:n]] = torch.as_tensor(-level, dtype=torch.float32)
    x = x.to({"f32": torch.float32, "bf16": torch.bfloat16}[dtype])
    for turn in range(8):
        us, near, ps = [], [], []
        for i in range(rows):
            ids, w = km.kept(x[i].float().numpy(), 0.7)
            p = np.cumsum(w) / w.sum()
            # ends of levels, where the next weight may be buckets away
            last = np.nonzero(np.append(np.diff(w) < 0, False))[0]
            at = int(r.choice(last[w[last] / w.sum() > 1e-5]))
            if turn % 2:  # top_p at the border, the draw at its end: the last token that top_p keeps
                ps.append(float(np.float32(p[at])))
                us.append(1.0)
            else:
                ps.append(1.0)
                us.append(float(np.float32(p[at])))
            # within 2^-19 of the whole, all that the weights' roundings and that of the number can move
            lo, hi = np.searchsorted(p, [p[at] - 2.0**-19, p[at] + 2.0**-19])
            near.append({int(v) for v in ids[lo : hi + 1]})
        got, _ = run(x, us, dtype, temperature=[float(np.float32(0.7))] * rows, top_p=ps if turn % 2 else None)
        for i in range(rows):
            assert int(got[i]) in near[i], (turn, i, int(got[i]))


def test_engine_keeps_no_logits_of_steps_that_were_not_asked_for():
    """After profiled or timed steps, or a call that failed on its way, there is nothing to sample from."""
    from work_llm_accelerator_b200 import host

    eng = host.Engine(0, 8, max_seqs=8, max_len=256)
    try:
        eng.init_synthetic(5)
        eng.set_option("logits", 1)
        for slot in range(8):
            eng.prefill(slot, [slot + 1, 7])

        def dropped(call, n, slots):
            eng.decode(slots, [3] * n)
            eng.sample([0.5] * n)
            call()
            with pytest.raises(host.EngineError, match="logits"):
                eng.sample([0.5] * n)

        def fails(call):
            with pytest.raises(host.EngineError):
                call()

        dropped(lambda: eng.profile_decode(0, 9, 2), 1, [0])
        dropped(lambda: eng.bench_decode([0], [9], 2, 1), 1, [0])
        dropped(lambda: eng.profile_batched(range(8), [9] * 8, 2), 8, range(8))
        dropped(lambda: fails(lambda: eng.decode([0, 99], [3, 3])), 2, [0, 1])
        dropped(lambda: fails(lambda: eng.prefill_chunk(0, [5] * 255)), 1, [0])
        dropped(lambda: fails(lambda: eng.prefill(0, [5])), 1, [0])  # the slot is not empty
        eng.set_option("batched", 0)
        # two groups, the second of which is refused after the first has run
        dropped(lambda: fails(lambda: eng.decode([0, 1, 2, 3, 99, 5, 6, 7], [3] * 8)), 4, [0, 1, 2, 3])
        eng.decode(range(6), [3] * 6)
        eng.sample([0.5, 0.5])  # the last group
        assert list(eng.sample([0.5, 0.5], temperature=[0.0, 0.0])[0]) == list(eng.read_logits(2).argmax(1))
    finally:
        eng.close()


def test_engine_rows_that_leave_settings_open():
    from work_llm_accelerator_b200 import host

    eng = host.Engine(0, 8, max_seqs=3, max_len=64)
    try:
        eng.init_synthetic(5)
        eng.set_option("logits", 1)
        for slot in range(3):
            eng.prefill(slot, [slot + 1, 7])
        eng.decode([0, 1, 2], [3, 3, 3])
        u = [0.9, 0.8, 0.999]
        want = eng.sample(u, temperature=[1.0, 0.0, 0.5], top_k=[0, 5, 9], top_p=[1.0, 1.0, 0.9], min_p=[0.1, 0.0, 0.0])
        got = eng.sample(u, temperature=[None, 0.0, 0.5], top_k=[None, 5, 9], top_p=[None, None, 0.9], min_p=[0.1, None, None])
        np.testing.assert_array_equal(got[0], want[0])
        np.testing.assert_array_equal(got[1], want[1])
    finally:
        eng.close()


@pytest.mark.parametrize("t,acts", [(2.0**-126, 2.0**-121), (1.5 * 2.0**-124, 2.0**-121), (2.0**-121, 2.0**-121), (1.3 * 2.0**-119, 1.3 * 2.0**-119)])
def test_the_smallest_temperatures(t, acts):
    """Logits as close to one another as the smallest temperatures are to 0: from 2^-126 to 2^-121 they act as 2^-121."""
    import torch

    step = 2.0**-121
    x = torch.tensor([[3 * step, 0.0, 1.5 * step, 3 * step]])
    ids, w = km.kept(x[0].numpy(), acts)
    for kw in ({}, {"min_p": [0.1]}):
        n = 4 if not kw else int((w >= 0.1).sum())
        p = w[:n] / w[:n].sum()
        for at in range(n):
            got, prob = run(x, [float(np.cumsum(p)[at] - p[at] / 2)], temperature=[t], **kw)
            assert got[0] == ids[at], (at, kw)
            np.testing.assert_allclose(prob, p[at], rtol=2.0**-18)
