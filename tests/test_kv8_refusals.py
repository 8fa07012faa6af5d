"""CPU tests of the 8-bit KV cache and sampling entry points: every argument that the host can check is refused with
status 1 and a message that names it, before any GPU work. And of the plain models themselves."""
from __future__ import annotations

import numpy as np
import pytest

import kv8_model as km

A = 1 << 20  # an aligned address that is never read


@pytest.fixture(scope="module")
def host(built_libs):
    from work_llm_accelerator_b200 import host as h

    return h


def cache(host, **kw):
    a = dict(k_codes_ptr=A, v_codes_ptr=A, k_scales_ptr=A, v_scales_ptr=A, n_blocks=4, n_kv_heads=2, block_table_ptr=A, n_seqs=1,
             max_blocks=4)
    return host.Kv8Cache(**{**a, **kw})


CACHE = [(dict(n_blocks=0), "n_blocks"), (dict(n_kv_heads=0), "n_kv_heads"), (dict(n_seqs=0), "n_seqs"),
         (dict(max_blocks=0), "max_blocks"), (dict(max_blocks=1 << 30), "max_blocks"), (dict(k_codes_ptr=0), "k_codes is null"),
         (dict(v_codes_ptr=A + 8), "v_codes is not 16-byte"), (dict(k_scales_ptr=A + 2), "k_scales is not 4-byte"),
         (dict(v_scales_ptr=0), "v_scales is null"), (dict(block_table_ptr=0), "block_table is null")]


def refused(host, call, text):
    with pytest.raises(host.EngineError, match="status 1:"):
        call()
    assert text in host.last_error(), host.last_error()


@pytest.mark.parametrize("name", ["kv8_append", "kv8_read"])
def test_rows_refusals(host, name):
    fn = getattr(host, name)
    good = dict(k_ptr=A, v_ptr=A if name == "kv8_append" else 2 * A, dtype=0, row_stride=256, n_rows=3, seqs_ptr=A, starts_ptr=A, offsets_ptr=A, n_segments=1)
    for kw, text in CACHE:
        refused(host, lambda: fn(cache(host, **kw), **good), text)
    for kw, text in [(dict(dtype=3), "dtype"), (dict(dtype=-1), "dtype"), (dict(row_stride=255), "row_stride"),
                     (dict(row_stride=257), "row_stride"), (dict(dtype=1, row_stride=260), "row_stride"), (dict(n_rows=-1), "n_rows"),
                     (dict(n_rows=1 << 40), "n_rows"), (dict(n_segments=-1), "n_segments"), (dict(k_ptr=0), "k is null"),
                     (dict(v_ptr=A + 4), "v is not 16-byte"), (dict(seqs_ptr=0), "seqs is null"),
                     (dict(starts_ptr=A + 1), "starts is not 4-byte"), (dict(offsets_ptr=0), "offsets is null")]:
        refused(host, lambda: fn(cache(host), **{**good, **kw}), text)
    if name == "kv8_read":
        refused(host, lambda: fn(cache(host), **{**good, "v_ptr": A}), "one buffer")
    fn(cache(host), **{**good, "n_rows": 0})  # nothing to do: no error, no GPU
    fn(cache(host), **{**good, "n_segments": 0})


def test_attention_refusals(host):
    good = dict(q_ptr=A, q_stride=1536, out_ptr=2 * A, out_stride=1536, dtype=0, n_rows=2, n_q_heads=12, row_seqs_ptr=A, row_lens_ptr=A,
                scale=0.1, workspace_ptr=A, workspace_bytes=1 << 30)
    for kw, text in CACHE:
        refused(host, lambda: host.kv8_attention(cache(host, **kw), **good), text)
    need = host.kv8_attention_workspace(2, 12, 2)
    for kw, text in [(dict(dtype=5), "dtype"), (dict(n_rows=-1), "n_rows"), (dict(n_q_heads=13, q_stride=1664, out_stride=1664), "multiple"),
                     (dict(n_q_heads=0), "n_q_heads"), (dict(q_stride=1535), "q_stride"), (dict(out_stride=1538), "out_stride"),
                     (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(workspace_bytes=need - 1), "workspace"),
                     (dict(workspace_ptr=0), "workspace is null"), (dict(workspace_ptr=A + 8), "workspace is not"),
                     (dict(out_ptr=A), "overlap"), (dict(q_ptr=0), "q is null"), (dict(out_ptr=A + 4), "out is not"),
                     (dict(row_seqs_ptr=0), "row_seqs is null"), (dict(row_lens_ptr=A + 2), "row_lens is not"),
                     (dict(lse_ptr=A + 1), "lse is not")]:
        refused(host, lambda: host.kv8_attention(cache(host), **{**good, **kw}), text)
    big = dict(n_rows=1 << 20, workspace_bytes=1 << 40)
    wide = dict(n_q_heads=64, q_stride=8192, out_stride=8192)
    refused(host, lambda: host.kv8_attention(cache(host, max_blocks=1 << 24), **{**good, **wide}), "n_q_heads * max_blocks")
    refused(host, lambda: host.kv8_attention(cache(host, max_blocks=1 << 16), **{**good, **big}), "n_rows * n_q_heads * max_blocks")
    host.kv8_attention(cache(host), **{**good, "n_rows": 0, "workspace_bytes": 0})
    for args in ((-1, 12, 2), (1, 0, 2), (1, 12, 0)):
        with pytest.raises(host.EngineError):
            host.kv8_attention_workspace(*args)


def test_sample_refusals(host):
    good = dict(logits_ptr=A, dtype=0, rows=2, vocab=100, row_stride=100, temperature_ptr=A, top_k_ptr=A, top_p_ptr=A, min_p_ptr=A,
                uniforms_ptr=A, tokens_ptr=A, probs_ptr=A)
    for kw, text in [(dict(dtype=3), "dtype"), (dict(rows=-1), "rows"), (dict(vocab=0), "vocab"),
                     (dict(vocab=262145, row_stride=1 << 20), "vocab"), (dict(row_stride=99), "row_stride"), (dict(logits_ptr=0), "logits"),
                     (dict(logits_ptr=A + 2), "logits is not 4-byte"), (dict(dtype=2, logits_ptr=A + 1), "logits is not 2-byte"),
                     (dict(uniforms_ptr=0), "uniforms is null"), (dict(tokens_ptr=0), "tokens is null"),
                     (dict(temperature_ptr=A + 1), "temperature"), (dict(top_k_ptr=A + 1), "top_k"), (dict(top_p_ptr=A + 1), "top_p"),
                     (dict(min_p_ptr=A + 1), "min_p"), (dict(probs_ptr=A + 1), "probs")]:
        refused(host, lambda: host.sample(**{**good, **kw}), text)
    host.sample(**{**good, "rows": 0})


def test_without_a_device_or_with_host_memory(host, gpu_available):
    """Sound arguments on a machine without a GPU: status 31 (host memory on one with a GPU: status 1); never computed."""
    x = np.zeros(8192, np.float32)
    p = x.ctypes.data // 16 * 16 + 16
    c = cache(host, k_codes_ptr=p, v_codes_ptr=p, k_scales_ptr=p, v_scales_ptr=p, block_table_ptr=p)
    want = "status 1:" if gpu_available else "status 31:"
    with pytest.raises(host.EngineError, match=want):
        host.kv8_append(c, p, p, 0, 256, 1, p, p, p, 1)
    with pytest.raises(host.EngineError, match=want):
        host.kv8_read(c, p, p + 4096, 0, 256, 1, p, p, p, 1)
    with pytest.raises(host.EngineError, match=want):
        host.kv8_attention(c, p, 1536, p + 16, 1536, 0, 1, 12, p, p, 0.1, p, 1 << 30)
    with pytest.raises(host.EngineError, match=want):
        host.sample(p, 0, 1, 10, 10, 0, 0, 0, 0, p, p)
    assert (x == 0).all()


def test_model_write_bound():
    """The model's codes keep the documented bounds, and a wrong growth rule would not."""
    r = np.random.RandomState(0)
    x = (r.randn(64, 1, 128) * np.exp(np.linspace(-3, 3, 64))[:, None, None]).astype(np.float32)
    table = np.zeros((1, 1), np.int64)
    blank = lambda: km.Model(np.zeros((1, 1, 64, 128)), np.zeros((1, 1), np.float32), table)  # noqa: E731
    whole, steps = blank(), blank()
    whole.append(x, 0, 0)
    for t in range(64):
        steps.append(x[t : t + 1], 0, t)
    s = whole.scales[0, 0]
    assert (np.abs(whole.values(0, 64) - x) <= s * (0.5 + 127 * 2.0**-23)).all()
    s = steps.scales[0, 0]
    assert whole.scales[0, 0] <= s < 2 * whole.scales[0, 0]
    assert (np.abs(steps.values(0, 64) - x) < s * (1 + 127 * 2.0**-23)).all()


def test_model_sampler():
    x = [1.0, 3.0, 2.0, 3.0]
    ids, w = km.kept(x)
    assert list(ids) == [1, 3, 2, 0]
    assert list(km.kept(x, top_k=3)[0]) == [1, 3, 2]
    assert list(km.kept(x, top_p=0.5)[0]) == [1, 3] and list(km.kept(x, top_p=0.39)[0]) == [1]  # shares .3995 .3995 .147 .054
    assert list(km.kept(x, min_p=0.3)[0]) == [1, 3, 2] and list(km.kept(x, min_p=0.4)[0]) == [1, 3]
    assert km.sample(x, 0.0)[0] == 1 and km.sample(x, 0.999)[0] == 0
    assert km.sample([-np.inf, np.nan], 0.5) == (-1, 0.0)


def test_rows_that_leave_a_setting_open(host):
    """None in a row: the value that turns the filter off, temperature 1 (a NaN would mean greedy)."""
    assert host._per_row(None, 1.0, np.float32) is None
    np.testing.assert_array_equal(host._per_row([None, 0.5, 0.0], 1.0, np.float32), np.float32([1.0, 0.5, 0.0]))
    np.testing.assert_array_equal(host._per_row((7, None), 0, np.int32), np.int32([7, 0]))
    np.testing.assert_array_equal(host._per_row(np.float32([0.25, 0.5]), 0.0, np.float32), np.float32([0.25, 0.5]))
