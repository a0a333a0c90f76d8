"""What the cache and scoring operators refuse, at the C ABI and in Python, before any device work."""
import ctypes

import pytest
import torch


def batch(p, **changes):
    from dscquant_b200 import _lib

    fields = dict(k_codes=p, k_affine=p, v_codes=p, v_affine=p, pages=4, kv_heads=2, page_size=64, head_dim=128,
                  dtype=_lib.BF16, page_table=p, ld_table=3, max_pages=3, q_start=p, lengths=p, seqs=2)
    fields.update(changes)
    return _lib.KV4_BATCH.pack(*(v or 0 for v in fields.values()))


@pytest.fixture
def buf():
    raw = ctypes.create_string_buffer(4096 + 16)
    at = (ctypes.addressof(raw) + 15) // 16 * 16
    yield at
    del raw


@pytest.mark.parametrize("changes,word", [
    (dict(k_codes=None), "null"), (dict(head_dim=96), "head_dim"), (dict(dtype=2), "bf16 or f16"),
    (dict(page_size=48), "page_size"), (dict(page_size=8), "page_size"), (dict(page_size=2048), "page_size"),
    (dict(kv_heads=0), "kv_heads"), (dict(pages=0), "pages"), (dict(pages=1 << 31), "pages"), (dict(seqs=-1), "sequences"),
    (dict(page_table=None), "null"), (dict(lengths=None), "null"), (dict(ld_table=2), "ld_table"),
    (dict(max_pages=1 << 26, ld_table=1 << 26), "max_pages")])
def test_batch_refusals(native, buf, changes, word):
    from dscquant_b200 import _lib

    b = batch(buf, **changes)
    for rc in (native.dscq_kv4_append(b, buf, 256, 128, buf, 256, 128, buf, 256, 128, 1, 2, buf, buf, 0, 10, buf, None),
               native.dscq_kv4_read(b, 1, buf, buf, None),
               native.dscq_kv4_attention(b, buf, 256, 128, 1, 2, 1, 1.0, buf, buf, 1 << 30, None)):
        assert rc == _lib.DSCQ_ERR_INVALID and word in _lib.last_error()


def test_misaligned_cache(native, buf):
    from dscquant_b200 import _lib

    assert native.dscq_kv4_read(batch(buf, v_codes=buf + 8), 1, buf, buf, None) == _lib.DSCQ_ERR_INVALID
    assert "aligned" in _lib.last_error()


def test_append_refusals(native, buf):
    from dscquant_b200 import _lib

    b = batch(buf)
    good = dict(q=buf, qt=256, qh=128, k=buf, kt=256, kh=128, v=buf, vt=256, vh=128, T=1, hq=2, cos=buf, sin=buf, td=0,
                rows=10, out=buf)
    for change, word in ((dict(hq=0), "q_heads"), (dict(td=1), "cos / sin"), (dict(rows=-1), "table rows"),
                         (dict(q=None), "q, k, v"), (dict(qt=257), "multiples"), (dict(kh=4), "multiples"),
                         (dict(v=buf + 2), "aligned"), (dict(out=None), "q_out"), (dict(cos=None), "cos"),
                         (dict(sin=buf + 4), "sin"), (dict(T=-1), "T"), (dict(T=1 << 31), "T")):
        a = {**good, **change}
        rc = native.dscq_kv4_append(b, *a.values(), None)
        assert rc == _lib.DSCQ_ERR_INVALID and word in _lib.last_error(), change
    assert native.dscq_kv4_append(None, *good.values(), None) == _lib.DSCQ_ERR_INVALID
    assert native.dscq_kv4_append(b, *{**good, "T": 0}.values(), None) == _lib.DSCQ_OK  # nothing to do


def test_attention_refusals(native, buf):
    from dscquant_b200 import _lib

    b = batch(buf)
    good = dict(q=buf, qt=256, qh=128, T=1, hq=2, max_q=1, scale=1.0, out=buf, ws=buf, bytes=1 << 30)
    for change, word in ((dict(hq=3), "multiple of kv_heads"), (dict(hq=0), "q_heads"), (dict(scale=float("nan")), "scale"),
                         (dict(scale=float("inf")), "scale"), (dict(q=None), "q and out"), (dict(qt=250), "multiples"),
                         (dict(out=buf + 8), "aligned"), (dict(max_q=-1), "max_q"), (dict(ws=None), "workspace"),
                         (dict(ws=buf + 4), "workspace")):
        rc = native.dscq_kv4_attention(b, *{**good, **change}.values(), None)
        assert rc == _lib.DSCQ_ERR_INVALID and word in _lib.last_error(), change
    assert native.dscq_kv4_attention(b, *{**good, "T": 0}.values(), None) == _lib.DSCQ_OK


def test_logprob_refusals(native, buf):
    from dscquant_b200 import _lib

    good = dict(x=buf, dt=0, rows=1, V=100, ld=100, t=buf, k=3, lp=buf, h=buf, top=buf, ids=buf)
    for change, word in ((dict(dt=3), "bf16, f16 or f32"), (dict(rows=-1), "rows"), (dict(V=0), "V"), (dict(ld=99), "ld"),
                         (dict(V=(1 << 24) + 1, ld=1 << 25), "V"), (dict(k=-1), "k"), (dict(k=65), "k"),
                         (dict(V=2, k=3), "k"), (dict(x=None), "null"), (dict(t=None), "null"), (dict(ids=None), "null"),
                         (dict(x=buf + 1), "aligned"), (dict(dt=2, x=buf + 2), "aligned")):
        rc = native.dscq_token_logprobs(*{**good, **change}.values(), None)
        assert rc == _lib.DSCQ_ERR_INVALID and word in _lib.last_error(), change
    assert native.dscq_token_logprobs(*{**good, "rows": 0}.values(), None) == _lib.DSCQ_OK


def test_valid_calls_without_gpu_fail_cleanly(native, buf):
    if torch.cuda.is_available():
        pytest.skip("GPU present")
    from dscquant_b200 import _lib

    b = batch(buf)
    failed = (_lib.DSCQ_ERR_CUDA, _lib.DSCQ_ERR_UNSUPPORTED)
    assert native.dscq_kv4_read(b, 1, buf, buf, None) in failed
    assert native.dscq_kv4_attention(b, buf, 256, 128, 1, 2, 1, 1.0, buf, buf, 1 << 30, None) in failed
    assert native.dscq_token_logprobs(buf, 0, 1, 10, 10, buf, 0, buf, buf, None, None, None) in failed


def test_cpu_tensors_are_refused():
    from dscquant_b200 import PagedKV4, ops

    with pytest.raises(RuntimeError, match="CUDA"):
        PagedKV4.allocate(4, 2, 128, 64, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.token_logprobs(torch.zeros(2, 10), torch.zeros(2, dtype=torch.int64))
    for bad in (dict(head_dim=96), dict(page_size=24), dict(page_size=8), dict(dtype=torch.float32)):
        with pytest.raises(RuntimeError):
            PagedKV4.allocate(**{**dict(pages=4, kv_heads=2, head_dim=128, device="cpu"), **bad})
