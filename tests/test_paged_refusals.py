"""What the paged cache's entry points refuse, before any device work (no GPU needed; dummy addresses, never read)."""

import ctypes

import pytest
import torch

from pollux_amd import _lib
from pollux_amd.paged import PagedBatch, PagedKV

A, B, C = 0x10000, 0x20000, 0x30000


def _kv(**change):
    f = dict(k=A, v=B, k_scale=A, v_scale=B, pages=10, heads=3, page_size=16, kv_type=_lib.KV_INT8)
    f.update(change)
    return _lib.PagedKVStruct(**f)


def _batch(**change):
    f = dict(table=A, table_stride=4, seqs=2, cu_q=B, kv_len=C, tokens=9, max_q=8, max_kv=64, singles=1)
    f.update(change)
    return _lib.PagedBatchStruct(**f)


def _all(kv, batch, message):
    lib = _lib.lib()
    k, b = ctypes.byref(kv), ctypes.byref(batch)
    for st in (lib.plx_paged_write(k, b, A, B, 0, 0, None, 0.0, None), lib.plx_paged_read(k, b, A, B, None),
               lib.plx_paged_attention(k, b, A, 0, 0, None, 0.0, B, C, 1 << 30, None)):
        assert st == _lib.PLX_EINVAL and message in lib.plx_last_error().decode()
    assert lib.plx_paged_attention_workspace_bytes(k, b) == 0


@pytest.mark.parametrize("change,message", [
    ({"kv_type": 3}, "unknown cache type"), ({"kv_type": -1}, "unknown cache type"), ({"pages": 0}, "pages"),
    ({"heads": 0}, "heads"), ({"heads": 70_000}, "heads"), ({"page_size": 24}, "power of two"),
    ({"page_size": 4}, "power of two"), ({"page_size": 8192}, "power of two"), ({"k": None}, "null"),
    ({"k_scale": None}, "scales"), ({"v_scale": None}, "scales"), ({"kv_type": _lib.KV_F16}, "scales"),
    ({"v": B + 8}, "aligned"), ({"k_scale": A + 4}, "aligned")])
def test_caches(change, message):
    _all(_kv(**change), _batch(), message)


@pytest.mark.parametrize("change,message", [
    ({"seqs": -1}, "sequences"), ({"tokens": -1}, "sequences"), ({"max_q": 10}, "new tokens"), ({"max_q": -1}, "new"),
    ({"max_kv": 65}, "does not hold"), ({"table_stride": -1}, "does not hold"), ({"max_kv": -1}, "does not hold"),
    ({"singles": 3}, "one-token"), ({"cu_q": None}, "null"), ({"kv_len": None}, "null"), ({"table": None}, "null")])
def test_batches(change, message):
    _all(_kv(), _batch(**change), message)


def test_largest():
    lib = _lib.lib()
    _all(_kv(), _batch(tokens=(1 << 30) + 1), "tokens")
    _all(_kv(), _batch(table_stride=1 << 62), "does not hold")  # (its product with the page size leaves 64 bits)
    _all(_kv(heads=65_535), _batch(seqs=40_000), "heads")
    kv, batch = ctypes.byref(_kv(heads=480)), ctypes.byref(_batch(seqs=60_000, tokens=1 << 30, max_q=1 << 20, singles=0))
    need = lib.plx_paged_attention_workspace_bytes(kv, batch)
    for st in (lib.plx_paged_write(kv, batch, A, B, 0, 0, None, 0.0, None), lib.plx_paged_read(kv, batch, A, B, None),
               lib.plx_paged_attention(kv, batch, A, 0, 0, None, 0.0, B, C, need, None)):
        assert st == _lib.PLX_EINVAL and "too many" in lib.plx_last_error().decode()


def test_rows_and_workspace():
    lib = _lib.lib()
    k, b = ctypes.byref(_kv()), ctypes.byref(_batch())

    def write(kp=A, vp=B, x_type=0, stride=0, norm=None):
        return lib.plx_paged_write(k, b, kp, vp, x_type, stride, norm, 0.0, None)

    for call, message in ((lambda: write(x_type=3), "dtype"), (lambda: write(stride=64), "apart"),
                          (lambda: write(stride=76), "apart"), (lambda: write(kp=A + 8), "aligned"),
                          (lambda: write(vp=None), "null"), (lambda: write(norm=A + 2), "norm weight"),
                          (lambda: lib.plx_paged_read(k, b, A, None, None), "null"),
                          (lambda: lib.plx_paged_read(k, b, A, B + 4, None), "aligned"),
                          (lambda: lib.plx_paged_attention(k, b, None, 0, 0, None, 0.0, B, C, 0, None), "null"),
                          (lambda: lib.plx_paged_attention(k, b, A, 0, 0, None, 0.0, B + 4, C, 0, None), "aligned")):
        assert call() == _lib.PLX_EINVAL and message in lib.plx_last_error().decode()
    # one long sequence is split over its keys: the states need room
    kv, long = _kv(), _batch(seqs=1, tokens=1, max_q=1, max_kv=1 << 16, table_stride=1 << 12, singles=0)
    k, b = ctypes.byref(kv), ctypes.byref(long)
    need = lib.plx_paged_attention_workspace_bytes(k, b)
    assert need > 0
    for ws, size in ((C, need - 1), (None, need), (C + 4, need)):
        assert lib.plx_paged_attention(k, b, A, 0, 0, None, 0.0, B, ws, size, None) == _lib.PLX_EINVAL
        assert "workspace" in lib.plx_last_error().decode()


def test_null_structures_and_nothing_to_do():
    lib = _lib.lib()
    kv, batch = ctypes.byref(_kv()), ctypes.byref(_batch())
    assert lib.plx_paged_read(None, batch, A, B, None) == _lib.PLX_EINVAL
    assert lib.plx_paged_write(kv, None, A, B, 0, 0, None, 0.0, None) == _lib.PLX_EINVAL
    for empty in (_batch(seqs=0, singles=0), _batch(max_q=0, tokens=0)):
        b = ctypes.byref(empty)
        assert lib.plx_paged_attention(kv, b, None, 0, 0, None, 0.0, None, None, 0, None) == _lib.PLX_OK
        assert lib.plx_paged_write(kv, b, None, None, 0, 0, None, 0.0, None) == _lib.PLX_OK


def test_python_checks():
    k = torch.zeros(2, 3, 16, 24)
    with pytest.raises(ValueError, match="ROCm device"):
        PagedKV(k, k.clone())
    for bad in (torch.zeros(2, 3, 16, 23), torch.zeros(2, 3, 16, 24, dtype=torch.bfloat16), torch.zeros(3, 16, 24)):
        with pytest.raises(ValueError, match="float32, float16 or int8"):
            PagedKV(bad, bad)
    with pytest.raises(ValueError, match="power of two"):
        PagedKV(torch.zeros(2, 3, 12, 24), torch.zeros(2, 3, 12, 24))
    with pytest.raises(ValueError, match="both scales"):
        PagedKV(k.to(torch.int8), k.to(torch.int8))
    with pytest.raises(ValueError, match="both scales"):
        PagedKV(k, k, k[..., 0], None)
    with pytest.raises(ValueError, match="per sequence"):
        PagedBatch.build([[0]], [3, 4], [1, 1], "cpu")
    with pytest.raises(ValueError, match="negative"):
        PagedBatch.build([[0]], [3], [-1], "cpu")
    with pytest.raises(ValueError, match="ROCm device"):
        PagedBatch.build([[0]], [3], [1], "cpu")


def test_short_page_lists_end_in_no_page(monkeypatch):
    # (0 is a page, another sequence's)
    monkeypatch.setattr(_lib, "require_device", lambda t, what: None)
    batch = PagedBatch.build([[5, 0, 2], [3], []], [40, 40, 0], [1, 1, 0], "cpu")
    assert batch.table.tolist() == [[5, 0, 2], [3, -1, -1], [-1, -1, -1]]
    given = torch.tensor([[5, 0], [3, 0]])
    assert PagedBatch.build(given, [20, 9], [1, 1]).table.tolist() == [[5, 0], [3, 0]]
