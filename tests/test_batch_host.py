"""CPU tests of the batched-decode operators' host side: workspace sizes and
refusals that need no GPU."""
import ctypes

import pytest
import torch

import lalmodel_b200 as lb
from lalmodel_b200 import _abi


def test_batch_ws_bytes_host_only():
    """Workspace sizes and shape checks of the batched-decode operators need no device."""
    L, n = _abi.lib(), ctypes.c_size_t()

    def cache(dtype=0, n_seq=2, max_ctx=64, n_kv=2, hd=64):
        return ctypes.byref(_abi.KVBatchDesc(dtype, n_seq, max_ctx, n_kv, hd, None, None, None, None))

    def attn(n_head=4, prefix=0):
        return ctypes.byref(_abi.AttnBatchDesc(n_head, 0.0, prefix, None, None, 0, 0.0))

    assert L.lalb_attention_batch_ws_bytes(cache(), attn(), ctypes.byref(n)) == 0 and n.value > 0
    assert L.lalb_kv_evict_ws_bytes(cache(), 32, ctypes.byref(n)) == 0 and n.value >= 4 * 4 + 2 * 4 * 32 * 4
    for bad in (dict(dtype=1), dict(dtype=9), dict(hd=48), dict(n_seq=1 << 20, max_ctx=1 << 12)):
        assert L.lalb_attention_batch_ws_bytes(cache(**bad), attn(), ctypes.byref(n)) == -4
        assert L.lalb_kv_evict_ws_bytes(cache(**bad), 1, ctypes.byref(n)) == -4
    for bad in (dict(n_seq=0), dict(max_ctx=-1), dict(n_kv=0)):
        assert L.lalb_attention_batch_ws_bytes(cache(**bad), attn(), ctypes.byref(n)) == -1
        assert L.lalb_kv_evict_ws_bytes(cache(**bad), 1, ctypes.byref(n)) == -1
    for bad in (dict(n_head=3), dict(n_head=0), dict(prefix=-1)):
        assert L.lalb_attention_batch_ws_bytes(cache(), attn(**bad), ctypes.byref(n)) == -1
    # more rows, query rows or tiles than 31-bit indices hold
    for bad in (dict(n_seq=1, max_ctx=2 ** 31 - 1), dict(n_seq=1, max_ctx=2 ** 30 + 1)):
        assert L.lalb_attention_batch_ws_bytes(cache(**bad), attn(), ctypes.byref(n)) == -4
    assert L.lalb_attention_batch_ws_bytes(cache(), attn(prefix=2 ** 31 - 1), ctypes.byref(n)) == -4
    assert L.lalb_attention_batch_ws_bytes(cache(n_seq=70000, max_ctx=8), attn(), ctypes.byref(n)) == -4
    for keep in (0, 65):
        assert L.lalb_kv_evict_ws_bytes(cache(), keep, ctypes.byref(n)) == -1
    assert L.lalb_kv_evict_ws_bytes(cache(), 8, None) == -1
    assert L.lalb_rope_append(None, None, None, 1, None, 0, 0, 1, None, None, None, None) == -1
    assert L.lalb_attention_batch(None, None, None, None, 0, None, None, None, None) == -1


def test_batch_python_refusals_need_no_device():
    with pytest.raises(lb.LalbError):
        lb.KVBatch(torch.zeros(2, 4, 64, dtype=torch.float64), torch.zeros(2, 4, 64, dtype=torch.float64), 1)
    with pytest.raises(lb.LalbError):
        lb.KVBatch(torch.zeros(2, 4, 64), torch.zeros(2, 4, 32), 1)
    with pytest.raises(lb.LalbError):
        lb.KVBatch(torch.zeros(2, 4, 64), torch.zeros(2, 4, 64), 3)
    with pytest.raises(lb.LalbError):
        lb.KVBatch(torch.zeros(2, 4, 64), torch.zeros(2, 4, 64), 1, row_weight=torch.zeros(2, 1, 3))
    with pytest.raises(lb.LalbError):
        lb.Rope(scaling="quadratic")


def test_a_cache_keeps_its_tensors():
    """Calls use the tensors' addresses as they were at first: another tensor in
    their place would leave calls on memory that is given back."""
    k = torch.zeros(2, 4, 64)
    cache = lb.KVBatch(k, k.clone(), 1)
    assert cache.k is k and cache.row_pos is None
    for name in ("k", "v", "row_pos", "row_weight"):
        with pytest.raises(AttributeError):
            setattr(cache, name, torch.zeros(2, 4, 64))
