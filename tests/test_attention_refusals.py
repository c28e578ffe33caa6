"""What AttentionBatch, kv_append, paged_attention and norm_residual pass on to
the library and what they refuse, beyond test_attention_abi.py (CPU only)."""
import ctypes

import pytest
import torch

from test_attention_abi import call, lib


@pytest.fixture
def on_cpu(monkeypatch):
    """The handles take CPU tensors: nothing is launched."""
    import nvfp4.attention as A

    monkeypatch.setattr(A, "_check_device", lambda t, **others: None)
    return A


def test_page_table_stride_is_the_tables_own(on_cpu):
    """A table expanded to all sequences has one row in memory, and the library
    must not step beyond it."""
    i = lambda *x: torch.tensor(x, dtype=torch.int32)
    stride = lambda table, B: on_cpu.AttentionBatch(torch.ones(B, dtype=torch.int32), table)._c.page_table_stride
    assert stride(i(4, 2, 7).expand(5, -1), 5) == 0
    assert stride(torch.zeros(5, 3, dtype=torch.int32), 5) == 3
    assert stride(torch.zeros(5, 8, dtype=torch.int32)[:, :3], 5) == 8
    assert stride(torch.zeros(5, 3, dtype=torch.int32)[:1].as_strided((1, 3), (1, 1)), 1) >= 3
    assert stride(torch.zeros(5, 0, dtype=torch.int32), 5) >= 0
    with pytest.raises(ValueError, match="overlap"):
        stride(torch.zeros(20, dtype=torch.int32).as_strided((5, 6), (2, 1)), 5)


def test_library_takes_one_table_row_for_all_sequences():
    _lib, _ = lib()
    for over in (dict(stride=0), dict(stride=0, B=1, T=1), dict(stride=2, B=1, T=1)):
        rc, msg = call(ws=None, **over)  # the table passes; the workspace is the next complaint
        assert rc == _lib.NVFP4_ERR_INVALID_ARG and "workspace" in msg, msg
    for stride in (-3, 1, 2):
        rc, msg = call(stride=stride)
        assert rc == _lib.NVFP4_ERR_INVALID_ARG and "page_table" in msg, msg
