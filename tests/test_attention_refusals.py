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


def spans(which, q, out, T, H, D=128, **over):
    """paged_attention's or kv_append's word on q at `q` and out (q_out) at
    `out`, each (address, token stride, head stride) in elements of 2 bytes."""
    _lib, L = lib()
    s3, r = ctypes.c_int64 * 3, ctypes.byref
    rows = lambda x: _lib.HeadRows(*x)
    big = 1 << 40  # far from every row
    cache = _lib.KvCache(big, over.get("v_cache", big + (1 << 30)), s3(65536, 256, 128), s3(65536, 256, 128), 4, 16, 2, D)
    b = _lib.AttnBatch(T, 1, T, None, 64, 64, 3, 3, 0, None, None)
    if which == "attention":
        d = _lib.AttnDesc(H, 2, D, 1, 0, 0.1, 0.0)
        gate = over.get("gate")
        rc = L.nvfp4_paged_attention(r(d), r(rows(q)), r(cache), r(b), None, None if gate is None else r(rows(gate)),
                                     r(rows(out)), over.get("lse"), None, 0, None)
    else:
        k = over.get("k", (big + (1 << 32), 256, 128))
        rc = L.nvfp4_kv_append(r(cache), r(b), None, None, r(rows(q)), r(rows(k)), r(rows(k)),
                               over.get("dtype", _lib.DTYPE_BF16), H, None, 0, 1, r(rows(out)), None)
    return rc, L.nvfp4_last_error_string().decode()


A = 1 << 20


# T = 4 tokens of H = 8 heads of 128: 256 bytes a row.
@pytest.mark.parametrize("which", ["attention", "append"])
@pytest.mark.parametrize("out", [
    (A, 0, 128), (A, 1024, 0), (A, 1024, 64), (A, 512, 128), (A, 128, 128),   # rows on rows
    (A + (1 << 24), 1024, 120), (A + (1 << 24), 1016, 128), (A + (1 << 24), 0, 128),  # also far from q
    (A + 256, 1024, 128), (A - 256, 1024, 128), (A + 2048, 1024, 128), (A + 16, 1024, 128),  # q, shifted
    (A + 6144, 1024, 128), (A + 8176, 1024, 128), (A - 8176, 1024, 128), (A + 2048, 2048, 128)])
def test_rows_that_overlap_are_refused(which, out):
    _lib, _ = lib()
    rc, msg = spans(which, (A, 1024, 128), out, 4, 8)
    assert rc == _lib.NVFP4_ERR_INVALID_ARG and ("overlap" in msg or "another" in msg), msg


@pytest.mark.parametrize("q,out", [
    ((A, 1024, 128), (A, 1024, 128)),                    # in place
    ((A, 1024, 128), (A + 8192, 1024, 128)), ((A + 8192, 1024, 128), (A, 1024, 128)),  # behind each other
    ((A, 2048, 256), (A + 256, 2048, 256)),              # the halves of [T, H, 2, D]
    ((A, 2048, 128), (A + 2048, 2048, 128)),             # of [T, 2 H, D]
    ((A, 4096, 256), (A + 4096, 4096, 128)),             # [T, H, 2, D] beside [T, H, D]
    ((A, 128, 512), (A + 8192, 1024, 128))])             # head by head
def test_rows_that_do_not_overlap_are_taken(q, out):
    _lib, _ = lib()
    rc, msg = spans("attention", q, out, 4, 8)
    assert "workspace" in msg, msg  # which is missing: the last check
    rc, msg = spans("append", q, out, 4, 8, v_cache=1 << 40)
    assert "cache" in msg, msg  # keys and values in one place: the last check


def test_other_operands_overlaps_are_refused():
    _lib, _ = lib()
    q, out = (A, 1024, 128), (A + (1 << 20), 1024, 128)
    gate = lambda by: (out[0] + by, 1024, 128)
    for over, word in ((dict(gate=gate(0)), "workspace"), (dict(gate=gate(8192)), "workspace"),
                       (dict(gate=gate(2048)), "gate"), (dict(gate=(out[0], 2048, 128)), "gate"),
                       (dict(lse=out[0] + 512), "lse"), (dict(lse=q[0] - 64), "lse"), (dict(lse=q[0] - 128), "workspace")):
        rc, msg = spans("attention", q, out, 4, 8, **over)
        assert rc == _lib.NVFP4_ERR_INVALID_ARG and word in msg, (over, msg)
    for over in (dict(k=(out[0] + 2048, 256, 128)), dict(k=(out[0], 1024, 128)), dict(k=(out[0] + 8000, 256, 128))):
        rc, msg = spans("append", q, out, 4, 8, **over)
        assert rc == _lib.NVFP4_ERR_INVALID_ARG and "k, v" in msg, (over, msg)
    # Parts of one projection [T, 12, 128], q turned in place.
    wide = lambda at: (A + 256 * at, 12 * 128, 128)
    assert "cache" in spans("append", wide(0), wide(0), 4, 8, k=wide(8), v_cache=1 << 40)[1]
    assert "k, v" in spans("append", wide(0), wide(0), 4, 8, k=wide(7))[1]
    # fp32 q under a bf16 q_out.
    assert "q_out" in spans("append", (A, 1024, 128), (A + 4096, 1024, 128), 4, 8, dtype=_lib.DTYPE_F32)[1]


def norm_word(rows, hidden, x, res=None, gate=None, ro=None, y=None, xd=1, rd=1, yd=1, gc=1):
    """norm_residual's word; x, res, gate, ro and y as (address, row stride)."""
    _lib, L = lib()
    at = lambda t: (None, 0) if t is None else t
    d = _lib.NormDesc(rows, hidden, xd, rd, yd, 1, 1.0, 1e-6, 0.0, at(x)[1], at(res)[1], at(ro)[1], at(y)[1],
                      at(gate)[1], gc)
    rc = L.nvfp4_norm_residual(ctypes.byref(d), at(x)[0], at(res)[0], None, at(gate)[0], 64 if y else None,
                               at(ro)[0], at(y)[0], None)
    assert rc == _lib.NVFP4_ERR_INVALID_ARG
    return L.nvfp4_last_error_string().decode()


def test_norm_outputs_that_overlap_are_refused():
    far = (1 << 30, 64)
    for kw in (dict(ro=(A + 128, 64)), dict(ro=(A - 128, 64)), dict(y=(A + 256, 64), ro=far), dict(ro=(A + 2, 64)),
               dict(res=far, ro=(far[0] + 128, 64)), dict(res=far, y=(far[0] - 128, 64), ro=(1 << 29, 64)),
               dict(gate=far, ro=(far[0] + 128, 64)), dict(gate=(far[0], 0), ro=far), dict(gate=(far[0] + 2, 64), ro=far, gc=0),
               dict(ro=far, y=(far[0] + 128, 64)), dict(ro=far, rd=0, y=(far[0] + 64, 64))):
        assert "overlap" in norm_word(8, 64, (A, 64), **kw), kw


@pytest.mark.parametrize("name", ["num_heads", "num_kv_heads", "head_dim", "window"])
@pytest.mark.parametrize("by", [2 ** 31, 2 ** 32, -2 ** 32])
def test_whole_numbers_that_do_not_fit_are_refused(name, by):
    """ctypes would pass on their low 32 bits, which may be an ordinary number."""
    import nvfp4

    good = dict(num_heads=8, num_kv_heads=2, head_dim=128, window=16)
    nvfp4.AttentionConfig(**good)
    with pytest.raises(ValueError, match=name):
        nvfp4.AttentionConfig(**{**good, name: good[name] + by})


def test_lengths_that_do_not_fit_are_refused(on_cpu):
    i = lambda *x: torch.tensor(x, dtype=torch.int32)
    make = lambda **kw: on_cpu.AttentionBatch(i(9, 9), torch.zeros(2, 4, dtype=torch.int32), q_start=i(0, 4, 9),
                                              num_tokens=9, **kw)
    make(max_q_len=5, prefix_len=3, prefix_pages=i(1))
    with pytest.raises(ValueError, match="max_q_len"):
        make(max_q_len=2 ** 32 + 5)
    with pytest.raises(ValueError, match="prefix_len"):
        make(max_q_len=5, prefix_len=2 ** 32 + 3, prefix_pages=i(1))


def test_norm_rows_that_do_not_fit_are_refused():
    import nvfp4

    for hidden in (32769, 2 ** 32 + 8):
        with pytest.raises(ValueError, match="hidden"):
            nvfp4.norm_residual(torch.empty(1, hidden, dtype=torch.bfloat16, device="meta"))
