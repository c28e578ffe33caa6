"""kv_append, paged_attention and norm_residual refuse bad calls on the host,
before any CUDA work (CPU only), and the ctypes structs match the headers."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parents[1]


def lib():
    from nvfp4 import _lib

    return _lib, _lib.load()


def test_struct_layouts(tmp_path):
    _lib, _ = lib()
    names = {"nvfp4_head_rows": _lib.HeadRows, "nvfp4_kv_cache": _lib.KvCache,
             "nvfp4_attention_batch": _lib.AttnBatch, "nvfp4_rotary": _lib.RotaryDesc,
             "nvfp4_qk_norm": _lib.QkNorm, "nvfp4_attention_desc": _lib.AttnDesc,
             "nvfp4_norm_desc": _lib.NormDesc}
    lines = []
    for c, t in names.items():
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f} %zu\\n", offsetof({c}, {f}));' for f, *_ in t._fields_]
    src = tmp_path / "s.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "nvfp4_attention.h"\n'
                   '#include "nvfp4_norm.h"\nint main(void) {' + "".join(lines) + "return 0; }\n")
    exe = tmp_path / "s"
    subprocess.run(["gcc", "-std=c99", "-I", str(ROOT / "include"), str(src), "-o", str(exe)], check=True)
    got = dict(l.rsplit(" ", 1) for l in subprocess.run([str(exe)], check=True, capture_output=True,
                                                        text=True).stdout.splitlines())
    for c, t in names.items():
        assert int(got[c]) == ctypes.sizeof(t), c
        for f, *_ in t._fields_:
            assert int(got[f"{c}.{f}"]) == getattr(t, f).offset, (c, f)


def call(**over):
    """A paged_attention call with plausible addresses and `over` changed."""
    _lib, L = lib()
    s3 = ctypes.c_int64 * 3
    v = dict(H=8, KV=2, D=128, page=16, pages=4, B=2, T=2, q_start=None, kv_len=4096, table=4096, stride=3, max_pages=3,
             max_q=1, prefix=0, prefix_pages=None, scale=0.1, softcap=0.0, window=0, q=4096, out=8192, qts=1024,
             qhs=128, ks=(4096, 256, 128), k=4096, ws=4096, ws_bytes=1 << 40, cKV=None, cD=None)
    v.update(over)
    cache = _lib.KvCache(v["k"], 4096, s3(*v["ks"]), s3(*v["ks"]), v["pages"], v["page"],
                         v["cKV"] or v["KV"], v["cD"] or v["D"])
    b = _lib.AttnBatch(v["B"], v["max_q"], v["T"], v["q_start"], v["kv_len"], v["table"], v["stride"], v["max_pages"],
                       v["prefix"], v["prefix_pages"], None)
    d = _lib.AttnDesc(v["H"], v["KV"], v["D"], 1, v["window"], v["scale"], v["softcap"])
    q, o = _lib.HeadRows(v["q"], v["qts"], v["qhs"]), _lib.HeadRows(v["out"], 1024, 128)
    r = ctypes.byref
    rc = L.nvfp4_paged_attention(r(d), r(q), r(cache), r(b), None, None, r(o), None, v["ws"], v["ws_bytes"], None)
    return rc, L.nvfp4_last_error_string().decode()


@pytest.mark.parametrize("over,status,word", [
    (dict(H=9), "INVALID_ARG", "multiple"), (dict(H=0), "INVALID_ARG", "multiple"),
    (dict(H=258, KV=2), "UNSUPPORTED", "128"), (dict(D=100), "UNSUPPORTED", "head_dim"),
    (dict(D=264), "UNSUPPORTED", "head_dim"), (dict(page=48), "UNSUPPORTED", "page_size"),
    (dict(page=8), "UNSUPPORTED", "page_size"), (dict(page=512), "UNSUPPORTED", "page_size"),
    (dict(scale=0.0), "INVALID_ARG", "scale"), (dict(scale=float("nan")), "INVALID_ARG", "scale"),
    (dict(softcap=-1.0), "INVALID_ARG", "softcap"), (dict(window=-1), "INVALID_ARG", "window"),
    (dict(cKV=4), "INVALID_ARG", "cache has"), (dict(pages=0), "INVALID_ARG", "pages"),
    (dict(k=None), "INVALID_ARG", "null"), (dict(k=4104), "INVALID_ARG", "aligned"),
    (dict(ks=(4096, 252, 128)), "INVALID_ARG", "strides"), (dict(ks=(4096, 0, 128)), "INVALID_ARG", "strides"),
    (dict(T=3), "INVALID_ARG", "one token"), (dict(T=3, q_start=64, max_q=0), "INVALID_ARG", "max_q_len"),
    (dict(B=-1), "INVALID_ARG", "batch"), (dict(kv_len=None), "INVALID_ARG", "kv_len"),
    (dict(table=None), "INVALID_ARG", "page_table"), (dict(stride=2), "INVALID_ARG", "page_table"),
    (dict(prefix=5), "INVALID_ARG", "prefix_pages"), (dict(prefix=-5), "INVALID_ARG", "lengths"),
    (dict(max_pages=1 << 27, stride=1 << 27), "INVALID_ARG", "lengths"),
    (dict(T=1 << 22, q_start=64, max_q=1 << 22, max_pages=1 << 24, stride=1 << 24), "UNSUPPORTED", "tokens against"),
    (dict(q=None), "INVALID_ARG", "null"), (dict(q=4100), "INVALID_ARG", "aligned"),
    (dict(qhs=4), "INVALID_ARG", "strides"), (dict(out=4096, qts=2048), "INVALID_ARG", "another stride"),
    (dict(ws=None), "INVALID_ARG", "workspace"), (dict(ws=4100), "INVALID_ARG", "workspace"),
    (dict(ws_bytes=1000), "WORKSPACE", "needed")])
def test_paged_attention_refuses(over, status, word):
    _lib, _ = lib()
    rc, msg = call(**over)
    assert rc == getattr(_lib, "NVFP4_ERR_" + status) and word in msg, (rc, msg)


def test_calls_without_work_are_accepted():
    assert call(B=0, T=0, kv_len=None, table=None)[0] == 0
    assert call(T=0, q_start=64, max_q=0, q=None, out=None, ws=None)[0] == 0


def test_workspace_size_grows_with_the_call():
    _lib, L = lib()

    def size(T, max_q, prefix, D=128):
        b = _lib.AttnBatch(4, max_q, T, 64, 64, 64, 4, 4, prefix, 64, None)
        return L.nvfp4_attention_workspace_size(ctypes.byref(_lib.AttnDesc(8, 2, D, 1, 0, 0.1, 0.0)), ctypes.byref(b))

    assert 0 < size(4, 1, 0) <= size(4, 1, 7) <= size(64, 16, 7)
    assert size(4, 1, 0, D=100) == 0


def append(**over):
    _lib, L = lib()
    s3 = ctypes.c_int64 * 3
    v = dict(D=128, rotary=128, inv=64, dtype=1, H=8, pos=None, pstride=0, axes=1, q=4096, qo=8192, qts=1024, eps=1e-6,
             T=2)
    v.update(over)
    cache = _lib.KvCache(4096, 4096, s3(4096, 256, 128), s3(4096, 256, 128), 4, 16, 2, v["D"])
    b = _lib.AttnBatch(v["T"], 1, v["T"], None, 64, 64, 3, 3, 0, None, None)
    rot, norm = _lib.RotaryDesc(v["inv"], None, v["rotary"], 0, 1.0), _lib.QkNorm(64, 64, v["eps"], 0.0)
    rows = lambda p, s=1024: _lib.HeadRows(p, s, 128)
    r = ctypes.byref
    rc = L.nvfp4_kv_append(r(cache), r(b), r(rot), r(norm), r(rows(v["q"], v["qts"])), r(rows(4096)), r(rows(4096)),
                           v["dtype"], v["H"], v["pos"], v["pstride"], v["axes"], r(rows(v["qo"])), None)
    return rc, L.nvfp4_last_error_string().decode()


@pytest.mark.parametrize("over,word", [
    (dict(rotary=130), "rotary_dim"), (dict(rotary=7), "rotary_dim"), (dict(rotary=0), "rotary_dim"),
    (dict(inv=None), "rotary_dim"), (dict(dtype=2), "dtype"), (dict(H=0), "num_heads"), (dict(q=None), "null"),
    (dict(qo=None), "null"), (dict(pos=64, axes=0), "positions"), (dict(pos=64, axes=3, pstride=1), "positions"),
    (dict(qo=4096, dtype=0), "q_out is q"), (dict(qo=4096, qts=4096), "q_out is q"), (dict(eps=-1.0), "eps"),
    (dict(D=12), "head_dim")])
def test_kv_append_refuses(over, word):
    rc, msg = append(**over)
    assert rc < 0 and word in msg, (rc, msg)


def norm(**over):
    _lib, L = lib()
    v = dict(rows=4, hidden=64, xd=1, rd=1, yd=1, act=1, eps=1e-6, xs=64, rs=64, ros=64, ys=64, gr=64, gc=1, x=4096,
             res=8192, post=64, gate=64, pre=64, ro=16384, y=32768)
    v.update(over)
    d = _lib.NormDesc(v["rows"], v["hidden"], v["xd"], v["rd"], v["yd"], v["act"], 1.0, v["eps"], 0.0, v["xs"], v["rs"],
                      v["ros"], v["ys"], v["gr"], v["gc"])
    rc = L.nvfp4_norm_residual(ctypes.byref(d), v["x"], v["res"], v["post"], v["gate"], v["pre"], v["ro"], v["y"], None)
    return rc, L.nvfp4_last_error_string().decode()


@pytest.mark.parametrize("over,word", [
    (dict(hidden=0), "shape"), (dict(hidden=32769), "shape"), (dict(rows=-1), "shape"), (dict(xd=5), "dtype"),
    (dict(act=7), "activation"), (dict(eps=float("nan")), "eps"), (dict(gc=2), "gate column"), (dict(xs=63), "strides"),
    (dict(y=None), "together"), (dict(pre=None), "together"), (dict(y=None, pre=None, ro=None), "nothing"),
    (dict(x=None), "null x"), (dict(ro=8192, ros=128), "another stride"), (dict(y=16384), "same buffer"),
    (dict(y=4096, yd=0, xs=64), "another stride or dtype"), (dict(gr=-1), "gate stride")])
def test_norm_refuses(over, word):
    rc, msg = norm(**over)
    assert rc < 0 and word in msg, (rc, msg)


def test_python_refuses_what_is_not_on_the_gpu_or_of_another_type():
    import nvfp4

    k = torch.zeros(4, 16, 2, 128, dtype=torch.bfloat16)
    i = lambda *x: torch.tensor(x, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        nvfp4.PagedKVCache(k, k)
    with pytest.raises(TypeError, match="bf16"):
        nvfp4.PagedKVCache(k.float(), k.float())
    with pytest.raises(ValueError, match="contiguous"):
        nvfp4.PagedKVCache(k[..., ::2], k[..., ::2])
    with pytest.raises(ValueError, match="num_pages"):
        nvfp4.PagedKVCache(k[0], k[0])
    with pytest.raises(TypeError, match="int32"):
        nvfp4.AttentionBatch(torch.zeros(2, dtype=torch.int64), i([0], [1]))
    with pytest.raises(ValueError, match="one token"):
        nvfp4.AttentionBatch(i(1, 2), i([0], [1]), num_tokens=3)
    with pytest.raises(ValueError, match="num_tokens"):
        nvfp4.AttentionBatch(i(1, 2), i([0], [1]), q_start=i(0, 1, 2))
    with pytest.raises(ValueError, match="go together"):
        nvfp4.AttentionBatch(i(1, 2), i([0], [1]), prefix_len=3)
    with pytest.raises(ValueError, match="page_table"):
        nvfp4.AttentionBatch(i(1, 2), i([0], [1], [2]))
    with pytest.raises(ValueError, match="inv_freq"):
        nvfp4.Rotary(torch.zeros(4, dtype=torch.float64))
    with pytest.raises(ValueError, match="CUDA"):
        nvfp4.norm_residual(torch.zeros(2, 64, dtype=torch.bfloat16))
