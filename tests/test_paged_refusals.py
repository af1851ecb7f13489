"""What the paged cache's entry points refuse, before anything touches the GPU, and its definitions'
own arithmetic."""
import ctypes
import os
import re

import pytest
import torch

import paged_reference as R
from deltaattention_amd import _native, ops, paged

A = 1 << 20
F32, BF16, I32 = 4, 1, 3


def _err():
    return _native.lib().da_last_error().decode()


def _refused(rc, code, text):
    assert rc == code, (rc, _err())
    assert text in _err(), _err()


def _kv(**change):
    at = dict(k=A, v=A, num_pages=10, page_size=16, sk_p=4096, sk_h=2048, sk_n=128, sv_p=4096, sv_h=2048, sv_n=128)
    at.update(change)
    return ctypes.byref(_native.PagedKVBlock(**at))


def _batch(**change):
    at = dict(table=A, lengths=A, cu=A, start=None, B=3, width=4, table_stride=4, max_seqlen=5)
    at.update(change)
    return ctypes.byref(_native.PagedBatchBlock(**at))


def _append(k=A, v=A, q=A, q_out=A, dt=BF16, T=8, Hq=4, Hkv=2, D=128, cos=A, sin=A, rt=F32, rows=64, s_rot=64, rot=128, tok=0,
            kv=None, batch=None, st=1024):
    return _native.lib().da_paged_append(k, st, 128, v, st, 128, q, st, 128, q_out, st, 128, dt, T, Hq, Hkv, D, cos, sin, rt,
                                         rows, s_rot, rot, 0, tok, kv or _kv(), batch or _batch(), None)


def _attend(q=A, out=A, dt=BF16, T=8, Hq=4, Hkv=2, D=128, scale=0.1, kv=None, batch=None, prefix=None, st=512):
    return _native.lib().da_paged_attention(q, st, 128, out, st, 128, dt, T, Hq, Hkv, D, scale, kv or _kv(),
                                            batch or _batch(), prefix, None, 0, None)


@pytest.mark.parametrize("call", [_append, _attend])
def test_pages_and_batches(call):
    for name in ("k", "v"):
        _refused(call(kv=_kv(**{name: None})), -1, "null pages")
        _refused(call(kv=_kv(**{name: A + 8})), -1, "aligned")
    _refused(call(kv=_kv(num_pages=0)), -1, "no pages")
    _refused(call(kv=_kv(num_pages=1 << 31)), -1, "no pages")
    for size in (0, 8, 24, 1 << 30):
        _refused(call(kv=_kv(page_size=size)), -1, "page_size")
    for name in ("sk_p", "sk_h", "sk_n", "sv_p", "sv_h", "sv_n"):
        _refused(call(kv=_kv(**{name: 132})), -1, "multiples of 8")
    for name in ("sk_n", "sv_n"):
        _refused(call(kv=_kv(**{name: 120})), -1, "row strides")
        _refused(call(kv=_kv(**{name: 1 << 23})), -1, "row strides")
    _refused(call(batch=_batch(table=None)), -1, "table")
    _refused(call(batch=_batch(lengths=None)), -1, "lengths")
    _refused(call(batch=_batch(B=0)), -1, "empty")
    _refused(call(batch=_batch(width=0)), -1, "empty")
    _refused(call(batch=_batch(table_stride=3)), -1, "overlap")
    _refused(call(batch=_batch(width=1 << 26, table_stride=1 << 26)), -1, "2^30")
    _refused(call(batch=_batch(max_seqlen=0)), -1, "max_seqlen")
    _refused(call(batch=_batch(cu=None, B=9)), -1, "a token for each")
    _refused(call(dt=I32), -2, "bf16, fp16 or fp32")
    for D in (0, 4, 60, 136):
        _refused(call(D=D), -2, "head_dim")
    _refused(call(T=0), -1, "empty")
    _refused(call(q=A + 8), -1, "aligned")
    _refused(call(st=516), -1, "multiples of 8")


def test_append_refuses():
    _refused(_append(k=None), -1, "null")
    _refused(_append(q_out=None), -1, "null")
    for rot in (2, 130, 132, -4):
        _refused(_append(rot=rot), -1, "rotated dims")
    _refused(_append(cos=None), -1, "cos and sin")
    _refused(_append(rows=0), -1, "cos and sin")
    _refused(_append(rt=2), -1, "pages' type")
    for s in (63, 1, -64):
        _refused(_append(s_rot=s), -1, "overlap")
    _refused(_append(tok=1, rows=7), -1, "every token")


def test_attention_refuses():
    _refused(_attend(out=None), -1, "null")
    _refused(_attend(Hq=3), -1, "multiple of Hkv")
    _refused(_attend(T=1 << 27, Hq=32, Hkv=8), -1, "2^31 rows")
    _refused(_attend(T=1 << 24, Hq=32, Hkv=8), -1, "2^24 tokens")
    _refused(_attend(scale=0.0), -1, "scale")
    _refused(_attend(prefix=_batch(cu=None, B=3)), -1, "cu")
    _refused(_attend(prefix=_batch(width=0)), -1, "empty")


def test_python_refuses():
    cpu = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        ops.PagedKV(cpu, cpu)
    with pytest.raises(ValueError, match="GPU"):
        ops.PagedBatch(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32))
    for name in paged.__all__:
        assert getattr(ops, name) is getattr(paged, name) and name in ops.__all__


def test_header_and_signatures():
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "deltaattn_paged.h")).read()
    plain = re.sub(r"/\*.*?\*/", "", text, flags=re.S)
    names = set(re.findall(r"\b(da_[a-z_0-9]+)\s*\(", plain))
    assert names == {"da_paged_append", "da_paged_attention_workspace_size", "da_paged_attention"}
    for n in names:
        assert n in _native.SIGNATURES and hasattr(_native.lib(), n)
    for struct, block in (("DaPagedKV", _native.PagedKVBlock), ("DaPagedBatch", _native.PagedBatchBlock)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % struct, plain, flags=re.S).group(1)
        fields = [f.strip(" *") for line in body.split(";") if line.strip() for f in
                  re.sub(r"^\s*(const\s+)?\w+\s*\*?", "", line.strip()).split(",")]
        assert fields == [n for n, _ in block._fields_]


def test_reference_is_attention():
    """The 64-bit definition against torch's softmax over rows gathered by hand."""
    gen = torch.Generator().manual_seed(0)
    k, v = (torch.randn(9, 2, 16, 8, generator=gen, dtype=torch.float64).float() for _ in range(2))
    q = torch.randn(4, 4, 8, generator=gen)
    out, tol = R.attention(q, k, v, [[3, 1], [2, 0]], [20, 5], [0, 3, 4], ([[8, 4]], [17], [0, 4]))
    own = torch.cat([k[3], k[1][:, :4]], 1), torch.cat([v[3], v[1][:, :4]], 1)
    common = torch.cat([k[8], k[4][:, :1]], 1), torch.cat([v[8], v[4][:, :1]], 1)
    for i in range(3):
        for h in range(4):
            kk = torch.cat([common[0][h // 2], own[0][h // 2][:18 + i]]).double()
            vv = torch.cat([common[1][h // 2], own[1][h // 2][:18 + i]]).double()
            w = torch.softmax(q[i, h].double() @ kk.T / 8 ** 0.5, 0)
            assert torch.allclose(out[i, h], w @ vv, atol=1e-12)
    assert (tol > 0).all() and (tol < 1e-4).all()
