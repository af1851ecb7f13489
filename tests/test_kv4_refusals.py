"""What the bounded cache's entry points refuse, before anything touches the GPU."""
import ctypes

import pytest
import torch

from deltaattention_amd import _native, kv4, ops

A = ctypes.c_void_p(1 << 20)
ODD = ctypes.c_void_p((1 << 20) + 8)


def _err():
    return _native.lib().da_last_error().decode()


def _kv(capacity=64, **change):
    names = ("k_codes", "k_scales", "v_codes", "v_scales", "counts", "timestamps", "lengths", "mass")
    at = {n: 1 << 20 for n in names}
    at.update(change)
    return ctypes.byref(_native.Kv4Block(*(at[n] for n in names), capacity))


def _refused(rc, code, text):
    assert rc == code, (rc, _err())
    assert text in _err(), _err()


def test_quantize_refuses():
    f = _native.lib().da_kv4_quantize

    def call(k=A, v=A, dt=1, B=1, H=2, N=64, D=128, sk=(0, 0, 128), sv=(0, 0, 128), index=None, M=64, out=None):
        return f(k, v, dt, B, H, N, D, *sk, *sv, None, None, None, None, index, M, out if out is not None else _kv(), None)
    _refused(call(k=None), -1, "null")
    _refused(call(out=_kv(k_codes=None)), -1, "null")
    _refused(call(dt=3), -2, "bf16")
    for D in (0, 4, 60, 136):
        _refused(call(D=D), -2, "head_dim")
    _refused(call(B=0), -1, "empty")
    _refused(call(M=63), -1, "M")
    _refused(call(M=65, index=A), -1, "capacity")
    _refused(call(k=ODD), -1, "aligned")
    _refused(call(sk=(0, 0, 129)), -1, "aligned")
    _refused(call(dt=4, sv=(0, 2, 128)), -1, "aligned")
    _refused(call(out=_kv(k_codes=(1 << 20) + 4)), -1, "aligned")
    _refused(call(out=_kv(v_scales=(1 << 20) + 2)), -1, "aligned")
    _refused(call(out=_kv(capacity=(1 << 26) + 1)), -2, "2^26")
    _refused(call(B=65536), -1, "65535")


def test_dequantize_refuses():
    f = _native.lib().da_kv4_dequantize
    _refused(f(_kv(), 1, 2, 65, 128, A, A, 1, None), -1, "capacity")
    _refused(f(_kv(), 1, 2, 64, 128, A, None, 1, None), -1, "aligned")
    _refused(f(_kv(), 1, 2, 64, 128, A, A, 3, None), -2, "bf16")
    _refused(f(None, 1, 2, 64, 128, A, A, 1, None), -1, "null")


def test_evict_and_rows_refuse():
    lib = _native.lib()
    need = lib.da_kv4_evict_workspace_size(1, 2, 64, 16)
    assert need == 0  # a small budget's choice stays on the chip
    other = dict(k_codes=1 << 22, v_codes=1 << 22, mass=1 << 22, counts=1 << 22, lengths=1 << 22)

    def evict(kv=None, out=None, budget=16, sinks=1, recent=1, ws=A, n=need):
        return lib.da_kv4_evict(kv if kv is not None else _kv(), 1, 2, 128, budget, sinks, recent,
                                out if out is not None else _kv(**other), None, ws, n, None)
    _refused(evict(kv=_kv(mass=None)), -1, "null")
    _refused(evict(out=_kv(**dict(other, mass=None))), -1, "null")
    _refused(evict(out=_kv()), -1, "other memory")
    for bad in (dict(budget=0), dict(sinks=-1), dict(recent=-1), dict(sinks=10, recent=7), dict(sinks=1 << 62, recent=1 << 62)):
        _refused(evict(**bad), -1, "budget")
    _refused(evict(budget=65), -1, "capacity")
    need = lib.da_kv4_evict_workspace_size(1, 2, 1024, 512)
    assert need > 0
    large = dict(kv=_kv(capacity=1024), out=_kv(**dict(other, capacity=1024)), budget=512)
    _refused(evict(**large, n=need - 1), -4, "workspace")
    _refused(evict(**large, ws=None, n=need), -4, "workspace")
    assert lib.da_kv4_evict_workspace_size(0, 2, 64, 16) == 0
    rows = lib.da_heavy_rows
    _refused(rows(None, None, 1, 2, 64, 16, 0, 0, A, A, A, need, None), -1, "null")
    _refused(rows(A, None, 1, 0, 64, 16, 0, 0, A, A, A, need, None), -1, "shape")
    _refused(rows(A, None, 1, 2, 64, 16, 9, 8, A, A, A, need, None), -1, "budget")
    _refused(rows(A, None, 1, 2, 1024, 512, 0, 0, A, A, None, 0, None), -4, "workspace")
    # a head longer than 16384 rows needs scratch for its chunks as well
    assert lib.da_kv4_evict_workspace_size(1, 2, 16385, 16) > lib.da_kv4_evict_workspace_size(1, 2, 16384, 16)


def test_attention_refuses():
    lib = _native.lib()
    need = lib.da_kv4_attention_workspace_size(1, 8, 2, 4096, 0)
    assert lib.da_kv4_attention_workspace_size(1, 8, 2, 4096, 1) > need > 0

    def call(q=A, dt=1, B=1, Hq=8, H=2, D=128, sq=(1024, 128), kv=None, kx=A, vx=A, sx=(0, 2048, 128), n=16, scale=0.1,
             acc=0, out=A, ws=A, size=need):
        return lib.da_kv4_attention(q, dt, B, Hq, H, D, *sq, kv if kv is not None else _kv(4096), kx, vx, *sx, n, scale,
                                    acc, out, 1024, 128, ws, size, None)
    _refused(call(q=None), -1, "null")
    _refused(call(kx=None), -1, "ring")
    _refused(call(kv=_kv(4096, mass=None), acc=1), -1, "null")
    _refused(call(dt=3), -2, "bf16")
    _refused(call(D=100), -2, "head_dim")
    _refused(call(Hq=7), -1, "head counts")
    _refused(call(Hq=130), -2, "group")
    _refused(call(n=-1), -1, "lengths")
    _refused(call(kv=_kv((1 << 24) + 1)), -2, "2^24")
    _refused(call(sq=(1024, 124)), -1, "aligned")
    _refused(call(q=ODD), -1, "aligned")
    _refused(call(sx=(0, 2048, 132)), -1, "aligned")
    _refused(call(scale=0.0), -1, "scale")
    _refused(call(scale=float("nan")), -1, "scale")
    _refused(call(size=need - 1), -4, "workspace")
    _refused(call(ws=ODD), -1, "aligned")


def test_mass_refuses():
    lib = _native.lib()
    need = lib.da_attention_mass_workspace_size(1, 8, 2, 16, 256)

    def call(q=A, k=A, dt=1, B=1, Hq=8, H=2, Nq=16, Nk=256, D=128, sq=(0, 128, 1024), sk=(0, 128, 256), start=240, scale=0.1,
             mass=A, ws=A, n=need):
        return lib.da_attention_mass(q, k, dt, B, Hq, H, Nq, Nk, D, *sq, *sk, None, None, None, start, scale, mass, ws, n,
                                     None)
    _refused(call(mass=None), -1, "null")
    _refused(call(dt=0), -2, "bf16")
    _refused(call(D=132), -2, "head_dim")
    _refused(call(Hq=9), -1, "shape")
    _refused(call(Nq=0), -1, "shape")
    _refused(call(Hq=130), -2, "group")
    _refused(call(Nk=(1 << 24) + 1), -2, "2^24")
    _refused(call(sk=(0, 128, 252)), -1, "aligned")
    _refused(call(scale=-1.0), -1, "scale")
    _refused(call(start=1 << 41), -1, "q_start")
    _refused(call(n=need - 4), -4, "workspace")
    assert lib.da_attention_mass_workspace_size(1, 2, 8, 16, 256) == 0


def test_update_refuses():
    f = _native.lib().da_kv4_update

    def call(nk=A, D=128, sn=(256, 128), kv=None, last=A, exact=5, total=9, W=8):
        return f(nk, A, 1, 1, 2, D, *sn, A, A, 0, 1024, 128, kv if kv is not None else _kv(), last, exact, total, W, 1.0, 0,
                 None)
    _refused(call(last=None), -1, "null")
    _refused(call(kv=_kv(counts=None)), -1, "null")
    _refused(call(D=12), -2, "head_dim")
    _refused(call(W=0), -1, "lengths")
    _refused(call(exact=-1), -1, "lengths")
    _refused(call(sn=(256, 127)), -1, "aligned")


def test_host_tensors_are_refused():
    t = torch.zeros(1, 2, 4, 64)
    for f in (lambda: ops.attention_mass(t, t), lambda: ops.quantize_kv4(t, t), lambda: ops.heavy_rows(t[..., 0], 2),
              lambda: ops.KV4(*(torch.zeros(1, 2, 4, 32, dtype=torch.uint8),) * 4, *(torch.zeros(1, 2, 4),) * 3, 64),
              lambda: ops.KV4.empty(1, 2, 4, 64, "cpu")):
        with pytest.raises(ValueError, match="GPU"):
            f()


def test_budget_arguments():
    for bad in ((0, 0, 0), (4, 3, 2), (4, -1, 0), (4, 0, -1)):
        with pytest.raises(ValueError):
            kv4._budget(*bad)
    assert kv4._budget(4, 2, 2) == (4, 2, 2)


def test_declared_symbols_have_signatures():
    import os
    import re
    text = open(os.path.join(os.path.dirname(__file__), "..", "include", "deltaattn_cache.h")).read()
    names = sorted(set(re.findall(r"\b(da_[a-z_0-9]+)\s*\(", re.sub(r"/\*.*?\*/", "", text, flags=re.S))))
    assert names == sorted(["da_kv4_quantize", "da_kv4_dequantize", "da_kv4_evict_workspace_size", "da_kv4_evict",
                            "da_kv4_update", "da_heavy_rows", "da_kv4_attention_workspace_size", "da_kv4_attention",
                            "da_attention_mass_workspace_size", "da_attention_mass"])
    for name in names:
        assert hasattr(_native.lib(), name) and name in _native.SIGNATURES
    # struct DaKv4: eight pointers and an int64
    assert ctypes.sizeof(_native.Kv4Block) == 72
