"""FourBitCompressedCache decoded on another stream than the one it was made on: the rows that a cut, a
growth or a new prompt replaces stay untouched until that stream has read them."""
import pytest
import torch

from conftest import announce
from test_gpu_fourbit_steps import W, _cache, _state, _token, knobs  # noqa: F401 (knobs: autouse)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("form", ["cut", "growth", "prompt"])
def test_replaced_rows_outlive_their_stream(gpu, form):
    from deltaattention_amd import kv4
    announce(f"four-bit streams: {form}")
    how = dict(initial_capacity=1, fill=1024) if form == "growth" else dict(budget=20, sinks=2, recent=4, slack=3, fill=3)
    cache, gen = _cache(gpu, **how)
    twin, _ = _cache(gpu, **how)
    token = _token(gpu, gen)
    prompt = [torch.randn(1, 2, 40, 64, generator=gen).bfloat16().to(gpu) for _ in range(2)]
    ones = torch.ones(1, 2, 40, dtype=torch.int32, device=gpu)
    weight = torch.rand(1, 2, 40, generator=gen).to(gpu)

    def step(c):
        got = [c.attend(token[0], 0)] if form == "prompt" else []
        if form == "prompt":
            c.initialize_from_prefill(0, *prompt, ones, ones.cumsum(-1).int(), *(x[:, :, -W:] for x in prompt), 40, mass=weight)
        return got + [c.decode_step(*token, 0)]

    want = step(twin)
    old = cache.anchors[0]
    at, size = old._own[1][torch.uint8].data_ptr(), old._own[1][torch.uint8].numel()
    busy = torch.randn(8192, 8192, device=gpu).bfloat16()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for _ in range(40):  # tens of milliseconds before the step's kernels begin
            busy = busy @ busy
        del old
        got = step(cache)
    assert cache.anchors[0].capacity == twin.anchors[0].capacity
    # what this stream allocates and writes meanwhile must not be those rows
    late = [torch.full((size,), 255, dtype=torch.uint8, device=gpu) for _ in range(4)]
    assert all(t.data_ptr() != at for t in late)
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    for x, y in zip(_state(cache), _state(twin)):
        assert torch.equal(x, y)
    assert isinstance(cache.anchors[0], kv4.KV4)


def test_record_stream_of_a_cache_of_tensors(gpu):
    """A KV4 built from tensors, with and without mass."""
    from deltaattention_amd import ops
    announce("KV4.record_stream")
    made = ops.KV4.empty(1, 2, 9, 64, gpu)
    side = torch.cuda.Stream()
    for mass in (made.mass, None):
        kv = ops.KV4(made.k_codes, made.k_scales, made.v_codes, made.v_scales, made.counts, made.timestamps, made.lengths,
                     64, mass)
        kv.record_stream(side)
    ops.KV4.empty(1, 2, 9, 64, gpu, mass=False).record_stream(side)
    torch.cuda.synchronize()
