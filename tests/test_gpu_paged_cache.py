"""PagedCache: through the model swap against transformers' own attention, and its pages by themselves."""
import copy
import types

import pytest
import torch

import paged_reference as R
from conftest import announce

pytestmark = pytest.mark.gpu


def _model(impl, seed=0, layers=2):
    from deltaattention_amd import llama_swap
    cfg = llama_swap.llama3_8b_config(impl, num_layers=layers)
    cfg.vocab_size, cfg.hidden_size, cfg.intermediate_size = 512, 512, 1024
    cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim = 8, 2, 64
    return llama_swap.random_llama(cfg, torch.device("cuda:0"), seed=seed)


def _ids(*shape, seed=1):
    return torch.randint(0, 512, shape, generator=torch.Generator().manual_seed(seed)).cuda()


def _exact(model):
    """The same weights in fp32 through transformers' eager attention."""
    from transformers import LlamaForCausalLM
    cfg = copy.deepcopy(model.config)
    cfg._attn_implementation = "eager"
    ref = LlamaForCausalLM(cfg).to("cuda:0", torch.float32).eval()
    ref.load_state_dict({k: v.float() for k, v in model.state_dict().items()})
    return ref


@torch.no_grad()
def _logits(model, ids, cache=None):
    return model(ids, past_key_values=cache, use_cache=cache is not None).logits.float()


def _near(got, want):
    # bf16 weights and activations against fp32 throughout, as in the swap's other tests
    err, scale = (got - want).abs(), want.abs()
    assert torch.isfinite(got).all()
    assert err.mean() <= 0.02 * scale.mean() and err.max() <= 0.25 * scale.max(), (err.mean(), err.max(), scale.mean())


def test_prompt_part_and_steps(gpu):
    """A prompt, a second part and single tokens through the dense path, two sequences."""
    from deltaattention_amd import llama_swap
    from deltaattention_amd.paged_cache import PagedCache
    announce("model over a PagedCache: 70 + 33 + 1 + 1 + 1 tokens, two sequences")
    model = _model(llama_swap.DENSE)
    ids = _ids(2, 106)
    want = _logits(_exact(model), ids)
    cache = PagedCache(model.config, 2, num_pages=4)
    at = 0
    for n in (70, 33, 1, 1, 1):
        got = _logits(model, ids[:, at:at + n], cache)
        _near(got, want[:, at:at + n])
        at += n
        assert cache.get_seq_length() == at and cache.get_seq_length(1) == at


def test_attention_of_every_layer(gpu, monkeypatch):
    """What a layer's attention gets and gives, against 64 bits: rotation, pages and both kernels."""
    from deltaattention_amd import llama_swap, paged
    from deltaattention_amd.paged_cache import PagedCache
    announce("model over a PagedCache: attention against 64 bits")
    model = _model(llama_swap.DENSE)
    calls = []
    real = paged.paged_attention

    def spy(q, kv, batch, scale=None, out=None):
        got = real(q, kv, batch, scale=scale, out=out)
        calls.append([t.detach().cpu().clone() for t in (q, kv.k_pages, kv.v_pages, batch.table, batch.lengths, got)])
        return got
    monkeypatch.setattr(paged, "paged_attention", spy)
    cache = PagedCache(model.config, 2)
    ids = _ids(2, 90)
    for a, b in ((0, 80), (80, 81), (81, 90)):
        _logits(model, ids[:, a:b], cache)
    assert len(calls) == 6
    for q, k, v, table, lengths, got in calls:
        n = q.shape[0] // 2
        want, tol = R.attention(q, k, v, table, lengths.tolist(), [0, n, 2 * n], None, 64 ** -0.5)
        assert ((got.double() - want).abs() <= tol).all()


def test_delta_prompt_then_steps(gpu, monkeypatch):
    """PATH 1 for the prompt (every key an anchor: dense attention), dense attention over the pages after."""
    from deltaattention_amd import globVR, llama_swap
    from deltaattention_amd.paged_cache import PagedCache
    announce("model over a PagedCache: delta prompt, then steps")
    monkeypatch.setattr(globVR, "packing_mode", "periodic")
    monkeypatch.setattr(globVR, "target_keep_rate", 1.0)
    model = _model(llama_swap.DELTA)
    ids = _ids(1, 305)
    want = _logits(_exact(model), ids)
    cache = PagedCache(model.config, 1)
    for a, b in ((0, 300), (300, 304), (304, 305)):
        _near(_logits(model, ids[:, a:b], cache), want[:, a:b])


def test_fork(gpu):
    """Answers behind a common prompt: each as if its sequence were alone; the parent goes on."""
    from deltaattention_amd import llama_swap
    from deltaattention_amd.paged_cache import PagedCache
    announce("PagedCache.fork: two prompts, three answers each")
    model = _model(llama_swap.DENSE)
    ref = _exact(model)
    prompts, tails = _ids(2, 45), _ids(6, 20, seed=7)
    whole = torch.cat([prompts.repeat_interleave(3, 0), tails], 1)
    want = _logits(ref, whole)
    cache = PagedCache(model.config, 2, num_pages=8)
    _logits(model, prompts, cache)
    fork = cache.fork(3)
    assert fork.get_seq_length() == 45
    at = 0
    for n in (1, 17, 1, 1):
        got = _logits(model, tails[:, at:at + n], fork)
        _near(got, want[:, 45 + at:45 + at + n])
        at += n
    more = _ids(2, 5, seed=9)
    _near(_logits(model, more, cache), _logits(ref, torch.cat([prompts, more], 1))[:, 45:])
    with pytest.raises(NotImplementedError):
        fork.fork(2)
    used = sum(x > 0 for x in cache._pool.holders)
    del fork
    assert sum(x > 0 for x in cache._pool.holders) == used - 6 * 2  # two pages an answer


def test_generate(gpu):
    """transformers' own generation loop over a PagedCache gives the tokens of step-by-step argmax."""
    from deltaattention_amd import llama_swap
    from deltaattention_amd.paged_cache import PagedCache
    announce("generate() over a PagedCache")
    model = _model(llama_swap.DENSE)
    ids = _ids(1, 40)
    cache = PagedCache(model.config, 1)
    step, at = [], ids
    for _ in range(6):
        at = _logits(model, at, cache)[:, -1:].argmax(-1)
        step.append(int(at))
    with torch.no_grad():
        got = model.generate(ids, attention_mask=torch.ones_like(ids), past_key_values=PagedCache(model.config, 1),
                             max_new_tokens=6, do_sample=False, pad_token_id=0, eos_token_id=None)
    assert got[0, 40:].tolist() == step


def _cfg(layers=1, heads=4, kv=2, dim=64):
    return types.SimpleNamespace(head_dim=dim, num_key_value_heads=kv, num_hidden_layers=layers, hidden_size=heads * dim,
                                 num_attention_heads=heads)


def _rand(*shape, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda").to(dtype)


def test_pages_grow_and_return(gpu):
    """The pool grows with its contents kept; reset and the end of a cache give pages back."""
    from deltaattention_amd.paged_cache import PagedCache
    announce("PagedCache: pages")
    cache = PagedCache(_cfg(), 3, num_pages=2)
    rows = []
    for n in (20, 1, 200, 1):
        k, v = _rand(3, 2, n, 64), _rand(3, 2, n, 64)
        assert cache.append(k, v, 0) is None
        rows.append((k, v))
    k, v = (torch.cat([r[i] for r in rows], 2) for i in (0, 1))
    table = cache._table[:, :len(cache._pages[0])].long()
    for pages, want in ((cache._pool.k[0], k), (cache._pool.v[0], v)):
        got = pages[table].transpose(1, 2).reshape(3, 2, -1, 64)[:, :, :222]
        assert torch.equal(got, want)
    assert sum(x > 0 for x in cache._pool.holders) == 3 * 14 == len(cache._pool.holders) - len(cache._pool.free)
    cache.reset()
    assert cache.get_seq_length() == 0 and not any(cache._pool.holders)
    q = _rand(3, 4, 5, 64)
    k, v = _rand(3, 2, 5, 64), _rand(3, 2, 5, 64)
    out = cache.attend(cache.append(k, v, 0, q), 0)
    mask = torch.ones(5, 5, device="cuda").tril().log()
    kk, vv = (x.float().repeat_interleave(2, 1) for x in (k, v))
    w = torch.softmax(torch.matmul(q.float(), kk.transpose(-1, -2).contiguous()) / 8 + mask, -1)
    assert (out.transpose(1, 2).float() - torch.matmul(w, vv)).abs().max() <= 0.03


def test_refused_calls_change_nothing(gpu):
    from deltaattention_amd.paged_cache import PagedCache
    announce("PagedCache: refusals")
    cache = PagedCache(_cfg(layers=2), 2)
    k, v, q = _rand(2, 2, 20, 64), _rand(2, 2, 20, 64), _rand(2, 4, 20, 64)
    cos = torch.ones(1, 20, 64, device="cuda")
    state = lambda: (cache._total, list(cache._seen), [list(p) for p in cache._pages], len(cache._pool.free))  # noqa: E731
    before = state()
    for bad in (dict(key=k.float()), dict(key=k[:1]), dict(value=v[:, :, :3]), dict(query=q[:, :, :3]), dict(query=q[:, :3]),
                dict(key=k[..., :32]), dict(cos=cos[:, :5]), dict(cos=cos.half()), dict(key=k.cpu())):
        args = dict(key=k, value=v, query=q, cos=cos, sin=cos)
        args.update(bad)
        if "cos" in bad:
            args["sin"] = args["cos"]
        with pytest.raises((ValueError, TypeError)):
            cache.append(args["key"], args["value"], 0, args["query"], args["cos"], args["sin"])
        assert state() == before
    with pytest.raises(RuntimeError):
        cache.attend(q.transpose(1, 2).reshape(-1, 4, 64), 0)
    with pytest.raises(ValueError):
        cache.fork(2)
    cache.append(k, v, 0)
    with pytest.raises(RuntimeError, match="same"):
        cache.append(k, v, 0)          # layer 1 has not had its turn
    with pytest.raises(RuntimeError, match="same"):
        cache.append(k[:, :, :3], v[:, :, :3], 1)
    cache.append(k, v, 1)
    assert cache._seen == [20, 20]
    for call in (lambda: cache.update(k, v, 0), lambda: cache.crop(3), lambda: cache.reorder_cache(None),
                 lambda: cache.batch_repeat_interleave(2), lambda: cache.batch_select_indices(None)):
        with pytest.raises(NotImplementedError):
            call()
