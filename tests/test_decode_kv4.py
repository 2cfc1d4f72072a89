"""The decode harness over a 4-bit key/value cache: every attention of a run against the oracle, captured against eager steps, refusals."""
import pytest
import torch

from oracle import kv4_oracle as oracle

SMALL = dict(hidden=256, intermediate=512, n_heads=4, n_kv_heads=2, n_layers=2, vocab=512)
OPTIONS = {"everything": {}, "window": dict(kv_window=9, kv_sinks=2), "eviction": dict(kv_keep=16, kv_slack=3, kv_sinks=2, kv_recent=5)}


def small_model(cuda, dtype, batch, **kv):
    from matgptq_b200 import decode
    return decode.PackedLlama(decode.LlamaShape(**SMALL), 4, dtype=dtype, batch=batch, max_seq=64, device=cuda, seed=3, kv_bits=4, **kv)


def prompt(cuda, batch, n):
    return torch.randint(0, SMALL["vocab"], (batch, n), generator=torch.Generator(device=cuda).manual_seed(batch), device=cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("option", OPTIONS)
def test_every_attention_of_a_run(cuda, dtype, batch, option):
    """Prefill and steps: what each layer's attention gives, and the weights it adds, is the oracle's over the entries that the layer's
    cache holds at that moment; after an eviction the lengths are cut."""
    kv = OPTIONS[option]
    model = small_model(cuda, dtype, batch, **kv)
    cache, real, calls = model.cache4, model.cache4.attend, []
    window, sinks = kv.get("kv_window", 0), kv.get("kv_sinks", 0)

    def attend(i, q, *args, **kwargs):
        before = cache.weights[i].clone() if cache.weights is not None else None
        out = real(i, q, *args, **kwargs)
        lengths = cache.lengths.tolist()
        want, added, near, added_near = oracle.attention(q, *cache.layer(i), lengths, window, sinks, 64 ** -0.5)
        half = torch.finfo(dtype).eps / 2
        bound = near * (1 + half) + want.abs() * half * (1 + half) + torch.finfo(dtype).smallest_normal * half * 2
        assert ((out.double() - want).abs() <= bound).all()
        if before is not None:
            off = (cache.weights[i].double() - before.double() - added).abs()
            assert (off <= added_near + 2.0 ** -23 * cache.weights[i].double()).all()
        calls.append(lengths[0])
        return out

    cache.attend = attend
    model.generate(prompt(cuda, batch, 11), 20, use_graph=False)
    got = calls[::SMALL["n_layers"]]
    if option == "eviction":  # 19 entries are the most that stay; the 20th cuts the sequence to 16
        assert got == [11, 12, 13, 14, 15, 16, 17, 18, 19, 20, 17, 18, 19, 20, 17, 18, 19, 20, 17, 18]
    else:
        assert got == list(range(11, 31))


@pytest.mark.gpu
@pytest.mark.parametrize("option", OPTIONS)
def test_captured_steps_are_the_eager_ones(cuda, option):
    """Tokens and the whole state of the cache after a run with replayed steps; then again on the same model."""
    runs = []
    for use_graph in (False, True):
        model = small_model(cuda, torch.float16, 2, **OPTIONS[option])
        for _ in range(2):
            tokens = model.generate(prompt(cuda, 2, 11), 30, use_graph=use_graph)["tokens"]
            runs.append((tokens, [t.clone() for t in model.cache4.tensors()]))
    for tokens, tensors in runs[1:]:
        assert torch.equal(tokens, runs[0][0])
        n = tensors[-1].tolist()
        assert n == runs[0][1][-1].tolist()
        for got, want in zip(tensors[:-1], runs[0][1][:-1]):
            rows = n[0] // 2 if got.dtype == torch.uint8 and got.shape[2] * 2 == model.cache4.capacity else n[0]
            assert torch.equal(got[:, :, :rows].contiguous().view(torch.uint8), want[:, :, :rows].contiguous().view(torch.uint8))


@pytest.mark.gpu
def test_a_full_cache_is_refused(cuda):
    model = small_model(cuda, torch.float16, 1)
    model.forward(prompt(cuda, 1, 60), torch.arange(60, device=cuda))
    with pytest.raises(RuntimeError, match="do not fit"):
        model.forward(prompt(cuda, 1, 5), torch.arange(59, 64, device=cuda))


@pytest.mark.parametrize("kv", [dict(kv_bits=8), dict(kv_bits=16, kv_window=4), dict(kv_bits=16, kv_keep=4),
                                dict(kv_bits=4, kv_keep=4, kv_sinks=3, kv_recent=2)])
def test_refusals(kv):
    from matgptq_b200 import decode
    shape = decode.LlamaShape(**{**SMALL, "n_layers": 0})
    with pytest.raises(ValueError, match="kv_"):
        decode.PackedLlama(shape, 4, max_seq=64, device="cpu", **kv)
