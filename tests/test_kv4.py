"""The 4-bit key/value cache on the CPU: refusals of the operators and of the C ABI, shapes of the fake implementations, and the oracle's
layout.  No kernel is launched here."""
import ctypes

import pytest
import torch

from oracle import kv4_oracle as oracle

CAPACITY, D, KV, H, B = 128, 64, 2, 4, 3


def cache(device="cpu", dtype=torch.float16, capacity=CAPACITY, d=D, b=B, kv=KV):
    new = lambda t, *s: torch.zeros(b, kv, *s, dtype=t, device=device)  # noqa: E731
    return [new(torch.uint8, capacity, d // 2), new(torch.uint8, capacity // 2, d), new(dtype, capacity, 4)]


def test_operators_refuse_host_tensors():
    from matgptq_b200 import ops
    lengths = torch.zeros(B, dtype=torch.int32)
    table = torch.zeros(16, D // 2)
    with pytest.raises(RuntimeError, match="k_codes to be a CUDA tensor"):
        ops.append_kv4(torch.zeros(B, (H + 2 * KV) * D, dtype=torch.float16), torch.zeros(1, dtype=torch.int64), table, table, lengths, *cache(), H, 1)
    with pytest.raises(RuntimeError, match="k_codes to be a CUDA tensor"):
        ops.attention_kv4(torch.zeros(B, 1, H, D, dtype=torch.float16), *cache(), lengths, 0, 0, 1.0, 1)
    with pytest.raises(RuntimeError, match="k_codes to be a CUDA tensor"):
        ops.evict_kv4(*cache(), torch.zeros(B, KV, CAPACITY), lengths, 8, 0, 0, 0, 1)
    with pytest.raises(RuntimeError, match="k_codes to be a CUDA tensor"):
        ops.dequantize_kv4(*cache(), lengths, 4, 1)


def test_fake_implementations_give_the_shapes():
    from matgptq_b200 import ops
    with torch._subclasses.FakeTensorMode():
        c = cache("cuda")
        lengths = torch.zeros(B, dtype=torch.int32, device="cuda")
        table = torch.zeros(16, D // 2, device="cuda")
        qkv = torch.zeros(B * 5, (H + 2 * KV) * D, dtype=torch.float16, device="cuda")
        q = ops.append_kv4(qkv, torch.zeros(5, dtype=torch.int64, device="cuda"), table, table, lengths, *c, H, 1)
        assert q.shape == (B, 5, H, D) and q.dtype == torch.float16
        assert ops.attention_kv4(q, *c, lengths, 0, 0, 1.0, 1).shape == q.shape
        new, kept = ops.evict_kv4(*c, torch.zeros(B, KV, CAPACITY, device="cuda"), lengths, 8, 0, 0, 0, 1)
        assert new.shape == (B,) and kept.shape == (B, KV, 8) and kept.dtype == new.dtype == torch.int32
        k, v = ops.dequantize_kv4(*c, lengths, 7, 1)
        assert k.shape == v.shape == (B, KV, 7, D) and k.dtype == torch.float16


def native_cache(**change):
    from matgptq_b200 import _native
    fields = dict(k_codes=1 << 20, v_codes=1 << 21, params=1 << 22, batch=B, n_kv_heads=KV, head_dim=D, capacity=CAPACITY)
    fields.update(change)
    return ctypes.byref(_native.Kv4Cache(**fields))


BAD_CACHES = [(dict(k_codes=None), 1), (dict(params=None), 1), (dict(batch=-1), 1), (dict(n_kv_heads=0), 1), (dict(capacity=0), 1),
              (dict(capacity=100), 1), (dict(capacity=1 << 31), 1), (dict(head_dim=96), 3), (dict(head_dim=256), 3), (dict(batch=40000), 3),
              (dict(v_codes=(1 << 21) + 8), 4)]


@pytest.mark.parametrize("change, status", BAD_CACHES)
def test_c_abi_refuses_bad_caches(lib, change, status):
    """Every entry point checks the cache before anything else; the addresses are never followed."""
    p = 1 << 23
    c = native_cache(**change)
    assert lib.matgptq_b200_append_kv4(c, p, p, 0, p, p, 16, p, p, 1, H, 0, None) == status
    assert lib.matgptq_b200_attention_kv4(c, p, 1, H, p, 0, 0, 1.0, None, p, None, 0, 0, None) == status
    assert lib.matgptq_b200_evict_kv4(c, p, p, 8, 0, 0, 0, p + 64, p, 0, None) == status
    assert lib.matgptq_b200_dequantize_kv4(c, p, 4, p, p, 0, None) == status


def test_c_abi_refuses_bad_arguments(lib):
    p, odd = 1 << 23, (1 << 23) + 2
    c = native_cache()
    append = lambda **k: lib.matgptq_b200_append_kv4(c, *{**dict(qkv=p, pos=p, stride=0, cos=p, sin=p, n=16, len=p, q=p, seq=1, heads=H,  # noqa: E731
                                                               flags=0, stream=None), **k}.values())
    for bad in (dict(qkv=None), dict(pos=None), dict(cos=None), dict(len=None), dict(q=None), dict(seq=-1), dict(heads=0), dict(n=0), dict(stride=-1)):
        assert append(**bad) == 1, bad
    assert append(qkv=odd) == 4 and append(q=odd) == 4 and append(cos=odd) == 4
    assert append(seq=0) == 0
    attend = lambda **k: lib.matgptq_b200_attention_kv4(c, *{**dict(q=p, seq=1, heads=H, len=p, window=0, sinks=0, scale=1.0, weights=None, out=p,  # noqa: E731
                                                                  ws=None, ws_bytes=0, flags=0, stream=None), **k}.values())
    for bad in (dict(q=None), dict(len=None), dict(out=None), dict(seq=-1), dict(heads=0), dict(heads=3), dict(window=-1), dict(sinks=-1),
                dict(seq=12, weights=p), dict(seq=12, weights=p, ws=p, ws_bytes=0)):
        assert attend(**bad) == 1, bad
    assert attend(q=odd) == 4 and attend(out=odd) == 4
    assert attend(seq=1 << 25) == 3
    assert attend(seq=0) == 0
    evict = lambda **k: lib.matgptq_b200_evict_kv4(c, *{**dict(w=p, len=p, keep=8, slack=0, sinks=0, recent=0, new=p + 64, kept=p, flags=0,  # noqa: E731
                                                             stream=None), **k}.values())
    for bad in (dict(w=None), dict(len=None), dict(new=None), dict(kept=None), dict(new=p), dict(keep=0), dict(keep=CAPACITY + 1), dict(slack=-1),
                dict(sinks=-1), dict(recent=-1), dict(sinks=9), dict(sinks=4, recent=5)):
        assert evict(**bad) == 1, bad
    assert lib.matgptq_b200_dequantize_kv4(c, None, 4, p, p, 0, None) == 1
    assert lib.matgptq_b200_dequantize_kv4(c, p, -1, p, p, 0, None) == 1
    assert lib.matgptq_b200_dequantize_kv4(c, p, 4, None, p, 0, None) == 1
    assert lib.matgptq_b200_dequantize_kv4(c, p, 4, p, odd, 0, None) == 4
    assert lib.matgptq_b200_dequantize_kv4(c, p, 0, None, None, 0, None) == 0
    assert lib.matgptq_b200_attention_kv4_workspace_bytes(c, 5, H, 0, 0, 0) == 0
    assert lib.matgptq_b200_attention_kv4_workspace_bytes(None, 5, H, 0, 0, 1) == 0
    for seq in (12, 17, 500):  # more rows than one CTA has: what it leaves for the weights goes through the workspace
        need = lib.matgptq_b200_attention_kv4_workspace_bytes(c, seq, H, 0, 0, 1)
        assert need >= B * seq * H * 4
        assert lib.matgptq_b200_attention_kv4_workspace_bytes(c, seq, H, 9, 1, 1) >= B * seq * H * 4
        assert attend(seq=seq, weights=p, ws=p, ws_bytes=need - 1) == 1 and attend(seq=seq, weights=p, ws=odd, ws_bytes=need) == 4


def test_long_caches_need_a_workspace(lib):
    """Few rows over many entries: the work is cut into shares, whose partial results go through the workspace."""
    p = 1 << 23
    c = native_cache(capacity=1 << 17)
    need = lib.matgptq_b200_attention_kv4_workspace_bytes(c, 1, H, 0, 0, 0)
    assert need > 0
    attend = lambda ws, n: lib.matgptq_b200_attention_kv4(c, p, 1, H, p, 0, 0, 1.0, None, p, ws, n, 0, None)  # noqa: E731
    assert attend(None, need) == 1 and attend(p, need - 1) == 1 and attend(p + 8, need) == 4
    assert lib.matgptq_b200_attention_kv4_workspace_bytes(c, 1, H, 100, 4, 0) == 0  # a window that one CTA takes as a whole


def test_cache_refuses_bad_shapes():
    from matgptq_b200.kv_cache import KV4Cache
    with pytest.raises(ValueError, match="head dimension"):
        KV4Cache(1, 1, 1, 96, 64, device="cpu")
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        KV4Cache(1, 1, 1, 64, 64, dtype=torch.float32, device="cpu")
    with pytest.raises(ValueError, match="at least 1"):
        KV4Cache(1, 0, 1, 64, 64, device="cpu")
    c = KV4Cache(2, 3, 2, 64, 100, device="cpu")
    assert c.capacity == 128 and len(c.k_codes) == 2
    c.advance(120)
    assert c.lengths.tolist() == [120] * 3
    with pytest.raises(RuntimeError, match="do not fit"):
        c.advance(9)
    with pytest.raises(RuntimeError, match="weights=True"):
        c.evict(8)
    c.reset()
    c.advance(8, torch.tensor([8, 3, 0], dtype=torch.int32))
    assert c.lengths.tolist() == [8, 3, 0] and c.most == 8


def test_oracle_layout():
    """Byte i of a K row holds channels 2i and 2i + 1; a V pair holds two bytes of one entry, then two of the other."""
    codes = torch.arange(2 * 128 * 64).view(1, 2, 128, 64) * 7 % 16
    k, v = oracle.pack_k(codes), oracle.pack_v(codes)
    assert k[0, 1, 5, 3] == codes[0, 1, 5, 6] + 16 * codes[0, 1, 5, 7]
    assert v[0, 1, 2, 4 * 3 + 0] == codes[0, 1, 4, 12] + 16 * codes[0, 1, 4, 13]
    assert v[0, 1, 2, 4 * 3 + 1] == codes[0, 1, 4, 14] + 16 * codes[0, 1, 4, 15]
    assert v[0, 1, 2, 4 * 3 + 2] == codes[0, 1, 5, 12] + 16 * codes[0, 1, 5, 13]
    assert torch.equal(oracle.unpack_k(k), codes) and torch.equal(oracle.unpack_v(v), codes)
