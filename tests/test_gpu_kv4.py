"""The 4-bit key/value cache on the GPU against the 64-bit oracle: writing, reading back, attention with window and first entries, eviction,
and a run of them as a model uses them."""
import math

import pytest
import torch

from oracle import kv4_oracle as oracle

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def flag_of(dtype):
    return 1 | (2 if dtype == torch.bfloat16 else 0)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def empty_cache(b, kv, capacity, d, dtype, dev):
    """A cache whose unused entries hold what must never be read: every code set, NaN for every scale."""
    return [torch.full((b, kv, capacity, d // 2), 255, dtype=torch.uint8, device=dev),
            torch.full((b, kv, capacity // 2, d), 255, dtype=torch.uint8, device=dev),
            torch.full((b, kv, capacity, 4), math.nan, dtype=dtype, device=dev)]


def filled_cache(b, kv, capacity, d, dtype, lengths, dev, gen, v_size=1.0):
    cache = empty_cache(b, kv, capacity, d, dtype, dev)
    x = torch.randn(b, kv, capacity, d, generator=gen, device=dev)
    x += torch.randn(b, kv, 1, d, generator=gen, device=dev)
    kc, ks, kl = oracle.quantise_rows(x.to(dtype))
    vc, vs, vl = oracle.quantise_rows((v_size * torch.randn(b, kv, capacity, d, generator=gen, device=dev)).to(dtype))
    k, v, p = oracle.pack_k(kc), oracle.pack_v(vc), torch.cat([ks, kl, vs, vl], -1).to(dtype)
    # what lies behind the last entry stays as it was; the second of a V pair by bytes
    behind = torch.arange(capacity, device=dev)[None] >= torch.tensor(lengths, device=dev)[:, None]
    k[behind[:, None].expand(-1, kv, -1)] = 255
    p[behind[:, None].expand(-1, kv, -1)] = math.nan
    cache[0].copy_(k), cache[1].copy_(v), cache[2].copy_(p)
    return cache


def lengths_tensor(lengths, dev):
    return torch.tensor(lengths, dtype=torch.int32, device=dev)


def status():
    from matgptq_b200 import _native
    return _native.device_status()


# ---- writing and reading back ----------------------------------------------------------------------------------------
def plain_tables(n, d, dev):
    """No rotation at all: what is written is what was given."""
    return torch.ones(n, d // 2, device=dev), torch.zeros(n, d // 2, device=dev)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b, seq, heads, kv, lengths", [(1, 1, 8, 2, [1]), (1, 1, 4, 4, [64]), (3, 5, 3, 1, [5, 17, 40]),
                                                        (4, 37, 6, 3, [37, 12, 0, 1]), (2, 64, 1, 1, [64, 63])])
def test_append_and_dequantize(cuda, dtype, d, b, seq, heads, kv, lengths):
    """Codes, scales and minima to the bit, nothing else touched, padding left out; the same bits read back."""
    from matgptq_b200 import ops
    capacity = 64
    gen = torch.Generator(device=cuda).manual_seed(seq * 7 + d)
    qkv = torch.randn(b, seq, heads + 2 * kv, d, generator=gen, device=cuda)
    qkv[:, ::3, heads:] *= 1e-3
    qkv[:, -1, heads + kv:] = 0.25  # a row of one value: scale 0
    qkv = qkv.to(dtype)
    cache = empty_cache(b, kv, capacity, d, dtype, cuda)
    want = [t.clone() for t in cache]
    n = lengths_tensor(lengths, cuda)
    cos, sin = plain_tables(7, d, cuda)
    positions = torch.randint(0, 7, (b, seq), generator=gen, device=cuda)
    q = ops.append_kv4(qkv.view(b * seq, -1), positions, cos, sin, n, *cache, heads, flag_of(dtype))

    units = [t.clone() for t in want]
    k_codes, k_scale, k_min = oracle.quantise_rows(qkv[:, :, heads:heads + kv])
    v_codes, v_scale, v_min = oracle.quantise_rows(qkv[:, :, heads + kv:])
    v_all = oracle.unpack_v(units[1])
    k_dense = torch.zeros(b, kv, seq, d, dtype=torch.float64, device=cuda)
    v_dense = torch.zeros_like(k_dense)
    q_want = qkv[:, :, :heads].clone()
    for i in range(b):
        for s in range(seq):
            slot = lengths[i] - seq + s
            if slot < 0:
                q_want[i, s] = 0
                continue
            want[0][i, :, slot] = oracle.pack_k(k_codes[i, s])
            v_all[i, :, slot] = v_codes[i, s]
            want[2][i, :, slot] = torch.cat([k_scale[i, s], k_min[i, s], v_scale[i, s], v_min[i, s]], -1).to(dtype)
            k_dense[i, :, s] = k_min[i, s] + k_scale[i, s] * k_codes[i, s]
            v_dense[i, :, s] = v_min[i, s] + v_scale[i, s] * v_codes[i, s]
    want[1] = oracle.pack_v(v_all)
    assert torch.equal(q, q_want)
    for name, got, expected in zip(("k_codes", "v_codes"), cache, want):
        assert torch.equal(got, expected), name
    assert torch.equal(cache[2].view(torch.int16), want[2].view(torch.int16))
    k, v = ops.dequantize_kv4(*cache, n, seq, flag_of(dtype))
    # an exact product, one addition in fp32, one rounding to the type: the 64-bit value rounded in the same two steps
    assert torch.equal(k, k_dense.float().to(dtype)) and torch.equal(v, v_dense.float().to(dtype))
    assert status() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_append_rotates(cuda, dtype):
    """q and k by the angles of their positions.  fp32 multiply-add of two products and one rounding: half a step of the type and
    2**-23 of the magnitudes; the entry read back is within half a code of that, plus the rounding of scale and value."""
    from matgptq_b200 import ops
    b, seq, heads, kv, d, capacity = 2, 19, 4, 2, 128, 64
    gen = torch.Generator(device=cuda).manual_seed(3)
    qkv = torch.randn(b, seq, heads + 2 * kv, d, generator=gen, device=cuda).to(dtype)
    positions = torch.randint(0, 500, (seq,), generator=gen, device=cuda)
    angle = torch.arange(500, device=cuda)[:, None] / 10000 ** (torch.arange(0, d, 2, device=cuda) / d)[None]
    cos, sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    cache = empty_cache(b, kv, capacity, d, dtype, cuda)
    n = lengths_tensor([seq, seq + 30], cuda)
    q = ops.append_kv4(qkv.view(b * seq, -1), positions, cos, sin, n, *cache, heads, flag_of(dtype))
    x = qkv[:, :, :heads + kv].double()
    c, s = cos[positions].double()[None, :, None], sin[positions].double()[None, :, None]
    turned = torch.empty_like(x)
    turned[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    turned[..., 1::2] = x[..., 1::2] * c + x[..., 0::2] * s
    size = x[..., 0::2].abs() + x[..., 1::2].abs()
    near = turned.abs() * half_step(dtype) + 2.0 ** -23 * size.repeat_interleave(2, -1) + torch.finfo(dtype).smallest_normal
    assert ((q.double() - turned[:, :, :heads]).abs() <= near[:, :, :heads]).all()
    k, v = ops.dequantize_kv4(*cache, n, seq, flag_of(dtype))
    k_want = turned[:, :, heads:].transpose(1, 2)
    spread = k_want.max(-1, keepdim=True).values - k_want.min(-1, keepdim=True).values
    # half a code, 15 codes of a scale that is off by half a step, and the value's own roundings
    bound = spread / 15 * 0.5 * (1 + half_step(dtype)) + 16 / 15 * spread * half_step(dtype) + 3 * k_want.abs().max(-1, keepdim=True).values * half_step(dtype)
    assert ((k.double() - k_want).abs() <= bound).all()
    v_codes, v_scale, v_min = oracle.quantise_rows(qkv[:, :, heads + kv:].transpose(1, 2))
    assert torch.equal(v, (v_min + v_scale * v_codes).float().to(dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_append_rounds_the_rotation_once(cuda, dtype):
    """Codes and scales are to the bit those of the rotation in 64 bits, rounded to fp32 and to the type: no code goes by an error of the
    rotation.  q has the bits that the 16-bit cache's operator gives it.  Zero coordinates, small and large values among them."""
    from matgptq_b200 import _native, ops
    b, seq, heads, kv, d, capacity = 4, 500, 6, 2, 128, 512
    gen = torch.Generator(device=cuda).manual_seed(4)
    qkv = torch.randn(b, seq, heads + 2 * kv, d, generator=gen, device=cuda)
    qkv[0, ::7, :, ::5] = 0
    qkv[1] *= 1e-4
    qkv[2, :, :, ::9] *= 500
    qkv = qkv.to(dtype)
    qkv = qkv.contiguous()
    positions = torch.arange(capacity - seq, capacity, device=cuda)
    angle = torch.arange(capacity, device=cuda)[:, None] / 500000 ** (torch.arange(0, d, 2, device=cuda) / d)[None]
    cos, sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    cache = empty_cache(b, kv, capacity, d, dtype, cuda)
    n = lengths_tensor([seq] * b, cuda)
    q = ops.append_kv4(qkv.view(b * seq, -1), positions, cos, sin, n, *cache, heads, flag_of(dtype))
    x = qkv[:, :, :heads + kv].double()
    c, s = cos[positions].double()[None, :, None], sin[positions].double()[None, :, None]
    turned = torch.empty_like(x)
    turned[..., 0::2] = x[..., 0::2] * c - x[..., 1::2] * s
    turned[..., 1::2] = x[..., 1::2] * c + x[..., 0::2] * s
    turned = turned.float().to(dtype)
    q16 = torch.empty(b, heads, seq, d, dtype=dtype, device=cuda)
    k16 = torch.zeros(b, kv, capacity, d, dtype=dtype, device=cuda)
    v16 = torch.zeros_like(k16)
    _native.check(_native.load().matgptq_b200_rope_kv(
        qkv.data_ptr(), positions.data_ptr(), cos.data_ptr(), sin.data_ptr(), q16.data_ptr(), k16.data_ptr(), v16.data_ptr(), b, seq, heads, kv, d,
        capacity, flag_of(dtype), torch.cuda.current_stream().cuda_stream), "rope_kv")
    assert torch.equal(q.transpose(1, 2), q16)
    k_codes, k_scale, k_min = oracle.quantise_rows(turned[:, :, heads:].transpose(1, 2))
    assert torch.equal(oracle.unpack_k(cache[0])[:, :, :seq], k_codes)
    assert torch.equal(cache[2][:, :, :seq, 0:2].double(), torch.cat([k_scale, k_min], -1))


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_are_not_finite_read_back_as_nan(cuda, dtype):
    from matgptq_b200 import ops
    b, seq, heads, kv, d = 1, 4, 1, 1, 64
    qkv = torch.randn(b, seq, 3, d, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(dtype)
    qkv[0, 0, 1, 5], qkv[0, 1, 2, 63], qkv[0, 2, 1, 0] = math.inf, math.nan, -math.inf
    cache = empty_cache(b, kv, 64, d, dtype, cuda)
    n = lengths_tensor([4], cuda)
    cos, sin = plain_tables(4, d, cuda)
    ops.append_kv4(qkv.view(seq, -1), torch.arange(4, device=cuda), cos, sin, n, *cache, heads, flag_of(dtype))
    k, v = ops.dequantize_kv4(*cache, n, 4, flag_of(dtype))
    assert k[0, 0].isnan().all(-1).tolist() == [True, False, True, False] and v[0, 0].isnan().all(-1).tolist() == [False, True, False, False]
    assert not k[0, 0, 1].isnan().any() and not v[0, 0, 0].isnan().any()


def test_what_is_out_of_range_is_reported_and_not_touched(cuda):
    """Entries past the capacity and positions past the tables: status 106, nothing written outside, the context stays usable."""
    from matgptq_b200 import ops
    dtype, b, seq, heads, kv, d, capacity = torch.float16, 2, 3, 2, 1, 64, 64
    qkv = torch.ones(b * seq, (heads + 2 * kv) * d, dtype=dtype, device=cuda)
    store = [torch.cat([t, t]) for t in empty_cache(b, kv, capacity, d, dtype, cuda)]
    cache = [t[:b] for t in store]
    cos, sin = plain_tables(5, d, cuda)
    status()
    ops.append_kv4(qkv, torch.arange(seq, device=cuda), cos, sin, lengths_tensor([capacity + 2, 2 ** 31 - 1], cuda), *cache, heads, 1)
    assert status() == 106
    assert (store[0][b:] == 255).all() and store[2][b:].isnan().all()
    assert (cache[0][1] == 255).all() and (cache[0][0, 0, :capacity - 1] == 255).all() and not (cache[0][0, 0, capacity - 1] == 255).any()
    q = ops.append_kv4(qkv, torch.tensor([0, 5, -1], device=cuda), cos, sin, lengths_tensor([3, 3], cuda), *cache, heads, 1)
    assert status() == 106
    assert q[:, 0].eq(1).all() and q[:, 1:].isnan().all()
    k, v = ops.dequantize_kv4(*cache, lengths_tensor([3, 3], cuda), 3, 1)
    assert k[:, 0, 0].eq(1).all() and k[:, 0, 1:].isnan().all() and v.eq(1).all()
    out = ops.attention_kv4(torch.ones(b, 1, heads, d, dtype=dtype, device=cuda), *cache, lengths_tensor([capacity + 1, 1], cuda), 0, 0, 1.0, 1)
    assert status() == 106 and out[1].eq(1).all()
    new, _ = ops.evict_kv4(*cache, torch.zeros(b, kv, capacity, device=cuda), lengths_tensor([capacity + 1, -5], cuda), capacity, 0, 0, 0, 1)
    assert status() == 106 and new.tolist() == [capacity, 0]


# ---- attention -------------------------------------------------------------------------------------------------------
def check_attention(cuda, dtype, d, b, seq, kv, group, lengths, window=0, sinks=0, capacity=None, seed=0, q_size=1.5, v_size=1.0, weighted=True):
    from matgptq_b200 import ops
    capacity = capacity or -(-max(max(lengths), 1) // 64) * 64
    gen = torch.Generator(device=cuda).manual_seed(seed)
    cache = filled_cache(b, kv, capacity, d, dtype, lengths, cuda, gen, v_size)
    q = (q_size * torch.randn(b, seq, kv * group, d, generator=gen, device=cuda)).to(dtype)
    scale = 1 / math.sqrt(d)
    n = lengths_tensor(lengths, cuda)
    weights = torch.rand(b, kv, capacity, generator=gen, device=cuda) if weighted else None
    before = weights.clone() if weighted else None
    out = ops.attention_kv4(q, *cache, n, window, sinks, scale, flag_of(dtype), weights)
    want, added, near, added_near = oracle.attention(q, *cache, lengths, window, sinks, scale)
    bound = near + want.abs() * half_step(dtype) * (1 + half_step(dtype)) + near * half_step(dtype) + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
    off = (out.double() - want).abs()
    assert not out.isnan().any()
    assert (off <= bound).all(), f"off by {(off / bound).max().item():.3g} times the bound"
    if weighted:
        off = (weights.double() - before.double() - added).abs()
        bound = added_near + 2.0 ** -23 * weights.double().abs()
        assert (off <= bound).all(), f"weights off by {(off / bound).max().item():.3g} times the bound"
        at = torch.arange(capacity, device=cuda)[None, None] >= n[:, None, None]
        assert torch.equal(weights[at.expand_as(weights)], before[at.expand_as(weights)])
        # without weights: the same bits
        assert torch.equal(out, ops.attention_kv4(q, *cache, n, window, sinks, scale, flag_of(dtype)))
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kv, group", [(1, 1), (2, 4), (3, 3), (1, 8), (2, 12), (1, 17)])
def test_attention_of_one_token(cuda, dtype, d, kv, group):
    check_attention(cuda, dtype, d, 6, 1, kv, group, [1, 0, 2, 15, 130, 257])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seq, group", [(2, 4), (3, 1), (5, 2), (5, 4), (17, 1), (33, 3), (70, 4), (130, 1)])
def test_attention_of_several_tokens(cuda, dtype, seq, group):
    """Prompts, pieces of prompts, prompts padded on the left (with rows that see nothing), sequences without any entry."""
    check_attention(cuda, dtype, 128, 5, seq, 2, group, [seq, seq + 61, max(1, seq // 2), 0, 1], seed=seq)


@pytest.mark.parametrize("seq", [1, 4, 40, 150])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 3), (16, 0), (17, 1), (48, 33), (300, 4), (1000, 5), (0, 7)])
def test_attention_with_a_window(cuda, seq, window, sinks):
    check_attention(cuda, torch.float16, 64, 4, seq, 2, 2, [seq + 300, seq + 31, seq, max(1, seq - 1)], window, sinks, capacity=512, seed=window)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_over_many_entries(cuda, dtype):
    """The split over the CTAs of a cluster, and their warps; one sequence far shorter than the others."""
    check_attention(cuda, dtype, 128, 2, 1, 2, 4, [9001, 40], seed=1)
    check_attention(cuda, dtype, 128, 2, 3, 1, 5, [5003, 640], window=700, sinks=9, seed=2)


def test_attention_has_one_order(cuda):
    """The same bits on every run: nothing is added up by atomics."""
    from matgptq_b200 import ops
    gen = torch.Generator(device=cuda).manual_seed(9)
    cache = filled_cache(3, 2, 2048, 128, torch.float16, [2048, 1000, 77], cuda, gen)
    n = lengths_tensor([2048, 1000, 77], cuda)
    for seq in (1, 50):
        q = torch.randn(3, seq, 8, 128, generator=gen, device=cuda).half()
        runs = []
        for _ in range(4):
            w = torch.zeros(3, 2, 2048, device=cuda)
            runs.append((ops.attention_kv4(q, *cache, n, 0, 0, 0.1, 1, w), w))
        for out, w in runs[1:]:
            assert torch.equal(out, runs[0][0]) and torch.equal(w, runs[0][1])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_size, v_size", [(30.0, 1.0), (1e-3, 1.0), (1.5, 1e-4), (1.5, 200.0), (0.0, 1.0)])
def test_attention_of_large_and_small_values(cuda, dtype, q_size, v_size):
    check_attention(cuda, dtype, 128, 2, 1, 2, 4, [300, 33], q_size=q_size, v_size=v_size, seed=5)
    check_attention(cuda, dtype, 128, 2, 40, 2, 4, [300, 60], q_size=q_size, v_size=v_size, seed=6)


def test_attention_of_scales_that_vary_widely(cuda):
    """bf16 entries whose V rows differ by powers of two from 2**-40 to 2**40: the largest ones set the rounding."""
    from matgptq_b200 import ops
    dtype, d, n = torch.bfloat16, 128, 200
    gen = torch.Generator(device=cuda).manual_seed(8)
    cache = filled_cache(1, 1, 256, d, dtype, [n], cuda, gen)
    power = 2.0 ** torch.randint(-40, 41, (n, 1), generator=gen, device=cuda)
    cache[2][0, 0, :n, 2:] = (cache[2][0, 0, :n, 2:].float() * power).to(dtype)
    for seq in (1, 60):
        q = torch.randn(1, seq, 4, d, generator=gen, device=cuda).to(dtype)
        out = ops.attention_kv4(q, *cache, lengths_tensor([n], cuda), 0, 0, 0.1, 3)
        want, _, near, _ = oracle.attention(q, *cache, [n], 0, 0, 0.1)
        assert ((out.double() - want).abs() <= near * 1.01 + want.abs() * half_step(dtype) * 1.01).all()


@pytest.mark.parametrize("seq", [1, 3, 40])
def test_nan_reaches_the_rows_that_see_it_and_no_others(cuda, seq):
    """A NaN in an entry's scale or minimum, of K or of V, in the middle of a sequence, seen or hidden by the causal border or the window."""
    from matgptq_b200 import ops
    dtype, d, kv, group, capacity = torch.float16, 64, 1, 2, 192
    n = [150, 150, 150, 150]
    for column in range(4):
        gen = torch.Generator(device=cuda).manual_seed(column)
        cache = filled_cache(4, kv, capacity, d, dtype, n, cuda, gen)
        q = torch.randn(4, seq, group, d, generator=gen, device=cuda).to(dtype)
        clean = ops.attention_kv4(q, *cache, lengths_tensor(n, cuda), 20, 2, 0.1, 1)
        bad = [150 - 1, 150 - seq, 150 - seq - 5, 60]  # the last token's own entry, the first token's, one in the window, one outside
        for i, j in enumerate(bad):
            cache[2][i, 0, j, column] = math.nan
        out = ops.attention_kv4(q, *cache, lengths_tensor(n, cuda), 20, 2, 0.1, 1)
        for i, j in enumerate(bad):
            seen = oracle.visible(150, seq, 20, 2)[:, j]
            assert out[i].isnan().all(-1).all(-1).cpu().tolist() == seen.tolist(), (column, i)
            assert torch.equal(out[i, ~seen], clean[i, ~seen]), (column, i)


@pytest.mark.parametrize("seq", [1, 40])
def test_infinite_queries_give_nan(cuda, seq):
    from matgptq_b200 import ops
    gen = torch.Generator(device=cuda).manual_seed(2)
    cache = filled_cache(1, 1, 64, 64, torch.float16, [50], cuda, gen)
    q = torch.randn(1, seq, 2, 64, generator=gen, device=cuda).half()
    q[0, 0, 1, 3] = math.inf
    q[0, seq - 1, 0, 9] = math.nan
    out = ops.attention_kv4(q, *cache, lengths_tensor([50], cuda), 0, 0, 0.1, 1)
    rows = out.isnan().all(-1)[0]
    want = torch.zeros_like(rows)
    want[0, 1] = want[seq - 1, 0] = True
    assert torch.equal(rows, want) and torch.equal(out.isnan().any(-1)[0], want)


def test_strides_streams_and_empty_batches(cuda):
    from matgptq_b200 import ops
    gen = torch.Generator(device=cuda).manual_seed(12)
    n = [100, 64]
    cache = filled_cache(2, 2, 128, 128, torch.float16, n, cuda, gen)
    lengths = lengths_tensor(n, cuda)
    q = torch.randn(2, 8, 3, 128, generator=gen, device=cuda).half().transpose(1, 2)  # heads outside in memory
    want = ops.attention_kv4(q.contiguous(), *cache, lengths, 0, 0, 0.1, 1)
    assert torch.equal(ops.attention_kv4(q, *cache, lengths, 0, 0, 0.1, 1), want)
    odd = torch.empty(q.numel() + 1, dtype=torch.float16, device=cuda)[1:].view(q.shape).copy_(q)  # 2 bytes past an aligned address
    assert torch.equal(ops.attention_kv4(odd, *cache, lengths, 0, 0, 0.1, 1), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.attention_kv4(q, *cache, lengths, 0, 0, 0.1, 1)
    side.synchronize()
    assert torch.equal(other, want)
    none = [t[:0] for t in cache]
    assert ops.attention_kv4(q[:0], *none, lengths[:0], 0, 0, 0.1, 1).shape == (0, 3, 8, 128)
    assert ops.attention_kv4(q[:, :0], *cache, lengths, 0, 0, 0.1, 1).shape == (2, 0, 8, 128)
    assert ops.dequantize_kv4(*cache, lengths, 0, 1)[0].shape == (2, 2, 0, 128)


# ---- many rows: enough of them, over all heads, that 256 rows share an entry's operands -----------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("b, seq, kv, group", [(20, 33, 5, 1), (5, 130, 3, 4), (3, 257, 4, 3), (10, 70, 2, 8), (1, 1200, 4, 1),
                                               (8, 300, 10, 2), (19, 33, 8, 8), (160, 35, 1, 1),
                                               (1, 700, 4, 1), (3, 100, 2, 5), (4, 130, 2, 4)])
def test_attention_of_many_rows(cuda, dtype, d, b, seq, kv, group):
    """Prompts of which some are padded on the left (rows that see nothing), later pieces, sequences of one entry and of none."""
    lengths = ([seq, seq + 61, max(1, seq // 2), 0, 1, 129, seq + 200] * 23)[:b]
    check_attention(cuda, dtype, d, b, seq, kv, group, lengths, seed=seq)


@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 3), (17, 1), (64, 0), (65, 64), (128, 129), (200, 4), (1000, 5), (0, 7)])
@pytest.mark.parametrize("kv", [2, 5, 8, 20])  # clusters of four and of two that share the entries, CTAs of 128 rows, more of 256
def test_attention_of_many_rows_with_a_window(cuda, window, sinks, kv):
    check_attention(cuda, torch.float16, 128, 4, 150, kv, 2, [450, 331, 150, 149], window, sinks, capacity=512, seed=window)
    check_attention(cuda, torch.bfloat16, 64, 4, 150, kv, 2, [450, 331, 20, 0], window, sinks, capacity=512, seed=window + 1)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_size, v_size", [(30.0, 1.0), (1e-3, 1.0), (1.5, 1e-4), (1.5, 200.0), (0.0, 1.0)])
@pytest.mark.parametrize("kv", [2, 4, 8, 26])
def test_attention_of_large_and_small_values_in_many_rows(cuda, dtype, q_size, v_size, kv):
    check_attention(cuda, dtype, 128, 2, 160, kv, 2, [300, 160], q_size=q_size, v_size=v_size, seed=6)


@pytest.mark.parametrize("kv", [4, 8, 40])
def test_attention_of_many_rows_over_scales_that_vary_widely(cuda, kv):
    """As test_attention_of_scales_that_vary_widely; the unit of a tile's weights rises and what was added up follows it."""
    from matgptq_b200 import ops
    dtype, d, n = torch.bfloat16, 128, 400
    gen = torch.Generator(device=cuda).manual_seed(8)
    cache = filled_cache(1, kv, 448, d, dtype, [n], cuda, gen)
    power = 2.0 ** torch.randint(-40, 41, (kv, n, 1), generator=gen, device=cuda)
    cache[2][0, :, :n, 2:] = (cache[2][0, :, :n, 2:].float() * power).to(dtype)
    q = torch.randn(1, 160, kv * 4, d, generator=gen, device=cuda).to(dtype)
    out = ops.attention_kv4(q, *cache, lengths_tensor([n], cuda), 0, 0, 0.1, 3)
    want, _, near, _ = oracle.attention(q, *cache, [n], 0, 0, 0.1)
    assert ((out.double() - want).abs() <= near * 1.01 + want.abs() * half_step(dtype) * 1.01).all()


@pytest.mark.parametrize("b, group", [(30, 3), (64, 2), (100, 4)])
def test_nan_reaches_the_rows_that_see_it_among_many(cuda, b, group):
    """As test_nan_reaches_the_rows_that_see_it_and_no_others.  Beside a NaN the other rows keep their bits.  An infinite score makes its
    warp take all its rows' weights against new maxima: by whole powers of two, so with the same error bound, but the exponents
    score - maximum are rounded elsewhere, by half a step of fp32 of the larger of the two: these rows are held to the bound, not the bits."""
    from matgptq_b200 import ops
    dtype, d, kv, capacity, seq = torch.float16, 64, 1, 192, 40
    n = [150] * b
    for column in range(4):
        gen = torch.Generator(device=cuda).manual_seed(column)
        cache = filled_cache(b, kv, capacity, d, dtype, n, cuda, gen)
        q = torch.randn(b, seq, group, d, generator=gen, device=cuda).to(dtype)
        clean = ops.attention_kv4(q, *cache, lengths_tensor(n, cuda), 20, 2, 0.1, 1)
        want, _, near, _ = oracle.attention(q, *cache, n, 20, 2, 0.1)
        bound = near + want.abs() * half_step(dtype) * (1 + half_step(dtype)) + near * half_step(dtype) + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
        bad = [(150 - 1, 150 - seq, 150 - seq - 5, 60, 1, 128)[i % 6] for i in range(b)]
        for i, j in enumerate(bad):
            cache[2][i, 0, j, column] = math.nan if i % 2 else math.inf
        out = ops.attention_kv4(q, *cache, lengths_tensor(n, cuda), 20, 2, 0.1, 1)
        for i, j in enumerate(bad):
            seen = oracle.visible(150, seq, 20, 2)[:, j]
            assert ((out[i].double() - want[i]).abs() <= bound[i])[~seen].all(), (column, i)
            if i % 2:
                assert torch.equal(out[i, ~seen], clean[i, ~seen]), (column, i)
                assert out[i].isnan().all(-1).all(-1).cpu().tolist() == seen.tolist(), (column, i)


@pytest.mark.parametrize("group", [1, 4, 8])
def test_attention_of_many_rows_has_one_order(cuda, group):
    from matgptq_b200 import ops
    gen = torch.Generator(device=cuda).manual_seed(9)
    n = [2048, 1000, 377]
    cache = filled_cache(3, 4, 2048, 128, torch.float16, n, cuda, gen)
    q = torch.randn(3, 300, 4 * group, 128, generator=gen, device=cuda).half()
    runs = []
    for _ in range(4):
        w = torch.zeros(3, 4, 2048, device=cuda)
        runs.append((ops.attention_kv4(q, *cache, lengths_tensor(n, cuda), 0, 0, 0.1, 1, w), w))
    for out, w in runs[1:]:
        assert torch.equal(out, runs[0][0]) and torch.equal(w, runs[0][1])


# ---- long caches: segments that are cut into pieces --------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("seq, group", [(1, 1), (1, 8), (1, 12), (2, 10), (9, 11)])
def test_attention_over_a_long_cache(cuda, dtype, seq, group):
    """One tile of rows and several, a sequence without entries and a short one beside the long one, everything and a window."""
    check_attention(cuda, dtype, 64, 1, seq, 1, group, [20001], seed=seq)
    check_attention(cuda, dtype, 64, 3, seq, 1, group, [33, 18000, 0], seed=seq + 1)
    check_attention(cuda, dtype, 128, 1, seq, 1, group, [20480], 17000, 70, seed=seq + 2)


@pytest.mark.parametrize("seq, group", [(1, 4), (4, 5)])
def test_attention_over_the_caches_of_many_sequences(cuda, seq, group):
    """More sequences than a warp has lanes, more segments than CTAs run at once, lengths from none to all."""
    b = 45
    lengths = [(i * 397) % 2241 for i in range(b)]
    check_attention(cuda, torch.bfloat16, 64, b, seq, 8, group, lengths, capacity=2240, seed=seq)
    check_attention(cuda, torch.float16, 64, b, seq, 1, group, lengths[:44] + [17000], capacity=17024, seed=seq + 1, weighted=seq > 1)


@pytest.mark.parametrize("b, seq, group, weighted", [(149, 1, 3, True), (149, 1, 16, False), (80, 4, 5, True)])
def test_attention_over_pieces_of_many_sequences(cuda, b, seq, group, weighted):
    """Long enough for pieces; more sequences than a warp has lanes, lengths from none to all."""
    lengths = [(i * 1237) % 5313 for i in range(b)]
    check_attention(cuda, torch.bfloat16, 64, b, seq, 1, group, lengths, capacity=5312, seed=b + seq, weighted=weighted)


def test_entries_past_four_gigabytes(cuda):
    """Offsets that pass 32 bits: the last entries of the second head of a cache of 2**26 entries do what they do in a small one."""
    from matgptq_b200 import ops
    d, kv, group, capacity, small = 128, 2, 2, 2 ** 26, 512
    if torch.cuda.mem_get_info()[0] < 24e9:
        pytest.skip("needs 24 GB")
    dtype, gen = torch.float16, torch.Generator(device=cuda).manual_seed(3)
    part = filled_cache(1, kv, small, d, dtype, [small - 3], cuda, gen)
    cache = [torch.empty(1, kv, capacity // r, t.shape[-1], dtype=t.dtype, device=cuda) for r, t in zip((1, 2, 1), part)]
    for t, s in zip(cache, part):
        t[:, :, -s.shape[2]:] = s
    scale = 0.1
    for seq in (1, 20, 1300):
        rows = min(seq, 100)
        q = torch.randn(1, seq, kv * group, d, generator=gen, device=cuda).half()
        n = capacity - 3
        if seq >= small:  # the first tokens' windows lie in front of what is compared
            for t, r in zip(cache, (1, 2, 1)):
                t[:, :, (capacity - 4096) // r:(capacity - small) // r] = 0
        out = ops.attention_kv4(q, *cache, lengths_tensor([n], cuda), 100, 0, scale, 1)[:, -rows:]
        want, _, near, _ = oracle.attention(q[:, -rows:].contiguous(), *part, [small - 3], 100, 0, scale)
        bound = near + want.abs() * half_step(dtype) * (1 + half_step(dtype)) + near * half_step(dtype) + torch.finfo(dtype).smallest_normal * half_step(dtype) * 2
        assert ((out.double() - want).abs() <= bound).all(), seq
    # three more, written and read back
    qkv = torch.randn(3, (kv * group + 2 * kv) * d, generator=gen, device=cuda).half()
    cos, sin = plain_tables(4, d, cuda)
    for t, length in ((cache, capacity), (part, small)):
        ops.append_kv4(qkv, torch.arange(3, device=cuda), cos, sin, lengths_tensor([length], cuda), *t, kv * group, 1)
    for big, little in zip(ops.dequantize_kv4(*cache, lengths_tensor([capacity], cuda), 20, 1), ops.dequantize_kv4(*part, lengths_tensor([small], cuda), 20, 1)):
        assert torch.equal(big, little)
    # and the last ones kept
    weights = torch.zeros(1, kv, capacity, device=cuda)
    weights[:, :, -small:] = 1 + torch.rand(1, kv, small, generator=gen, device=cuda)
    order = weights[0, :, -small:].clone()
    rows = oracle.unpack_k(part[0])
    new, kept = ops.evict_kv4(*cache, weights, lengths_tensor([capacity], cuda), 100, 0, 0, 0, 1)
    for head in range(kv):
        at = order[head].topk(100).indices.sort().values
        assert (kept[0, head] == at + capacity - small).all()
        assert torch.equal(oracle.unpack_k(cache[0][:, :, :128])[0, head, :100], rows[0, head, at])
    assert new.tolist() == [100] and status() == 0


# ---- ways to call ------------------------------------------------------------------------------------------------------
def test_the_operators_with_and_without_a_dispatch_mode(cuda):
    """A mode sees every one of them, and what they answer is the same; what they write to is marked as written."""
    from torch.utils._python_dispatch import TorchDispatchMode

    from matgptq_b200 import ops

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(func._schema.name.split("::")[-1])
            return func(*args, **(kwargs or {}))

    b, seq, heads, kv, d, capacity = 2, 3, 4, 2, 64, 64
    gen = torch.Generator(device=cuda).manual_seed(5)
    qkv = torch.randn(b * seq, (heads + 2 * kv) * d, generator=gen, device=cuda).half()
    cos, sin = plain_tables(seq, d, cuda)
    n, positions = lengths_tensor([9, 5], cuda), torch.arange(seq, device=cuda)

    def run():
        start = torch.Generator(device=cuda).manual_seed(6)
        cache = filled_cache(b, kv, capacity, d, torch.float16, [6, 2], cuda, start)
        weights = torch.zeros(b, kv, capacity, device=cuda)
        versions = [t._version for t in (*cache, weights)]
        q = ops.append_kv4(qkv, positions, cos, sin, n, *cache, heads, 1)
        out = ops.attention_kv4(q, *cache, n, 4, 1, 0.125, 1, weights)
        new, kept = ops.evict_kv4(*cache, weights, n, 4, 0, 1, 1, 1)
        k, v = ops.dequantize_kv4(*cache, new, 4, 1)
        assert all(t._version > old for t, old in zip((*cache, weights), versions))
        return q, out, new, kept, k, v, weights

    plain = run()
    with Seen() as mode:
        moded = run()
    assert all(torch.equal(x, y) for x, y in zip(plain, moded))
    assert all(any(name == want for name in mode.names) for want in ("append_kv4", "attention_kv4", "evict_kv4", "dequantize_kv4"))


def test_two_streams_at_once(cuda):
    """Calls in flight at the same time have workspaces of their own."""
    from matgptq_b200 import ops
    gen = torch.Generator(device=cuda).manual_seed(13)
    n = lengths_tensor([20000], cuda)
    caches = [filled_cache(1, 1, 20032, 64, torch.float16, [20000], cuda, gen) for _ in range(2)]
    qs = [torch.randn(1, 1, 8, 64, generator=gen, device=cuda).half() for _ in range(2)]
    want = [ops.attention_kv4(q, *c, n, 0, 0, 0.1, 1) for q, c in zip(qs, caches)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(ops.attention_kv4(qs[i], *caches[i], n, 0, 0, 0.1, 1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, want[i]) for i in range(2) for x in got[i])


def test_two_graphs_replayed_in_turn(cuda):
    """Captured calls with workspaces, in two graphs of one pool, replayed one after the other and again with other lengths."""
    from matgptq_b200 import ops
    gen = torch.Generator(device=cuda).manual_seed(14)
    cache = filled_cache(2, 1, 20032, 64, torch.float16, [20000, 19000], cuda, gen)
    q1, q2 = (torch.randn(2, s, 8, 64, generator=gen, device=cuda).half() for s in (1, 70))
    n = lengths_tensor([20000, 17000], cuda)
    ws = [torch.zeros(2, 1, 20032, device=cuda) for _ in range(2)]

    def eager():
        w = [torch.zeros_like(x) for x in ws]
        return [ops.attention_kv4(q, *cache, n, 0, 0, 0.1, 1, x) for q, x in zip((q1, q2), w)] + w

    eager()
    graphs, outs = [], []
    for q, w in zip((q1, q2), ws):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(ops.attention_kv4(q, *cache, n, 0, 0, 0.1, 1, w))
        graphs.append(g)
    for lengths in ([20000, 17000], [100, 19000], [0, 71]):
        n.copy_(lengths_tensor(lengths, cuda))
        for w in ws:
            w.zero_()
        want = eager()
        for g, out, expected in zip(graphs, outs, want):
            g.replay()
            assert torch.equal(out, expected)
        assert all(torch.equal(x, y) for x, y in zip(ws, want[2:]))


# ---- eviction --------------------------------------------------------------------------------------------------------
def check_eviction(cuda, weights, lengths, keep, slack=0, sinks=0, recent=0, d=64, dtype=torch.float16):
    from matgptq_b200 import ops
    b, kv, capacity = weights.shape
    gen = torch.Generator(device=cuda).manual_seed(keep)
    cache = filled_cache(b, kv, capacity, d, dtype, lengths, cuda, gen)
    before = [t.clone() for t in cache]
    k_rows, v_rows = oracle.unpack_k(cache[0]), oracle.unpack_v(cache[1])
    w = weights.clone()
    new, kept = ops.evict_kv4(*cache, w, lengths_tensor(lengths, cuda), keep, slack, sinks, recent, flag_of(dtype))
    k_now, v_now = oracle.unpack_k(cache[0]), oracle.unpack_v(cache[1])
    host = weights.cpu()
    for i in range(b):
        cut = lengths[i] > keep + slack
        assert new[i].item() == (keep if cut else lengths[i])
        for j in range(kv):
            stay = oracle.evict(host[i, j], lengths[i], keep, slack, sinks, recent)
            assert (stay is not None) == cut
            if not cut:
                assert (kept[i, j] == -1).all()
                assert torch.equal(w[i, j].view(torch.int32), weights[i, j].view(torch.int32))
                assert all(torch.equal(a[i, j].view(torch.uint8), c[i, j].view(torch.uint8)) for a, c in zip(cache, before))
                continue
            at = torch.tensor(stay, device=cuda)
            assert kept[i, j].tolist() == stay
            assert torch.equal(k_now[i, j, :keep], k_rows[i, j, at]) and torch.equal(v_now[i, j, :keep], v_rows[i, j, at])
            assert torch.equal(cache[2][i, j, :keep].view(torch.int16), before[2][i, j, at].view(torch.int16))
            assert torch.equal(w[i, j, :keep].view(torch.int32), weights[i, j, at].view(torch.int32))
            assert (w[i, j, keep:lengths[i]] == 0).all()
            assert torch.equal(w[i, j, lengths[i]:].view(torch.int32), weights[i, j, lengths[i]:].view(torch.int32))
            # what lies behind the last entry is as it was
            assert torch.equal(k_now[i, j, keep:], k_rows[i, j, keep:]) and torch.equal(v_now[i, j, keep:], v_rows[i, j, keep:])
            assert torch.equal(cache[2][i, j, keep:].view(torch.int16), before[2][i, j, keep:].view(torch.int16))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("keep, slack, sinks, recent", [(1, 0, 0, 0), (1, 0, 1, 0), (40, 0, 4, 16), (41, 0, 0, 41), (63, 3, 2, 0), (64, 0, 60, 4),
                                                        (100, 20, 5, 31), (128, 0, 0, 0)])
def test_evict(cuda, dtype, d, keep, slack, sinks, recent):
    gen = torch.Generator(device=cuda).manual_seed(keep + recent)
    weights = torch.rand(5, 2, 128, generator=gen, device=cuda)
    check_eviction(cuda, weights, [128, 101, 65, 1, 0], keep, slack, sinks, recent, d, dtype)


def test_evict_ties_and_odd_weights(cuda):
    """Equal weights stay from the front; zeros of both signs are equal; NaN is the largest; infinities and negative weights have their order."""
    gen = torch.Generator(device=cuda).manual_seed(1)
    weights = torch.randint(0, 4, (6, 2, 192), generator=gen, device=cuda).float()
    weights[1] = 0.5
    weights[2] = torch.where(torch.rand(2, 192, generator=gen, device=cuda) < 0.5, -0.0, 0.0)
    weights[3, :, ::7] = math.nan
    weights[3, :, 1::7] = -math.nan
    weights[4, :, ::5] = math.inf
    weights[4, :, 1::5] = -math.inf
    weights[5] -= 2
    check_eviction(cuda, weights, [192, 192, 191, 192, 190, 189], 77, 0, 3, 20)
    check_eviction(cuda, weights, [192, 192, 191, 192, 190, 189], 20)


def test_evict_many_entries(cuda):
    gen = torch.Generator(device=cuda).manual_seed(2)
    weights = torch.randn(2, 3, 8192, generator=gen, device=cuda).exp()
    weights[0, 1] = weights[0, 1].half().float()  # many equal ones
    check_eviction(cuda, weights, [8191, 5003], 3001, 0, 4, 1000, 128)
    check_eviction(cuda, weights, [8191, 5003], 8190, 0, 4, 100, 128)


# ---- refusals --------------------------------------------------------------------------------------------------------
def test_refusals(cuda):
    from matgptq_b200 import ops
    b, kv, h, d, capacity = 2, 2, 4, 64, 64
    cache = empty_cache(b, kv, capacity, d, torch.float16, cuda)
    n = lengths_tensor([1, 1], cuda)
    q = torch.zeros(b, 1, h, d, dtype=torch.float16, device=cuda)
    w = torch.zeros(b, kv, capacity, device=cuda)
    attend = lambda q=q, c=cache, n=n, window=0, sinks=0, flag=1, w=None: ops.attention_kv4(q, *c, n, window, sinks, 1.0, flag, w)  # noqa: E731
    attend()
    for bad, match in ((dict(q=q.float()), "q must be"), (dict(q=q[:1]), "q must be"), (dict(q=q[:, :, :3]), "multiple of the cache's"),
                       (dict(q=q[..., :32]), "q must be"), (dict(q=q.cpu()), "on the GPU"), (dict(n=n.long()), "lengths"), (dict(n=n[:1]), "lengths"),
                       (dict(n=n.cpu()), "same GPU"), (dict(flag=3), "params must be"), (dict(window=-1), "negative"), (dict(sinks=-1), "negative"),
                       (dict(w=w.half()), "weights"), (dict(w=w[:, :, :63]), "weights"), (dict(w=w.cpu()), "weights"),
                       (dict(c=[cache[0][:, :, :60], *cache[1:]]), "multiple of 64"), (dict(c=[cache[0][..., :24], *cache[1:]]), "head dimension"),
                       (dict(c=[cache[0], cache[1][:, :1], cache[2]]), "v_codes"), (dict(c=[cache[0], cache[1], cache[2][..., :3]]), "params"),
                       (dict(c=[cache[0].expand(b, kv, capacity, d // 2).transpose(0, 1), cache[1], cache[2]]), "contiguous")):
        with pytest.raises(RuntimeError, match=match):
            attend(**bad)
    evict = lambda w=w, keep=8, slack=0, sinks=0, recent=0: ops.evict_kv4(*cache, w, n, keep, slack, sinks, recent, 1)  # noqa: E731
    for bad, match in ((dict(w=w[:1]), "weights"), (dict(keep=0), "keep"), (dict(keep=65), "keep"), (dict(slack=-1), "slack"), (dict(sinks=5, recent=4), "fit"),
                       (dict(recent=-1), "fit")):
        with pytest.raises(RuntimeError, match=match):
            evict(**bad)
    cos, sin = plain_tables(4, d, cuda)
    pos = torch.zeros(1, dtype=torch.int64, device=cuda)
    qkv = torch.zeros(b, (h + 2 * kv) * d, dtype=torch.float16, device=cuda)
    append = lambda qkv=qkv, pos=pos, cos=cos, sin=sin, h=h: ops.append_kv4(qkv, pos, cos, sin, n, *cache, h, 1)  # noqa: E731
    append()
    for bad, match in ((dict(qkv=qkv[:, :64]), "qkv"), (dict(qkv=torch.cat([qkv, qkv[:1]])), "same number"), (dict(qkv=qkv.float()), "qkv"),
                       (dict(pos=pos.int()), "positions"), (dict(pos=torch.zeros(2, dtype=torch.int64, device=cuda)), "positions"), (dict(cos=cos.half()), "cos_table"),
                       (dict(sin=sin[:2]), "cos_table"), (dict(h=5), "qkv"), (dict(cos=cos[:, :16], sin=sin[:, :16]), "cos_table")):
        with pytest.raises(RuntimeError, match=match):
            append(**bad)
    with pytest.raises(RuntimeError, match="negative"):
        ops.dequantize_kv4(*cache, n, -1, 1)


def test_gradients_are_refused_and_writes_are_counted(cuda):
    from matgptq_b200 import ops
    cache = empty_cache(1, 1, 64, 64, torch.float16, cuda)
    n = lengths_tensor([1], cuda)
    cos, sin = plain_tables(4, 64, cuda)
    versions = [t._version for t in cache]
    qkv = torch.randn(1, 3 * 64, device=cuda).half().requires_grad_()
    q = ops.append_kv4(qkv, torch.zeros(1, dtype=torch.int64, device=cuda), cos, sin, n, *cache, 1, 1)
    assert [t._version for t in cache] == [v + 1 for v in versions]
    w = torch.zeros(1, 1, 64, device=cuda)
    out = ops.attention_kv4(q, *cache, n, 0, 0, 1.0, 1, w)
    assert w._version == 1
    with pytest.raises(RuntimeError, match="derivative"):
        out.float().sum().backward()


# ---- a run of them ---------------------------------------------------------------------------------------------------
def run_steps(cuda, use_graph, dtype=torch.float16):
    """A prompt of unequal lengths, padded on the left, then single tokens with eviction; every step's output, weights and lengths."""
    from matgptq_b200.kv_cache import KV4Cache
    layers, b, heads, kv, d, keep, slack = 2, 3, 4, 2, 64, 40, 6
    gen = torch.Generator(device=cuda).manual_seed(21)
    cache = KV4Cache(layers, b, kv, d, 128, dtype=dtype, device=cuda, weights=True)
    angle = torch.arange(200, device=cuda)[:, None] / 10000 ** (torch.arange(0, d, 2, device=cuda) / d)[None]
    cos, sin = angle.cos().float().contiguous(), angle.sin().float().contiguous()
    seq, valid = 30, torch.tensor([30, 11, 1], dtype=torch.int32, device=cuda)
    cache.advance(seq, valid)
    positions = (torch.arange(seq, device=cuda)[None] - (seq - valid[:, None])).clamp(min=0)
    outs = []
    for i in range(layers):
        x = torch.randn(b * seq, (heads + 2 * kv) * d, generator=gen, device=cuda).to(dtype)
        outs.append(cache.attend(i, cache.append(i, x, positions, cos, sin, heads), window=25, sinks=2))
    inputs = torch.randn(30, layers, b, (heads + 2 * kv) * d, generator=gen, device=cuda).to(dtype)
    x, at = inputs[0].clone(), valid.long()[:, None].clone()

    def step():
        cache.lengths.add_(1)
        got = [cache.attend(i, cache.append(i, x[i], at, cos, sin, heads, pdl=True), window=25, sinks=2, pdl=True) for i in range(layers)]
        cache.evict(keep, slack, sinks=2, recent=10, pdl=True)
        at.add_(1)
        return torch.stack(got)

    graph, out = None, None
    if use_graph:
        saved = [t.clone() for t in cache.tensors()], at.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        for t, s in zip(cache.tensors(), saved[0]):
            t.copy_(s)
        at.copy_(saved[1])
    for s in range(30):
        x.copy_(inputs[s])
        if graph is not None:
            graph.replay()
            outs.append(out.clone())
        else:
            outs.append(step())
    return outs, [t.clone() for t in cache.tensors()], cache


def test_steps_eager_and_captured(cuda):
    eager, tensors, cache = run_steps(cuda, False)
    captured, tensors_captured, _ = run_steps(cuda, True)
    assert all(torch.equal(a, c) for a, c in zip(eager, captured))
    assert all(torch.equal(a.view(torch.uint8), c.view(torch.uint8)) for a, c in zip(tensors, tensors_captured))
    # the first: 30 + 17 = 47 is over keep + slack and cut to 40, so is 40 + 7 in the 24th step; six more steps
    assert cache.lengths.tolist() == [46, 41, 31]
    assert not any(t.isnan().any() for t in eager)
    assert status() == 0


def test_two_captured_graphs_do_not_share_state(cuda):
    """Attention with weights needs a workspace: two graphs that are replayed at the same time on two streams have one each."""
    from matgptq_b200 import ops
    gen = torch.Generator(device=cuda).manual_seed(31)
    n = lengths_tensor([500], cuda)
    sides = []
    for _ in range(2):
        cache = filled_cache(1, 2, 512, 128, torch.float16, [500], cuda, gen)
        q = torch.randn(1, 60, 8, 128, generator=gen, device=cuda).half()
        w = torch.zeros(1, 2, 512, device=cuda)
        want = ops.attention_kv4(q, *cache, n, 0, 0, 0.1, 1, w)
        want_w = w.clone()
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = ops.attention_kv4(q, *cache, n, 0, 0, 0.1, 1, w)
        sides.append((graph, out, w, want, want_w, cache, q))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(10):
        for _, out, w, *_ in sides:
            out.zero_(), w.zero_()
        torch.cuda.synchronize()
        for (graph, *_), stream in zip(sides, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, out, w, want, want_w, *_ in sides:
            assert torch.equal(out, want) and torch.equal(w, want_w)


def test_a_cache_without_heads_is_refused(cuda):
    """By a message: the number of heads is divided by the cache's."""
    from matgptq_b200 import ops
    cache = [t[:, :0] for t in empty_cache(2, 1, 64, 64, torch.float16, cuda)]
    n = lengths_tensor([1, 1], cuda)
    for call in (lambda: ops.attention_kv4(torch.zeros(2, 1, 4, 64, dtype=torch.float16, device=cuda), *cache, n, 0, 0, 1.0, 1),
                 lambda: ops.dequantize_kv4(*cache, n, 1, 1), lambda: ops.evict_kv4(*cache, torch.zeros(2, 0, 64, device=cuda), n, 1, 0, 0, 0, 1)):
        with pytest.raises(RuntimeError, match="at least one key/value head"):
            call()


@pytest.mark.parametrize("name", ["append_kv4", "attention_kv4", "evict_kv4", "dequantize_kv4"])
def test_schema_and_fake_agree(cuda, name):
    gen = torch.Generator(device=cuda).manual_seed(41)
    cache = filled_cache(2, 2, 64, 64, torch.float16, [20, 7], cuda, gen)
    n = lengths_tensor([20, 7], cuda)
    cos, sin = plain_tables(8, 64, cuda)
    w = torch.rand(2, 2, 64, generator=gen, device=cuda)
    args = {"append_kv4": (torch.randn(4, 8 * 64, generator=gen, device=cuda).half(), torch.zeros(2, dtype=torch.int64, device=cuda), cos, sin, n, *cache, 4, 1),
            "attention_kv4": (torch.randn(2, 2, 4, 64, generator=gen, device=cuda).half(), *cache, n, 3, 1, 0.1, 1, w),
            "evict_kv4": (*cache, w, n, 9, 0, 1, 2, 1), "dequantize_kv4": (*cache, n, 5, 1)}[name]
    torch.library.opcheck(getattr(torch.ops.matgptq_cuda, name).default, args, test_utils=("test_schema", "test_faketensor"))
