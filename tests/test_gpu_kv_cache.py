"""The 8-bit key/value cache and the attention over it, on the GPU, against oracle/kv_cache.py in 64 bits.

Bounds, from the roundings made (eps / 2 of a type: bf16 2^-8, fp16 2^-11, fp32 2^-24):
 * whole numbers are equal, scales equal to the correctly rounded fp32 quotient;
 * a value read back is the fp32 product of whole number and scale, rounded to bf16: equal bit for bit;
 * attention: a score is an fp32 sum of D products times a scale, so it is off by at most e_s = (D + 4) 2^-24 of
   scale sum_d |q_d k_d|; q in fp16 adds 2^-24 of the row's largest q per value, within (D + 4) 2^-24 of the same
   sum's bound with |q| at its largest, which the tests allow for by 2^-23 |q|max sum_d |k_d| scale.  A weight is off
   by 2 e_s + 2^-21 (exponential) + 2^-11 (fp16) relative, the normaliser by as much without the 2^-11, and sums of
   n terms by n 2^-24; the output by 2^-8 relative for bf16.
"""
from __future__ import annotations

import pytest
import torch

import hlm_attn
from oracle import kv_cache as oracle

pytestmark = [pytest.mark.gpu]
BF16 = torch.bfloat16


def _rand(g, *shape, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).bfloat16()


def plain_of(cache) -> tuple:
    """The device cache's contents as plain ones: (codes, scales) of k and of v."""
    B, Hkv, S, D = cache.batch, cache.n_kv_head, cache.capacity, cache.kernel_dim
    k = cache.k.cpu().long() - 128  # token / 16, dim / 16, token % 16, dim % 16
    k = k.permute(0, 1, 2, 4, 3, 5).reshape(B, Hkv, S, D)
    v = cache.v.cpu().long().view(B, Hkv, S // 64, D // 16, 4, 16, 4, 4) - 128  # block, dim / 16, g, dim % 16, t, i: token 16 t + 4 g + i
    v = v.permute(0, 1, 2, 6, 4, 7, 3, 5).reshape(B, Hkv, S, D)
    return (k, cache.k_scale.cpu().double()), (v, cache.v_scale.cpu().double())


def filled(g, B, capacity, Hkv, D, k=None, v=None):
    """A cache with all positions written, and its plain form."""
    cache = hlm_attn.KVCache(B, capacity, Hkv, D)
    k = _rand(g, B, cache.capacity, Hkv, D) if k is None else k
    v = _rand(g, B, cache.capacity, Hkv, D) if v is None else v
    hlm_attn.kv_cache_write_hip(cache, k.cuda(), v.cuda(), 0)
    return cache, [tuple(t.transpose(1, 2) for t in oracle.encode(x)) for x in (k, v)]


def int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check_attention(out, q, k, v, starts, counts, window=None, scale=None, prefix=None):
    o, a, reach = oracle.attention(q, k, v, starts, counts, window, scale, prefix)
    D = q.shape[3]
    n = k[0].shape[2] + (prefix[0][0].shape[2] if prefix else 0)
    kmax = max((c[0].abs().sum(-1) * c[1]).nan_to_num().max().item() for c in ([k] + ([prefix[0]] if prefix else [])))
    e_s = (D + 4) * 2.0**-24 * reach + 2.0**-23 * q.double().abs().amax(-1) * kmax * (D**-0.5 if scale is None else scale)
    rel = 4 * e_s + 2.0**-20 + 2.0**-11 + n * 2.0**-23
    tol = 2.0**-8 * o.abs() + a * rel[..., None] * (1 + 2.0**-8) + 1e-30
    err = (out.double().cpu() - o).abs()
    assert out.dtype == BF16 and out.shape == q.shape
    assert torch.isfinite(out).all()
    worst = (err / tol).max().item() if err.numel() else 0.0
    assert worst <= 1.0, f"error {worst:.3f} of its bound, at {(err / tol).argmax().item()}"


# --- writing and reading -------------------------------------------------------------


WRITES = [
    # B, T, Hkv, D, capacity, starts, counts
    (1, 1, 1, 64, 64, [0], None),
    (3, 1, 2, 64, 192, [0, 63, 130], None),
    (2, 1, 3, 128, 128, [64, 127], [1, 0]),
    (2, 63, 2, 64, 256, [0, 65], None),
    (2, 64, 1, 128, 256, [64, 3], None),
    (3, 130, 3, 64, 320, [0, 61, 190], [130, 77, 130]),
    (2, 200, 4, 128, 448, [1, 248], [199, 200]),
    (4, 70, 2, 64, 128, [-5, 100, 128, -80], [70, 70, 70, 70]),  # partly or wholly outside
    (1, 300, 12, 64, 384, [17], None),
]


@pytest.mark.parametrize("B,T,Hkv,D,capacity,starts,counts", WRITES)
def test_write_stores_the_nearest_whole_numbers_and_nothing_else(B, T, Hkv, D, capacity, starts, counts):
    g = torch.Generator().manual_seed(B * 1000 + T)
    cache, plain = filled(g, B, capacity, Hkv, D)
    k = _rand(g, B, T, Hkv, D, scale=3.0)
    fused = _rand(g, B, T, (2 * Hkv + 1) * D)
    v = fused[..., D : (Hkv + 1) * D].view(B, T, Hkv, D)
    hlm_attn.kv_cache_write_hip(cache, k.cuda(), fused.cuda()[..., D : (Hkv + 1) * D].view(B, T, Hkv, D), int32(starts),
                                None if counts is None else int32(counts))
    n = [T] * B if counts is None else counts
    for (codes, scales), x in zip(plain, (k, v)):
        oracle.write(codes, scales, x, starts, n)
    for (codes, scales), (want_c, want_s) in zip(plain_of(cache), plain):
        assert torch.equal(codes, want_c) and torch.equal(scales, want_s)
    got = hlm_attn.kv_cache_read_hip(cache, int32(starts), T, None if counts is None else int32(counts))
    for x, (codes, scales) in zip(got, plain):
        want = oracle.read(codes, scales, T, starts, n).float().bfloat16()
        assert torch.equal(x.cpu(), want)


def test_rows_that_are_zero_tiny_huge_tied_or_not_finite():
    D = 64
    x = torch.zeros(1, 9, 1, D)
    g = torch.Generator().manual_seed(5)
    x[0, 1] = 1e-37 * torch.randn(D, generator=g)  # below 2^-119
    x[0, 2] = 2.0**-119
    x[0, 3] = 3.38e38 * torch.rand(D, generator=g)
    x[0, 4] = torch.arange(D) * 2.0 - 63  # odd values of a row whose largest is 254: ties
    x[0, 4, 0, 0] = 254.0
    x[0, 5, 0, 7] = float("inf")
    x[0, 6, 0, 9] = float("nan")
    x[0, 7] = torch.randn(D, generator=g)
    x[0, 7, 0, 63] = -1e4
    x[0, 8, 0, 1] = -0.0
    x = x.bfloat16()
    cache = hlm_attn.KVCache(1, 64, 1, D)
    hlm_attn.kv_cache_write_hip(cache, x.cuda(), x.cuda(), 3)
    codes, scales = oracle.encode(x)
    for got_c, got_s in plain_of(cache):
        assert torch.equal(got_c[:, :, 3:12], codes.transpose(1, 2))
        assert torch.equal(torch.isnan(got_s[:, :, 3:12]), torch.isnan(scales.transpose(1, 2)))
        assert torch.equal(got_s[:, :, 3:12].nan_to_num(), scales.transpose(1, 2).nan_to_num())
    k, v = hlm_attn.kv_cache_read_hip(cache, 3, 9)
    assert torch.isnan(k[0, 5:7]).all() and torch.isnan(v[0, 5:7]).all()
    assert torch.isfinite(k[0, [0, 1, 2, 3, 4, 7, 8]]).all() and not k[0, [0, 1, 8]].any()


def test_unwritten_positions_read_as_zeros():
    cache = hlm_attn.KVCache(2, 100, 2, 64)
    assert cache.capacity == 128
    cache.k.fill_(255), cache.v.fill_(255)
    for x in hlm_attn.kv_cache_read_hip(cache, 0, 128):
        assert not x.any()
    assert hlm_attn.kv_cache_read_hip(cache, 0, 0)[0].shape == (2, 0, 2, 64)


# --- attention -----------------------------------------------------------------------


ATTENDS = [
    # B, T, H, Hkv, D, capacity, starts, counts, window
    (1, 1, 1, 1, 64, 64, [0], None, None),
    (1, 1, 4, 4, 64, 128, [63], None, None),
    (1, 1, 12, 4, 128, 192, [64], None, None),
    (3, 1, 6, 2, 64, 512, [0, 300, 511], None, None),
    (2, 1, 12, 12, 64, 1024, [1000, 700], None, 512),
    (2, 1, 8, 1, 128, 640, [639, 64], None, 1),
    (2, 4, 6, 2, 64, 320, [100, 316], [4, 3], None),
    (2, 5, 16, 4, 128, 320, [0, 200], None, 65),
    (1, 33, 4, 4, 64, 192, [70], None, None),
    (2, 70, 6, 2, 64, 320, [13, 100], [70, 41], 50),
    (2, 70, 3, 1, 128, 320, [13, 100], [70, 41], None),
    (3, 7, 4, 2, 64, 64, [-3, 60, 200], None, None),  # queries at positions outside the cache
    (2, 6, 4, 2, 64, 128, [50, 90], [0, 6], None),  # a sequence without queries
    (1, 20, 4, 1, 64, 4096, [4000], None, None),
    (1, 1, 16, 16, 128, 2048, [2047], None, 1000),
]


@pytest.mark.parametrize("B,T,H,Hkv,D,capacity,starts,counts,window", ATTENDS)
def test_attention_over_a_cache(B, T, H, Hkv, D, capacity, starts, counts, window):
    g = torch.Generator().manual_seed(T * 100 + H)
    cache, (k, v) = filled(g, B, capacity, Hkv, D)
    q = _rand(g, B, T, H, D, scale=1.5)
    out = hlm_attn.cached_attention_hip(q.cuda(), cache, int32(starts), None if counts is None else int32(counts), window)
    check_attention(out, q, k, v, starts, [T] * B if counts is None else counts, window)
    if len(set(starts)) == 1 and starts[0] + T <= capacity:  # one place that the host knows
        same = hlm_attn.cached_attention_hip(q.cuda(), cache, starts[0], None if counts is None else int32(counts), window)
        check_attention(same, q, k, v, starts, [T] * B if counts is None else counts, window)


PREFIXES = [
    # B, T, H, Hkv, D, capacity, starts, counts, window, P
    (1, 1, 2, 2, 64, 64, [0], None, None, 1),
    (3, 1, 6, 2, 64, 128, [0, 64, 100], None, None, 200),
    (4, 9, 4, 4, 64, 64, [0, 0, 0, 0], [9, 1, 0, 5], None, 333),
    (4, 9, 4, 4, 64, 64, [0, 0, 0, 0], [9, 1, 0, 5], 40, 333),
    (2, 5, 12, 4, 128, 192, [3, 150], None, 100, 64),  # the second sequence is past the prefix
    (5, 3, 8, 1, 128, 64, [1, 2, 3, 4, 61], None, None, 1000),
    (2, 40, 6, 2, 64, 128, [10, 20], None, 130, 190),
    (2, 3, 4, 2, 64, 64, [-1, 62], None, None, 100),  # outside the own cache
    (40, 1, 4, 2, 64, 64, list(range(40)), None, None, 130),
]


@pytest.mark.parametrize("B,T,H,Hkv,D,capacity,starts,counts,window,P", PREFIXES)
def test_attention_with_a_shared_prefix(B, T, H, Hkv, D, capacity, starts, counts, window, P):
    g = torch.Generator().manual_seed(P)
    cache, (k, v) = filled(g, B, capacity, Hkv, D)
    shared, plain = filled(g, 1, P, Hkv, D)
    q = _rand(g, B, T, H, D, scale=1.5)
    out = hlm_attn.cached_attention_hip(
        q.cuda(), cache, int32(starts), None if counts is None else int32(counts), window, prefix=shared, prefix_length=P
    )
    prefix = [(c[:, :, :P], s[:, :, :P]) for c, s in plain]
    check_attention(out, q, k, v, starts, [T] * B if counts is None else counts, window, prefix=prefix)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,window", [(1, None), (1, 70), (40, None), (40, 33)])
def test_masked_slots_may_hold_anything(D, T, window):
    """Slots behind a sequence, and before its window, hold NaN scales and any bytes."""
    g = torch.Generator().manual_seed(3)
    B, H, Hkv, starts = 2, 4, 2, [90, 5]
    cache, (k, v) = filled(g, B, 192, Hkv, D)
    q = _rand(g, B, T, H, D)
    clean = hlm_attn.cached_attention_hip(q.cuda(), cache, int32(starts), None, window)
    for b, s in enumerate(starts):
        dead = list(range(s + T, 192)) + (list(range(0, max(0, s - window + 1))) if window else [])
        cache.k_scale[b, :, dead] = float("nan")
        cache.v_scale[b, :, dead] = float("nan")
        cache.k[b, :, [i for i in range(192 // 16) if all(p in dead for p in range(16 * i, 16 * i + 16))]] = 255
    out = hlm_attn.cached_attention_hip(q.cuda(), cache, int32(starts), None, window)
    assert torch.equal(out, clean)
    check_attention(out, q, k, v, starts, [T] * B, window)


def test_a_key_that_is_nan_reaches_the_rows_that_see_it_and_no_other():
    g = torch.Generator().manual_seed(4)
    cache, (k, v) = filled(g, 2, 128, 2, 64)
    q = _rand(g, 2, 6, 4, 64)
    cache.k_scale[0, 1, 93] = float("nan")
    cache.v_scale[1, 0, 92] = float("nan")
    out = hlm_attn.cached_attention_hip(q.cuda(), cache, 90)
    nan = torch.isnan(out).all(-1).cpu()
    want = torch.zeros(2, 6, 4, dtype=torch.bool)
    want[0, 3:, 2:] = True
    want[1, 2:, :2] = True
    assert torch.equal(nan, want) and torch.equal(torch.isnan(out).any(-1).cpu(), want)


@pytest.mark.parametrize("D", [64, 128])
def test_scales_far_apart_and_one_key_that_takes_it_all(D):
    g = torch.Generator().manual_seed(7)
    S, Hkv = 512, 2
    k = _rand(g, 1, S, Hkv, D)
    v = torch.randn(1, S, Hkv, D, generator=g) * 10.0 ** torch.randint(-6, 7, (1, S, Hkv, 1), generator=g)
    v = v.bfloat16()
    q = _rand(g, 1, 5, 4, D)
    k[0, 77, 0] = q[0, 1, 0] * 8  # far above the others for one row
    q[0, 2] = 0
    q[0, 3] *= 1e-30
    cache, (kp, vp) = filled(g, 1, S, Hkv, D, k, v)
    out = hlm_attn.cached_attention_hip(q.cuda(), cache, S - 5)
    check_attention(out, q, kp, vp, [S - 5], [5])
    big = (q.float() * 1e20).bfloat16()
    out = hlm_attn.cached_attention_hip(big.cuda(), cache, S - 5, scale=1e-20)
    check_attention(out, big, kp, vp, [S - 5], [5], scale=1e-20)


@pytest.mark.parametrize("T", [1, 30, 70])
def test_values_at_the_ends_of_the_range(T):
    g = torch.Generator().manual_seed(2)
    D, S = 64, 256
    for size in (2.0**-118, 2.0**100):
        v = (torch.randn(1, S, 1, D, generator=g) * size).bfloat16()
        v[0, :, 0, 0] = size  # no row below 2^-119
        cache, (kp, vp) = filled(g, 1, S, 1, D, None, v)
        q = _rand(g, 1, T, 2, D)
        out = hlm_attn.cached_attention_hip(q.cuda(), cache, S - T)
        o, _, _ = oracle.attention(q, kp, vp, [S - T], [T])
        # outputs below the smallest normal bf16 may come out as zeros
        assert ((out.double().cpu() - o).abs() <= 2.0**-6 * size + 2.0**-125).all()
        assert (out[..., 0].double().cpu() / size - 1).abs().max() <= 2.0**-7
    zeros = hlm_attn.KVCache(1, S, 1, D)  # all scales zero
    assert not hlm_attn.cached_attention_hip(_rand(g, 1, T, 2, D).cuda(), zeros, S - T).any()


def test_many_small_weights_are_not_lost():
    """One key at weight 1 and 16000 of 2^-20 each: together a hundredth, below fp16's smallest normal each."""
    S, D = 16384, 64
    q = torch.zeros(1, 1, 1, D)
    q[..., 0] = 1.0
    k = torch.zeros(1, S, 1, D)
    k[0, 100, 0, 0] = 1.0
    k[0, :, 0, 1] = 1.0
    k, q = k.bfloat16(), q.bfloat16()
    scale = 20 * 0.6931471805599453
    v = torch.ones(1, S, 1, D)
    v[0, 100] = 0
    g = torch.Generator().manual_seed(1)
    cache, (kp, vp) = filled(g, 1, S, 1, D, k, v.bfloat16())
    out = hlm_attn.cached_attention_hip(q.cuda(), cache, S - 1, scale=scale)
    check_attention(out, q, kp, vp, [S - 1], [1], scale=scale)


@pytest.mark.parametrize("D", [32, 80, 96])
def test_other_head_dims_and_types(D):
    g = torch.Generator().manual_seed(D)
    cache, (k, v) = filled(g, 2, 128, 2, D)
    q = _rand(g, 2, 3, 4, D).float()
    out = hlm_attn.cached_attention_hip(q.cuda(), cache, int32([10, 90]))
    check_attention(out, q, k, v, [10, 90], [3, 3])
    back = hlm_attn.kv_cache_read_hip(cache, 0, 128)
    for x, (c, s) in zip(back, (k, v)):
        assert torch.equal(x.cpu(), oracle.read(c, s, 128, [0, 0], [128, 128]).float().bfloat16())


def test_strided_queries_and_int64_places():
    g = torch.Generator().manual_seed(8)
    cache, (k, v) = filled(g, 2, 128, 2, 64)
    fused = _rand(g, 2, 3, 8 * 64).cuda()
    q = fused[..., 64 : 5 * 64].view(2, 3, 4, 64)
    starts = torch.tensor([20, 100], device="cuda")
    out = hlm_attn.cached_attention_hip(q, cache, starts)
    check_attention(out, q.cpu(), k, v, [20, 100], [3, 3])
    odd = _rand(g, 2, 3, 4, 65).cuda()[..., :64]  # no layout that the kernels read in place
    check_attention(hlm_attn.cached_attention_hip(odd, cache, starts), odd.cpu(), k, v, [20, 100], [3, 3])
    far = hlm_attn.cached_attention_hip(q, cache, torch.tensor([2**40, -(2**40)], device="cuda"))
    assert not far.any()
    empty = hlm_attn.cached_attention_hip(q[:, :0], cache, starts)
    assert empty.shape == (2, 0, 4, 64)
