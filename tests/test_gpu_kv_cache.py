"""The 8-bit key/value cache and the attention over it, on the GPU, against oracle/kv_cache.py in 64 bits.

Bounds, from the roundings made (eps / 2 of a type: bf16 2^-8, fp16 2^-11, fp32 2^-24):
 * whole numbers are equal, scales equal to the correctly rounded fp32 quotient;
 * a value read back is the fp32 product of whole number and scale, rounded to bf16: equal bit for bit;
 * attention: a score is an fp32 sum of D products times a scale, so it is off by at most e_s = (D + 4) 2^-24 of
   scale sum_d |q_d k_d|; q in fp16 adds 2^-24 of the row's largest q per value, within (D + 4) 2^-24 of the same
   sum's bound with |q| at its largest, which the tests allow for by 2^-23 |q|max sum_d |k_d| scale.  A weight is off
   by 2 e_s + 2^-21 (exponential) + 2^-11 (fp16) relative, the normaliser by as much without the 2^-11, and sums of
   n terms by n 2^-24; the output by 2^-8 relative for bf16.  Weights are held relative to the row's largest value scale vs,
   2^11 at p = 1, so below fp16's normal range one is off by half its spacing there, 2^-25, that is by 2^-36 vs times a
   whole number of at most 127 in the output: n 127 2^-36 vs in all (the sum of p is at least 1).
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
    o, a, reach, top = oracle.attention(q, k, v, starts, counts, window, scale, prefix)
    D = q.shape[3]
    n = k[0].shape[2] + (prefix[0][0].shape[2] if prefix else 0)
    kmax = max((c[0].abs().sum(-1) * c[1]).nan_to_num().max().item() for c in ([k] + ([prefix[0]] if prefix else [])))
    e_s = (D + 4) * 2.0**-24 * reach + 2.0**-23 * q.double().abs().amax(-1) * kmax * (D**-0.5 if scale is None else scale)
    rel = 4 * e_s + 2.0**-20 + 2.0**-11 + n * 2.0**-23
    tol = 2.0**-8 * o.abs() + (a * rel[..., None] + (n * 127 * 2.0**-36 * top)[..., None]) * (1 + 2.0**-8) + 1e-30
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


@pytest.mark.parametrize("T", [3, 200])
def test_negative_counts_are_none(T):
    g = torch.Generator().manual_seed(T)
    cache, plain = filled(g, 2, 256, 2, 64)
    x = _rand(g, 2, T, 2, 64).cuda()
    starts, counts = int32([5, 40]), torch.tensor([-(2**40), -1], device="cuda")
    hlm_attn.kv_cache_write_hip(cache, x, x, starts, counts)
    for (codes, scales), (want_c, want_s) in zip(plain_of(cache), plain):
        assert torch.equal(codes, want_c) and torch.equal(scales, want_s)
    for got in hlm_attn.kv_cache_read_hip(cache, starts, T, counts):
        assert not got.any()
    assert not hlm_attn.cached_attention_hip(_rand(g, 2, T, 4, 64).cuda(), cache, starts, counts).any()


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


JOINT = [
    # B, T, H, Hkv, starts, counts, window, P
    (1, 1, 2, 2, [0], None, None, 1),
    (5, 1, 6, 2, [0, 63, 64, 100, 190], None, None, 63),
    (5, 2, 6, 2, [0, 63, 64, 100, 190], [2, 1, 0, 2, 2], None, 64),
    (3, 3, 4, 4, [-1, 60, 189], None, None, 65),
    (3, 1, 4, 4, [3, 60, 150], None, 61, 100),  # windows that end in the prefix, at the first own key, behind it
    (3, 1, 4, 4, [59, 60, 61], None, 61, 100),
    (2, 40, 4, 2, [0, 90], [40, 17], None, 70),
    (2, 40, 4, 2, [0, 90], [40, 17], 50, 70),
    (8, 64, 3, 1, [0, 10, 20, 30, 40, 50, 60, 70], None, None, 50),
    (8, 150, 2, 2, [0] * 8, [150, 149, 1, 0, 64, 65, 128, 150], 30, 100),
    (8, 150, 2, 2, [0] * 8, [150, 149, 1, 0, 64, 65, 128, 150], None, 100),
    (32, 65, 16, 16, list(range(32)), None, None, 70),  # tiles of 128 rows
    (32, 65, 16, 16, list(range(32)), [65, 1] * 16, 80, 70),
]


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("B,T,H,Hkv,starts,counts,window,P", JOINT)
def test_a_short_prefix_and_the_own_keys_in_one_pass(B, T, H, Hkv, starts, counts, window, P, D):
    """The prefix's last block ends in slots that belong to nobody, whatever these hold."""
    g = torch.Generator().manual_seed(B * T + P)
    cache, (k, v) = filled(g, B, 192, Hkv, D)
    shared, whole = filled(g, 1, 192, Hkv, D)
    for scale, fill in ((shared.k_scale, float("nan")), (shared.v_scale, float("inf"))):
        scale[:, :, P:] = fill
    q = _rand(g, B, T, H, D, scale=1.5)
    n = [T] * B if counts is None else counts
    out = hlm_attn.cached_attention_hip(q.cuda(), cache, int32(starts), None if counts is None else int32(counts), window,
                                        prefix=shared, prefix_length=P)
    check_attention(out, q, k, v, starts, n, window, prefix=[(c[:, :, :P], s[:, :, :P]) for c, s in whole])


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


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,window", [(5, None), (5, 40), (60, None), (60, 30), (100, 50)])
def test_rows_keep_clear_of_values_that_they_do_not_see(D, T, window):
    """Values 2^80 above the others, behind some rows' positions and before others' windows, and after a prefix: rows that do
    not see them lose nothing."""
    g = torch.Generator().manual_seed(6)
    S, start = 256, 120
    v = _rand(g, 1, S, 2, D)
    for at in (start + T // 2, start + T - 2, start - 25):
        v[0, at] = (v[0, at].float() * 2.0**80).bfloat16()
    cache, (kp, vp) = filled(g, 1, S, 2, D, None, v)
    shared, whole = filled(g, 1, 150, 2, D)
    q = _rand(g, 1, T, 4, D)
    check_attention(hlm_attn.cached_attention_hip(q.cuda(), cache, start, None, window), q, kp, vp, [start], [T], window)
    out = hlm_attn.cached_attention_hip(q.cuda(), cache, 0, None, window, prefix=shared, prefix_length=150)
    check_attention(out, q, kp, vp, [0], [T], window, prefix=[(c[:, :, :150], s[:, :, :150]) for c, s in whole])


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
        o = oracle.attention(q, kp, vp, [S - T], [T])[0]
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
    flat = torch.zeros(2 * 3 * 4 * 64 + 4, dtype=BF16, device="cuda")
    flat[4:] = q.flatten()
    moved = flat[4:].view(2, 3, 4, 64)  # contiguous, but 8 bytes off
    assert moved.data_ptr() % 16 == 8 and torch.equal(hlm_attn.cached_attention_hip(moved, cache, starts), out)
    assert torch.equal(hlm_attn.cached_attention_hip(q, cache, starts, window_size=2**32 + 5), out)
    far = hlm_attn.cached_attention_hip(q, cache, torch.tensor([2**40, -(2**40)], device="cuda"))
    assert not far.any()
    empty = hlm_attn.cached_attention_hip(q[:, :0], cache, starts)
    assert empty.shape == (2, 0, 4, 64)


# --- a run of them together, graphs, streams, tracing --------------------------------------


@pytest.mark.parametrize("layer,prefix_tokens", [(0, 0), (1, 0), (0, 70), (1, 70)])
def test_a_generation_run_through_the_attention_core(layer, prefix_tokens):
    """Prompts of different lengths in two chunks, drafted tokens, then single ones, in a local layer (window 96) and a full
    one, with and without a shared context: each step against the oracle over the cache as it then is."""
    g = torch.Generator().manual_seed(layer)
    cfg = hlm_attn.AttentionConfig(n_layer=2, n_head=6, n_kv_head=2, attention_window=96, attention_full_every=2)
    core = hlm_attn.AttentionCore(cfg, layer)
    B, H, Hkv, D, S = 3, 6, 2, 64, 320
    cache = hlm_attn.KVCache(B, S, Hkv, D)
    plain = [(torch.zeros(B, Hkv, S, D, dtype=torch.long), torch.zeros(B, Hkv, S, dtype=torch.float64)) for _ in "kv"]
    shared, prefix = (None, None)
    if prefix_tokens:
        shared, whole = filled(g, 1, prefix_tokens, Hkv, D)
        prefix = [(c[:, :, :prefix_tokens], s[:, :, :prefix_tokens]) for c, s in whole]
    lengths = [0, 0, 0]
    for T, counts in ((130, [130, 57, 99]), (70, [20, 70, 0]), (4, [4, 4, 4]), (4, [1, 3, 4]), (1, [1, 1, 1]), (1, [1, 1, 1])):
        q, k, v = _rand(g, B, T, H, D), _rand(g, B, T, Hkv, D), _rand(g, B, T, Hkv, D)
        with torch.no_grad():
            out = core.forward_cached(q.cuda(), k.cuda(), v.cuda(), cache, int32(lengths), int32(counts), shared, prefix_tokens)
        for (c, s), x in zip(plain, (k, v)):
            oracle.write(c, s, x, lengths, counts)
        check_attention(out, q, *plain, lengths, counts, core.attention_window, prefix=prefix)
        lengths = [n + m for n, m in zip(lengths, counts)]
    for x, (c, s) in zip(hlm_attn.kv_cache_read_hip(cache, 0, S), plain):
        assert torch.equal(x.cpu(), oracle.read(c, s, S, [0] * B, [S] * B).float().bfloat16())


def test_a_cached_sequence_follows_the_uncached_attention():
    """Token by token over the cache against attention() of the whole sequence: apart by the cache's rounding, half a step of
    max|x| / 127 for each value and key (scores: 2^-8.9 of sum|q| max|k| scale at most)."""
    g = torch.Generator().manual_seed(3)
    B, T, H, Hkv, D, W = 2, 150, 4, 2, 64, 64
    q, k, v = (_rand(g, B, T, h, D) for h in (H, Hkv, Hkv))
    whole = hlm_attn.attention(q.cuda(), k.cuda(), v.cuda(), window_size=W).float()
    cache = hlm_attn.KVCache(B, T, Hkv, D)
    rows = []
    for t in range(T):
        hlm_attn.kv_cache_write_hip(cache, k[:, t : t + 1].cuda(), v[:, t : t + 1].cuda(), t)
        rows.append(hlm_attn.cached_attention_hip(q[:, t : t + 1].cuda(), cache, t, window_size=W))
    step = k.float().abs().amax() / 254
    e = (q.float().abs().sum(-1).max() * step * D**-0.5).item()  # of a score
    v_top = v.float().abs().max().item()
    bound = v_top / 254 + v_top * 2 * (torch.tensor(e).exp().item() - 1) + 2**-7 * v_top
    assert (torch.cat(rows, 1).float() - whole).abs().max().item() <= bound
    assert ((torch.cat(rows, 1).float() - whole).norm() / whole.norm()).item() <= 0.03


def test_a_step_is_captured_once_and_replayed_at_other_places():
    """Write, attend and read back in one graph; starts, counts and the new tokens change between replays, with eager calls on
    another cache and synchronisations in between."""
    g = torch.Generator().manual_seed(11)
    B, T, H, Hkv, D, S = 3, 2, 8, 2, 64, 1024
    cache, plain = filled(g, B, S, Hkv, D)
    other, other_plain = filled(g, B, S, Hkv, D)
    shared, whole = filled(g, 1, 200, Hkv, D)
    prefix = [(c[:, :, :200], s[:, :, :200]) for c, s in whole]
    q, k, v = (torch.zeros(B, T, h, D, dtype=BF16, device="cuda") for h in (H, Hkv, Hkv))
    starts, counts = int32([0] * B), int32([T] * B)

    def step():
        hlm_attn.kv_cache_write_hip(cache, k, v, starts, counts)
        return (hlm_attn.cached_attention_hip(q, cache, starts, counts, 500),
                hlm_attn.cached_attention_hip(q, cache, starts, counts, prefix=shared, prefix_length=200),
                *hlm_attn.kv_cache_read_hip(cache, starts, T, counts))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    hlm_attn.kv_cache_write_hip(cache, torch.zeros(B, T, Hkv, D, dtype=BF16, device="cuda"), torch.zeros(B, T, Hkv, D, dtype=BF16, device="cuda"), starts)
    for c, s in plain:
        c[:, :, :T], s[:, :, :T] = 0, 0
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for places, n in (([0, 500, 1022], [2, 1, 2]), ([2, 501, 3], [2, 2, 0]), ([900, 64, 63], [1, 2, 2]), ([-1, 1023, 700], [2, 2, 2])):
        new = [_rand(g, B, T, h, D) for h in (H, Hkv, Hkv)]
        for to, x in zip((q, k, v), new):
            to.copy_(x)
        starts.copy_(int32(places)), counts.copy_(int32(n))
        graph.replay()
        for (c, s), x in zip(plain, new[1:]):
            oracle.write(c, s, x, places, n)
        eager = hlm_attn.cached_attention_hip(q, other, starts, counts)
        check_attention(outs[0], new[0], *plain, places, n, 500)
        check_attention(outs[1], new[0], *plain, places, n, prefix=prefix)
        for x, (c, s) in zip(outs[2:], plain):
            assert torch.equal(x.cpu(), oracle.read(c, s, T, places, n).float().bfloat16())
        check_attention(eager, new[0], *other_plain, places, n)
        torch.cuda.synchronize()


def test_two_streams_over_one_cache():
    """Calls that only read may overlap: each has its own workspace."""
    g = torch.Generator().manual_seed(12)
    cache, (k, v) = filled(g, 1, 4096, 4, 64)
    qs = [_rand(g, 1, 1, 8, 64) for _ in range(2)]
    on_gpu = [x.cuda() for x in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in qs]
    outs = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(hlm_attn.cached_attention_hip(on_gpu[i], cache, 4095 - 64 * i))
    torch.cuda.synchronize()
    for i, x in enumerate(qs):
        assert all(torch.equal(o, outs[i][0]) for o in outs[i])
        check_attention(outs[i][0], x, k, v, [4095 - 64 * i], [1])


@pytest.mark.parametrize("T", [1, 30])
def test_results_do_not_change_from_call_to_call(T):
    g = torch.Generator().manual_seed(13)
    cache, _ = filled(g, 2, 2048, 4, 128)
    shared, _ = filled(g, 1, 700, 4, 128)
    q = _rand(g, 2, T, 12, 128).cuda()
    first = hlm_attn.cached_attention_hip(q, cache, int32([1500, 77]), prefix=shared, prefix_length=700)
    for _ in range(5):
        assert torch.equal(first, hlm_attn.cached_attention_hip(q, cache, int32([1500, 77]), prefix=shared, prefix_length=700))


def test_compiled_calls_run_the_kernels():
    g = torch.Generator().manual_seed(14)
    cache, plain = filled(g, 2, 128, 2, 64)
    q, k, v = (_rand(g, 2, 3, h, 64) for h in (4, 2, 2))

    def step(q, k, v, starts):
        hlm_attn.kv_cache_write_hip(cache, k, v, starts)
        return hlm_attn.cached_attention_hip(q * 2, cache, starts, window_size=50) + 1

    with torch.no_grad():
        out = torch.compile(step, fullgraph=True)(q.cuda(), k.cuda(), v.cuda(), int32([5, 100]))
    for (c, s), x in zip(plain, (k, v)):
        oracle.write(c, s, x, [5, 100], [3, 3])
    eager = hlm_attn.cached_attention_hip((q * 2).cuda(), cache, int32([5, 100]), window_size=50)
    assert torch.equal(out, eager + 1)
    check_attention(eager, q * 2, *plain, [5, 100], [3, 3], 50)
    for got, want in zip(plain_of(cache), plain):
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_without_the_torch_extension(monkeypatch):
    """The general path through the C ABI gives the same results, bit for bit."""
    from hlm_attn import _lib

    g = torch.Generator().manual_seed(15)
    cache, _ = filled(g, 2, 256, 2, 64)
    twin, _ = filled(torch.Generator().manual_seed(15), 2, 256, 2, 64)
    shared, _ = filled(g, 1, 100, 2, 64)
    q, k, v = (_rand(g, 2, 5, h, 64).cuda() for h in (4, 2, 2))
    starts, counts = int32([100, 3]), int32([5, 4])

    def run(c):
        hlm_attn.kv_cache_write_hip(c, k, v, starts, counts)
        return (hlm_attn.cached_attention_hip(q, c, starts, counts, 60), hlm_attn.cached_attention_hip(q, c, 20, prefix=shared, prefix_length=99),
                *hlm_attn.kv_cache_read_hip(c, starts, 5, counts))

    fast = run(cache)
    monkeypatch.setattr(_lib, "_torch_fwd", False)
    for a, b in zip(fast, run(twin)):
        assert torch.equal(a, b)


def test_refusals_on_the_device():
    cache = hlm_attn.KVCache(2, 128, 2, 64)
    x = torch.zeros(2, 3, 2, 64, dtype=BF16, device="cuda")
    with pytest.raises(RuntimeError, match="do not fit"):
        hlm_attn.kv_cache_write_hip(cache, x, x, 126)
    with pytest.raises(RuntimeError, match="do not fit"):
        hlm_attn.cached_attention_hip(x, cache, -1)
    with pytest.raises(RuntimeError, match="do not fit"):
        hlm_attn.kv_cache_read_hip(cache, 0, 129)
    with pytest.raises(RuntimeError, match="starts"):
        hlm_attn.kv_cache_write_hip(cache, x, x, torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="starts"):
        hlm_attn.cached_attention_hip(x, cache, torch.zeros(2, dtype=torch.int32))  # on the CPU
    with pytest.raises(RuntimeError, match="multiple of kv heads"):
        hlm_attn.cached_attention_hip(torch.zeros(2, 1, 3, 64, dtype=BF16, device="cuda"), cache, 0)
    with pytest.raises(RuntimeError, match="does not match a cache"):
        hlm_attn.cached_attention_hip(x[:1], cache, 0)
    with pytest.raises(RuntimeError, match="do not match"):
        hlm_attn.kv_cache_write_hip(cache, x[:, :, :1], x[:, :, :1], 0)
    with pytest.raises(RuntimeError, match="does not match"):
        hlm_attn.cached_attention_hip(x, cache, 0, prefix=cache, prefix_length=5)  # two sequences
    with pytest.raises(RuntimeError, match="scale"):
        hlm_attn.cached_attention_hip(x, cache, 0, scale=-1.0)
    padded = hlm_attn.KVCache(2, 128, 2, 48)  # held in 64 dims, which is no head dim of its callers
    for call in (lambda: hlm_attn.cached_attention_hip(x, padded, 0), lambda: hlm_attn.kv_cache_write_hip(padded, x, x, 0)):
        with pytest.raises(RuntimeError, match="heads of 48"):
            call()


def test_a_cache_beyond_4_gib_of_keys():
    """Byte offsets pass 2^31 and 2^32: all sequences of a cache of 5 GiB of keys, near their ends."""
    g = torch.Generator().manual_seed(16)
    B, Hkv, S, D, T, W = 5, 2, 1 << 22, 128, 80, 100
    cache = hlm_attn.KVCache(B, S, Hkv, D)
    assert cache.k.numel() > 4 << 30
    starts = [S - 300, 5, S - 190, S - 250, S - 190]
    k, v = _rand(g, B, 190, Hkv, D), _rand(g, B, 190, Hkv, D)
    hlm_attn.kv_cache_write_hip(cache, k.cuda(), v.cuda(), int32(starts))
    got = hlm_attn.kv_cache_read_hip(cache, int32(starts), 190)
    plain = [oracle.encode(x) for x in (k, v)]
    for x, (c, s) in zip(got, plain):
        assert torch.equal(x.cpu(), (c.double() * s[..., None]).float().bfloat16())
    for n in (1, T):  # the last n of those tokens
        q = _rand(g, B, n, 4, D)
        out = hlm_attn.cached_attention_hip(q.cuda(), cache, int32([s + 190 - n for s in starts]), window_size=W)
        rows = [(c.transpose(1, 2), s.transpose(1, 2)) for c, s in plain]
        check_attention(out, q, *rows, [190 - n] * B, [n] * B, W)


def test_many_sequences_heads_and_rows():
    """More workgroups than one wave of them, several tiles per unit, all variants of the prefix's and the own rows."""
    g = torch.Generator().manual_seed(17)
    for B, T, H, Hkv, D, P in ((20, 2, 8, 4, 64, 500), (5, 25, 6, 2, 64, 300), (3, 90, 4, 2, 64, 200), (9, 3, 4, 4, 128, 260), (2, 100, 6, 2, 128, 150)):
        cache, (k, v) = filled(g, B, 192, Hkv, D)
        shared, whole = filled(g, 1, P, Hkv, D)
        q = _rand(g, B, T, H, D)
        starts = [i * 7 % (192 - T) for i in range(B)]
        out = hlm_attn.cached_attention_hip(q.cuda(), cache, int32(starts), prefix=shared, prefix_length=P)
        check_attention(out, q, k, v, starts, [T] * B, prefix=[(c[:, :, :P], s[:, :, :P]) for c, s in whole])


def test_the_producer_at_positions():
    """QKVProjection with the tables of its tokens' positions: the rows that the producer gives those positions."""
    cfg = hlm_attn.AttentionConfig(n_layer=1, n_head=4, n_kv_head=2, n_embd=64)
    g = torch.Generator().manual_seed(18)
    proj = hlm_attn.QKVProjection(cfg, 0)
    with torch.no_grad():
        proj.qkv_proj.weight.copy_(torch.randn(proj.qkv_proj.weight.shape, generator=g) * 0.1)
        proj = proj.to("cuda", BF16)
        proj.rope = hlm_attn.RotaryEmbedding(64).to("cuda")
        x = _rand(g, 2, 5, 64).cuda()
        pos = torch.tensor([[0, 1, 2, 3, 4], [40, 41, 42, 43, 44]], device="cuda")
        q, k, v = proj(x, proj.rope.at(pos, BF16))
        q0, k0, v0 = proj(x)
        assert torch.equal(q[0], q0[0]) and torch.equal(k[0], k0[0]) and torch.equal(v, v0)
        raw_q, raw_k, _, cos, sin = proj._project(x)
        cos, sin = (t[0, 0] for t in proj.rope(50, x.device, BF16))
        want = hlm_attn.qk_norm_rope_hip(raw_q[1:], raw_k[1:], cos[40:45].contiguous(), sin[40:45].contiguous(), cfg.norm_eps)
        assert torch.equal(q[1:], want[0]) and torch.equal(k[1:], want[1])


# --- calls that something watches -------------------------------------------------------------


def test_traced_calls_hold_the_write_and_run_again():
    """make_fx and jit.trace record the write and the attention; the recorded step run on other tokens does both."""
    from torch.fx.experimental.proxy_tensor import make_fx

    B, T, H, Hkv, D, S = 2, 3, 4, 2, 64, 128
    for trace in (lambda f, a: make_fx(f)(*a), lambda f, a: torch.jit.trace(f, a, check_trace=False)):
        g = torch.Generator().manual_seed(21)
        cache, plain = filled(g, B, S, Hkv, D)

        def step(q, k, v, starts):
            hlm_attn.kv_cache_write_hip(cache, k, v, starts)
            return hlm_attn.cached_attention_hip(q, cache, starts, window_size=50)

        with torch.no_grad():
            first = [_rand(g, B, T, h, D) for h in (H, Hkv, Hkv)]
            recorded = trace(step, (*(x.cuda() for x in first), int32([5, 60])))
            for (c, s), x in zip(plain, first[1:]):  # tracing ran the step
                oracle.write(c, s, x, [5, 60], [T, T])
            q, k, v = (_rand(g, B, T, h, D) for h in (H, Hkv, Hkv))
            out = recorded(q.cuda(), k.cuda(), v.cuda(), int32([100, 20]))
        for (c, s), x in zip(plain, (k, v)):
            oracle.write(c, s, x, [100, 20], [T, T])
        for got, want in zip(plain_of(cache), plain):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        check_attention(out, q, *plain, [100, 20], [T, T], 50)


def test_attention_over_vmap_is_that_of_its_parts():
    g = torch.Generator().manual_seed(22)
    cache, plain = filled(g, 2, 128, 2, 64)
    q = _rand(g, 3, 2, 1, 4, 64)
    with torch.no_grad():
        out = torch.func.vmap(lambda x: hlm_attn.cached_attention_hip(x, cache, 100))(q.cuda())
        for a, b in zip(out, q):
            assert torch.equal(a, hlm_attn.cached_attention_hip(b.cuda(), cache, 100))
        with pytest.raises(RuntimeError, match="[Bb]atching rule"):
            torch.func.vmap(lambda x: (hlm_attn.kv_cache_write_hip(cache, x, x, 0), x)[1])(_rand(g, 3, 2, 1, 2, 64).cuda())


# --- each kernel of the plan ------------------------------------------------------------------


def plan_of(B, T, H, Hkv, D, slots, prefix, window):
    """The plan's kernels, with places on the device: of the own keys and of the prefix (see hlm_attn_cached_fwd_plan)."""
    import ctypes

    from hlm_attn import _lib

    plan = (ctypes.c_int32 * 6)()
    assert _lib.load().hlm_attn_cached_fwd_plan(B, T, H, Hkv, D, slots, ctypes.c_void_p(16), 0, None, prefix, window or 0, plan) == 0
    return plan[0], plan[3]


def check_rows(out, q, k, v, starts, counts, rows, window=None, prefix=None, scale=None):
    """check_attention of the rows (sequence, token) alone, each as a sequence of one token."""
    out = out.cpu()
    for b, t in rows:
        check_attention(out[b : b + 1, t : t + 1], q[b : b + 1, t : t + 1], *([x[b : b + 1] for x in pair] for pair in (k, v)),
                        [starts[b] + t], [int(t < counts[b])], window, scale, prefix)


KERNELS = [
    # own kernel, prefix's (-1: no prefix; -2: the prefix's keys with the own ones), B, T, H, Hkv, D, capacity, window, P
    (0, 0, 1, 1, 3, 1, 64, 128, None, 852),
    (0, 0, 2, 1, 3, 1, 64, 960, 964, 55),
    (0, 0, 1, 1, 4, 1, 64, 64, None, 4650),
    (0, 0, 4, 1, 3, 1, 128, 64, None, 451),
    (0, 0, 2, 1, 3, 1, 128, 512, 460, 39),
    (0, 1, 66, 1, 4, 4, 64, 64, None, 424),
    (0, 1, 55, 1, 3, 1, 64, 128, 933, 1127),
    (0, 1, 64, 1, 12, 4, 64, 512, None, 8000),
    (0, 1, 8, 4, 3, 1, 128, 128, None, 393),
    (0, 1, 5, 4, 3, 1, 128, 256, 489, 265),
    (1, 1, 2, 28, 3, 1, 64, 128, None, 194),
    (1, 1, 6, 12, 3, 1, 64, 128, 271, 194),
    (1, 1, 5, 73, 3, 1, 128, 192, None, 72),
    (1, 1, 7, 6, 3, 1, 128, 64, 330, 267),
    (1, 2, 35, 36, 4, 4, 64, 64, None, 5344),
    (1, 2, 93, 9, 6, 2, 64, 64, None, 7000),
    (1, 2, 108, 23, 3, 1, 128, 256, None, 2314),
    (1, 2, 53, 14, 4, 2, 128, 640, 6606, 10190),
    (2, 2, 29, 185, 3, 1, 64, 1216, None, 845),
    (2, 2, 36, 98, 4, 4, 64, 768, 884, 269),
    (2, 2, 34, 159, 3, 1, 128, 1216, None, 426),
    (2, 2, 10, 209, 8, 1, 128, 960, 1160, 311),
    (2, -1, 109, 37, 8, 4, 64, 64, None, 0),
    (2, -1, 1, 5000, 12, 4, 64, 5056, None, 0),
    (2, -1, 101, 43, 8, 4, 64, 64, 20, 0),
    (2, -1, 101, 23, 12, 4, 128, 64, None, 0),
    (2, -1, 102, 25, 12, 4, 128, 64, 9, 0),
    (2, -1, 1, 5000, 12, 4, 128, 5056, 1000, 0),
    (2, -2, 32, 65, 16, 16, 64, 192, 80, 70),
    (2, -2, 32, 65, 16, 16, 128, 192, None, 70),
]


@pytest.mark.parametrize("own,shared,B,T,H,Hkv,D,capacity,window,P", KERNELS)
def test_each_kernel_of_the_plan(own, shared, B, T, H, Hkv, D, capacity, window, P):
    """A ragged batch at places of its own, the slots behind the prefix holding anything: forty rows of it."""
    assert plan_of(B, T, H, Hkv, D, capacity, P, window) == (own, shared)
    g = torch.Generator().manual_seed(B * T + P)
    cache, (k, v) = filled(g, B, capacity, Hkv, D)
    prefix = pre = None
    if P:
        pre, whole = filled(g, 1, P, Hkv, D)
        for scale, fill in ((pre.k_scale, float("nan")), (pre.v_scale, float("inf"))):
            scale[:, :, P:] = fill
        prefix = [(c[:, :, :P], s[:, :, :P]) for c, s in whole]
    q = _rand(g, B, T, H, D, scale=1.5)
    starts = [b * 37 % (capacity - T + 1) for b in range(B)]
    starts[-1] = capacity - T
    counts = [T - b * 5 % (T + 1) for b in range(B)]
    out = hlm_attn.cached_attention_hip(q.cuda(), cache, int32(starts), int32(counts), window, prefix=pre, prefix_length=P)
    ends = [(b, t) for b in (0, 1 % B, B - 1) for t in {0, counts[b] - 1, min(T - 1, counts[b]), T // 2, T - 1} if t >= 0]
    some = [(int(b), int(t)) for b, t in zip(torch.randint(B, (25,), generator=g), torch.randint(T, (25,), generator=g))]
    check_rows(out, q, k, v, starts, counts, ends + some, window, prefix)
    dead = torch.arange(T)[None] >= torch.tensor(counts)[:, None]
    assert not out.cpu()[dead].any() and torch.isfinite(out).all()


# --- values far above others, with little weight ----------------------------------------------


def check_by_weight(out, q, k, v, starts, counts, window=None, scale=None, prefix=None):
    """check_attention with the fp16 weights' absolute error relative to the row's largest weight p vs instead of its largest
    value scale: what weights are relative to is at most 2^8 of the former, so one is off by at most 2^-36 2^8 of it, times a
    whole number of at most 127."""
    o, a, reach, _ = oracle.attention(q, k, v, starts, counts, window, scale, prefix)
    B, T, H, D = q.shape
    scale = D**-0.5 if scale is None else scale
    P = prefix[0][0].shape[2] if prefix else 0
    n = k[0].shape[2] + P
    heavy = torch.zeros(B, T, H, dtype=torch.float64)
    for b in range(B):
        for h in range(H):
            g = h // (H // k[0].shape[1])
            kr, ks, vs = (torch.cat([x[i][0, g] for x in (prefix[j],)] + [own[i][b, g]]) if P else own[i][b, g]
                          for own, i, j in ((k, 0, 0), (k, 1, 0), (v, 1, 1)))
            s = (q[b, :, h].double() @ kr.double().T) * ks * scale
            lag = (torch.arange(T) + starts[b] + P)[:, None] - torch.arange(n)
            s = s.masked_fill((lag < 0) | (lag >= (window or n + 1)), -float("inf"))
            heavy[b, :, h] = (torch.softmax(s, -1) * vs).amax(-1)
    kmax = max((c[0].abs().sum(-1) * c[1]).max().item() for c in ([k] + ([prefix[0]] if prefix else [])))
    e_s = (D + 4) * 2.0**-24 * reach + 2.0**-23 * q.double().abs().amax(-1) * kmax * scale
    rel = 4 * e_s + 2.0**-20 + 2.0**-11 + n * 2.0**-23
    tol = 2.0**-8 * o.abs() + (a * rel[..., None] + (n * 127 * 2.0**-28 * heavy)[..., None]) * (1 + 2.0**-8)
    err = (out.double().cpu() - o).abs()
    assert torch.isfinite(out).all()
    assert (err <= tol).all(), f"error {(err / tol).max().item():.3f} of its bound"


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,window", [(1, None), (5, None), (5, 100), (60, None), (60, 70), (130, 90)])
def test_a_visible_value_far_above_the_others_with_little_weight(D, T, window):
    """Values near 1, and single ones of 2^40 whose keys' logits are 40 and 100 below: the others keep their bits, wherever
    the large ones stand, in the cache and in a prefix."""
    g = torch.Generator().manual_seed(T)
    S, start, H, P = 320, 150, 4, 100
    for below in (40.0, 100.0):
        for spots in ((start,), (0, 70), (start - 3, start - 60, 5)):
            q = _rand(g, 1, T, H, D)
            q[..., 0] = 8.0
            k, v = _rand(g, 1, S, 2, D), _rand(g, 1, S, 2, D)
            k[..., 0] = 0.0
            for at in spots:
                k[0, at, :, 0] = -below * D**0.5 / 8
                v[0, at] = (v[0, at].float() * 2.0**40).bfloat16()
            cache, (kp, vp) = filled(g, 1, S, 2, D, k, v)
            out = hlm_attn.cached_attention_hip(q.cuda(), cache, start, None, window)
            check_by_weight(out, q, kp, vp, [start], [T], window)
            pre, whole = filled(g, 1, P, 2, D, *(torch.nn.functional.pad(x[:, :P], (0, 0, 0, 0, 0, 128 - P)) for x in (k, v)))
            prefix = [(c[:, :, :P], s[:, :, :P]) for c, s in whole]
            out = hlm_attn.cached_attention_hip(q.cuda(), cache, start, None, window, prefix=pre, prefix_length=P)
            check_by_weight(out, q, kp, vp, [start], [T], window, prefix=prefix)


@pytest.mark.parametrize("T,H", [(1, 2), (40, 2), (300, 12)])
def test_weights_and_values_over_many_powers_of_two(T, H):
    """Logits that rise and fall by tens along the keys, values of 10^-6 to 10^6: each row to its own weights."""
    g = torch.Generator().manual_seed(T)
    S, D = 1024, 64
    q = _rand(g, 1, T, H, D)
    q[..., 0] = 8.0
    k = _rand(g, 1, S, 2, D)
    k[0, :, :, 0] = (torch.randn(S, 2, generator=g).cumsum(0) * 3).bfloat16()
    v = (torch.randn(1, S, 2, D, generator=g) * 10.0 ** torch.randint(-6, 7, (1, S, 2, 1), generator=g)).bfloat16()
    cache, (kp, vp) = filled(g, 1, S, 2, D, k, v)
    out = hlm_attn.cached_attention_hip(q.cuda(), cache, S - T)
    check_by_weight(out, q, kp, vp, [S - T], [T])


def test_one_key_that_takes_it_all_with_a_small_value():
    """A first key with nearly all the weight and a value of 2^-20, as models learn: the others' share is kept."""
    g = torch.Generator().manual_seed(23)
    for T in (1, 20, 100):
        q, k, v = _rand(g, 1, T, 4, 64), _rand(g, 1, 512, 2, 64), _rand(g, 1, 512, 2, 64)
        q[..., 0], k[..., 0] = 8.0, 0.0
        k[0, 0, :, 0] = 9.0
        v[0, 0] = (v[0, 0].float() * 2.0**-20).bfloat16()
        cache, (kp, vp) = filled(g, 1, 512, 2, 64, k, v)
        out = hlm_attn.cached_attention_hip(q.cuda(), cache, 512 - T)
        check_by_weight(out, q, kp, vp, [512 - T], [T])


# --- logits far from zero ---------------------------------------------------------------------


@pytest.mark.parametrize("T,Hkv", [(1, 2), (40, 2), (70, 1), (2000, 2)])
def test_equal_logits_give_the_mean_however_large_they_are(T, Hkv):
    """All keys alike in one dim: the probabilities are equal, the kernels' scores bit for bit, so that of a weight and of the
    normaliser only the exponential of 0 and the fp16 weight are roundings.  Logits of 2^20 to 2^125, of either sign."""
    g = torch.Generator().manual_seed(T)
    S, D, H, P = 4096, 64, 4, 150
    v = _rand(g, 1, S, Hkv, D) + 2
    q, k = torch.zeros(1, T, H, D), torch.zeros(1, S, Hkv, D)
    q[..., 0], k[..., 0] = 1.6875, 3.0
    for sign in (1, -1):
        cache, (_, (c, s)) = filled(g, 1, S, Hkv, D, (sign * k).bfloat16(), v)
        pre, (_, (pc, ps)) = filled(g, 1, P, Hkv, D, (sign * k[:, :192]).bfloat16(), v[:, :192])
        own, shared = c[0] * s[0, ..., None], pc[0, :, :P] * ps[0, :, :P, None]  # (Hkv, keys, D)
        for power in (20, 26, 31, 60, 100, 122):
            for prefix in (None, pre):
                out = hlm_attn.cached_attention_hip(q.bfloat16().cuda(), cache, 333, scale=2.0**power, prefix=prefix, prefix_length=P if prefix else 0)
                for t in {0, T // 2, T - 1}:
                    for h in range(H):
                        rows = own[h * Hkv // H, : 334 + t]
                        rows = torch.cat((shared[h * Hkv // H], rows)) if prefix else rows
                        n = rows.shape[0]
                        want, size = rows.mean(0), rows.abs().mean(0)
                        err = (out[0, t, h].double().cpu() - want).abs()
                        assert (err <= 2.0**-8 * want.abs() + (2.0**-11 + 2.0**-20 + n * 2.0**-23) * size).all(), (power, t, h)


@pytest.mark.parametrize("T", [1, 40, 300])
def test_a_far_larger_logit_takes_it_all(T):
    """Logits that differ by 2^20 and more: each row's output is the value of its largest visible key."""
    g = torch.Generator().manual_seed(T)
    S, D, H, Hkv = 1024, 64, 4, 2
    q, k = torch.zeros(1, T, H, D), torch.zeros(1, S, Hkv, D)
    q[..., 0] = 1.25
    k[0, :, :, 0] = torch.stack([torch.randperm(S, generator=g) for _ in range(Hkv)], 1) / 8 + 1.0  # apart by 2^-10 at least
    k = k.bfloat16().float()
    cache, ((kc, ks), (vc, vs)) = filled(g, 1, S, Hkv, D, k.bfloat16())
    for scale in (2.0**34, 2.0**90):
        for window in (None, 100):
            out = hlm_attn.cached_attention_hip(q.bfloat16().cuda(), cache, S - T, window_size=window, scale=scale)
            for t in {0, T // 2, T - 1}:
                p = S - T + t
                first = 0 if window is None else max(0, p - window + 1)
                for h in range(H):
                    g_ = h // (H // Hkv)
                    logits = (kc[0, g_, first : p + 1, 0] * ks[0, g_, first : p + 1]) * 1.25
                    best = (logits == logits.max()).nonzero()[:, 0] + first  # keys that bf16 made equal share it
                    want = (vc[0, g_, best] * vs[0, g_, best, None]).mean(0)
                    size = (vc[0, g_, best] * vs[0, g_, best, None]).abs().mean(0)
                    err = (out[0, t, h].double().cpu() - want).abs()
                    assert (err <= 2.0**-8 * want.abs() + (2.0**-10 + len(best) * 2.0**-23) * size + 1e-30).all(), (scale, t, h)


@pytest.mark.parametrize("prefix_tokens", [0, 70])
def test_a_layer_step_is_captured_once_and_replayed(prefix_tokens):
    """Projection, rotary tables at the tokens' places, forward_cached and the places' advance in one graph: each replay equals
    the eager step of a twin cache, bit for bit, with that step between the replays."""
    g = torch.Generator().manual_seed(24)
    B, T, S = 3, 2, 192
    cfg = hlm_attn.AttentionConfig(n_layer=2, n_head=4, n_kv_head=2, n_embd=64, attention_window=40, attention_full_every=2)
    core, proj = hlm_attn.AttentionCore(cfg, 0), hlm_attn.QKVProjection(cfg, 0)
    shared = filled(g, 1, prefix_tokens, 2, 64)[0] if prefix_tokens else None
    with torch.no_grad():
        proj.qkv_proj.weight.copy_(torch.randn(proj.qkv_proj.weight.shape, generator=g) * 0.1)
        proj = proj.to("cuda", BF16)
        proj.rope = hlm_attn.RotaryEmbedding(64).to("cuda")
        places = torch.arange(T, device="cuda")
        x, counts = torch.zeros(B, T, 64, dtype=BF16, device="cuda"), int32([T] * B)

        def step(cache, starts):
            rotary = proj.rope.at(starts[:, None] + places + prefix_tokens, BF16)
            y = core.forward_cached(*proj(x, rotary), cache, starts, counts, shared, prefix_tokens)
            starts += counts
            return y

        cache, twin = (hlm_attn.KVCache(B, S, 2, 64) for _ in range(2))
        starts, twin_starts = int32([0] * B), int32([0] * B)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(twin, twin_starts)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(cache, starts)
        twin_starts.zero_()
        for n in ([2, 2, 2], [1, 2, 0], [2, 2, 2], [0, 1, 2], [2, 1, 1], [2, 2, 2]) * 3:
            x.copy_(_rand(g, B, T, 64))
            counts.copy_(int32(n))
            graph.replay()
            want = step(twin, twin_starts)
            torch.cuda.synchronize()
            assert torch.equal(out, want) and torch.equal(starts, twin_starts)
        for a, b in zip(hlm_attn.kv_cache_read_hip(cache, 0, S, starts), hlm_attn.kv_cache_read_hip(twin, 0, S, starts)):
            assert torch.equal(a, b) and a.any()


@pytest.mark.parametrize("T", [1, 40])
@pytest.mark.parametrize("power,scale", [(-110, 2.0**-40), (-60, 2.0**-149), (-126, 2.0**-130), (-126, 2.0**20), (120, 2.0**-149), (127, 2.0**-140)])
def test_queries_and_scales_at_the_ends_of_the_range(T, power, scale):
    """Keys of 2^118 that all have the query's direction, half of them turned round: logits of +-scale |q.k|, from far below 2^-24
    (the mean of all values) to a few units."""
    g = torch.Generator().manual_seed(25)
    S, D = 256, 128
    q = torch.full((1, T, 2, D), 1.0) * 2.0**power
    turned = torch.where(torch.arange(S) % 3 == 0, -1.0, 1.0)[None, :, None, None]
    logit = scale * 2.0**power * D
    size = 2.0**118 if logit * 2.0**118 < 8 else 4.0 / logit  # a power of two: exact codes
    k = (turned * size).expand(1, S, 1, D)
    cache, (kp, vp) = filled(g, 1, S, 1, D, k.bfloat16())
    out = hlm_attn.cached_attention_hip(q.bfloat16().cuda(), cache, S - T, scale=scale)
    values = vp[0][0, 0] * vp[1][0, 0, :, None]
    for t in range(T):
        p = torch.softmax((kp[0][0, 0, :, 0] * kp[1][0, 0] * scale * 2.0**power * D)[: S - T + t + 1], 0)
        want, size_ = p @ values[: len(p)], p @ values[: len(p)].abs()
        # logits up to 4: fp32 to (D + 4) 2^-24 of them, q in fp16 exact or, for the smallest, lost with logits below 2^-20
        err = (out[0, t].double().cpu() - want).abs()
        assert (err <= 2.0**-8 * want.abs() + (2.0**-11 + 2.0**-13) * size_ + 1e-30).all(), t


def test_a_prefix_of_no_tokens_many_query_heads_and_counts_past_the_end():
    g = torch.Generator().manual_seed(26)
    cache, (k, v) = filled(g, 3, 128, 1, 64)
    q = _rand(g, 3, 2, 32, 64)
    shared, _ = filled(g, 1, 64, 1, 64)
    out = hlm_attn.cached_attention_hip(q.cuda(), cache, int32([5, 126, 60]), prefix=shared, prefix_length=0)
    check_attention(out, q, k, v, [5, 126, 60], [2, 2, 2])
    assert torch.equal(out, hlm_attn.cached_attention_hip(q.cuda(), cache, int32([5, 126, 60])))
    # a place that the host knows, and more tokens than fit it: counts tell which are real, the cache's end which lie in it
    for T in (12, 40):
        q, counts = _rand(g, 3, T, 4, 64), [T, 3, 0]
        out = hlm_attn.cached_attention_hip(q.cuda(), cache, 120, int32(counts))
        check_attention(out, q, k, v, [120] * 3, counts)
        x = _rand(g, 3, T, 1, 64)
        hlm_attn.kv_cache_write_hip(cache, x.cuda(), x.cuda(), 120, int32(counts))
        for c, s in (k, v):
            oracle.write(c, s, x, [120] * 3, counts)
        for got, (c, s) in zip(hlm_attn.kv_cache_read_hip(cache, 120, T, int32(counts)), (k, v)):
            assert torch.equal(got.cpu(), oracle.read(c, s, T, [120] * 3, counts).float().bfloat16())
