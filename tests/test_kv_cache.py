"""CPU tests of the 8-bit key/value cache: its oracle, the C ABI's and the Python entry points' refusals, the plan of the
attention's workspace, and the layout that KVCache describes.  Nothing here launches a kernel."""
from __future__ import annotations

import ctypes
from fractions import Fraction

import pytest
import torch

import hlm_attn
from hlm_attn import _lib, kernels, ops
from oracle import kv_cache as oracle

P = ctypes.c_void_p
BF16 = torch.bfloat16


# --- the oracle -----------------------------------------------------------------------


def test_oracle_rounds_to_the_nearest_whole_number_ties_to_even():
    """Against exact fractions, over every significand of the row's largest value."""
    for a in range(128, 256):
        x = torch.tensor([[float(a), a / 2, -a / 2, 1.0, 37.0, 63.5, -126.5, a / 4]]).bfloat16()
        codes, scales = oracle.encode(x)
        for c, v in zip(codes[0].tolist(), x[0].tolist()):
            assert c == round(127 * Fraction(v) / a)  # Fraction rounds half to even
        assert codes[0, 1] == 64 and codes[0, 2] == -64  # 63.5
        assert scales[0].item() == torch.tensor(float(a)).div(torch.tensor(127.0)).item()


def test_kernel_arithmetic_gives_the_same_whole_numbers():
    """x r with r = 127 / a rounded up to fp32 and the product exact (a fused multiply-add): every pair of significands and
    every power of two between them gives the nearest whole number to 127 x / a."""
    import numpy as np

    for a in range(128, 256):
        r = np.float32(127) / np.float32(a)
        if Fraction(float(r)) * a < 127:
            r = np.nextafter(r, np.float32(np.inf), dtype=np.float32)
        up = Fraction(float(r))
        assert 127 <= up * a
        for shift in range(10):
            for m in range(128, 256):
                if m <= a << shift:
                    x = Fraction(m, 1 << shift)
                    assert round(x * up) == round(127 * x / a)


def test_oracle_zero_tiny_and_not_finite_rows():
    x = torch.zeros(4, 8)
    x[1] = 1e-37
    x[2, 3] = float("inf")
    x[3, 5] = float("nan")
    codes, scales = oracle.encode(x)
    assert not codes.any() and scales[0] == 0 and scales[1] == 0 and torch.isnan(scales[2:]).all()


def test_oracle_attention_is_the_dense_one():
    """Over a cache that holds its values exactly: softmax over the visible keys, for every kind of place."""
    g = torch.Generator().manual_seed(0)
    B, T, H, Hkv, D, S, Pn = 3, 4, 4, 2, 8, 32, 5
    codes = [torch.randint(-127, 128, (n, Hkv, s, D), generator=g) for n, s in ((B, S), (B, S), (1, Pn), (1, Pn))]
    scales = [torch.rand(c.shape[:3], generator=g).double() / 100 for c in codes]
    q = torch.randn(B, T, H, D, generator=g).bfloat16()
    starts, counts = [0, 10, 30], [4, 2, 4]
    for window in (None, 1, 6, 100):
        for prefix in (None, [(codes[2], scales[2]), (codes[3], scales[3])]):
            o, a, _, top = oracle.attention(q, (codes[0], scales[0]), (codes[1], scales[1]), starts, counts, window, None, prefix)
            n = Pn if prefix else 0
            for b in range(B):
                for t in range(T):
                    p = starts[b] + t
                    if t >= counts[b] or p >= S:
                        assert not o[b, t].any()
                        continue
                    for h in range(H):
                        k = torch.cat(([codes[2][0, h // 2] * scales[2][0, h // 2, :, None]] if prefix else []) + [codes[0][b, h // 2] * scales[0][b, h // 2, :, None]])
                        v = torch.cat(([codes[3][0, h // 2] * scales[3][0, h // 2, :, None]] if prefix else []) + [codes[1][b, h // 2] * scales[1][b, h // 2, :, None]])
                        lag = p + n - torch.arange(S + n)
                        s = (k @ q[b, t, h].double()) * D**-0.5
                        s[(lag < 0) | (lag >= (window or 10**6))] = -float("inf")
                        want = torch.softmax(s, 0) @ v
                        assert (o[b, t, h] - want).abs().max() <= 1e-12
                        assert (a[b, t, h] >= o[b, t, h].abs() - 1e-12).all()
                        seen = torch.cat(([scales[3][0, h // 2]] if prefix else []) + [scales[1][b, h // 2]])[(lag >= 0) & (lag < (window or 10**6))]
                        assert top[b, t, h] == seen.max()


# --- the C ABI --------------------------------------------------------------------------


def _strides(*s):
    return (ctypes.c_int64 * 3)(*s)


def _write(lib, ptr=0x1000, slots=128, starts=None, start=0, counts=None, B=1, T=16, Hkv=2, D=64, strides=(2048, 128, 64)):
    s = _strides(*strides)
    p = P(ptr) if ptr else None
    return lib.hlm_attn_cache_write(p, p, s, s, p, p, p, p, slots, starts, start, counts, B, T, Hkv, D, None)


def _read(lib, ptr=0x1000, slots=128, starts=None, start=0, counts=None, B=1, T=16, Hkv=2, D=64, strides=None):
    p = P(ptr) if ptr else None
    return lib.hlm_attn_cache_read(p, p, p, p, slots, p, p, starts, start, counts, B, T, Hkv, D, None)


CACHE_REFUSALS = [
    (dict(D=96), -2, "head_dim 96"),
    (dict(Hkv=0), -1, "bad shape"),
    (dict(B=-1), -1, "bad shape"),
    (dict(ptr=None), -1, "16-byte aligned"),
    (dict(ptr=0x1008), -1, "16-byte aligned"),
    (dict(slots=100), -1, "multiple of 64"),
    (dict(slots=0), -1, "do not fit"),
    (dict(slots=0, starts=P(0x1000)), -1, "multiple of 64"),
    (dict(slots=(1 << 24) + 64), -1, "multiple of 64"),
    (dict(start=113), -1, "do not fit"),
    (dict(start=-1), -1, "do not fit"),
    (dict(start=129, counts=P(0x1000)), -1, "do not fit"),
    (dict(B=1 << 16, T=1 << 15), -2, "too many rows"),
    (dict(B=1 << 14, T=1 << 13), -2, "too many rows"),  # 2^28 rows
    (dict(B=1 << 21, T=16, Hkv=2, D=128, strides=(2048, 128, 128)), -2, "too many rows"),  # 2^23 blocks of 512 threads
]


@pytest.mark.parametrize("kwargs,code,msg", CACHE_REFUSALS)
@pytest.mark.parametrize("call", [_write, _read])
def test_cache_calls_reject_bad_arguments_before_touching_the_device(call, kwargs, code, msg):
    lib = _lib.load()
    if "T" in kwargs:
        kwargs = dict(kwargs, starts=P(0x1000))
    assert call(lib, **kwargs) == code
    assert msg in lib.hlm_attn_last_error().decode()


def test_cache_write_rejects_strides_that_it_cannot_read():
    lib = _lib.load()
    assert _write(lib, strides=(2048, 100, 64)) == -1 and b"multiple of 8" in lib.hlm_attn_last_error()
    assert _write(lib, strides=(2048, -128, 64)) == -1
    assert _write(lib, T=0) == 0 and _write(lib, B=0) == 0 and _read(lib, T=0) == 0
    assert lib.hlm_attn_last_error() == b""


def _attend(lib, ptr=0x1000, ws=0x1000, ws_bytes=1 << 40, slots=128, starts=None, start=0, counts=None, prefix=None,
            prefix_slots=0, prefix_length=0, B=1, T=1, H=2, Hkv=2, D=64, window=0, scale=0.125, strides=(2048, 128, 64)):
    p = P(ptr) if ptr else None
    w = P(ws) if ws else None
    return lib.hlm_attn_cached_fwd(p, _strides(*strides), p, p, p, p, p, slots, starts, start, counts, prefix, prefix, prefix, prefix,
                                   prefix_slots, prefix_length, B, T, H, Hkv, D, window, scale, w, ws_bytes, None)


def test_cached_attention_rejects_bad_arguments_before_touching_the_device():
    lib = _lib.load()
    for kwargs, code, msg in [
        (dict(D=96), -2, "head_dim 96"),
        (dict(H=3), -1, "bad shape"),
        (dict(H=0), -1, "bad shape"),
        (dict(ptr=None), -1, "16-byte aligned"),
        (dict(ptr=0x1008), -1, "16-byte aligned"),
        (dict(slots=96), -1, "multiple of 64"),
        (dict(start=128), -1, "do not fit"),
        (dict(scale=0.0), -1, "scale"),
        (dict(scale=float("inf")), -1, "scale"),
        (dict(T=2, strides=(2048, 100, 64)), -1, "multiple of 8"),
        (dict(prefix_length=-1), -1, "prefix length"),
        (dict(prefix_length=10), -1, "multiple of 64"),
        (dict(prefix_length=10, prefix_slots=64), -1, "prefix tensor is null"),
        (dict(prefix_length=65, prefix_slots=64, prefix=P(0x1000)), -1, "beyond its 64 slots"),
        (dict(prefix_length=8192, prefix_slots=8192, prefix=P(0x1000), ws=None), -1, "workspace"),
        (dict(prefix_length=8192, prefix_slots=8192, prefix=P(0x1000), ws=0x1008), -1, "workspace"),
        (dict(prefix_length=8192, prefix_slots=8192, prefix=P(0x1000), ws_bytes=8), -1, "needed"),
        (dict(B=1 << 20, T=1 << 11, starts=P(0x1000)), -2, "too many query rows"),
        (dict(B=1 << 24, T=1, H=4, Hkv=4, starts=P(0x1000)), -2, "too many query rows"),  # 2^26 workgroups
    ]:
        assert _attend(lib, **kwargs) == code, kwargs
        assert msg in lib.hlm_attn_last_error().decode(), (kwargs, lib.hlm_attn_last_error())
    assert _attend(lib, T=0) == 0 and _attend(lib, B=0) == 0


@pytest.mark.parametrize("D", [64, 128])
def test_workspace_is_a_whole_number_of_partial_outputs_and_bounded(D):
    """(splits) x (B T H) x (D + 2) floats: at most 64 of the own keys and 64 of the prefix's."""
    fn = _lib.load().hlm_attn_cached_fwd_workspace_bytes
    some = P(0x1000)
    for B in (1, 3, 64, 500):
        for T in (1, 2, 5, 17, 64, 500, 2000):
            for H, Hkv in ((1, 1), (12, 12), (12, 4), (16, 1)):
                for slots in (64, 2048, 1 << 17):
                    for window in (0, 1, 512):
                        for prefix in (0, 1, 5000):
                            n = fn(B, T, H, Hkv, D, slots, some, 0, None, prefix, window)
                            row = B * T * H * (D + 2) * 4
                            assert n >= 0 and n % row == 0
                            assert n // row <= (128 if prefix else 64)
    assert fn(1, 1, 12, 12, D, 1 << 17, some, 0, None, 0, 64) == 0  # a short window needs no splits
    assert fn(1, 1, 4, 4, D, 1 << 17, None, 63, None, 0, 0) == 0  # nor does a short cache that the host knows of
    assert fn(1, 1, 4, 4, D, 1 << 17, some, 0, None, 0, 0) > 0
    assert fn(1, 1, 4, 4, D, 64, some, 0, None, 60, 0) == 0  # a short prefix is taken with the own keys
    for prefix, window, n in ((8000, 0, 2), (60, 0, 0)):  # many samples: a long one once for all of them
        assert fn(64, 1, 12, 12, D, 64, some, 0, None, prefix, window) >= n * 64 * 12 * (D + 2) * 4
    assert fn(1, 0, 4, 4, D, 64, some, 0, None, 0, 0) == 0 and fn(1, 1, 4, 4, 96, 64, some, 0, None, 0, 0) == -2


# --- Python ---------------------------------------------------------------------------------


def test_cache_rounds_its_capacity_and_pads_its_heads():
    c = hlm_attn.KVCache(2, 100, 3, 80, device="cpu")
    assert (c.capacity, c.kernel_dim, c.head_dim) == (128, 128, 80)
    assert c.k.shape == (2, 3, 8, 8, 16, 16) and c.v.shape == (2, 3, 2, 8, 4, 16, 16) and c.k_scale.shape == (2, 3, 128)
    assert c.nbytes == 2 * 2 * 3 * 128 * (128 + 4)
    assert not c.k_scale.any() and not c.v_scale.any()
    for bad in ((0, 64, 1, 64), (1, 0, 1, 64), (1, 64, 0, 64), (1, 64, 1, 129), (1, 64, 1, 0), (1, (1 << 24) + 1, 1, 64)):
        with pytest.raises(RuntimeError):
            hlm_attn.KVCache(*bad, device="meta")


def test_entry_points_refuse_cpu_tensors_gradients_and_mismatches():
    c = hlm_attn.KVCache(2, 64, 2, 64, device="cpu")
    x = torch.zeros(2, 3, 2, 64, dtype=BF16)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        hlm_attn.kv_cache_write_hip(c, x, x, 0)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        hlm_attn.kv_cache_read_hip(c, 0, 3)
    with pytest.raises(RuntimeError, match="ROCm devices only"):
        hlm_attn.cached_attention_hip(x, c, 0)
    g = x.clone().requires_grad_(True)
    for call in (lambda: hlm_attn.kv_cache_write_hip(c, g, x, 0), lambda: hlm_attn.kv_cache_write_hip(c, x, g, 0),
                 lambda: hlm_attn.cached_attention_hip(g, c, 0)):
        with pytest.raises(RuntimeError, match="no backward"):
            call()
    with pytest.raises(RuntimeError, match="heads of 64"):
        hlm_attn.cached_attention_hip(torch.zeros(2, 3, 2, 32), c, 0)
    with pytest.raises(RuntimeError, match="differ"):
        hlm_attn.kv_cache_write_hip(c, x, x[:, :2], 0)
    with pytest.raises(RuntimeError, match="window_size"):
        hlm_attn.cached_attention_hip(x, c, 0, window_size=0)
    with pytest.raises(RuntimeError, match="without a prefix"):
        hlm_attn.cached_attention_hip(x, c, 0, prefix_length=5)
    with pytest.raises(RuntimeError, match="outside 0"):
        hlm_attn.cached_attention_hip(x, c, 0, prefix=c, prefix_length=65)
    with pytest.raises(RuntimeError, match="heads of 32"):
        hlm_attn.cached_attention_hip(x, c, 0, prefix=hlm_attn.KVCache(1, 64, 2, 32, device="cpu"), prefix_length=5)


def test_places_and_windows_beyond_32_bits():
    """They would wrap in the C ABI's ints: refused, or held as the longest window there is."""
    c = hlm_attn.KVCache(1, 64, 1, 64, device="cpu")
    x = torch.zeros(1, 1, 1, 64, dtype=BF16)
    for start in (2**32, 2**32 + 5, -(2**31) - 1, 2**31):
        for call in (lambda: hlm_attn.kv_cache_write_hip(c, x, x, start), lambda: hlm_attn.kv_cache_read_hip(c, start, 1),
                     lambda: hlm_attn.cached_attention_hip(x, c, start)):
            with pytest.raises(RuntimeError, match="no position"):
                call()
    assert kernels._places(7) == (None, 7)


def test_places_that_are_no_whole_numbers_are_refused():
    c = hlm_attn.KVCache(1, 64, 1, 64, device="cpu")
    x = torch.zeros(1, 1, 1, 64, dtype=BF16)
    for call in (lambda: hlm_attn.kv_cache_write_hip(c, x, x, 1.5), lambda: hlm_attn.kv_cache_read_hip(c, 0.0, 1),
                 lambda: hlm_attn.kv_cache_read_hip(c, 0, 1.5), lambda: hlm_attn.cached_attention_hip(x, c, 2.0)):
        with pytest.raises(TypeError):
            call()


def test_per_sequence_places_are_checked_and_converted():
    cpu = torch.device("cpu")
    assert ops._per_sequence("starts", None, 2, cpu) is None
    t = torch.tensor([1, 2], dtype=torch.int32)
    assert ops._per_sequence("starts", t, 2, cpu) is t
    far = ops._per_sequence("starts", torch.tensor([2**40, -(2**40)]), 2, cpu)
    assert far.dtype == torch.int32 and far.tolist() == [2**31 - 1, -(2**31)]
    for bad in (torch.tensor([1.0, 2.0]), torch.tensor([1, 2, 3]), torch.tensor([[1], [2]])):
        with pytest.raises(RuntimeError, match="starts"):
            ops._per_sequence("starts", bad, 2, cpu)


def test_tensors_that_are_no_cache_are_refused():
    c = hlm_attn.KVCache(1, 64, 2, 64, device="cpu")
    assert ops._cache_dims("cache", *c.tensors()) == (1, 2, 64, 64)
    k, v, ks, vs = c.tensors()
    for bad in ((v, k, ks, vs), (k.to(torch.int8), v, ks, vs), (k, v, ks.double(), vs), (k, v, ks, vs[:, :, :32]),
                (k[:, :1], v, ks, vs), (k.transpose(4, 5), v, ks, vs)):
        with pytest.raises(RuntimeError, match="not those of a KVCache"):
            ops._cache_dims("cache", *bad)
    ext = _lib.load_torch_fwd()
    x = torch.zeros(1, 1, 2, 64, dtype=BF16)
    assert ext.kv_cache_write(x, x, k, v, ks, vs, None, 0, None) is False  # CPU tensors: the general path's
    assert ext.kv_cache_read(k, v, ks, vs, None, 0, None, 1) is None
    assert ext.cached_attn(x, k, v, ks, vs, None, 0, None, None, None, None, None, 0, 0, 0.125) is None


def test_fake_implementations_describe_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        c = hlm_attn.KVCache(2, 64, 2, 128, device="cuda")
        q = torch.empty(2, 3, 4, 128, dtype=BF16, device="cuda")
        k = torch.empty(2, 3, 2, 128, dtype=BF16, device="cuda")
        hlm_attn.kv_cache_write_hip(c, k, k, 0)
        a, b = hlm_attn.kv_cache_read_hip(c, 0, 5)
        assert a.shape == b.shape == (2, 5, 2, 128) and a.dtype == BF16
        o = hlm_attn.cached_attention_hip(q, c, 0)
        assert o.shape == q.shape and o.dtype == BF16


def test_rotary_tables_at_positions_are_the_sequence_tables_rows():
    rope = hlm_attn.RotaryEmbedding(64)
    cos, sin = rope(50, torch.device("cpu"), BF16)
    pos = torch.tensor([[3, 4, 49], [0, 7, 20]])
    c, s = rope.at(pos, BF16)
    assert c.shape == (2, 3, 16) and torch.equal(c, cos[0, 0][pos]) and torch.equal(s, sin[0, 0][pos])


def test_attention_core_caches_on_the_hip_backend_only(monkeypatch):
    cfg = hlm_attn.AttentionConfig(n_layer=4, n_head=4, n_kv_head=2, attention_window=32, attention_full_every=2)
    calls = []
    monkeypatch.setattr(kernels, "kv_cache_write_hip", lambda *a: calls.append(("write", a)))
    monkeypatch.setattr(kernels, "cached_attention_hip", lambda *a, **kw: calls.append(("attend", a, kw)) or "out")
    for layer, window in ((0, 32), (1, None), (3, None)):
        calls.clear()
        core = hlm_attn.AttentionCore(cfg, layer)
        assert core.forward_cached("q", "k", "v", "cache", 7, None, "prefix", 9) == "out"
        assert calls[0] == ("write", ("cache", "k", "v", 7, None))
        assert calls[1] == ("attend", ("q", "cache", 7, None), dict(window_size=window, prefix="prefix", prefix_length=9))
    core.config.attention_backend = "torch"
    with pytest.raises(RuntimeError, match="no cached attention"):
        core.forward_cached("q", "k", "v", "cache", 0)


# --- calls that something watches -------------------------------------------------------------


class _Seen(torch.utils._python_dispatch.TorchDispatchMode):
    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


class _Functions(torch.overrides.TorchFunctionMode):
    def __torch_function__(self, func, types, args=(), kwargs=None):
        return func(*args, **(kwargs or {}))


def _watched(f):
    """f(x) under each thing that has to see the ops themselves."""
    from torch.autograd import forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.zeros(2, 3, 2, 64, dtype=BF16)
    with _Seen():
        f(x)
    with _Functions():
        f(x)
    with forward_ad.dual_level():
        f(x)
    make_fx(lambda x: (f(x), x + 1)[1])(x)
    torch.jit.trace(lambda x: (f(x), x + 1)[1], (x,), check_trace=False)
    torch.func.vmap(lambda x: (f(x), x)[1])(x[None])
    torch.func.functionalize(lambda x: (f(x), x + 1)[1])(x)


@pytest.mark.parametrize("extension", [True, False])
def test_direct_calls_stand_aside_where_the_op_must_be_seen(monkeypatch, extension):
    ext = _lib.load_torch_fwd()
    monkeypatch.setattr(_lib, "_torch_fwd", ext if extension else False)
    x = torch.zeros(2, 3, 2, 64, dtype=BF16)
    taken = []
    with torch.no_grad():
        _watched(lambda x: taken.append(ops.direct_call_ok(x, x)))
        assert taken == [False] * 7
        with torch.device("cpu"):  # a default device is a function mode that changes nothing for them
            assert ops.direct_call_ok(x)
        assert ops.direct_call_ok(x) and not ext.watched()
        taken.clear()
        _watched(lambda x: taken.append(ext.watched()))
        assert taken == [True] * 7


def test_cache_calls_reach_their_ops_where_something_watches(monkeypatch):
    """A traced write that launches at once would be missing from the trace, and the attention's output a constant in it."""
    c = hlm_attn.KVCache(2, 64, 2, 64, device="cpu")
    seen, direct = [], []
    for name in ("write", "read", "attn"):
        op, impl = (f"hip_kv_cache_{name}", f"kv_cache_{name}_impl") if name != "attn" else ("hip_cached_attn", "cached_attn_impl")
        monkeypatch.setattr(ops, op, lambda *a, name=name: seen.append(name))
        monkeypatch.setattr(ops, impl, lambda *a, name=name: direct.append(name))
    monkeypatch.setattr(ops, "hip_attn_fwd", lambda *a: (seen.append("attention"), None))
    monkeypatch.setattr(ops, "attn_fwd_impl", lambda *a: (direct.append("attention"), None))

    def step(x):
        hlm_attn.kv_cache_write_hip(c, x, x, 0)
        hlm_attn.cached_attention_hip(x, c, 0)
        hlm_attn.kv_cache_read_hip(c, 0, 3)
        hlm_attn.attention(x, x, x)

    with torch.no_grad():
        _watched(step)
        assert seen == ["write", "attn", "read", "attention"] * 7 and not direct
        step(torch.zeros(2, 3, 2, 64, dtype=BF16))
        assert direct == ["write", "attn", "read", "attention"]


# --- sizes --------------------------------------------------------------------------------


def test_sizes_that_are_no_whole_numbers_are_refused():
    """A window of 512.5 is none: it was cut to 512."""
    import numpy as np

    c = hlm_attn.KVCache(2, 64, 2, 64, device="cpu")
    x = torch.zeros(2, 3, 2, 64, dtype=BF16)
    one = hlm_attn.KVCache(1, 64, 2, 64, device="cpu")
    for call in (lambda: hlm_attn.cached_attention_hip(x, c, 0, window_size=512.5), lambda: hlm_attn.cached_attention_hip(x, c, 0, window_size=20.0),
                 lambda: hlm_attn.cached_attention_hip(x, c, 0, prefix=one, prefix_length=3.5),
                 lambda: hlm_attn.KVCache(1.5, 64, 2, 64, device="meta"), lambda: hlm_attn.KVCache(1, 100.5, 2, 64, device="meta"),
                 lambda: hlm_attn.KVCache(1, 64, 2.0, 64, device="meta"), lambda: hlm_attn.KVCache(1, 64, 2, 64.0, device="meta")):
        with pytest.raises(TypeError):
            call()
    whole = hlm_attn.KVCache(np.int64(1), np.int64(100), np.int32(2), np.int16(80), device="cpu")
    assert (whole.batch, whole.capacity, whole.n_kv_head, whole.head_dim) == (1, 128, 2, 80)
    with pytest.raises(RuntimeError, match="ROCm devices only"):  # whole numbers of any type pass
        hlm_attn.cached_attention_hip(x, c, np.int64(0), window_size=np.int64(20), prefix=one, prefix_length=np.int32(3))


def test_compiled_calls_take_whole_numbers_that_vary():
    """torch.compile traces the checks, as constants and as sizes that change: on the CPU the call ends at the op itself."""
    c = hlm_attn.KVCache(2, 64, 2, 64, device="cpu")
    one = hlm_attn.KVCache(1, 64, 2, 64, device="cpu")
    x = torch.zeros(2, 3, 2, 64, dtype=BF16)

    def attend(x, start, window, n):
        return hlm_attn.cached_attention_hip(x, c, start, window_size=window, prefix=one, prefix_length=n)

    run = torch.compile(attend, fullgraph=True, backend="eager")
    for start, window, n in ((0, 5, 7), (1, 6, 8), (2, 9, 10)):
        with pytest.raises(RuntimeError, match="ROCm devices only"), torch.no_grad():
            run(x, start, window, n)


@pytest.mark.parametrize("D", [64, 128])
def test_rows_whose_join_would_have_too_many_threads_are_refused(D):
    """256 threads to 8 rows (head dim 128): 2^27 - 7 rows would be 2^32."""
    lib = _lib.load()
    fn = lib.hlm_attn_cached_fwd_workspace_bytes
    some = P(0x1000)
    for rows, ok in (((1 << 27) - 8, True), ((1 << 27) - 7, False), ((1 << 27) - 1, False)):
        n = fn(1, rows, 1, 1, D, 64, some, 0, None, 5000, 64)
        assert n % (rows * (D + 2) * 4) == 0 and n > 0 if ok else n == -2
    assert b"too many query rows" in lib.hlm_attn_last_error()


# --- the plan -----------------------------------------------------------------------------


def plan_of(B, T, H, Hkv, D, slots, prefix, window, starts=P(0x1000), start=0):
    """(own kernel, tiles, splits, prefix kernel, tiles, splits) of hlm_attn_cached_fwd."""
    lib = _lib.load()
    plan = (ctypes.c_int32 * 6)()
    assert lib.hlm_attn_cached_fwd_plan(B, T, H, Hkv, D, slots, starts, start, None, prefix, window, plan) == 0
    return tuple(plan)


def test_plan_of_long_and_short_prefixes():
    """64 samples: a prefix of 60 goes with the own keys, without a join; a long one is read once for all of them."""
    fn = _lib.load().hlm_attn_cached_fwd_workspace_bytes
    some = P(0x1000)
    assert fn(64, 1, 12, 12, 64, 64, some, 0, None, 60, 0) == 0
    assert plan_of(64, 1, 12, 12, 64, 64, 60, 0) == (0, 1, 1, -2, 0, 0)
    assert plan_of(64, 1, 12, 12, 64, 64, 8000, 0)[3] == 1
    assert fn(64, 1, 12, 12, 64, 64, some, 0, None, 8000, 0) >= 2 * 64 * 12 * (64 + 2) * 4
    assert plan_of(1, 1, 4, 4, 64, 64, 0, 0) == (0, 1, 1, -1, 0, 0)
    assert plan_of(0, 1, 4, 4, 64, 64, 0, 0) == (0,) * 6


@pytest.mark.parametrize("D", [64, 128])
def test_plan_names_a_kernel_that_exists_and_agrees_with_the_workspace(D):
    """The own keys' kernel alone, with the prefix in one pass, or beside the prefix's: (0, 0), (0, 1), (1, 1), (1, 2), (2, 2)."""
    import random

    fn = _lib.load().hlm_attn_cached_fwd_workspace_bytes
    rng = random.Random(D)
    seen = set()
    for _ in range(4000):
        H = rng.choice((1, 3, 4, 12, 16))
        Hkv = rng.choice([g for g in (1, 2, 3, 4, 16) if H % g == 0])
        B, T = int(2 ** rng.uniform(0, 8)), int(2 ** rng.choice((0, rng.uniform(0, 11))))
        slots, prefix, window = 64 * int(2 ** rng.uniform(0, 10)), rng.choice((0, int(2 ** rng.uniform(0, 14)))), rng.choice((0, 1, 700))
        v, tiles, splits, vp, ptiles, psplits = plan_of(B, T, H, Hkv, D, slots, prefix, window)
        seen.add((v, vp))
        rows = T * (H // Hkv)
        assert tiles == -(-rows // (16, 64, 128)[v]) and 1 <= splits <= 64
        if vp >= 0:
            assert prefix and ptiles == -(-rows * B // (16, 64, 128)[vp]) and 1 <= psplits <= 64
        else:
            assert vp == (-2 if prefix else -1) and ptiles == psplits == 0
        n = splits + psplits
        assert fn(B, T, H, Hkv, D, slots, P(0x1000), 0, None, prefix, window) == (0 if n == 1 else n * B * T * H * (D + 2) * 4)
    assert seen <= {(v, vp) for v in (0, 1, 2) for vp in (-1, -2)} | {(0, 0), (0, 1), (1, 1), (1, 2), (2, 2)}
    assert len(seen) >= 8


def test_plan_refuses_what_the_call_refuses():
    lib = _lib.load()
    plan = (ctypes.c_int32 * 6)()
    args = lambda **kw: [{**dict(B=1, T=1, H=2, Hkv=2, D=64, slots=64, starts=None, start=0, counts=None, prefix=0, window=0), **kw}[n]
                         for n in ("B", "T", "H", "Hkv", "D", "slots", "starts", "start", "counts", "prefix", "window")]
    assert lib.hlm_attn_cached_fwd_plan(*args(), None) == -1 and b"plan" in lib.hlm_attn_last_error()
    for kw, code in ((dict(D=96), -2), (dict(H=3), -1), (dict(slots=65), -1), (dict(start=64), -1), (dict(prefix=-1), -1)):
        assert lib.hlm_attn_cached_fwd_plan(*args(**kw), plan) == code


# --- the library's kernels --------------------------------------------------------------------


def _kernels_of_library():
    """The metadata of each kernel in the built library, by name: the notes of the code objects in its offload bundles."""
    import struct

    msgpack = pytest.importorskip("msgpack")
    data = _lib.LIB_PATH.read_bytes()
    found, magic = {}, b"__CLANG_OFFLOAD_BUNDLE__"
    at = data.find(magic)
    while at >= 0:
        (n,) = struct.unpack_from("<Q", data, at + 24)
        p = at + 32
        for _ in range(n):
            offset, size, length = struct.unpack_from("<QQQ", data, p)
            target = data[p + 24 : p + 24 + length]
            p += 24 + length
            if b"gfx950" not in target:
                continue
            elf = data[at + offset : at + offset + size]
            (sections,) = struct.unpack_from("<Q", elf, 0x28)
            entry, count = struct.unpack_from("<HH", elf, 0x3A)
            for i in range(count):
                kind, _, _, start, length_ = struct.unpack_from("<IQQQQ", elf, sections + i * entry + 4)
                if kind != 7:  # a note
                    continue
                name, desc, _ = struct.unpack_from("<III", elf, start)
                text = start + 12 + (name + 3) // 4 * 4
                for k in msgpack.unpackb(elf[text : text + desc], strict_map_key=False)["amdhsa.kernels"]:
                    found[k[".name"]] = k
        at = data.find(magic, at + 1)
    return found


def test_the_attention_kernels_fit_their_registers():
    """No scratch memory anywhere, four waves a SIMD (128 registers) for the 16- and 64-row kernels at head dim 64, and no
    kernel that no plan names."""
    import re

    seen = set()
    for name, k in _kernels_of_library().items():
        if "cached_attn_kernel" not in name:
            continue
        D, v, vp = (int(x.replace("n", "-")) for x in re.search(r"cached_attn_kernelILi(\d+)ELi(\d+)ELi(n?\d+)EE", name).groups())
        seen.add((D, v, vp))
        assert k[".private_segment_fixed_size"] == 0 and k[".vgpr_spill_count"] == 0, name
        assert k[".vgpr_count"] + k.get(".agpr_count", 0) <= (128 if D == 64 and v < 2 and vp < 2 else 256), name
    assert seen == {(D, v, vp) for D in (64, 128) for v, vp in
                    [(v, vp) for v in (0, 1, 2) for vp in (-1, -2)] + [(0, 0), (0, 1), (1, 1), (1, 2), (2, 2)]}
