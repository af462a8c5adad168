"""Refusals of the int8 operators, on the CPU: the C entry points reject bad
sizes, pointers and workspaces before they touch a device, and the tensor-level
ops reject wrong shapes and dtypes before the device check."""
import pytest
import torch

from oxide_b200 import OxideError, ops

FAKE, FAK2, FAK3 = 0x1000, 0x2000, 0x3000  # never dereferenced: every case fails validation first
f32, bf16, i8, i32 = torch.float32, torch.bfloat16, torch.int8, torch.int32


def _append(l, b=1, h=2, m=64, d=16, block=16, cur=0, cl=None, n=4, nl=None, ptrs=None):
    p = ptrs or (FAKE, FAK2, FAKE, FAK2, FAKE, FAK2)
    return l.oxide_kv_cache_append_q8_f32(*p, b, h, m, d, block, cur, cl, n, nl, None)


def _read(l, b=1, h=2, m=64, d=16, block=16, start=0, n=4, ptrs=None):
    p = ptrs or (FAKE, FAK2, FAKE, FAK2, FAKE, FAK2)
    return l.oxide_kv_cache_read_q8_bf16(*p, b, h, m, d, block, start, n, None, None)


def _attend(l, b=1, hq=4, hkv=2, m=64, d=16, block=16, ws=FAK3, wb=None, out=FAK2, q=FAKE):
    need = l.oxide_decode_attention_q8_workspace_bytes(b, hq, max(hkv, 1), d) if wb is None else wb
    return l.oxide_decode_attention_q8_f32(q, FAKE, FAK2, FAKE, FAK2, None, out, b, hq, hkv, m, d, block, 0.25, ws,
                                           need, None)


@pytest.mark.parametrize("call", [
    lambda l: l.oxide_rms_norm_q8_f32(FAKE, FAKE, FAK2, None, 4, 8, 1e-5, None),
    lambda l: l.oxide_rms_norm_q8_f32(FAKE, FAKE, FAK2, FAK3, 4, 0, 1e-5, None),
    lambda l: l.oxide_rms_norm_q8_bf16(FAKE, FAKE, FAKE, FAK3, 4, 8, 1e-5, None),  # codes over x
    lambda l: l.oxide_rms_norm_q8_f32(FAKE, FAKE, FAK2, FAK3, 1 << 40, 1 << 30, 1e-5, None),
    lambda l: l.oxide_add_rms_norm_q8_f32(FAKE, FAKE, FAKE, None, FAK2, FAK3, 4, 8, 1e-5, None),
    lambda l: l.oxide_add_rms_norm_q8_f32(FAKE, FAKE, FAKE, FAK2, FAK2, FAK3, 4, 8, 1e-5, None),  # codes over h
    lambda l: _append(l, block=0),
    lambda l: _append(l, block=24),
    lambda l: _append(l, block=256),
    lambda l: _append(l, cur=61),                       # 61 + 4 > 64
    lambda l: _append(l, n=65, cl=FAKE),                # more than the cache holds
    lambda l: _append(l, m=1 << 31),
    lambda l: _append(l, d=1 << 16),
    lambda l: _append(l, b=1 << 20, h=1 << 20),
    lambda l: _append(l, b=1 << 15, h=1 << 15, m=1 << 30, d=1 << 15),
    lambda l: _append(l, ptrs=(FAKE, FAK2, FAKE, None, FAKE, FAK2)),
    lambda l: _append(l, ptrs=(FAKE, FAKE, FAKE, FAK2, FAKE, FAK2)),  # one buffer for both caches
    lambda l: _read(l, start=61),
    lambda l: _read(l, n=65),
    lambda l: _read(l, block=3),
    lambda l: _read(l, ptrs=(FAKE, FAK2, FAKE, FAK2, FAKE, FAKE)),
    lambda l: _attend(l, hq=5),
    lambda l: _attend(l, hkv=0),
    lambda l: _attend(l, d=257),
    lambda l: _attend(l, d=0),
    lambda l: _attend(l, m=0),
    lambda l: _attend(l, b=4097),
    lambda l: _attend(l, block=12),
    lambda l: _attend(l, b=4096, hq=64, hkv=64, m=1 << 24),
    lambda l: _attend(l, out=FAKE),
    lambda l: _attend(l, q=None),
])
def test_invalid_arguments(olib, call):
    assert call(olib.lib()) == olib.ERR_INVALID_ARG
    assert olib.last_error() != ""


def test_workspace_is_checked(olib):
    l = olib.lib()
    need = l.oxide_decode_attention_q8_workspace_bytes(1, 4, 2, 16)
    assert _attend(l, wb=need - 1) == olib.ERR_WORKSPACE
    assert _attend(l, ws=None) == olib.ERR_WORKSPACE
    assert _attend(l, ws=FAK3 + 4) == olib.ERR_WORKSPACE


def test_empty_calls_do_nothing(olib):
    l = olib.lib()
    none = (None,) * 6
    assert l.oxide_rms_norm_q8_f32(None, None, None, None, 0, 8, 1e-5, None) == 0
    assert l.oxide_add_rms_norm_q8_bf16(None, None, None, None, None, None, 0, 8, 1e-5, None) == 0
    assert l.oxide_kv_cache_append_q8_f32(*none, 1, 2, 64, 16, 16, 64, None, 0, None, None) == 0
    assert l.oxide_kv_cache_append_q8_bf16(*none, 0, 2, 64, 16, 16, 0, None, 4, None, None) == 0
    assert l.oxide_kv_cache_read_q8_f32(*none, 1, 2, 64, 16, 16, 64, 0, None, None) == 0
    assert l.oxide_decode_attention_q8_f32(None, None, None, None, None, None, None, 0, 4, 2, 64, 16, 16, 1.0, None, 0,
                                           None) == 0


@pytest.mark.parametrize("name", ["oxide_rms_norm_q8_f32", "oxide_kv_cache_append_q8_bf16",
                                  "oxide_kv_cache_read_q8_f32", "oxide_decode_attention_q8_f32"])
def test_injected_failure(olib, name):
    l = olib.lib()
    l.oxide_debug_fail_next(name.encode())
    args = [0 if t is olib.u64 else 0.0 if t is olib.f32 else None for t in olib.SIGNATURES[name][1]]
    assert getattr(l, name)(*args) == olib.ERR_INJECTED


def raises(match, fn, *a, **k):
    with pytest.raises(OxideError, match=match):
        fn(*a, **k)


def t(*shape, dtype=f32):
    return torch.zeros(shape, dtype=dtype)


def test_norm_shapes():
    x, w = t(4, 32), t(32)
    raises("weight dtype", ops.rms_norm_q8, x, t(32, dtype=bf16), 1e-5)
    raises("last dim", ops.rms_norm_q8, x, t(16), 1e-5)
    raises("out must be int8", ops.rms_norm_q8, x, w, 1e-5, out=t(4, 32))
    raises("out must be int8", ops.rms_norm_q8, x, w, 1e-5, out=t(4, 31, dtype=i8))
    raises("scale must be", ops.rms_norm_q8, x, w, 1e-5, scale=t(3))
    raises("rows must not be empty", ops.rms_norm_q8, t(4, 0), t(0), 1e-5)
    raises("residual", ops.add_rms_norm_q8, x, t(4, 16), w, 1e-5)
    raises("h must be", ops.add_rms_norm_q8, x, x, w, 1e-5, h=t(4, 32, dtype=bf16))
    raises("scale must be", ops.add_rms_norm_q8, x, x, w, 1e-5, scale=t(4, dtype=bf16))
    raises("CUDA device", ops.rms_norm_q8, x, w, 1e-5)


def _caches(b=2, h=2, m=40, d=16, block=16):
    s = (b, h, -(-m // block))
    return t(b, h, m, d, dtype=i8), t(b, h, m, d, dtype=i8), t(*s), t(*s)


def test_append_shapes():
    c, k = _caches(), t(2, 2, 3, 16)
    raises("block must be", ops.kv_cache_append_q8, *c, k, k, 0, 20)
    raises("k_scale must be", ops.kv_cache_append_q8, *c, k, k, 0, 8)
    raises("caches must be int8", ops.kv_cache_append_q8, t(2, 2, 40, 16), *c[1:], k, k, 0, 16)
    raises("do not match", ops.kv_cache_append_q8, *c, k, t(2, 2, 3, 16, dtype=bf16), 0, 16)
    raises("do not match", ops.kv_cache_append_q8, *c, t(2, 1, 3, 16), t(2, 1, 3, 16), 0, 16)
    raises("overflow", ops.kv_cache_append_q8, *c, k, k, 38, 16)
    raises("cur_len must be", ops.kv_cache_append_q8, *c, k, k, -1, 16)
    raises("cur_len must be int32", ops.kv_cache_append_q8, *c, k, k, torch.zeros(2, dtype=torch.int64), 16)
    raises("new_lens must be int32", ops.kv_cache_append_q8, *c, k, k, 0, 16, new_lens=torch.zeros(1, dtype=i32))
    raises("CUDA device", ops.kv_cache_append_q8, *c, k, k, 0, 16)


def test_read_shapes():
    c = _caches()
    raises("out of range", ops.kv_cache_read_q8, *c, 16, 39, 2)
    raises("out of range", ops.kv_cache_read_q8, *c, 16, -1)
    raises("not float32/bfloat16", ops.kv_cache_read_q8, *c, 16, dtype=torch.float16)
    raises("k must be", ops.kv_cache_read_q8, *c, 16, 0, 4, k=t(2, 2, 5, 16))
    raises("v must be", ops.kv_cache_read_q8, *c, 16, 0, 4, k=t(2, 2, 4, 16), v=t(2, 2, 4, 16, dtype=bf16))
    raises("lens must be", ops.kv_cache_read_q8, *c, 16, lens=torch.zeros(3, dtype=i32))


def test_attend_shapes():
    c, q = _caches(), t(2, 4, 16)
    raises("do not match", ops.decode_attention_q8, t(1, 4, 16), *c, 16)
    raises("not a multiple", ops.decode_attention_q8, t(2, 3, 16), *c, 16)
    raises("lens must be", ops.decode_attention_q8, q, *c, 16, lens=torch.zeros(2))
    raises("out must be", ops.decode_attention_q8, q, *c, 16, out=t(2, 4, 16, dtype=bf16))
    raises("workspace must hold", ops.decode_attention_q8, q, *c, 16, workspace=torch.zeros(8, dtype=torch.uint8))
    raises("v_scale must be", ops.decode_attention_q8, q, *c[:3], t(2, 2, 2), 16)


def test_cache_class_refuses():
    c = ops.KvCacheQ8(1, 2, 2, 16, 40, block=16, device="cpu")
    raises("out of range", c.update, 1, t(2, 2, 1, 16), t(2, 2, 1, 16))
    raises("overflow", c.update, 0, t(2, 2, 41, 16), t(2, 2, 41, 16))
    raises("block must be", ops.KvCacheQ8, 1, 2, 2, 16, 40, block=48, device="cpu")
    assert c.get(0) is None and c.current_seq_len() == 0
    assert c.get_cache_size() == 2 * (2 * 2 * 40 * 16 + 2 * 2 * 3 * 4)


def test_work_division_formulas():
    """Host restatement of oxide_attn_q8.cuh's two divisions: worker c of W begins
    at floor(c T / W), and tile t belongs to floor(((t + 1) W - 1) / T) -- from an
    f64 product with 1 / W and from an f32 quotient off by up to two units in
    the last place, each put right by its remainder."""
    import random

    import numpy as np

    f = np.float32

    def corrected(n, d, q):
        r = n - q * d
        return q - 1 if r < 0 else q + 1 if r >= d else q

    rng = random.Random(5)
    for _ in range(20000):
        T = rng.choice([rng.randrange(1, 1 << 31), rng.randrange(1, 5000), (1 << 31) - 1])
        W = rng.choice([1, 148, rng.randrange(1, 2561), 2560])
        c = rng.choice([0, W, rng.randrange(0, W + 1)])
        assert corrected(c * T, W, int(float(c * T) * (1.0 / W))) == c * T // W
        t = rng.choice([0, T - 1, rng.randrange(0, T)])
        n = (t + 1) * W - 1
        for ulps in range(-2, 3):
            q = f(f(n) / f(T)) * f(1 + ulps * 2.0 ** -23)
            owner = corrected(n, T, int(q))
            assert owner == n // T and owner * T // W <= t
