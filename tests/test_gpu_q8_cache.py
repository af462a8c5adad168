"""kv_cache_append_q8 / kv_cache_read_q8 against their definitions in 64 bits.

Scales are one correctly rounded f32 division and codes are decided exactly:
both caches and both scale arrays have to be equal bit for bit, the parts that
an append does not write included.  A value read back is one f32 product,
rounded once more for bf16."""
import pytest
import torch

import _q8
from oxide_b200 import ops

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _cache(dev, b, h, m, d, block, seed):
    """Caches full of other tokens' codes and scales, NaN among the scales."""
    g = torch.Generator(device=dev).manual_seed(seed)
    codes = [torch.randint(-127, 128, (b, h, m, d), generator=g, device=dev, dtype=torch.int8) for _ in range(2)]
    scales = [torch.rand((b, h, -(-m // block)), generator=g, device=dev) * 0.02 for _ in range(2)]
    return [*codes, *scales], g


def _tokens(g, dev, b, h, n, d, dtype):
    x = [torch.randn((b, h, n, d), generator=g, device=dev) for _ in range(2)]
    for t in x:  # tokens of very different sizes: scales grow inside blocks
        t *= torch.exp2(torch.randint(-3, 4, (b, h, n, 1), generator=g, device=dev).float())
    return [t.to(DT[dtype]) for t in x]


def _bits(t):
    return t.view(torch.int32) if t.dtype == torch.float32 else t


def _same(got, want):
    for name, a, b in zip(("k codes", "v codes", "k scales", "v scales"), got, want):
        a, b = a.cpu(), b.cpu()
        if a.dtype == torch.float32:
            assert torch.equal(torch.isnan(a), torch.isnan(b)), name
            a, b = torch.nan_to_num(a), torch.nan_to_num(b)
        bad = (_bits(a) != _bits(b)).nonzero()
        assert bad.numel() == 0, f"{name}: {len(bad)} differ, first at {bad[0].tolist()}"


def _append(cache, x, cur, new, block, tensors=True):
    dev = cache[0].device
    want = [t.cpu() for t in cache]
    _q8.append(*want, x[0].cpu(), x[1].cpu(), cur, new, block)
    lens = torch.tensor(cur, dtype=torch.int32, device=dev) if tensors else cur[0]
    news = torch.tensor(new, dtype=torch.int32, device=dev) if tensors else None
    ops.kv_cache_append_q8(*cache, *x, lens, block, new_lens=news)
    _same(cache, want)


# head sizes and blocks that take every kernel: a warp, a CTA of 256 and of
# 1024 threads an item, and their element-wise forms
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,block", [(128, 1), (128, 4), (128, 16), (128, 64), (128, 128), (64, 32), (80, 8),
                                     (256, 128), (37, 1), (37, 16), (1, 128), (20, 64), (250, 128)])
def test_against_definition(cuda, dtype, d, block):
    b, h, m = 3, 2, 300
    cache, g = _cache(cuda, b, h, m, d, block, d * 1000 + block)
    _append(cache, _tokens(g, cuda, b, h, 131, d, dtype), [0, 77, 169], [131, 100, 131], block)
    _append(cache, _tokens(g, cuda, b, h, 1, d, dtype), [131, 177, 299], [1, 1, 1], block)
    _append(cache, _tokens(g, cuda, b, h, 7, d, dtype), [132, 178, 290], [7, 0, 3], block)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("block", [1, 16, 128])
def test_one_length_for_all(cuda, dtype, block):
    cache, g = _cache(cuda, 2, 3, 256, 128, block, block)
    cur = 0
    for n in (5, 1, 1, 130, 1, 118):  # to the last position
        _append(cache, _tokens(g, cuda, 2, 3, n, 128, dtype), [cur] * 2, [n] * 2, block, tensors=False)
        cur += n
    assert cur == 256


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_exact_ties(cuda, dtype):
    """x / scale at half-integers (amax 127: scale 1) and restated codes at
    half-integers (the scale doubles)."""
    cache, _ = _cache(cuda, 1, 1, 32, 128, 32, 5)
    x = (torch.arange(4 * 128, device=cuda).view(1, 1, 4, 128) % 255 - 127).float() + 0.5
    x = x.clamp(-126.5, 126.5)
    x[..., 0] = 127.0
    x = x.to(DT[dtype])
    _append(cache, [x, -x], [0], [4], 32)
    assert float(cache[2][0, 0, 0]) == 1.0
    y = torch.full((1, 1, 1, 128), 254.0, device=cuda).to(DT[dtype])
    _append(cache, [y, y], [4], [1], 32)
    assert float(cache[2][0, 0, 0]) == 2.0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d", [128, 33])
def test_zero_tiny_huge_and_not_finite(cuda, dtype, d):
    """Zero blocks, subnormal and near-overflow values, NaN and infinities: a
    block that holds one reads as NaN, and stays so until it is written anew."""
    block, m = 8, 64
    cache, g = _cache(cuda, 1, 2, m, d, block, 11)
    x = _tokens(g, cuda, 1, 2, 56, d, dtype)
    x[0][:, :, 0:8] = 0
    x[0][:, :, 8:16] = (x[0][:, :, 8:16].double() * 1e-39).to(x[0].dtype)
    x[0][:, :, 16:24] = (x[0][:, :, 16:24].double().clamp(-9, 9) * 3e37).to(x[0].dtype)
    x[0][:, :, 24:32] = (x[0][:, :, 24:32].double() * 1e-44).to(x[0].dtype)
    x[0][0, 0, 33, 0] = float("nan")
    x[0][0, 1, 34, d - 1] = float("inf")
    x[1][0, 0, 55, 0] = float("-inf")
    _append(cache, x, [0], [56], block)
    ks, vs = cache[2][0], cache[3][0]
    assert bool(torch.isnan(ks[:, 4]).all()) and bool(torch.isnan(vs[0, 6])) and int(torch.isnan(ks[:, :7]).sum()) == 2
    k, v = ops.kv_cache_read_q8(*cache, block, 0, 56, dtype=torch.float32)
    assert bool(torch.isnan(k[0, 0, 32:40]).all()) and not bool(torch.isnan(k[0, 0, :32]).any())
    # behind the NaN in its block, then the block anew
    y = _tokens(g, cuda, 1, 2, 2, d, dtype)
    _append(cache, y, [36], [2], block)
    assert bool(torch.isnan(cache[2][0, :, 4]).all())
    _append(cache, y, [32], [2], block)
    assert not bool(torch.isnan(cache[2][0, :, 4]).any())


@pytest.mark.parametrize("d", [128, 20])
def test_sequences_left_alone(cuda, d):
    """Negative lengths, tokens that do not fit, and no tokens: nothing of the
    sequence changes; padding behind new_lens may hold anything."""
    cache, g = _cache(cuda, 6, 2, 96, d, 16, 3)
    x = _tokens(g, cuda, 6, 2, 10, d, "bf16")
    for t in x:
        t[4, :, 3:] = float("nan")
    _append(cache, x, [-1, 87, 96, 50, 7, -2 ** 31], [10, 10, 1, 0, 3, 10], 16)


def test_poisoned_cache_behind_the_tokens(cuda):
    """Scales and codes behind the cached length may hold anything."""
    cache, g = _cache(cuda, 1, 2, 64, 64, 16, 8)
    cache[2][:, :, 1:] = float("nan")
    cache[3][:, :, 1:] = float("inf")
    _append(cache, _tokens(g, cuda, 1, 2, 40, 64, "bf16"), [16], [40], 16)
    assert bool(torch.isfinite(cache[2][:, :, 1:4]).all())


def test_unaligned(cuda):
    """Caches and tokens off every vector boundary."""
    b, h, m, d, block = 2, 2, 48, 64, 16
    cache, g = _cache(cuda, b, h, m, d, block, 4)
    codes = []
    for t in cache[:2]:
        buf = torch.empty(t.numel() + 1, dtype=torch.int8, device=cuda)
        buf[1:] = t.reshape(-1)
        codes.append(buf[1:].view(t.shape))
    x = _tokens(g, cuda, b, h, 20, d, "bf16")
    off = []
    for t in x:
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)
        buf[1:] = t.reshape(-1)
        off.append(buf[1:].view(t.shape))
    _append([*codes, *cache[2:]], off, [3, 28], [20, 20], block)
    k, v = ops.kv_cache_read_q8(*codes, *cache[2:], block, 5, 30, dtype=torch.float32)
    assert torch.equal(k, _q8.values(codes[0], cache[2], block)[:, :, 5:35].float())
    assert torch.equal(v, _q8.values(codes[1], cache[3], block)[:, :, 5:35].float())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,block,start,n", [(128, 64, 0, 300), (128, 1, 5, 1), (64, 32, 77, 200), (80, 8, 31, 33),
                                             (37, 16, 1, 299), (1, 128, 0, 300), (256, 4, 299, 1), (36, 2, 0, 0)])
@pytest.mark.parametrize("ragged", [False, True])
def test_read_back(cuda, dtype, d, block, start, n, ragged):
    b, h, m = 4, 3, 300
    cache, _ = _cache(cuda, b, h, m, d, block, d + block)
    lens = torch.tensor([0, start + n // 2, 400, -5], dtype=torch.int32, device=cuda) if ragged else None
    if ragged:
        cache[2][0] = float("nan")  # an empty sequence's scales are not read
        cache[3][3] = float("inf")
    got = ops.kv_cache_read_q8(*cache, block, start, n, lens=lens, dtype=DT[dtype])
    at = torch.arange(start, start + n, device=cuda)
    for t, codes, scales in ((got[0], *cache[0::2]), (got[1], *cache[1::2])):
        want = _q8.values(codes, scales, block)[:, :, start:start + n].float()  # the f32 product: 7 x 24 bits, one rounding
        if ragged:
            want = torch.where((at[None, :] < lens[:, None])[:, None, :, None], want, 0.0)
        assert t.shape == (b, h, n, d) and torch.equal(t, want.to(DT[dtype]))


def test_read_into_given_outputs(cuda):
    cache, _ = _cache(cuda, 1, 2, 32, 64, 16, 2)
    k, v = (torch.full((1, 2, 8, 64), 5.0, device=cuda) for _ in range(2))
    got = ops.kv_cache_read_q8(*cache, 16, 4, 8, k=k, v=v)
    assert got[0] is k and got[1] is v and torch.equal(k, _q8.values(cache[0], cache[2], 16)[:, :, 4:12].float())


def test_offsets_past_32_bits(cuda):
    """A cache whose later heads start behind 2^32 codes (two sequences of 2^25
    positions)."""
    m, d, block = 1 << 25, 128, 128
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 18 GB")
    kc = torch.zeros((2, 1, m, d), dtype=torch.int8, device=cuda)
    vc = torch.zeros_like(kc)
    ks = torch.zeros((2, 1, m // block), device=cuda)
    vs = torch.zeros_like(ks)
    g = torch.Generator(device=cuda).manual_seed(1)
    x = _tokens(g, cuda, 2, 1, 200, d, "bf16")
    cur = [m - 200, m - 333]
    ops.kv_cache_append_q8(kc, vc, ks, vs, *x, torch.tensor(cur, dtype=torch.int32, device=cuda), block)
    for i in range(2):
        small = [torch.zeros((1, 1, 512, d), dtype=torch.int8) for _ in range(2)]
        scales = [torch.zeros((1, 1, 4)) for _ in range(2)]
        _q8.append(*small, *scales, x[0][i:i + 1].cpu(), x[1][i:i + 1].cpu(), [cur[i] - (m - 512)], [200], block)
        _same([t[i:i + 1, :, -512:] for t in (kc, vc)] + [t[i:i + 1, :, -4:] for t in (ks, vs)], small + scales)
    k, v = ops.kv_cache_read_q8(kc, vc, ks, vs, block, m - 300, 300, dtype=torch.float32)
    assert torch.equal(k, _q8.values(kc[:, :, -384:], ks[:, :, -3:], block)[:, :, 84:].float())
    assert torch.equal(v, _q8.values(vc[:, :, -384:], vs[:, :, -3:], block)[:, :, 84:].float())
    # and the attention over it: two heads of the second sequence's last keys
    q = torch.randn((2, 2, d), generator=g, device=cuda)
    # all other keys are zero codes: score 0, value 0 -- the definition over the
    # last 512 keys with the others' mass added
    out = ops.decode_attention_q8(q, kc, vc, ks, vs, block, torch.tensor([m, m - 7], dtype=torch.int32, device=cuda))
    for i, n in enumerate((m, m - 7)):
        lo = m - 512
        tail = (q[i:i + 1], *[t[i:i + 1, :, lo:n] for t in (kc, vc)], *[t[i:i + 1, :, lo // block:] for t in (ks, vs)])
        want, mag, tol = _q8.attend(*tail, None, block, d ** -0.5)
        k = _q8.values(tail[1], tail[3], block)[0, 0]
        s = q[i].double() @ k.T * d ** -0.5
        share = torch.exp(torch.logsumexp(s, -1) - torch.logaddexp(torch.logsumexp(s, -1),
                                                                    torch.tensor(float(lo), device=cuda).double().log()))
        # the tail's tolerance, and the mass of the others: each worker adds up
        # to 2^25 / 128 equal weights one after another, half a rounding each
        tol = (tol + mag * 2.0 ** -24 * 2 ** 18) * share[:, None]
        assert bool(((out[i].double() - want[0] * share[:, None]).abs() <= tol[0]).all())


def test_class_round_trip(cuda):
    """KvCacheQ8 as the f32 cache is used: two layers, prompt and tokens."""
    c = ops.KvCacheQ8(2, 2, 3, 64, 100, block=32, dtype=torch.float32)
    g = torch.Generator(device=cuda).manual_seed(2)
    kept = {0: [], 1: []}
    for n in (37, 1, 1, 20):
        for layer in (0, 1):
            x = _tokens(g, cuda, 2, 3, n, 64, "f32")
            c.update(layer, *x)
            kept[layer].append(x)
    assert c.current_seq_len() == 59 and not c.is_full()
    for layer in (0, 1):
        got = c.get(layer)
        for i in (0, 1):
            x = torch.cat([t[i] for t in kept[layer]], 2)
            scale = (c.k_scale, c.v_scale)[i][layer].repeat_interleave(32, 2)[:, :, :59, None]
            # half a step at each rounding: when written, and at most at four restatements
            assert bool(((got[i] - x).abs() <= 2.5 * scale * 1.001).all())
    c.clear()
    assert c.get(0) is None


def test_graph_of_decode_steps(cuda):
    """A captured append whose lengths live on the device, replayed as the
    sequences grow."""
    b, h, m, d, block = 3, 2, 64, 128, 16
    cache, g = _cache(cuda, b, h, m, d, block, 21)
    want = [t.cpu() for t in cache]
    lens = torch.tensor([0, 30, 13], dtype=torch.int32, device=cuda)
    k, v = _tokens(g, cuda, b, h, 1, d, "bf16")
    graph = torch.cuda.CUDAGraph()
    warm = [t.clone() for t in cache]
    ops.kv_cache_append_q8(*warm, k, v, lens, block)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        ops.kv_cache_append_q8(*cache, k, v, lens, block)
        lens += 1
    for step in range(20):
        a, c = _tokens(g, cuda, b, h, 1, d, "bf16")
        k.copy_(a)
        v.copy_(c)
        _q8.append(*want, a.cpu(), c.cpu(), [step, 30 + step, 13 + step], [1] * 3, block)
        graph.replay()
    torch.cuda.synchronize()
    _same(cache, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("d,block", [(128, 1), (128, 16), (128, 64), (128, 128), (256, 128), (37, 1), (37, 16), (20, 64)])
def test_scales_of_fresh_blocks_hold_anything(cuda, dtype, d, block):
    """NaN, infinities and anything else among the scales of blocks at or behind
    each sequence's length: blocks that receive tokens get their own scale, the
    others keep what they hold."""
    b, h, m, cur = 3, 2, 300, [0, 77, 169]
    cache, g = _cache(cuda, b, h, m, d, block, d * 1000 + block)
    for scales in cache[2:]:
        for i, n in enumerate(cur):
            fresh = scales[i, :, -(-n // block):]
            fresh[:, 0::3] = float("nan")
            fresh[:, 1::3] = float("inf")
    _append(cache, _tokens(g, cuda, b, h, 131, d, dtype), cur, [131, 100, 120], block)
    for scales in cache[2:]:
        for i, n in enumerate((131, 177, 289)):
            assert bool(torch.isfinite(scales[i, :, :-(-n // block)]).all())
    _append(cache, _tokens(g, cuda, b, h, 9, d, dtype), [131, 177, 289], [9, 0, 5], block)
