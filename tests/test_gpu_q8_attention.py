"""decode_attention_q8 against the attention over the values the codes stand
for, in 64 bits, element by element within what f32 arithmetic allows
(_q8.attend's tolerance), bf16 outputs with their own rounding on top."""
import pytest
import torch

import _q8
from oxide_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _case(dev, b, hq, hkv, d, m, block, dtype, seed=0, sharp=1.0):
    g = torch.Generator(device=dev).manual_seed(seed + b * 7 + hq * 31 + d * 1009 + m)
    c = [torch.randn((b, hkv, m, d), generator=g, device=dev).mul_(40).round_().clamp_(-127, 127).to(torch.int8)
         for _ in range(2)]
    s = [(torch.rand((b, hkv, -(-m // block)), generator=g, device=dev) + 0.5) / 40 for _ in range(2)]
    q = (torch.randn((b, hq, d), generator=g, device=dev) * sharp).to(DT[dtype])
    return q, c[0], c[1], s[0], s[1]


def _lens(dev, v):
    return torch.tensor(v, dtype=torch.int32, device=dev)


def _close(got, want, tol):
    if got.dtype == torch.bfloat16:
        tol = tol + want.abs() * 2.0 ** -8 + 2.0 ** -134
    err = (got.double() - want).abs()
    assert bool(torch.isfinite(got).all())
    assert bool((err <= tol + 2.0 ** -149).all()), float((err / (tol + 2.0 ** -149)).max())


def _run(case, block, lens, **kw):
    q = case[0]
    got = ops.decode_attention_q8(*case, block, lens, **kw)
    scale = kw.get("scale") or q.shape[2] ** -0.5
    want, mag, tol = _q8.attend(*case, lens, block, scale)
    _close(got, want, tol)
    return got, want


# every group size (and pieces of more than eight), head size and kernel
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 128), (4, 2, 128), (8, 2, 128), (16, 2, 128), (6, 2, 128), (24, 2, 128),
                                      (4, 4, 64), (6, 2, 80), (8, 1, 96), (3, 1, 256), (8, 1, 256), (5, 5, 37),
                                      (12, 4, 20), (34, 2, 36), (2, 1, 1)])
@pytest.mark.parametrize("block", [1, 64])
def test_shapes(cuda, dtype, hq, hkv, d, block):
    case = _case(cuda, 5, hq, hkv, d, 517, block, dtype)
    _run(case, block, _lens(cuda, [517, 0, 1, 129, 300]))


EDGES = [0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 383, 384, 385, 511, 512]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (2, 2, 128), (6, 2, 64)])
@pytest.mark.parametrize("block", [1, 2, 4, 8, 16, 32, 128])
def test_lengths(cuda, dtype, hq, hkv, d, block):
    case = _case(cuda, len(EDGES), hq, hkv, d, 512, block, dtype)
    _run(case, block, _lens(cuda, EDGES))


@pytest.mark.parametrize("d", [128, 80])
def test_lengths_out_of_range_and_all_positions(cuda, d):
    """Lengths are held to [0, max_seq].  The work is divided over all sequences'
    tiles, so another sequence's length changes the order of the sums, not more:
    both calls are within the tolerance of the same definition."""
    case = _case(cuda, 3, 4, 2, d, 300, 16, "f32")
    _run(case, 16, None)
    odd, want = _run(case, 16, _lens(cuda, [-1, 301, 2 ** 31 - 1]))
    assert bool((odd[0] == 0).all()) and bool((want[1:] != 0).all())


@pytest.mark.parametrize("hq,hkv,d,b,m", [(8, 2, 128, 1, 1), (8, 2, 128, 1, 40000), (32, 8, 128, 2, 9000),
                                          (4, 4, 128, 300, 130), (4, 1, 64, 1, 30000), (2, 2, 48, 700, 40),
                                          (67, 1, 128, 1, 5000), (67, 1, 37, 2, 900)])
def test_work_division(cuda, hq, hkv, d, b, m):
    """One sequence over every worker, and many sequences to a worker."""
    case = _case(cuda, b, hq, hkv, d, m, 32, "bf16")
    lens = [m - (i * 37) % m for i in range(b)]
    _run(case, 32, _lens(cuda, lens))


@pytest.mark.parametrize("hq,hkv,d", [(12, 3, 128), (20, 2, 128), (8, 2, 256), (2, 2, 176)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_short_sequences(cuda, hq, hkv, d, dtype):
    """Several sequences to a worker, none, one and two tiles long, in a cache of
    less than two tiles; the query heads change with every one of them."""
    case = _case(cuda, 500, hq, hkv, d, 200, 16, dtype)
    _run(case, 16, _lens(cuda, [(i * 83) % 201 for i in range(500)]))
    case = _case(cuda, 400, hq, hkv, d, 7, 4, dtype)
    _run(case, 4, _lens(cuda, [i % 8 for i in range(400)]))


@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 128), (12, 3, 64), (8, 2, 37), (3, 1, 256)])
def test_a_long_sequence_among_short_ones(cuda, hq, hkv, d):
    """Its parts are many, the others' few, in the same launch; the batch does not
    fill the last group of heads, and most sequences are empty in the end."""
    b, m = 381, 5000 if d > 64 else 20000
    case = _case(cuda, b, hq, hkv, d, m, 128, "bf16")
    lens = [(i * 7) % 40 for i in range(b)]
    lens[b // 2], lens[b - 1] = m, m - 77
    _run(case, 128, _lens(cuda, lens))
    lens = [0] * b
    lens[3] = m
    _run(case, 128, _lens(cuda, lens))


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (2, 2, 128), (16, 2, 128), (6, 2, 80), (3, 3, 33), (8, 2, 256)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_anything_behind_the_length(cuda, hq, hkv, d, dtype):
    """Codes and scales behind a sequence's end may hold anything, -128 and NaN
    among them."""
    block, lens = 8, [200, 8, 0, 131]
    case = _case(cuda, 4, hq, hkv, d, 260, block, dtype)
    clean = ops.decode_attention_q8(*case, block, _lens(cuda, lens))
    for i, n in enumerate(lens):
        for codes, scales in ((case[1], case[3]), (case[2], case[4])):
            codes[i, :, n:] = -128
            scales[i, :, -(-n // block):] = float("nan") if i % 2 else float("inf")
    assert torch.equal(ops.decode_attention_q8(*case, block, _lens(cuda, lens)), clean)
    _run([*case[:3], *[torch.nan_to_num(s, nan=0.0, posinf=0.0) for s in case[3:]]], block, _lens(cuda, lens))


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (2, 2, 128), (6, 2, 80), (8, 2, 256)])
def test_not_finite_inside(cuda, hq, hkv, d):
    """A block with the scale NaN among a sequence's keys, in k or in v, and a
    query head with a NaN or an infinity make exactly their heads NaN."""
    block, lens = 16, _lens(cuda, [200, 200, 200])
    case = _case(cuda, 3, hq, hkv, d, 256, block, "f32")
    clean = ops.decode_attention_q8(*case, block, lens)
    case[3][0, 0, 5] = float("nan")
    case[4][1, 1, 12] = float("nan")
    case[0][2, 0, 3] = float("nan")
    case[0][2, hq - 1, 0] = float("inf")
    got = ops.decode_attention_q8(*case, block, lens)
    rep = hq // hkv
    bad = torch.zeros(3, hq, dtype=torch.bool, device=cuda)
    bad[0, :rep] = True
    bad[1, rep:] = True
    bad[2, 0] = bad[2, hq - 1] = True
    assert torch.equal(torch.isnan(got).all(-1), bad) and torch.equal(torch.isnan(got).any(-1), bad)
    assert torch.equal(got[~bad], clean[~bad])


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (2, 2, 128), (6, 2, 80)])
def test_zero_and_uneven_scales(cuda, hq, hkv, d):
    """Blocks of zeros, scales 60 orders of magnitude apart, and a cache of
    zeros only (the weights are even then, the values zero)."""
    block = 4
    case = _case(cuda, 2, hq, hkv, d, 300, block, "f32")
    case[4][0, :, ::3] = 0.0
    case[3][0, :, 1::3] = 0.0
    e = torch.arange(case[4].shape[2], device=cuda) % 7
    case[4][1] = torch.pow(10.0, e.double() * 10 - 30).float()
    _run(case, block, _lens(cuda, [300, 290]))
    case[4].zero_()
    assert bool((ops.decode_attention_q8(*case, block) == 0).all())


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 2, 128), (6, 2, 80)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_key_takes_all(cuda, hq, hkv, d, dtype):
    """Scores of some hundred: one key holds the weight, wherever its tile is."""
    case = _case(cuda, 4, hq, hkv, d, 1030, 64, dtype, sharp=20.0)
    _run(case, 64, _lens(cuda, [1030, 700, 129, 128]))


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 64)])
def test_faint_keys_add_up(cuda, hq, hkv, d):
    """One key far above a long even rest whose weights are 2^-24 to 2^-20 of it:
    the rest still counts."""
    m, block = 20000, 64
    case = _case(cuda, 1, hq, hkv, d, m, block, "f32")
    q, kc, vc, ks, vs = case
    q.fill_(1.0)
    kc.zero_()
    kc[:, :, 777] = 100
    vc[:, :, :, :] = 100
    vc[:, :, 777] = -100
    ks.fill_(15.0 / 100 / d ** 0.5)  # the key's score is 15: the others' weights are e^-15
    vs.fill_(0.01)
    _run(case, block, None)


@pytest.mark.parametrize("scale", [0.0, -0.5, 3.0])
def test_scale(cuda, scale):
    for d, hq in ((128, 8), (64, 8)):
        case = _case(cuda, 2, hq, 2, d, 200, 16, "f32")
        got = ops.decode_attention_q8(*case, 16, scale=scale)
        want, mag, tol = _q8.attend(*case, None, 16, scale)
        _close(got, want, tol)


def test_repeats_and_own_outputs(cuda):
    """The same call twice gives the same bits; given outputs and workspaces are
    used; a workspace may hold anything before."""
    for d, hq in ((128, 8), (96, 6)):
        case = _case(cuda, 3, hq, 2, d, 3000, 32, "bf16")
        lens = _lens(cuda, [3000, 17, 1999])
        a = ops.decode_attention_q8(*case, 32, lens)
        n = int(_lib.lib().oxide_decode_attention_q8_workspace_bytes(3, hq, 2, d))
        ws = torch.full((n,), 255, dtype=torch.uint8, device=cuda)
        out = torch.empty_like(case[0])
        assert ops.decode_attention_q8(*case, 32, lens, workspace=ws, out=out) is out
        assert torch.equal(out, a)


def test_nothing_behind_the_workspace(cuda):
    for b, hq, hkv, d in ((3, 8, 2, 128), (2, 24, 2, 64)):
        case = _case(cuda, b, hq, hkv, d, 700, 32, "bf16")
        n = int(_lib.lib().oxide_decode_attention_q8_workspace_bytes(b, hq, hkv, d))
        buf = torch.full((n + 4096,), 171, dtype=torch.uint8, device=cuda)
        ops.decode_attention_q8(*case, 32, workspace=buf[:n])
        assert bool((buf[n:] == 171).all())


def test_two_streams(cuda):
    """Two calls at once, each with a workspace of its own."""
    cases = [_case(cuda, 4, 8, 2, 128, 5000, 64, "bf16", seed=s) for s in (1, 2)]
    want = [ops.decode_attention_q8(*c, 64) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(ops.decode_attention_q8(*c, 64))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_graph_replay_with_growing_lengths(cuda):
    case = _case(cuda, 3, 8, 2, 128, 900, 64, "bf16")
    lens = _lens(cuda, [1, 400, 890])
    out = ops.decode_attention_q8(*case, 64, lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.decode_attention_q8(*case, 64, lens, out=out)
    for add in (0, 1, 9):
        lens += add
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.decode_attention_q8(*case, 64, lens))


@pytest.mark.parametrize("b,hq,hkv,d", [(3, 8, 2, 128), (299, 3, 1, 128), (301, 1, 1, 37), (151, 6, 2, 256),
                                        (1201, 2, 2, 20), (1, 1, 1, 16), (4096, 2, 1, 16)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_nothing_around_output_and_workspace(cuda, b, hq, hkv, d, dtype):
    """Guards around both, whichever way the heads are merged."""
    case = _case(cuda, b, hq, hkv, d, 150, 16, dtype)
    lens = _lens(cuda, [(i * 47) % 151 for i in range(b)])
    n = int(_lib.lib().oxide_decode_attention_q8_workspace_bytes(b, hq, hkv, d))
    ws = torch.full((n + 4096,), 171, dtype=torch.uint8, device=cuda)
    out = torch.full((b * hq * d + 64,), 7.0, dtype=case[0].dtype, device=cuda)
    _run(case, 16, lens, workspace=ws[2048:2048 + n], out=out[32:32 + b * hq * d].view(b, hq, d))
    assert bool((ws[:2048] == 171).all()) and bool((ws[2048 + n:] == 171).all())
    assert bool((out[:32] == 7).all()) and bool((out[32 + b * hq * d:] == 7).all())


@pytest.mark.parametrize("d", [128, 36, 37, 256, 1])
@pytest.mark.parametrize("k_off,v_off,q_off", [(1, 0, 0), (0, 2, 0), (3, 5, 1), (4, 8, 0), (0, 0, 1), (16, 16, 8)])
def test_unaligned(cuda, d, k_off, v_off, q_off):
    """Tensors that start anywhere give the same values."""
    case = _case(cuda, 3, 4, 2, d, 333, 8, "bf16")

    def moved(t, off):
        buf = torch.full((t.numel() + off + 16,), 99, dtype=t.dtype, device=cuda)
        buf[off:off + t.numel()] = t.reshape(-1)
        return buf[off:off + t.numel()].view(t.shape)

    lens = _lens(cuda, [333, 64, 100])
    out = moved(torch.zeros_like(case[0]), q_off)
    _run((moved(case[0], q_off), moved(case[1], k_off), moved(case[2], v_off), *case[3:]), 8, lens, out=out)


def test_two_graphs_at_once(cuda):
    """Two captured steps, replayed on two streams."""
    cases = [_case(cuda, b, 8, 2, 128, 3000, 64, "bf16", seed=b) for b in (2, 5)]
    want = [ops.decode_attention_q8(*c, 64) for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.decode_attention_q8(*c, 64))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_matches_bf16_attention_of_the_values(cuda):
    """Against the unquantised operator over the values read back (exact in bf16
    when the scales are powers of two)."""
    case = _case(cuda, 2, 8, 2, 128, 640, 16, "bf16")
    for s in case[3:]:
        s.copy_(torch.exp2(torch.round(torch.log2(s))))
    lens = _lens(cuda, [640, 333])
    k, v = ops.kv_cache_read_q8(*case[1:], 16)
    a = ops.decode_attention_q8(*case, 16, lens).double()
    b = ops.decode_attention(case[0], k, v, lens).double()
    want, mag, tol = _q8.attend(*case, lens, 16, 128 ** -0.5)
    # both round to bf16 once; the bf16 kernel holds its weights in 16 bits
    assert bool(((a - b).abs() <= want.abs() * 2.0 ** -7 + mag * 2.0 ** -13).all())


def test_a_decode_loop(cuda):
    """The operators as they are used together: the layer's normalisation hands
    int8 rows to a product, keys and values go into the int8 cache, attention
    reads it; several steps, against the same steps in 64 bits."""
    b, hq, hkv, d, hidden, block = 3, 8, 2, 128, 256, 16
    g = torch.Generator(device=cuda).manual_seed(0)
    wq, wk, wv = (torch.randn((n * d, hidden), generator=g, device=cuda) / 16 for n in (hq, hkv, hkv))
    w = (torch.rand(hidden, generator=g, device=cuda) + 0.5).bfloat16()
    cache = ops.KvCacheQ8(1, b, hkv, d, 96, block=block)
    mine = [torch.zeros((b, hkv, 96, d), dtype=torch.int8), torch.zeros((b, hkv, 96, d), dtype=torch.int8),
            torch.zeros((b, hkv, 6)), torch.zeros((b, hkv, 6))]
    x = torch.randn((b, 33, hidden), generator=g, device=cuda).bfloat16()
    at = 0
    for step in range(6):
        r = torch.randn(x.shape, generator=g, device=cuda).bfloat16()
        h, codes, scale = ops.add_rms_norm_q8(x, r, w, 1e-5)
        ref = _q8.norm_q8(x, r, w, 1e-5)
        assert torch.equal(h, ref[0]) and torch.equal(codes, ref[1])
        y = codes.float() * scale[..., None]
        n = y.shape[1]
        q, k, v = ((y @ m.T).view(b, n, -1, d).transpose(1, 2).contiguous().bfloat16() for m in (wq, wk, wv))
        cache.update(0, k, v)
        _q8.append(*mine, k.cpu(), v.cpu(), [at] * b, [n] * b, block)
        at += n
        assert torch.equal(cache.k_cache[0].cpu(), mine[0]) and torch.equal(cache.v_scale[0].cpu(), mine[3])
        last = q[:, :, -1].contiguous()
        got = cache.attend(0, last)
        want, mag, tol = _q8.attend(last, *[t.to(cuda) for t in mine], [at] * b, block, d ** -0.5)
        _close(got, want, tol)
        x = torch.randn((b, 1, hidden), generator=g, device=cuda).bfloat16()


def _on_path(path, case, block, lens):
    _lib.lib().oxide_debug_decode_attention_path(path)
    try:
        out = ops.decode_attention_q8(*case, block, lens)
        torch.cuda.synchronize()
    finally:
        _lib.lib().oxide_debug_decode_attention_path(0)
    return out


@pytest.mark.parametrize("hq,hkv,d", [(1, 1, 128), (4, 2, 128), (8, 2, 128), (16, 2, 128), (6, 2, 128), (24, 2, 128),
                                      (8, 2, 64), (8, 2, 16), (4, 4, 112), (8, 2, 256), (3, 1, 144), (16, 1, 208)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_both_kernels(cuda, hq, hkv, d, dtype):
    """Shapes that the tensor-core kernel takes, on it and on the other one."""
    case = _case(cuda, 4, hq, hkv, d, 1000, 32, dtype)
    lens = _lens(cuda, [1000, 999, 3, 514])
    want, mag, tol = _q8.attend(*case, lens, 32, d ** -0.5)
    for path in (0, 1):
        _close(_on_path(path, case, 32, lens), want, tol)


def test_query_magnitudes(cuda):
    """Queries of every magnitude: the digits follow the head's largest element,
    subnormal ones included; a head of zeros weighs its keys evenly."""
    case = _case(cuda, 1, 8, 1, 128, 400, 16, "f32")
    for h, s in enumerate((1e-44, 1e-38, 1e-25, 1e-18, 1.0, 1e3, 0.0, 1e-30)):
        case[0][0, h] = (case[0][0, h].double() * s).float()
    _run(case, 16, None)
    big = case[0].clone()
    big[0, 0] = 3e38 * torch.sign(big[0, 1])
    got = ops.decode_attention_q8(big, *case[1:], 16, scale=1e-38)
    want, mag, tol = _q8.attend(big, *case[1:], None, 16, 1e-38)
    _close(got, want, tol)


@pytest.mark.parametrize("b,hq,hkv,d,m", [(2, 8, 2, 128, 1024), (3, 16, 2, 256, 700), (300, 4, 2, 64, 200)])
def test_a_wait_that_runs_out(cuda, b, hq, hkv, d, m):
    """With its copies withheld every wait of the tensor-core kernel runs out:
    NaN outputs and the sticky flag, then the context works on."""
    case = _case(cuda, b, hq, hkv, d, m, 64, "bf16")
    flags = _lib.C.c_uint32()
    _lib.call("oxide_device_status", 1, _lib.C.byref(flags))
    out = _on_path(2, case, 64, None)
    assert bool(torch.isnan(out).all())
    _lib.call("oxide_device_status", 1, _lib.C.byref(flags))
    assert flags.value == _lib.DEVICE_WAIT_TIMEOUT
    _run(case, 64, None)
    _lib.call("oxide_device_status", 0, _lib.C.byref(flags))
    assert flags.value == 0


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (2, 2, 128), (6, 2, 80), (8, 2, 256), (4, 2, 37), (6, 3, 20)])
@pytest.mark.parametrize("block", [1, 16])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), -0.01])
def test_scales_that_are_not_sound(cuda, hq, hkv, d, block, bad):
    """A key or value scale that is NaN, infinite or negative makes exactly the
    heads NaN that read its block, on either kernel."""
    lens, rep = _lens(cuda, [200, 200, 200]), hq // hkv
    case = _case(cuda, 3, hq, hkv, d, 256, block, "f32")
    clean = [_on_path(path, case, block, lens) for path in (0, 1)]
    case[3][0, 0, 77 // block] = bad
    case[4][1, hkv - 1, 199 // block] = bad
    case[3][2, 0, 255 // block] = case[4][2, 0, 240 // block] = bad  # behind the length
    want = torch.zeros(3, hq, dtype=torch.bool, device=cuda)
    want[0, :rep] = want[1, -rep:] = True
    for path in (0, 1):
        got = _on_path(path, case, block, lens)
        assert torch.equal(torch.isnan(got).all(-1), want) and torch.equal(torch.isnan(got).any(-1), want)
        assert torch.equal(got[~want], clean[path][~want])


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (2, 2, 128), (6, 2, 80), (8, 2, 256), (4, 2, 37), (6, 3, 20)])
@pytest.mark.parametrize("m", [1, 40, 300])
def test_scores_of_minus_infinity(cuda, hq, hkv, d, m):
    """A head whose every score is -infinity (an infinite query element over codes
    of the other sign; products beyond f32) has no softmax: NaN, not the zeros of
    an empty sequence.  Where one key has a finite score, it takes all."""
    case = _case(cuda, 4, hq, hkv, d, m, 16, "f32")
    q, kc, vc, ks, vs = case
    q[0, 0, 3] = float("inf")
    q[1, hq - 1, 3] = float("-inf")
    kc[0, :, :, 3] = -7
    kc[1, :, :, 3] = 7
    q[2] = 3e38
    kc[2] = -100
    q[3] = 3e38
    kc[3] = -100
    kc[3, :, m // 2] = 0
    lens = _lens(cuda, [m, m, m, m])
    bad = torch.zeros(4, hq, dtype=torch.bool, device=cuda)
    bad[0, 0] = bad[1, hq - 1] = bad[2] = True
    only = (vc[3, :, m // 2].double() * vs[3, :, m // 2 // 16, None]).repeat_interleave(hq // hkv, 0)
    for path in (0, 1):
        got = _on_path(path, case, 16, lens)
        assert torch.equal(torch.isnan(got).all(-1), bad) and torch.equal(torch.isnan(got).any(-1), bad)
        # one weight of 1: the product code * scale, and at most four roundings and two base-2 functions
        assert bool(((got[3] - only).abs() <= (4 * 2.0 ** -24 + 2 * 2.0 ** -22) * only.abs()).all())
        assert bool((_on_path(path, case, 16, _lens(cuda, [0, 0, 0, 0])) == 0).all())


def _sink_case(dev, hq, hkv, d, m, dtype, gap):
    """One key (position 5) whose score is about `gap` above the others' and whose
    values are zero, so that the others make up the output.  Queries are whole
    numbers of a few bits, which every form of the kernels holds exactly."""
    g = torch.Generator(device=dev).manual_seed(hq * 31 + d * 1009 + m)
    q = torch.randint(1, 8, (2, hq, d), generator=g, device=dev).to(DT[dtype])
    kc = torch.randint(-6, 7, (2, hkv, m, d), generator=g, device=dev).to(torch.int8)
    vc = torch.randint(-127, 128, (2, hkv, m, d), generator=g, device=dev).to(torch.int8)
    kc[:, :, 5] = 100
    vc[:, :, 5] = 0
    ks = torch.full((2, hkv, -(-m // 16)), 1.0, device=dev)
    scale = gap / (4.0 * d * 100)  # q . k of the strong key: about 4 d 100
    vs = torch.rand((2, hkv, -(-m // 16)), generator=g, device=dev) + 0.5
    return (q, kc, vc, ks, vs), scale


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv,d,m", [(2, 2, 128, 100), (4, 2, 128, 300), (8, 2, 128, 100), (16, 2, 128, 1000), (6, 2, 64, 100),
                                        (8, 2, 256, 129), (16, 2, 256, 100), (2, 2, 37, 100), (3, 1, 144, 700)])
@pytest.mark.parametrize("gap", [4, 8, 12, 16, 20, 24, 30])
def test_a_sink_without_values(cuda, hq, hkv, d, m, dtype, gap):
    """The weights of the other keys keep their bits however far the strongest key
    is above them: f32's tolerance relative to sum p |v|, on either kernel.  u =
    2^-24 a rounding: scores of at most d products and eight roundings more, three
    base-2 functions of 2^-22 and 16 roundings in the sums and the quotient, twice
    (numerator and denominator).  The tensor-core kernel holds a weight to 2^-61 of
    the largest p vs of its tile beside that."""
    (q, kc, vc, ks, vs), scale = _sink_case(cuda, hq, hkv, d, m, dtype, gap)
    want, mag, _ = _q8.attend(q, kc, vc, ks, vs, None, 16, scale)
    u, rep = 2.0 ** -24, hq // hkv
    k = _q8.values(kc, ks, 16)
    size = (q.double().view(2, hkv, rep, d).abs() @ k.abs().transpose(2, 3)).amax(-1).view(2, hq, 1) * scale
    held = 2.0 ** -61 * vs.double().amax(-1) * vc.double().abs().sum(2).amax(-1)
    tol = mag * (2 * (d + 8) * u * size + 2 * (3 * 2.0 ** -22 + 16 * u)) + held.repeat_interleave(rep, 1)[..., None]
    for path in (0, 1):
        _lib.lib().oxide_debug_decode_attention_path(path)
        try:
            got = ops.decode_attention_q8(q, kc, vc, ks, vs, 16, scale=scale)
        finally:
            _lib.lib().oxide_debug_decode_attention_path(0)
        _close(got, want, tol)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 128), (4, 2, 128), (8, 2, 128), (16, 2, 128), (6, 2, 64), (8, 2, 256), (16, 2, 256),
                                      (2, 2, 37), (3, 1, 144)])
@pytest.mark.parametrize("strong", [100.0, 1e4, 1e6])
def test_a_strong_channel_over_zero_codes(cuda, hq, hkv, d, dtype, strong):
    """One query element far above the others, and keys that are zero there: the
    scores come from the small elements, which keep their bits.  u = 2^-24 a
    rounding: scores of d products and eight roundings more, relative to sum |q k|;
    three base-2 functions of 2^-22 and 16 roundings in sums and quotient; twice.
    (bf16 elements are whole units of 2^-30 of the largest down to 2^-23 of it, f32
    ones of 2^-61 down to 2^-37: nothing is left out.)"""
    block = 16
    q, kc, vc, ks, vs = _case(cuda, 2, hq, hkv, d, 300, block, dtype, seed=int(strong))
    q[:, :, 7] = strong
    kc[..., 7] = 0
    # elements of at least 2^-10, so that bf16's and f32's lie in whole units
    q.copy_(torch.where(q.abs() < 2.0 ** -10, torch.full_like(q, 2.0 ** -10), q))
    lens = _lens(cuda, [300, 77])
    want, mag, _ = _q8.attend(q, kc, vc, ks, vs, lens, block, d ** -0.5)
    u, rep = 2.0 ** -24, hq // hkv
    size = (q.double().view(2, hkv, rep, d).abs() @ _q8.values(kc, ks, block).abs().transpose(2, 3)).amax(-1)
    size = size.view(2, hq, 1) * d ** -0.5
    held = 2.0 ** -61 * vs.double().amax(-1) * vc.double().abs().sum(2).amax(-1)
    tol = mag * (2 * (d + 8) * u * size + 2 * (3 * 2.0 ** -22 + 16 * u)) + held.repeat_interleave(rep, 1)[..., None]
    for path in (0, 1):
        _close(_on_path(path, (q, kc, vc, ks, vs), block, lens), want, tol)


@pytest.mark.parametrize("hq,hkv,d", [(2, 2, 128), (4, 2, 128), (8, 2, 128), (16, 2, 128), (8, 2, 256), (2, 2, 37), (6, 2, 64)])
@pytest.mark.parametrize("n", [1, 100, 400])
@pytest.mark.parametrize("score", [-3000.0, -70.0, 40.0, 300.0, 5000.0])
def test_scores_far_from_zero(cuda, hq, hkv, d, n, score):
    """Keys that are alike have weights of exactly 1 / n however large their score
    is, so its rounding is nobody's excuse: the output is the mean of the values
    within three base-2 functions (2^-22), 16 roundings in the sums and the
    quotient and a sum of n values, twice, and 2^-61 of the tile's largest."""
    g = torch.Generator(device=cuda).manual_seed(n + d)
    q = torch.full((2, hq, d), 0.7, device=cuda)
    kc = torch.full((2, hkv, n, d), 91, dtype=torch.int8, device=cuda)
    vc = torch.randint(-127, 128, (2, hkv, n, d), generator=g, device=cuda).to(torch.int8)
    blocks = -(-n // 16)
    ks = torch.full((2, hkv, blocks), 0.013, device=cuda)
    vs = (torch.rand((2, hkv, blocks), generator=g, device=cuda) + 0.1) * 0.02
    scale = score / (0.7 * 91 * 0.013 * d)
    v = _q8.values(vc, vs, 16)
    want, mag = (t.mean(2).repeat_interleave(hq // hkv, 1) for t in (v, v.abs()))
    held = 2.0 ** -61 * vs.double().amax(-1) * vc.double().abs().sum(2).amax(-1)
    tol = mag * 2 * (3 * 2.0 ** -22 + (16 + n / 32) * 2.0 ** -24) + held.repeat_interleave(hq // hkv, 1)[..., None]
    for path in (0, 1):
        _lib.lib().oxide_debug_decode_attention_path(path)
        try:
            got = ops.decode_attention_q8(q, kc, vc, ks, vs, 16, scale=scale)
        finally:
            _lib.lib().oxide_debug_decode_attention_path(0)
        _close(got, want, tol)


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (2, 2, 128), (6, 2, 80), (16, 2, 256), (4, 2, 37), (6, 3, 20)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_queries_that_are_not_finite(cuda, hq, hkv, d, dtype):
    """A NaN or an infinity in a query head makes that head NaN and no other, on
    either kernel."""
    case = _case(cuda, 3, hq, hkv, d, 300, 16, dtype)
    lens = _lens(cuda, [300, 1, 129])
    clean = [_on_path(path, case, 16, lens) for path in (0, 1)]
    for b, h, i, v in ((0, 0, d - 1, "nan"), (1, hq - 1, 0, "inf"), (2, 1, d // 2, "-inf")):
        case[0][b, h, i] = float(v)
    bad = ~torch.isfinite(case[0]).all(-1)
    for path in (0, 1):
        got = _on_path(path, case, 16, lens)
        assert torch.equal(torch.isnan(got).all(-1), bad) and torch.equal(torch.isnan(got).any(-1), bad)
        assert torch.equal(got[~bad], clean[path][~bad])
