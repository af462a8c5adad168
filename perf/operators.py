"""Cases of the 8-bit serving operators: the normalisation that hands its rows
on as int8, the KV cache held as int8, and the decode attention over it.

Every 8-bit tensor here is symmetric int8: a code c stands for c * s with an
f32 scale s = amax / 127 of its group, and c is the integer nearest to x / s
(ties to even).  The operators:

  norm    h = x + r (as stored), y = rms_norm(h) * w, y as codes with one
          scale a row: scale = max|y| / 127, code = nearest(y / scale).  The
          row's rms cancels in y / scale, so the codes are decided by the
          products h * w alone: nearest(127 h w / max|h w|).
  append  new keys and values written into int8 caches [batch, kv_heads,
          max_seq, head_dim] with one scale for each block of tokens and head
          ([batch, kv_heads, blocks]).  A block that already holds tokens of
          its sequence keeps the larger of its scale and the new tokens'; if
          the scale grows, the codes it holds are restated in the new one.
  read    a range of cached positions as keys and values again, c * s, zeros
          behind each sequence's length.
  attend  one query token a sequence against the int8 cache: softmax over the
          keys below lens[b], grouped query heads, zeros for an empty sequence.

Codes are whole numbers and are returned as they are held, beside their
scales: both sides decide them from exact quotients, so they have to be equal.
"""
import os
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}


def _ops():
    """The framework's tensor-level entry points."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    pkg = os.path.join(root, "mistralrs-oxide_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from oxide_b200 import ops
    return ops


# ---- the cases ------------------------------------------------------------------
def _norm(rows, cols, dtype, residual):
    return {"op": "norm", "rows": rows, "cols": cols, "dtype": dtype, "residual": residual}


def _append(batch, kv_heads, head_dim, max_seq, block, new, cur, ragged, dtype):
    return {"op": "append", "batch": batch, "kv_heads": kv_heads, "head_dim": head_dim, "max_seq": max_seq,
            "block": block, "new": new, "cur": cur, "ragged": ragged, "dtype": dtype}


def _read(batch, kv_heads, head_dim, max_seq, block, start, n, ragged, dtype):
    return {"op": "read", "batch": batch, "kv_heads": kv_heads, "head_dim": head_dim, "max_seq": max_seq,
            "block": block, "start": start, "n": n, "ragged": ragged, "dtype": dtype}


def _attend(batch, q_heads, kv_heads, head_dim, max_seq, block, shortest, longest, dtype):
    return {"op": "attend", "batch": batch, "q_heads": q_heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "max_seq": max_seq, "block": block, "shortest": shortest, "longest": longest, "dtype": dtype}


def listed():
    return [
        # one decode step of eight sequences: latency
        {"name": "norm decode", **_norm(8, 4096, "bf16", True)},
        # a prefill of eight prompts of 2048 tokens
        {"name": "norm prefill", **_norm(16384, 4096, "bf16", True)},
        # f32 activations with an odd row length, no residual (a first layer's norm)
        {"name": "norm f32 odd", **_norm(2047, 4097, "f32", False)},
        # every decode step writes one token a sequence, each at its own length
        {"name": "append decode", **_append(64, 8, 128, 4096, 64, 1, 1, True, "bf16")},
        # a padded prefill of eight prompts into empty caches
        {"name": "append prefill", **_append(8, 8, 128, 4096, 64, 2048, 0, True, "bf16")},
        # a chunk of a prompt that starts and ends inside a block, f32, another head size
        {"name": "append f32 chunk", **_append(3, 5, 80, 2048, 16, 333, 777, False, "f32")},
        # whole caches read back for a prefill's products
        {"name": "read bf16", **_read(8, 8, 128, 8192, 64, 0, 8192, True, "bf16")},
        # an odd range of a small f32 cache
        {"name": "read f32 odd", **_read(3, 5, 64, 1500, 32, 77, 1001, True, "f32")},
        # the decode step of eight sequences of 1024 to 32768 tokens
        {"name": "attend long batch", **_attend(8, 32, 8, 128, 32768, 64, 1024, 32768, "bf16")},
        # one long sequence alone: the work is split over its keys
        {"name": "attend one long", **_attend(1, 32, 8, 128, 131072, 128, 131072, 131072, "bf16")},
        # short sequences, an empty one among them, no head groups, f32: latency
        {"name": "attend short f32", **_attend(16, 8, 8, 128, 512, 16, 0, 500, "f32")},
        # three query heads a group and another head size
        {"name": "attend odd heads", **_attend(5, 12, 4, 80, 4000, 8, 1, 3999, "bf16")},
    ]


def _span(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    import math
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "norm", "append", "append", "read", "attend", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if op == "norm":
        cols = rng.choice([_span(rng, 1, 16384), 16 * _span(rng, 1, 1024), 4096])
        rows = _span(rng, 1, max(1, min(16384, (16 << 20) // cols)))
        return _norm(rows, cols, dtype, rng.random() < 0.7)
    head_dim = rng.choice([128, 128, 64, 80, 96, 256, 37])
    kv_heads = _span(rng, 1, 16)
    batch = _span(rng, 1, 32)
    block = rng.choice([1, 4, 8, 16, 32, 64, 128])
    if op == "attend":
        max_seq = _span(rng, 1, max(2, min(65536, (96 << 20) // (batch * kv_heads * head_dim))))
        longest = rng.randint(0, max_seq)
        shortest = rng.randint(0, longest)
        return _attend(batch, kv_heads * rng.choice([1, 2, 3, 4, 8]), kv_heads, head_dim, max_seq, block,
                       shortest, longest, dtype)
    blocks = max(2, _span(rng, 1, max(2, min(8192, (24 << 20) // (batch * kv_heads * head_dim)))) // block)
    max_seq = block * blocks
    if op == "append":
        new = _span(rng, 1, max_seq)
        return _append(batch, kv_heads, head_dim, max_seq, block, new, rng.randint(0, max_seq - new),
                       rng.random() < 0.5, dtype)
    start = rng.randint(0, max_seq - 1)
    return _read(batch, kv_heads, head_dim, max_seq, block, start, rng.randint(1, max_seq - start),
                 rng.random() < 0.5, dtype)


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, not in order."""
    if n == 1:
        return [hi]
    v = [lo + (hi - lo) * i // (n - 1) for i in range(n)]
    return v[1::2] + v[0::2]


def _places(case):
    """append: (cached length, new tokens) of each sequence."""
    b, m, new, cur = case["batch"], case["max_seq"], case["new"], case["cur"]
    if not case["ragged"]:
        return [cur] * b, [new] * b
    return _spread(cur, m - new, b), _spread(max(1, new // 2), new, b)


def _read_lens(case):
    b, last = case["batch"], case["start"] + case["n"]
    return _spread(case["start"], last, b) if case["ragged"] else [last] * b


def _attend_lens(case):
    return _spread(case["shortest"], case["longest"], case["batch"])


# ---- inputs ---------------------------------------------------------------------
def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 2654435761 % (1 << 62) + 1)


def _rows(g, *shape):
    """Activations: N(0, 1) with a few strong channels."""
    x = torch.randn(shape, generator=g, device="cuda")
    gain = 1.0 + 7.0 * (torch.rand(shape[-1], generator=g, device="cuda") > 0.97)
    return x * gain


def _cache(g, batch, kv_heads, max_seq, head_dim, block):
    """A filled cache: codes as absolute-maximum scales leave them (about
    N(0, 36), the largest +-127) and scales of N(0, 1) rows."""
    blocks = (max_seq + block - 1) // block
    codes = torch.randn((batch, kv_heads, max_seq, head_dim), generator=g, device="cuda")
    codes = codes.mul_(36.0).round_().clamp_(-127, 127).to(torch.int8)
    scales = (0.7 + 0.6 * torch.rand((batch, kv_heads, blocks), generator=g, device="cuda")) / 36.0
    return codes, scales


def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = _generator(seed)
    dt = _DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "norm":
        s["x"] = _rows(g, case["rows"], case["cols"]).to(dt)
        s["r"] = _rows(g, case["rows"], case["cols"]).to(dt) if case["residual"] else None
        s["w"] = (0.5 + torch.rand(case["cols"], generator=g, device="cuda")).to(dt)
        return s
    b, hkv, d, m, block = (case[k] for k in ("batch", "kv_heads", "head_dim", "max_seq", "block"))
    s["kc"], s["ks"] = _cache(g, b, hkv, m, d, block)
    s["vc"], s["vs"] = _cache(g, b, hkv, m, d, block)
    if case["op"] == "append":
        s["k"] = _rows(g, b, hkv, case["new"], d).to(dt)
        s["v"] = _rows(g, b, hkv, case["new"], d).to(dt)
        cur, new = _places(case)
        s["cur"], s["new"] = (_int32(cur), _int32(new)) if case["ragged"] else (case["cur"], None)
    elif case["op"] == "read":
        s["lens"] = _int32(_read_lens(case)) if case["ragged"] else None
    else:
        s["q"] = torch.randn((b, case["q_heads"], d), generator=g, device="cuda").to(dt)
        s["lens"] = _int32(_attend_lens(case))
    return s


def work(case):
    e = _SIZE[case["dtype"]]
    if case["op"] == "norm":
        n = case["rows"] * case["cols"]
        return {"bytes": n * (e + (2 * e if case["residual"] else 0) + 1) + case["cols"] * e + case["rows"] * 4,
                "flops": 6 * n}
    d, hkv, block = case["head_dim"], case["kv_heads"], case["block"]
    if case["op"] == "append":
        cur, new = _places(case)
        blocks = sum((c + n - 1) // block - c // block + 1 for c, n in zip(cur, new))
        n = sum(new) * hkv * d
        return {"bytes": 2 * (n * (e + 1) + blocks * hkv * 4), "flops": 2 * 4 * n}
    if case["op"] == "read":
        total = sum(max(0, min(n, case["start"] + case["n"]) - case["start"]) for n in _read_lens(case))
        out = case["batch"] * case["n"] * hkv * d
        return {"bytes": 2 * (total * hkv * d + out * e + total * hkv * 4 // block), "flops": 2 * total * hkv * d}
    total = sum(_attend_lens(case))
    hq = case["q_heads"]
    return {"bytes": 2 * total * hkv * (d + 4 / block) + 2 * case["batch"] * hq * d * e, "flops": 4 * total * hq * d}


# ---- the plain forms ---------------------------------------------------------------
def _plain_norm(s, eps):
    x, w = s["x"], s["w"]
    h = x if s["r"] is None else (x.float() + s["r"].float()).to(x.dtype)
    hd = h.double()
    p = hd * w.double()                       # next to a border: in 64 bits
    top = p.abs().amax(-1, keepdim=True)
    codes = torch.where(top > 0, torch.round(p * 127.0 / top), 0.0).to(torch.int8)
    rms = torch.sqrt((hd * hd).mean(-1) + eps)
    scale = (top.squeeze(-1) / (127.0 * rms)).float()
    return (codes, scale) if s["r"] is None else (h, codes, scale)


def _plain_append(s, codes, scales, x):
    """The window of blocks around the new tokens, taken out, restated, put back."""
    case = s["case"]
    b, hkv, d, m, block, new = (case[k] for k in ("batch", "kv_heads", "head_dim", "max_seq", "block", "new"))
    dev = codes.device
    cur = s["cur"].long() if case["ragged"] else torch.full((b,), case["cur"], device=dev)
    cnt = s["new"].long() if case["ragged"] else torch.full((b,), new, device=dev)
    blocks = scales.shape[-1]
    wide = min(blocks, (new + block - 2) // block + 1)
    first = torch.clamp(cur // block, max=blocks - wide)
    at_block = first[:, None] + torch.arange(wide, device=dev)                       # [b, wide]
    pos = first[:, None] * block + torch.arange(wide * block, device=dev)            # [b, wide * block]
    is_new = (pos >= cur[:, None]) & (pos < (cur + cnt)[:, None])
    is_old = pos < cur[:, None]
    idx = pos[:, None, :, None].expand(b, hkv, wide * block, d)
    src = (pos - cur[:, None]).clamp(0, new - 1)[:, None, :, None].expand(b, hkv, wide * block, d)
    old = codes.gather(2, idx)
    fresh = torch.where(is_new[:, None, :, None], x.float().gather(2, src), 0.0)
    top = fresh.abs().view(b, hkv, wide, block * d).amax(-1)
    need = (top.double() / torch.tensor(127.0, dtype=torch.float64, device=dev)).float()
    block_idx = at_block[:, None, :].expand(b, hkv, wide)
    had = scales.gather(2, block_idx)
    holds = (at_block * block < cur[:, None])[:, None, :]
    touched = is_new.view(b, wide, block).any(-1)[:, None, :]
    scale = torch.where(touched, torch.where(holds, torch.maximum(had, need), need), had)
    per = scale.double().repeat_interleave(block, 2)[..., None]
    was = had.double().repeat_interleave(block, 2)[..., None]
    put = torch.where(per > 0, torch.round(fresh.double() / per), 0.0).clamp(-127, 127).to(torch.int8)
    grown = (touched & holds & (scale > had)).repeat_interleave(block, 2)[..., None] & is_old[:, None, :, None]
    again = torch.where(grown, torch.round(old.double() * was / per), 0.0).to(torch.int8)
    put = torch.where(is_new[:, None, :, None], put, torch.where(grown, again, old))
    codes.scatter_(2, idx, put)
    scales.scatter_(2, block_idx, scale)


def _plain_read(s, codes, scales):
    case = s["case"]
    start, n, block = case["start"], case["n"], case["block"]
    pos = torch.arange(start, start + n, device=codes.device)
    x = codes[:, :, start:start + n].float() * scales[:, :, pos // block][..., None]
    if s["lens"] is not None:
        x = torch.where((pos[None, :] < s["lens"][:, None])[:, None, :, None], x, 0.0)
    return x.to(_DTYPES[case["dtype"]])


def _plain_attend(s, scale):
    case = s["case"]
    b, hq, hkv, d, m, block = (case[k] for k in ("batch", "q_heads", "kv_heads", "head_dim", "max_seq", "block"))
    q = s["q"].float().view(b, hkv, hq // hkv, d)
    at = torch.arange(m, device=q.device)
    k = s["kc"].float() * s["ks"][:, :, at // block][..., None]
    scores = torch.matmul(q, k.transpose(2, 3)) * scale
    del k
    live = (at[None, :] < s["lens"][:, None])[:, None, None, :]
    top = torch.where(live, scores, -torch.inf).amax(-1, keepdim=True)
    p = torch.where(live, torch.exp(scores - top), 0.0)
    total = p.sum(-1, keepdim=True)
    v = s["vc"].float() * s["vs"][:, :, at // block][..., None]
    out = torch.where(total > 0, torch.matmul(p, v) / total, 0.0)
    return out.view(b, hq, d).to(s["q"].dtype)


_EPS = 1e-5


def _scale(head_dim):
    """The attention's default: 1 / sqrt(head_dim) in f32."""
    return float(torch.tensor(float(head_dim), dtype=torch.float32).sqrt().reciprocal())


def run(state):
    s, case = state, state["case"]
    if case["op"] == "norm":
        if not own:
            return _plain_norm(s, _EPS)
        if s["r"] is None:
            return _ops().rms_norm_q8(s["x"], s["w"], _EPS)
        return _ops().add_rms_norm_q8(s["x"], s["r"], s["w"], _EPS)
    if case["op"] == "append":
        if own:
            _ops().kv_cache_append_q8(s["kc"], s["vc"], s["ks"], s["vs"], s["k"], s["v"], s["cur"], case["block"],
                                      new_lens=s["new"])
        else:
            _plain_append(s, s["kc"], s["ks"], s["k"])
            _plain_append(s, s["vc"], s["vs"], s["v"])
        return s["kc"], s["vc"], s["ks"], s["vs"]
    if case["op"] == "read":
        if own:
            return _ops().kv_cache_read_q8(s["kc"], s["vc"], s["ks"], s["vs"], case["block"], case["start"], case["n"],
                                           lens=s["lens"], dtype=_DTYPES[case["dtype"]])
        return _plain_read(s, s["kc"], s["ks"]), _plain_read(s, s["vc"], s["vs"])
    if own:
        return _ops().decode_attention_q8(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], case["block"], s["lens"])
    return _plain_attend(s, _scale(case["head_dim"]))


# ---- the definitions in 64 bits ------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x, w = s["x"].double(), s["w"].double()
        h = x if s["r"] is None else x + s["r"].double()
        held = h if s["r"] is None else h.to(torch.float32).to(s["x"].dtype).double()  # the norm reads h as stored
        y = held / torch.sqrt(held.square().sum(-1, keepdim=True) / case["cols"] + _EPS) * w
        scale = y.abs().amax(-1) / 127.0
        return (None, scale) if s["r"] is None else (h, None, scale)
    block = case["block"]
    if case["op"] == "append":
        if case["batch"] * (case["new"] // block) > 8192:
            return None                                   # block by block below: too long
        cur, cnt = _places(case)
        out = []
        for codes, scales, x in ((s["kc"], s["ks"], s["k"]), (s["vc"], s["vs"], s["v"])):
            sc = scales.double()
            for b in range(case["batch"]):
                c, n = cur[b], cnt[b]
                for j in range(c // block, (c + n - 1) // block + 1):
                    lo, hi = max(c, j * block), min(c + n, (j + 1) * block)
                    need = x[b, :, lo - c:hi - c].double().abs().amax((-1, -2)) / 127.0
                    sc[b, :, j] = torch.maximum(sc[b, :, j], need) if j * block < c else need
            out.append(sc)
        return None, None, out[0], out[1]
    if case["op"] == "read":
        start, n = case["start"], case["n"]
        lens = _read_lens(case)
        out = []
        for codes, scales in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
            x = torch.zeros((case["batch"], case["kv_heads"], n, case["head_dim"]), dtype=torch.float64, device="cuda")
            for b in range(case["batch"]):
                end = min(start + n, lens[b])
                if end > start:
                    per = scales[b].double().repeat_interleave(block, 1)[:, start:end, None]
                    x[b, :, :end - start] = codes[b, :, start:end].double() * per
            out.append(x)
        return out[0], out[1]
    hq, hkv, d = case["q_heads"], case["kv_heads"], case["head_dim"]
    out = torch.zeros((case["batch"], hq, d), dtype=torch.float64, device="cuda")
    for b, n in enumerate(_attend_lens(case)):
        for j in range(hkv if n else 0):
            k = s["kc"][b, j, :n].double() * s["ks"][b, j].double().repeat_interleave(block)[:n, None]
            v = s["vc"][b, j, :n].double() * s["vs"][b, j].double().repeat_interleave(block)[:n, None]
            heads = slice(j * (hq // hkv), (j + 1) * (hq // hkv))
            t = s["q"][b, heads].double() @ k.T * _scale(d)
            out[b, heads] = torch.softmax(t, -1) @ v
    return out
