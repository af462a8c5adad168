"""The int8 operators by their definitions, in 64 bits, for the parity tests:
torch on whatever device the inputs are on, nothing of the library."""
import torch

F64 = torch.float64


def norm_q8(x, r, w, eps):
    """(h or None, codes, scale in f64) of add + rms_norm with int8 rows."""
    h = x if r is None else (x.float() + r.float()).to(x.dtype)
    p = h.to(F64) * w.to(F64)
    top = p.abs().amax(-1, keepdim=True)
    fine = torch.isfinite(top) & (top > 0)
    codes = torch.where(fine, torch.round(p * 127 / top), 0.0)
    codes = torch.nan_to_num(codes, nan=0.0).to(torch.int8)
    rms = torch.sqrt(h.to(F64).square().mean(-1) + eps)
    scale = top[..., 0] / (127 * rms)
    scale = torch.where(torch.isfinite(top[..., 0]), scale, torch.nan)
    return (None if r is None else h), codes, scale


def _nearest(x, s):
    """The code of x under the f32 scale s, in 64 bits."""
    if not (s > 0) or s == float("inf"):
        return torch.zeros_like(x, dtype=torch.int8)
    return torch.round(x.to(F64) / s).clamp(-127, 127).to(torch.int8)


def append_one(codes, scales, x, cur, n, block):
    """Append x[:n] ([new, d]) at cur to one head's codes [max_seq, d] and scales
    [nblk], in place, block by block."""
    for j in range(cur // block, (cur + n - 1) // block + 1):
        lo, hi = max(cur, j * block), min(cur + n, (j + 1) * block)
        part = x[lo - cur:hi - cur].float()
        top = float(part.abs().max()) if bool(torch.isfinite(part).all()) else float("nan")
        need = float(torch.tensor(top / 127.0, dtype=F64).float())  # one rounding: 53 bits >= 2 * 24 + 2
        had = float(scales[j])
        if j * block < cur:
            if need != need or need > had:
                if need == need:
                    old = codes[j * block:lo]
                    codes[j * block:lo] = torch.round(old.to(F64) * had / need).to(torch.int8)
                s = need
            else:
                s = had
        else:
            s = need
        scales[j] = s
        codes[lo:hi] = _nearest(part, s)


def append(kc, vc, ks, vs, k, v, cur, new, block):
    """The whole append, in place; cur and new one number a sequence.  A sequence
    whose tokens do not fit is left alone."""
    for codes, scales, x in ((kc, ks, k), (vc, vs, v)):
        for b in range(codes.shape[0]):
            n = min(max(new[b], 0), x.shape[2])
            if n == 0 or cur[b] < 0 or cur[b] + n > codes.shape[2]:
                continue
            for h in range(codes.shape[1]):
                append_one(codes[b, h], scales[b, h], x[b, h], cur[b], n, block)


def values(codes, scales, block):
    """What the codes stand for, in 64 bits."""
    m = codes.shape[2]
    per = scales.to(F64).repeat_interleave(block, 2)[:, :, :m, None]
    return codes.to(F64) * per


# Half a step of the tensor-core kernel's integers: of the weights (1 / 8e6 of the
# largest), and of the queries.  Those count units 2^(e - 22) where the head's
# largest element lies in [2^e, 1.992 2^e], else 2^(e - 21): half a unit is at
# most 2^-23 of it either way (2^(e - 22) / (1.992 2^e) < 2^-22.99).
GRID, GRID_Q = 0.5 / 8.0e6, 2.0 ** -22.99


def attend(q, kc, vc, ks, vs, lens, block, scale):
    """(out, sum p |v|, tolerance) of the decode attention in f64.  The tolerance
    is how far f32 arithmetic may be from the definition, element by element:
    u = 2^-24 a rounding.
    Scores sum head_dim products and take eight more roundings (the factors, the
    log2(e) factor, the difference from the maximum), each at most u of
    sum |q k| scale.  The tensor-core kernel writes q in integers, so a score is
    off by GRID_Q max|q| sum |k| scale more.  Both act on numerator and denominator: twice, relative to sum p |v|.
    Weights: three base-2 functions (2^-22 each) and 16 roundings in the sums of
    the parts and the quotient, again twice.  And the kernel writes p vs of a
    tile of 128 keys in integers of 1 / 8e6 of the tile's largest: an output is
    off by GRID max(p vs) sum |code| of each tile, whatever its own size."""
    b, hq, d = q.shape
    hkv, m = kc.shape[1], kc.shape[2]
    rep = hq // hkv
    u = 2.0 ** -24
    out = torch.zeros((b, hq, d), dtype=F64, device=q.device)
    mag, tol = torch.zeros_like(out), torch.zeros_like(out)
    for i in range(b):
        n = m if lens is None else max(0, min(int(lens[i]), m))
        if n == 0:
            continue
        nb = -(-n // block)
        k = values(kc[i:i + 1, :, :n], ks[i:i + 1, :, :nb], block)[0]
        v = values(vc[i:i + 1, :, :n], vs[i:i + 1, :, :nb], block)[0]
        qi = q[i].to(F64).view(hkv, rep, d)
        p = torch.softmax(qi @ k.transpose(1, 2) * scale, -1)
        one = p @ v.abs()
        size = (qi.abs() @ k.abs().transpose(1, 2)).amax(-1, keepdim=True) * abs(scale)
        wide = qi.abs().amax(-1, keepdim=True) * k.abs().sum(-1).amax(-1)[:, None, None] * abs(scale)
        t = one * (2 * ((d + 8) * u * size + GRID_Q * wide) + 2 * (3 * 2.0 ** -22 + 16 * u))
        pv = p * vs[i, :, :nb].to(F64).repeat_interleave(block, 1)[:, None, :n]
        for j in range(0, n, 128):
            top = pv[:, :, j:j + 128].amax(-1, keepdim=True)
            t += GRID * top * vc[i, :, None, j:j + 128].to(F64).abs().sum(2)
        out[i], mag[i], tol[i] = (p @ v).view(hq, d), one.view(hq, d), t.view(hq, d)
    return out, mag, tol
