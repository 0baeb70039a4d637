"""Cases and 64-bit forms for the FP8 cache with a power-of-two scale per (block, head)."""
import torch

FP8 = torch.float8_e4m3fn
BS = 16


def nearest_e4m3(x):
    """The e4m3 number next to each of ``x`` (fp64), ties to the even one, largest magnitude 448."""
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return (torch.round(x / step) * step).clamp(-448.0, 448.0)


def power_scale(amax):
    """Smallest 2^e, -60 <= e <= 60, with amax <= 448 * 2^e, by trying them."""
    e = torch.arange(-60, 61, dtype=torch.float64)
    fits = amax.double()[..., None] <= 448.0 * 2.0 ** e
    first = torch.where(fits.any(-1), fits.double().argmax(-1), torch.full(amax.shape, 120))
    return 2.0 ** e[first]


def make_cache(nb, hkv, d, gen, device, spread=3.0, kernel_layout=True):
    """Random codes, scales of powers of two over ``2 ** (+-spread)``; returns (k, v, k_scale, v_scale), logical [nb, 16, hkv, d] views."""
    out = []
    for which in "kv":
        x = torch.randn(nb, hkv, BS, d, generator=gen).clamp(-4, 4) * 100.0
        c = x.to(FP8)
        phys = c if which == "k" else c.view(torch.uint8).transpose(2, 3).contiguous().view(FP8)
        if kernel_layout:
            phys = phys.to(device)
            out.append(phys.permute(0, 2, 1, 3) if which == "k" else phys.permute(0, 3, 1, 2))
        else:
            out.append(c.view(torch.uint8).permute(0, 2, 1, 3).contiguous().view(FP8).to(device))
    scales = [torch.ldexp(torch.full((nb, hkv), 2.0 ** -7), torch.randint(-int(spread), int(spread) + 1, (nb, hkv), generator=gen)).to(device)
              for _ in range(2)]
    return out[0], out[1], scales[0], scales[1]


def tables_for(lens, gen, device, extra_cols=0):
    """Shuffled block tables of the given lengths: (tables, blocks used)."""
    need = [(n + BS - 1) // BS for n in lens]
    nb = sum(need)
    order = torch.randperm(max(nb, 1), generator=gen)
    t = torch.zeros(len(lens), max(max(need), 1) + extra_cols, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = order[at:at + n]
        at += n
    return t.to(device), max(nb, 1)


def dequant(cache, scales, table, n):
    """fp64 [n, hkv, d] of one sequence (CPU)."""
    blocks = table[:(n + BS - 1) // BS].long().cpu()
    c = cache.view(torch.uint8).cpu()[blocks].view(FP8).double() * scales.cpu().double()[blocks][:, None, :, None]
    return c.reshape(-1, *c.shape[2:])[:n]


def attention64(q, k, v, ks, vs, tables, lens, rows, scale, window=0):
    """Returns (out, sum of p |v|, bound of the scores' sums of magnitudes, weights [list of (hkv, L)])."""
    T, hq, d = q.shape
    hkv = k.shape[2]
    g = hq // hkv
    q = q.double().cpu()
    out, mag = torch.zeros(T, hq, d, dtype=torch.float64), torch.zeros(T, hq, d, dtype=torch.float64)
    amp = torch.zeros(T, hq, dtype=torch.float64)
    weights = []
    r0 = 0
    for i, (n, r) in enumerate(zip(lens, rows)):
        if n and r:
            kk, vv = dequant(k, ks, tables[i], n), dequant(v, vs, tables[i], n)
            qq = q[r0:r0 + r].view(r, hkv, g, d)
            s = torch.einsum("rhgd,nhd->hgrn", qq, kk) * scale
            size = torch.einsum("rhgd,nhd->hgrn", qq.abs(), kk.abs()) * abs(scale)
            pos, key = torch.arange(n - r, n)[:, None], torch.arange(n)[None]
            dead = key > pos
            if window:
                dead |= key <= pos - window
            p = torch.softmax(s.masked_fill(dead, float("-inf")), -1)
            out[r0:r0 + r] = torch.einsum("hgrn,nhd->rhgd", p, vv).reshape(r, hq, d)
            mag[r0:r0 + r] = torch.einsum("hgrn,nhd->rhgd", p, vv.abs()).reshape(r, hq, d)
            amp[r0:r0 + r] = size.masked_fill(dead, 0.0).amax(-1).permute(2, 0, 1).reshape(r, hq)
            weights.append(p.sum((1, 2)))
        else:
            weights.append(torch.zeros(hkv, n, dtype=torch.float64))
        r0 += r
    return out, mag, amp, weights


def attention_bound(out, mag, amp, d):
    """What the kernels may be off by.  Scores: d products, exact, summed in fp32 in groups of 16 (2^-23 a step of the running magnitude
    covers truncation) and a handful of fp32 operations on the exponent: relative error of p and of the sum l, twice.  p to f16: 2^-11 of
    each term (half of eps), 2^-24 of the largest one below f16's normal range, exp2 2^-22.  The result to bf16: 2^-8."""
    ds = (d / 16 + 8) * 2.0 ** -23 * (amp + 2.0)
    return 2.0 ** -8 * out.abs() + (2.0 ** -11 + 2.0 ** -14 + 2 * ds[..., None]) * mag * 1.01 + 1e-30


def evict64(weights, n, keep, sink, recent):
    """Kept positions of one sequence and head by sorting (weight descending, position ascending)."""
    if n <= keep:
        return list(range(n))
    mid = sorted(range(sink, n - recent), key=lambda j: (-float(weights[j]) if weights[j] == weights[j] else float("inf"), j))
    return sorted(list(range(sink)) + mid[:keep - sink - recent] + list(range(n - recent, n)))


def attention64_over(q, kk, vv, scale, window=0, there=None):
    """``q [r, hq, d]``, ``kk`` and ``vv [n, hkv, d]`` of one sequence, its last ``r`` tokens the queries'; ``there [n]``: tokens that are not
    skipped.  Returns (out, sum of p |v|, largest sum of magnitudes of a visible score, weights [hkv, n])."""
    r, hq, d = q.shape
    n, hkv, _ = kk.shape
    qq = q.double().cpu().view(r, hkv, hq // hkv, d)
    s = torch.einsum("rhgd,nhd->hgrn", qq, kk) * scale
    size = torch.einsum("rhgd,nhd->hgrn", qq.abs(), kk.abs()) * abs(scale)
    pos, key = torch.arange(n - r, n)[:, None], torch.arange(n)[None]
    see = key <= pos
    if window:
        see &= key > pos - window
    if there is not None:
        see &= there[None]
    p = torch.softmax(s.masked_fill(~see, float("-inf")), -1).nan_to_num(0.0)
    back = lambda x: x.permute(2, 0, 1, 3).reshape(r, hq, -1)
    out, mag = (back(torch.einsum("hgrn,nhd->hgrd", p, x)) for x in (vv, vv.abs()))
    return out, mag, back(size.masked_fill(~see, 0.0).amax(-1, keepdim=True))[..., 0], p.sum((1, 2))
