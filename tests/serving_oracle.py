"""What the operators of a serving step compute, in 64 bits and plain loops."""
import numpy as np

E4M3_MAX = 448.0


def e4m3_table():
    """The value of each of the 256 codes."""
    c = np.arange(256)
    sign, e, m = np.where(c & 128, -1.0, 1.0), (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e.astype(np.float64) - 10))
    v = np.where((c & 127) == 127, np.nan, v)
    return sign * v


def e4m3_round(x):
    """The nearest e4m3 value, ties to even; saturates, keeps NaN."""
    x = np.asarray(x, dtype=np.float64)
    _, e = np.frexp(x)
    step = np.exp2(np.maximum(np.where(np.isfinite(x), e, 0) - 4, -9).astype(np.float64))
    with np.errstate(invalid="ignore"):
        return np.where(np.isinf(x), np.sign(x) * E4M3_MAX, np.clip(np.rint(x / step) * step, -E4M3_MAX, E4M3_MAX))


def scale_for(amax):
    e = -64
    while amax > E4M3_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


def tables(cached, added, free, count, table, page, tokens):
    table, starts, slots, left, missing = table.copy(), [0], [], count, 0
    cached, added = np.maximum(cached, 0), np.maximum(added, 0)
    for b in range(len(cached)):
        for pos in range(cached[b], cached[b] + added[b]):
            j = pos // page
            if pos % page == 0:
                if j >= table.shape[1]:
                    missing += 1
                elif left > 0:
                    left -= 1
                    table[b, j] = free[left]
                else:
                    missing += 1
                    table[b, j] = -1
            held = table[b, j] if j < table.shape[1] else -1
            slots.append(held * page + pos % page if held >= 0 else -1)
        starts.append(len(slots))
    slots = (slots + [-1] * tokens)[:tokens]
    return dict(table=table, lengths=cached + added, starts=np.array(starts), slots=np.array(slots, dtype=np.int64), counts=np.array([left, missing]))


def write(x, slots, codes, scales):
    """codes [pages, heads, page, dim] as values; returns (codes, scales)."""
    codes, scales, (pages, _, page, _) = codes.copy(), scales.astype(np.float64).copy(), codes.shape
    t = 0
    while t < len(slots):
        n = 1
        if slots[t] < 0 or slots[t] // page >= pages:
            t += 1
            continue
        p, low = divmod(int(slots[t]), page)
        while t + n < len(slots) and slots[t + n] == slots[t] + n and low + n < page:
            n += 1
        for h in range(codes.shape[1]):
            new = x[t:t + n, h]
            finite = np.abs(new[np.isfinite(new)])
            need = scale_for(finite.max() if finite.size else 0.0)
            s = max(scales[p, h], need) if low > 0 else need
            if low > 0:
                codes[p, h, :low] = e4m3_round(codes[p, h, :low] * (scales[p, h] / s))
            codes[p, h, low:low + n] = e4m3_round(new / s)
            scales[p, h] = s
        t += n
    return codes, scales


def attention(q, k, v, v_scales, limits, scale):
    """One head of one request: q [n, dim], k and v [length, dim], v_scales [length], limits[i] keys seen by query i.
    Returns the result and how far a kernel may be from it before it rounds its result, from
      the weights' rounding to fp16: 2^-11 of a weight, or 2^-25 of the largest one where that is more (fp16 has 11 bits
        down to 2^-14 and steps of 2^-24 below; the largest weight, with its value scale, stands for 1)
      the exponents: dim products summed in fp32 in steps of 32 of a matrix instruction, times a scale, plus the value
        scale's logarithm (up to 64); once in the weights and once in their sum
      the sums over the keys in fp32, 32 at a time, joined at the end."""
    n, dim = q.shape
    o, tol = np.zeros((n, dim)), np.zeros((n, dim))
    codes = np.abs(v) / np.where(v_scales > 0, v_scales, 1.0)[:, None]
    for i in range(n):
        m = int(limits[i])
        if m <= 0:
            continue
        z = (k[:m] @ q[i]) * scale
        exponent = ((dim / 32 + 8) * 2.0 ** -24 * (np.abs(k[:m]) @ np.abs(q[i])) * scale + 8 * 2.0 ** -24 * (np.abs(z) + 64)).max()
        p = np.exp(z - z.max())
        p /= p.sum()
        o[i] = p @ v[:m]
        tol[i] = (2.0 ** -11 + 2 * exponent + (m / 32 + 16) * 2.0 ** -24) * (p @ np.abs(v[:m])) + 2.0 ** -25 * codes[:m].sum(axis=0) * (p * v_scales[:m]).max()
    return o, tol


def matvec4(x, codes, scales, zeros, group, offset):
    """x [m, k], codes [n, k / 2], scales and zeros [k / group, n].  Returns the result and how far fp32 sums may be from it
    when they are taken of x (offset + q) and of x, group by group: a matrix instruction adds 32 products and its
    accumulator, at most 8 roundings deep, group / 32 times; so does the sum of x, which counts offset + zero times; and
    the groups' sums are added up, in eight parts."""
    q = np.stack([codes & 15, codes >> 4], axis=2).reshape(codes.shape[0], -1).astype(np.float64)
    y, tol = np.zeros((x.shape[0], codes.shape[0])), np.zeros((x.shape[0], codes.shape[0]))
    size = np.zeros_like(y)
    for g in range(scales.shape[0]):
        part = slice(g * group, (g + 1) * group)
        dots, sums = x[:, part] @ q[:, part].T, x[:, part].sum(axis=1, keepdims=True)
        y += scales[g] * (dots - zeros[g] * sums)
        most = np.abs(x[:, part]) @ (offset + q[:, part]).T + (offset + zeros[g]) * np.abs(x[:, part]).sum(axis=1, keepdims=True)
        tol += np.abs(scales[g]) * (8 + group / 32) * 2.0 ** -24 * most
        size += np.abs(scales[g]) * np.abs(dots - zeros[g] * sums)
    return y, tol + (scales.shape[0] / 8 + 9) * 2.0 ** -24 * size
