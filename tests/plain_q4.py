"""A cache in 4 bits, plainly: the format's definition and packing, and attention over it, on the host in 64 bits."""
import numpy as np
import torch

GROUP = 32


def round5(x):
    """Five significant bits, ties to even (normal 32-bit numbers in, 64 bits out)."""
    fraction, exponent = np.frexp(np.asarray(x, dtype=np.float64))
    return np.ldexp(np.rint(fraction * 32), exponent - 5)


def quantise(x):
    """Codes and scales of rows [..., d]; a group with a value that is not finite has the scale NaN and codes 0."""
    x = np.asarray(x, dtype=np.float64)
    groups = x.reshape(*x.shape[:-1], -1, GROUP)
    with np.errstate(invalid="ignore", divide="ignore"):
        high, low = groups.max(-1), groups.min(-1)
        scale = round5(np.where(high >= -low, high, low) / -8)
        scale = np.where(np.isfinite(groups).all(-1), scale, np.nan)
        codes = np.clip(np.rint(groups / scale[..., None]), -8, 7)
    return np.where((scale == 0)[..., None] | np.isnan(codes), 0, codes).astype(np.int64), scale


def stand_for(codes, scales):
    values = codes.astype(np.float64) * scales[..., None]
    return values.reshape(*codes.shape[:-2], -1)


def pack(codes, keys):
    """Codes [..., groups, 32] to bytes [..., d / 2], one nibble at a time."""
    groups = codes.shape[-2]
    nibbles = np.zeros((*codes.shape[:-2], groups * GROUP), dtype=np.uint8)
    for g in range(groups):
        for c in range(GROUP):
            if keys:
                t, j, e = c // 8, c % 8 // 2, c % 2
                at = 8 * (t * groups + g) + j + 4 * e
            else:
                r, j = c // 4, c % 4
                at = 4 * (r * groups + g) + j
            nibbles[..., at] = codes[..., g, c] + 8
    return nibbles[..., 0::2] | nibbles[..., 1::2] << 4


def unpack(data, keys):
    data = np.asarray(data)
    groups = data.shape[-1] // 16
    nibbles = np.stack([data & 15, data >> 4], -1).reshape(*data.shape[:-1], -1)
    codes = np.zeros((*data.shape[:-1], groups, GROUP), dtype=np.int64)
    for g in range(groups):
        for c in range(GROUP):
            at = 8 * (c // 8 * groups + g) + c % 8 // 2 + 4 * (c % 2) if keys else 4 * (c // 4 * groups + g) + c % 4
            codes[..., g, c] = nibbles[..., at].astype(np.int64) - 8
    return codes


def rows_of(codes, scales, keys):
    """Pages as numbers: [pages, kv_heads, page_size, d]."""
    return stand_for(unpack(codes.cpu().numpy(), keys), scales.float().cpu().numpy().astype(np.float64))


def make_pages(num_pages, page_size, kv_heads, d, seed, device="cpu"):
    """Random pages: (codes and scales of keys, of values) as torch tensors."""
    rng = np.random.default_rng(seed)
    out = []
    for keys in (True, False):
        x = rng.standard_normal((num_pages, kv_heads, page_size, d)) * np.exp(0.7 * rng.standard_normal(d))
        codes, scales = quantise(x.astype(np.float32))
        out.append(torch.from_numpy(pack(codes, keys)).to(device))
        out.append(torch.from_numpy(scales).to(torch.bfloat16).to(device))
    return out


def attend(q, k_rows, v_rows, *, counts, history, tables, page_size, num_heads, num_kv_heads, d, scale, window=0, keep_first=0,
           sink=False, sink_values=None, gate=None, k_steps=None, v_steps=None):
    """(output [tokens, heads, d], parts): `parts` is what errors of the run's arithmetic are multiples of, for each output or head:
    ``spread`` sum_j p_j |v_j| / l, ``steps`` the same with the values' scales in the place of |v|, ``reach`` the largest sum over
    channels of |q k| scale that a score of the row has, ``full`` the same with 16 steps of the key's groups in the place of |k|."""
    q = np.asarray(q, dtype=np.float64).reshape(-1, num_heads, d)
    out, spread, steps = np.zeros_like(q), np.zeros_like(q), np.zeros_like(q)
    reach, full = np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    token = 0
    for e, (count, held) in enumerate(zip(counts, history)):
        for i in range(count):
            position = held + i
            seen = [j for j in range(position + 1) if not window or j > position - window or j < keep_first]
            page = np.asarray([tables[e][j // page_size] for j in seen])
            place = np.asarray(seen) % page_size
            for h in range(num_heads):
                kv = h // (num_heads // num_kv_heads)
                k, v = k_rows[page, kv, place], v_rows[page, kv, place]
                s = k @ q[token, h] * scale
                best = max(s.max(), 0.0) if sink and sink_values is None else s.max()
                p = np.exp(s - best)
                total = p.sum()
                if sink or sink_values is not None:
                    total += np.exp((0.0 if sink_values is None else float(sink_values[h])) - best)
                out[token, h] = p @ v / total
                spread[token, h] = p @ np.abs(v) / total
                if v_steps is not None:
                    steps[token, h] = np.repeat(p @ np.abs(v_steps[page, kv, place]) / total, GROUP)
                reach[token, h] = (np.abs(k) @ np.abs(q[token, h])).max() * scale
                if k_steps is not None:
                    full[token, h] = (np.abs(k_steps[page, kv, place]) @ np.abs(q[token, h]).reshape(-1, GROUP).sum(-1)).max() * 16 * scale
            if gate is not None:
                factor = 1 / (1 + np.exp(-np.asarray(gate[token], dtype=np.float64).reshape(num_heads, -1)))
                for part in (out, spread, steps):
                    part[token] *= factor
            token += 1
    return out, dict(spread=spread, steps=steps, reach=reach, full=full)


def allowed(out, parts, keys, d, dtype):
    """How far each output may be off.  Scores are sums of d products and weights and sums run over `keys` keys in 32 bits, a product
    or sum off by 2^-24 of its size, on tensor cores by 2^-22: a score by (d + 8) of these times its reach, a weight and the sum by e
    to that, a sum by one for each key.  2^-30 is for outputs next to 0.  In bfloat16 further:
    a weight (times the scale, where it is taken there) is rounded once and the output once, each by half a step, 2^-8;
    codes c meet the query as c + 8, below 16, in half precision's smallest numbers, whose products' sums the tensor cores were seen to
    have off by 2^-16.7 of their terms' sizes: a score by 2^-16 of `full`, a weight and the sum by e to that;
    values are summed as codes + 136 (144 steps at most) with 136 times the weights' sum taken off: of the 2^-20 that a product of
    17 terms may be off, one for each 16 keys that a warp walks (a quarter of its block's) and four to join the parts."""
    unit = 2.0 ** -22
    relative = 2 * (d + 8) * parts["reach"] * unit + 2 * (keys + 16) * unit
    if dtype == torch.bfloat16:
        relative = relative + 2 * 2.0 ** -16 * parts["full"]
        return (parts["spread"] * (2.0 ** -8 + 2.0 ** -15 + relative[..., None]) + np.abs(out) * 2.0 ** -8
                + parts["steps"] * (keys / 64 + 4) * 144 * 2.0 ** -20 + 2.0 ** -30)
    return parts["spread"] * relative[..., None] + 2.0 ** -30
