"""Block-scaled caches for the tests: inputs on the host, and what the operators
give for them in 64 bits (parity unpinned: the reference has no such cache)."""
import math

import numpy as np

DIM, BLOCK = 512, 32
ALL = 1 << 30
LARGEST = {"int8": 127.0, "e4m3": 448.0}


def e4m3_values():
    """The value of each of the 256 codes (NaN for the two that are none)."""
    code = np.arange(256)
    exponent, mantissa = code >> 3 & 15, code & 7
    value = np.where(exponent == 0, mantissa * 2.0 ** -9, (8 + mantissa) * 2.0 ** (exponent - 10.0))
    value = np.where(code & 128, -value, value)
    value[[127, 255]] = np.nan
    return value


E4M3 = e4m3_values()


def decode(codes, kind):
    """Codes (bytes) as numbers in 64 bits."""
    return E4M3[codes] if kind == "e4m3" else codes.view(np.int8).astype(np.float64)


def encode(x, kind):
    """The nearest code of numbers within the type's range, ties to even, as bytes."""
    if kind != "e4m3":
        return np.rint(x).astype(np.int8).view(np.uint8)
    size = np.abs(x)
    step = 2.0 ** (np.frexp(np.maximum(size, 2.0 ** -6))[1] - 4.0)
    size = np.rint(size / step) * step
    code = np.searchsorted(E4M3[:127], size)
    assert np.array_equal(E4M3[code], size)
    return (code + np.where(np.signbit(x), 128, 0)).astype(np.uint8)


def table_of(rng, first, last, pad=0, spare=3):
    """(block table with pages first[b] .. last[b] - 1 in mixed order and -1 elsewhere, pages)."""
    total = max(1, sum(b - a for a, b in zip(first, last)) + spare)
    order = rng.permutation(total)
    table = np.full((len(first) + pad, max(1, max(last)) + 1), -1, np.int32)
    at = 0
    for b, (lo, hi) in enumerate(zip(first, last)):
        table[b, lo:hi] = order[at:at + hi - lo]
        at += hi - lo
    return table, total


class Pool:
    """Pages of codes [pages, 32, heads, 512] (bytes) and their scales, on the host and on the device."""

    def __init__(self, rng, pages, heads, kind, *, behind=0, spread=1.0):
        self.kind, self.behind = kind, behind
        top = LARGEST[kind]
        x = np.clip(rng.standard_normal((pages, BLOCK, heads, DIM)) * (top / 4), -top, top)
        self.codes = encode(x, kind)
        self.scale = (np.exp(rng.uniform(-spread, spread, (pages, heads))) / top * 4).astype(np.float32)

    def device(self):
        """(cache, scales): pages `behind` bytes apart in one backing, scales in front of the last of those bytes."""
        import torch
        pages, _, heads, _ = self.codes.shape
        payload = BLOCK * heads * DIM
        stride = payload + self.behind
        self.backing = torch.full((pages * stride,), 77, dtype=torch.int8, device="cuda")
        cache = self.backing.as_strided((pages, BLOCK, heads, DIM), (stride, heads * DIM, DIM, 1))
        cache.copy_(torch.from_numpy(self.codes.view(np.int8)))
        if self.kind == "e4m3":
            cache = self.backing.view(torch.float8_e4m3fn).as_strided(cache.shape, cache.stride())
        scale = torch.from_numpy(self.scale).cuda()
        if self.behind >= 4 * heads + 16:
            inside = self.backing.view(torch.float32).as_strided((pages, heads), (stride // 4, 1), payload // 4 + 2)
            inside.copy_(scale)
            scale = inside
        return cache, scale


# ------------------------------------------------------------ append

def rotated(x, table, positions, pairs):
    """x [T, heads, 512] in 64 bits, the last channels rotated."""
    if table is None:
        return x
    half = table.shape[1] // 2
    turn = table[positions].astype(np.float64)
    turn = (turn[:, :half] + 1j * turn[:, half:])[:, None]
    out, end = x.copy(), x[..., DIM - 2 * half:]
    with np.errstate(invalid="ignore", over="ignore"):
        if pairs:
            a, b = end[..., 0::2], end[..., 1::2]
        else:
            a, b = end[..., :half], end[..., half:]
        c, s = turn.real, turn.imag
        a, b = a * c - b * s, a * s + b * c
    if pairs:
        out[..., DIM - 2 * half::2], out[..., DIM - 2 * half + 1::2] = a, b
    else:
        out[..., DIM - 2 * half:DIM - half], out[..., DIM - half:] = a, b
    return out


def append(codes, scale, kind, x, table, cu, lens, *, inverse=None, skip=()):
    """Appends rows x [T, heads, 512] (64 bits, rotated already) to codes and scale, in place."""
    pages, top, large = len(codes), LARGEST[kind], np.float32(np.finfo(np.float32).max)
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        for column in range(max(0, length - n) // BLOCK, -(-length // BLOCK) if n and length > 0 else 0):
            rows = [r for r in range(max(0, length - n, column * BLOCK), min(length, column * BLOCK + BLOCK))]
            page = table[b, column] if column < table.shape[1] else -1
            tokens = [cu[b] + r - (length - n) for r in rows]
            low = rows[0] % BLOCK
            keep = [i for i, t in enumerate(tokens) if t not in skip]
            rows, tokens = [rows[i] for i in keep], [tokens[i] for i in keep]
            if not 0 <= page < pages:
                continue
            at = [r % BLOCK for r in rows]
            if inverse is not None:
                v = x[tokens].astype(np.float32) * inverse
                codes[page, at] = encode(np.clip(np.where(np.isnan(v), 0, v), -127, 127), kind)
                continue
            for h in range(codes.shape[2]):
                v = x[tokens, h]
                with np.errstate(over="ignore"):
                    peak = np.abs(v).astype(np.float32)
                peak = min(np.max(peak, initial=0, where=~np.isnan(peak)), large)
                need = max(np.float32(peak / np.float32(top)), np.float32(1e-8))
                old = scale[page, h]
                if low and 0 < old < np.inf:
                    power = 0
                    while np.ldexp(old, power) < need:
                        power += 1
                    scale[page, h] = np.ldexp(old, power)
                    if power:
                        codes[page, :low, h] = encode(decode(codes[page, :low, h], kind) * 2.0 ** -power, kind)
                else:
                    scale[page, h] = need
                q = np.clip(np.clip(v, -float(large), float(large)) / np.float64(scale[page, h]), -top, top)
                code = encode(np.where(np.isnan(q), 0, q), kind)
                codes[page, at, h] = np.where(np.isnan(v), 127 if kind == "e4m3" else 0, code)


# ------------------------------------------------------------ attention

class Attend:
    """Inputs of a launch on the host."""

    def __init__(self, seed, new, lengths, *, heads=8, kv_heads=1, ratio=1, window=ALL, kind="int8", behind=0,
                 pad_tokens=0, pad_batch=0, softmax_scale=1 / math.sqrt(DIM), q_size=1.0, spread=1.0):
        rng = self.rng = np.random.default_rng(seed)
        self.new, self.lengths, self.heads, self.kv_heads, self.ratio, self.window = new, lengths, heads, kv_heads, ratio, window
        self.kind, self.softmax_scale = kind, softmax_scale
        live = sum(new)
        self.tokens = live + pad_tokens
        self.cu = np.array([0] + list(np.cumsum(new)) + [live] * pad_batch, np.int32)
        self.lens = np.array(list(lengths) + [0] * pad_batch, np.int32)
        self.q = rng.standard_normal((self.tokens, heads, DIM)).astype(np.float32) * q_size
        self.sink = rng.standard_normal(heads).astype(np.float32)
        first = [max(0, n - t - window + 1) // BLOCK for t, n in zip(new, lengths)]
        last = [max(a, -(-n // BLOCK)) for a, n in zip(first, lengths)]
        self.ori_table, pages = table_of(rng, first, last, pad_batch)
        self.ori = Pool(rng, pages, kv_heads, kind, behind=behind, spread=spread)
        self.cmp = self.cmp_table = None
        if ratio > 1:
            self.cmp_table, pages = table_of(rng, [0] * len(new), [-(-(n // ratio) // BLOCK) for n in lengths], pad_batch)
            self.cmp = Pool(rng, pages, kv_heads, kind, behind=behind, spread=spread)

    def device(self):
        import torch
        from npu_sparse_attn_sharedkv_int8 import SharedKVCase
        ori, ori_scale = self.ori.device()
        cmp, cmp_scale = self.cmp.device() if self.cmp else (None, None)
        put = lambda x: None if x is None else torch.from_numpy(x).cuda()  # noqa: E731
        case = SharedKVCase(put(self.q).to(torch.bfloat16), ori, put(self.ori_table), put(self.cu), put(self.lens),
                            put(self.sink), cmp, put(self.cmp_table), None, ratio=self.ratio, window=self.window,
                            softmax_scale=self.softmax_scale)
        return case, ori_scale, cmp_scale

    def rows(self, pool, table, b, rows, head):
        """(codes in 64 bits, scales) of the logical rows that lie on a page."""
        entry = rows // BLOCK
        page = np.where(entry < table.shape[1], table[b, np.minimum(entry, table.shape[1] - 1)], -1)
        good = (page >= 0) & (page < len(pool.codes))
        page, rows = page[good], rows[good]
        return decode(pool.codes[page, rows % BLOCK, head], self.kind), pool.scale[page, head].astype(np.float64)

    def expect(self):
        """(out, allowed |difference|, lse, allowed) in 64 bits.

        Bounds (derived, none fitted).  Q is held relative to its row's largest
        |q| = peak: as whole numbers of at least peak * 2^15 / 32512 / 2 a unit,
        off by half a unit at most, |q| below peak / 15000 (INT8), or in two e4m3
        terms, off by 2^-21 peak at most, so a score is off by
          d = softmax_scale * unit * max_j scale_j sum_c |code_j[c]|,  unit = peak / 15872 / 2 or 2^-21 peak
        and by the sums' roundings (exact for INT8 but for the last, at most
        sixteen of 2^-24 each of sum_c |q code| in FP32), and those of the
        score, its lift log2 scale and their differences from the running
        maximum, 2^-21 (1.5 max|s| + max|lift| + 24).  A weight relative to the
        sum is off by twice that and by FP16's 2^-11, the exponential, the
        logarithm of the scale, the sums and quotients by less than 2^-17
        together; the output's rounding adds 2^-8 |out|.  FP16 weights start at
        2^8 for a row's largest e^s scale and are multiples of 2^-24 at the low
        end: off by 2^-33 of that largest besides.  The log-sum-exp is off by
        the score's error, and its own roundings.
        """
        q = bf16(self.q).astype(np.float64)
        group = self.heads // self.kv_heads
        out = np.zeros((self.tokens, self.heads, DIM))
        near, lse, lse_near = np.zeros_like(out), np.zeros(out.shape[:2]), np.zeros(out.shape[:2])
        for b, (n, length) in enumerate(zip(self.new, self.lengths)):
            for i in range(n if length > 0 else 0):
                t, place = self.cu[b] + i, length - n + i
                for kv in range(self.kv_heads):
                    mine = slice(kv * group, (kv + 1) * group)
                    code, scale = self.rows(self.ori, self.ori_table, b, np.arange(max(0, place - self.window + 1), place + 1), kv)
                    if self.ratio > 1:
                        more = self.rows(self.cmp, self.cmp_table, b, np.arange(max(0, place + 1) // self.ratio), kv)
                        code, scale = np.concatenate([more[0], code]), np.concatenate([more[1], scale])
                    sink = self.sink[mine].astype(np.float64)
                    if not len(code):
                        lse[t, mine], lse_near[t, mine] = sink, 2 ** -20 + 2 ** -22 * np.abs(sink)
                        continue
                    s = q[t, mine] @ code.T * scale * self.softmax_scale
                    top = np.maximum(s.max(1), sink)
                    e = np.exp(s - top[:, None])
                    total = e.sum(1) + np.exp(sink - top)
                    p, v = e / total[:, None], code * scale[:, None]
                    out[t, mine] = p @ v
                    peak = np.abs(q[t, mine]).max(1)
                    unit = peak * 2.0 ** -21 if self.kind == "e4m3" else peak / 31744
                    d = abs(self.softmax_scale) * unit * (np.abs(code).sum(1) * scale).max()
                    d += abs(self.softmax_scale) * 2.0 ** -20 * (np.abs(q[t, mine]) @ np.abs(code).T * scale).max(1)
                    size, lift = np.abs(s).max(1), np.abs(np.log2(scale)).max()
                    d += 2.0 ** -21 * (1.5 * size + lift + 24)
                    slack = 2 * d + 2.0 ** -11 + 2.0 ** -17
                    near[t, mine] = 2.0 ** -8 * np.abs(out[t, mine]) + slack[:, None] * (p @ np.abs(v)) \
                        + 2.0 ** -33 * (p * scale).max(1)[:, None] * np.abs(code).sum(0)
                    lse[t, mine] = top + np.log(total)
                    lse_near[t, mine] = d + 2.0 ** -21 * np.abs(lse[t, mine]) + 2.0 ** -19
        return out, near, lse, lse_near


def bf16(x):
    """FP32 values rounded to BF16, as FP32."""
    import torch
    return torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(torch.bfloat16).float().numpy()
