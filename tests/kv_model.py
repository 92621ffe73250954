"""Plain models of the paged 8-bit cache in numpy: its layout, append in exact arithmetic, the page operations, and
attention in 64 bits with a bound on what the kernels may be off by."""
import math

import numpy as np

BLOCK = 32


def to_bf16(x):
    """float32 -> bfloat16 bits, nearest even."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u >> 16) & 1) + 0x7FFF
    out = ((u + r) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), out)


def from_bf16(b):
    return (b.astype(np.uint32) << 16).view(np.float32)


def encode(x, name):
    """Values as the array that a call takes, and the values it holds."""
    if name == "bf16":
        b = to_bf16(x)
        return b, from_bf16(b)
    with np.errstate(over="ignore"):
        a = x.astype({"f32": np.float32, "f16": np.float16}[name])
    return a, a.astype(np.float32)


def decode(a, name):
    return (from_bf16(a) if name == "bf16" else a).astype(np.float64)


HALF_STEP = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def k_bytes(D):
    """[32][D] byte of (token, dimension) in a K block"""
    t, d = np.arange(BLOCK)[:, None], np.arange(D)[None]
    return (d // 16) * (BLOCK * 16) + t * 16 + d % 16


def v_bytes(D):
    t, d = np.arange(BLOCK)[:, None], np.arange(D)[None]
    a, h, b = t // 8, t // 4 % 2, t % 4
    return (h * D + d) * 16 + 8 * (a & 1) + 4 * (a >> 1) + b


class Cache:
    """The cache's memory on the host: codes, scales, table, len, ref."""

    def __init__(self, layers, pages, P, H, D, seqs, most):
        self.shape = (layers, pages, P, H, D, seqs, most)
        self.L, self.N, self.P, self.H, self.D, self.S, self.M = self.shape
        self.codes = np.zeros((layers, pages, 2, H, P // BLOCK, BLOCK * D), np.int8)
        self.scales = np.zeros(self.codes.shape[:-1], np.float32)
        self.table = np.zeros((seqs, most), np.int32)
        self.len = np.zeros(seqs, np.int32)
        self.ref = np.zeros(pages, np.int32)
        self.bytes = (k_bytes(D), v_bytes(D))

    def pages(self, n):
        return -(-n // self.P)

    def free(self):
        return [p for p in range(self.N) if self.ref[p] == 0]

    def reserve(self, slots, n_new):
        free, need = self.free(), 0
        for s, n in zip(slots, n_new):
            need += self.pages(int(self.len[s]) + n) - self.pages(int(self.len[s]))
        if need > len(free):
            return False
        for s, n in zip(slots, n_new):
            for k in range(self.pages(int(self.len[s])), self.pages(int(self.len[s]) + n)):
                self.table[s, k] = free.pop(0)
                self.ref[self.table[s, k]] += 1
            self.len[s] += n
        return True

    def copy_page(self, src, dst):
        self.codes[:, dst] = self.codes[:, src]
        self.scales[:, dst] = self.scales[:, src]

    def trim(self, slots, new_len):
        for s, n in zip(slots, new_len):
            n = min(max(n, 0), int(self.len[s]))
            for k in range(self.pages(n), self.pages(int(self.len[s]))):
                self.ref[self.table[s, k]] -= 1
            self.len[s] = n
        free = self.free()
        shared = [s for s in slots if self.len[s] % self.P and self.ref[self.table[s, self.len[s] // self.P]] > 1]
        for s in shared:
            k, p = self.len[s] // self.P, free.pop(0)
            self.copy_page(self.table[s, k], p)
            self.ref[self.table[s, k]] -= 1
            self.ref[p] = 1
            self.table[s, k] = p

    def fork(self, src, dst):
        free, table, length = self.free(), self.table.copy(), self.len.copy()
        for s, d in zip(src, dst):
            if s != d:
                for k in range(self.pages(int(length[d]))):
                    self.ref[table[d, k]] -= 1
        copies = []
        for s, d in zip(src, dst):
            if s == d:
                continue
            n = int(length[s])
            for k in range(n // self.P):
                self.table[d, k] = table[s, k]
                self.ref[table[s, k]] += 1
            if n % self.P:
                p = free.pop(0)
                self.table[d, n // self.P] = p
                self.ref[p] += 1
                copies.append((table[s, n // self.P], p))
            self.len[d] = n
        for a, b in copies:
            self.copy_page(a, b)

    def compact(self):
        live = [p for p in range(self.N) if self.ref[p] > 0]
        n = len(live)
        high, low = [p for p in live if p >= n], [p for p in range(n) if self.ref[p] == 0]
        new = dict(zip(high, low))
        for a, b in new.items():
            self.copy_page(a, b)
            self.ref[b], self.ref[a] = self.ref[a], 0
        for s in range(self.S):
            for k in range(self.pages(int(self.len[s]))):
                self.table[s, k] = new.get(int(self.table[s, k]), self.table[s, k])
        return n

    def cell(self, slot, t):
        return int(self.table[slot, t // self.P]), t % self.P // BLOCK

    def tokens(self, layer, slot, which, codes=None, scales=None):
        """[len][H][D] values of a slot in 64 bits, from the host's or other memory of the same shape."""
        codes, scales = (self.codes, self.scales) if codes is None else (codes, scales)
        n = int(self.len[slot])
        out = np.zeros((n, self.H, self.D))
        for t0 in range(0, n, BLOCK):
            p, b = self.cell(slot, t0)
            m = min(BLOCK, n - t0)
            c = codes[layer, p, which, :, b][:, self.bytes[which][:m]]  # [H][m][D]
            with np.errstate(invalid="ignore"):
                out[t0:t0 + m] = (c.astype(np.float64) * scales[layer, p, which, :, b].astype(np.float64)[:, None, None]).transpose(1, 0, 2)
        return out

    def append(self, layer, slot, k, v):
        """k, v: [n][H][D] float32 values of the slot's last n tokens (in exact arithmetic: 64 bits hold every quotient's
        side of the middle of two codes, since value and scale have 24 bits)."""
        n, end = k.shape[0], int(self.len[slot])
        begin = end - n
        for t0 in range(begin // BLOCK * BLOCK, end, BLOCK):
            p, b = self.cell(slot, t0)
            lo, hi = max(t0, begin), min(t0 + BLOCK, end)
            for which, x in ((0, k), (1, v)):
                for head in range(self.H):
                    new = x[lo - begin:hi - begin, head]
                    before = self.scales[layer, p, which, head, b] if lo > t0 else np.float32(0)
                    with np.errstate(over="ignore", invalid="ignore"):
                        s = np.float32(np.abs(new).max() / np.float32(127))
                    cells, at = self.codes[layer, p, which, head, b], self.bytes[which]
                    if not np.isfinite(new).all() or np.isnan(before):
                        self.scales[layer, p, which, head, b] = np.nan
                        continue
                    s = np.float32(0) if s < np.float32(2.0 ** -120) else s
                    now = max(before, s)
                    if now > before and lo > t0:
                        old = cells[at[:lo - t0]].astype(np.float64)
                        cells[at[:lo - t0]] = np.rint(old * np.float64(before) / np.float64(now)).astype(np.int8)
                    q = np.rint(new.astype(np.float64) / np.float64(now)) if now > 0 else np.zeros_like(new)
                    cells[at[lo - t0:hi - t0]] = np.clip(q, -127, 127).astype(np.int8)
                    self.scales[layer, p, which, head, b] = now


def attention(cache, layer, slots, rows, q, *, scale, softcap=0.0, window=0, causal=True, alibi=None, dtype="f32"):
    """(out, bound): attention of q [n_rows][heads][D] (float32 values) in 64 bits, and what a kernel may be off by.

    Bound of a row, with M the largest |V| of its visible tokens and T their number.  A score may be off by
      d = scale * (unit / 2) * max_t sum |K_t|   q is held in units of its largest value / TOP
        + 2^-21 * max |x|                        a handful of 32-bit roundings of a score, in units of log2
        + softcap * 2^-22 (an absolute error of 2^-23 of tanh, doubled)   + alibi: 2^-22 * |bias|
    A weight's relative error is e^d - 1 and 2^-22 of the exponential, and its rounding for the product with V is 2^-11
    (f32: 2^-22); where a weight is below fp16's normal range it is off by 2^-25 of 2^9 times the largest one at most.
    Sums of T products in 32 bits add T * 2^-24.  Numerator and denominator both have the weights' errors: twice.
    At last the rounding to the type of the output."""
    top_unit = 127.0 * (16384 if dtype == "f32" else 128)
    p_round = 2.0 ** -22 if dtype == "f32" else 2.0 ** -11
    out, bound, row = np.zeros(q.shape), np.zeros(q.shape[:2]), 0
    for slot, n in zip(slots, rows):
        k, v, length = cache.tokens(layer, slot, 0), cache.tokens(layer, slot, 1), int(cache.len[slot])
        t = np.arange(length)
        G = q.shape[1] // cache.H
        for i in range(n):
            p = length - n + i
            seen = np.ones(length, bool)
            if causal:
                seen &= t <= p
            if window:
                seen &= t > p - window
            if not seen.any():
                continue
            for j in range(q.shape[1]):
                kj, vj = k[seen, j // G], v[seen, j // G]
                qj = q[row + i, j].astype(np.float64)
                with np.errstate(invalid="ignore", over="ignore"):
                    x = kj @ qj * scale
                    big = np.abs(x).max()
                    unit = np.abs(qj).max() / top_unit
                    d = scale * unit / 2 * np.abs(kj).sum(1).max() + 2.0 ** -21 * big
                    if softcap:
                        x = softcap * np.tanh(x / softcap)
                        d += softcap * 2.0 ** -22
                    if alibi is not None:
                        bias = np.float64(alibi[j]) * (t[seen] - p)
                        x = x + bias
                        d += 2.0 ** -22 * np.abs(bias).max()
                    w = np.exp(x - x.max())
                    out[row + i, j] = (w @ vj) / w.sum()
                    M, T = np.abs(vj).max(), len(x)
                    bound[row + i, j] = M * (2 * (math.expm1(min(d, 20.0)) + 2.0 ** -22) + p_round + T * (2.0 ** -33 + 2.0 ** -24))
        row += n
    return out, bound[..., None] + HALF_STEP[dtype] * np.abs(out) + (2.0 ** -25 if dtype == "f16" else 0.0)
