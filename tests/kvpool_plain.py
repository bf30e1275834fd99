"""The operators on a cache in pages and sampling, plainly, in 64 bits (numpy), and what the GPU tests of them share."""
import ctypes as C
import math

import numpy as np

F32, F16, BF16 = 0, 1, 2
SMALLEST = 2.0 ** -60
HALF_STEP = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
BYTES = {F32: 4, F16: 2, BF16: 2}


# ---- 16-bit types ---------------------------------------------------------------------------------------------


def bf16_bits(x):
    """float32 -> the bits of the nearest bfloat16, ties to even."""
    b = np.ascontiguousarray(x, np.float32).view(np.uint32)
    up = ((b >> 16) & 1) + np.uint32(0x7FFF)
    out = ((b + up) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), out)


def to_type(x, t):
    """What an array of type t holds, as its bytes' array."""
    with np.errstate(over="ignore"):
        return np.ascontiguousarray(x, np.float32) if t == F32 else np.asarray(x, np.float32).astype(np.float16) if t == F16 else bf16_bits(x)


def from_type(a, t):
    return a.astype(np.float32) if t != BF16 else (a.astype(np.uint32) << 16).view(np.float32)


def rounded(x, t):
    return from_type(to_type(x, t), t)


# ---- the cache ------------------------------------------------------------------------------------------------


def e4m3(y):
    """The nearest float of four exponent and three mantissa bits, ties to even (64-bit in and out)."""
    e = np.frexp(y)[1] - 1
    step = np.exp2(np.maximum(e, -6) - 3.0)
    return np.clip(np.rint(y / step) * step, -448.0, 448.0)


def held(x, kv_type):
    """The float32 values that a pool stands for once rows x (over the last axis) are written."""
    x = np.asarray(x, np.float32)
    if kv_type == "f16":
        return rounded(x, F16)
    if kv_type == "bf16":
        return rounded(x, BF16)
    most = np.float32(127 if kv_type == "i8" else 448)
    a = np.abs(x).max(-1, keepdims=True)
    fine = np.isfinite(a)
    s = np.where(fine & (a >= SMALLEST), a, 0).astype(np.float32) / most
    with np.errstate(all="ignore"):
        y = np.where(s > 0, x.astype(np.float64) / s.astype(np.float64), 0.0)
    c = e4m3(y) if kv_type == "e4m3" else np.rint(y)
    out = (c.astype(np.float32) * s).astype(np.float32)
    return np.where(fine, out, np.float32(np.nan))


def seen(pos, length, window, sinks):
    """Which of the positions 0..length-1 the row of position pos sees."""
    t = np.arange(length)
    m = t <= pos
    if window:
        m &= (t > pos - window) | (t < sinks)
    return m


def attention_row(q, k, v, scale):
    """One query head's row over the keys and values that it sees: the output, sum of p |v|, and the largest sum of |q k| scale."""
    if len(k) == 0:
        z = np.zeros(v.shape[-1])
        return z, z, 0.0
    q, k, v = q.astype(np.float64), k.astype(np.float64), v.astype(np.float64)
    with np.errstate(all="ignore"):
        s = k @ q * scale
        p = np.exp(s - s.max())
        p /= p.sum()
        return p @ v, p @ np.abs(v), float((np.abs(k) @ np.abs(q)).max() * abs(scale))


def attention_bound(kv_type, t, size, at_most, n, head_size, out):
    """How far fp32 arithmetic may be off, element by element.  A score is a sum of head_size products (each off by its pieces' 2^-22 in
    fp32 rows) in fp32: within at_most * (head_size * 2^-24 + 2^-21), and its product with a scale and the exponent another three roundings of
    it; a weight is off by twice that (itself and the sum), by the exponential's own 2^-22, by the rounding that it enters the product with, and
    the sum over n positions adds n roundings."""
    score = at_most * ((head_size + 4) * 2.0 ** -24 + 2.0 ** -21)
    weight = {F32: 2.0 ** -21, F16: 2.0 ** -11, BF16: 2.0 ** -11}[t]
    if kv_type == "bf16" and t != F32:
        weight = 2.0 ** -8
    off = size * (2 * score + weight + 2.0 ** -21 + (n + 64) * 2.0 ** -24)
    # a 16-bit result below its type's normal numbers is off by half of their smallest step
    return off * 1.01 + (np.abs(out) + off) * HALF_STEP[t] + (2.0 ** -25 if t == F16 else 2.0 ** -130)


# ---- sampling -------------------------------------------------------------------------------------------------


def sample(row, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0):
    """The id, and how near (of the whole) a border between two answers is."""
    x = np.where(np.isnan(row), -np.inf, row).astype(np.float64)
    order = np.lexsort((np.arange(len(x)), -x))
    top = x[order[0]]
    if top == -np.inf:
        return -1, 1.0
    if not temperature > 0:
        return int(order[0]), 1.0
    with np.errstate(all="ignore"):
        d = np.where(x == top, 0.0, x - top)
        w = np.where(x == -np.inf, 0.0, np.exp(d / np.float64(np.float32(temperature))))
    near = 1.0
    if 0 < top_k < len(x):
        order = order[:top_k]
    if top_p < 1:
        c = np.cumsum(w[order])
        target = float(np.float32(top_p)) * c[-1]
        near = min(near, float(np.abs(c - target).min() / c[-1]))
        order = order[:int(np.searchsorted(c, target)) + 1]
    if min_p > 0:
        least = min(float(np.float32(min_p)), 1.0)
        off = np.abs(w[order] - least)[x[order] != top]  # the largest weight is 1 exactly
        near = min(near, float(off.min()) if len(off) else 1.0)
        order = order[w[order] >= least]
    ids = np.sort(order)
    c = np.cumsum(w[ids])
    target = min(max(float(np.float32(u)), 0.0), 1.0) * c[-1]
    i = int(np.searchsorted(c, target, side="right"))
    if i < len(ids) and target > 0:
        near = min(near, float(np.abs(c - target).min() / c[-1]))
    if np.all((w == 0) | (w == 1)):  # weights that are whole: sums, and their products with a number of 24 bits, are exact on both sides
        near = 1.0
    last = int(np.flatnonzero(w[ids])[-1])
    return int(ids[min(i, last)]), near


# ---- on the GPU -----------------------------------------------------------------------------------------------


class Device:
    """Device memory for the tests' arrays."""

    def __init__(self):
        from tests.test_zz_no_alloc import _Hip
        self.hip = _Hip()
        self.rt = self.hip.rt

    def put(self, a):
        a = np.ascontiguousarray(a)
        return self.hip.upload(a) if a.nbytes else self.hip.empty(16)

    def set(self, p, a):
        a = np.ascontiguousarray(a)
        assert self.rt.hipMemcpy(C.c_void_p(p), a.ctypes.data_as(C.c_void_p), a.nbytes, 1) == 0

    def empty(self, n):
        return self.hip.empty(max(n, 16))

    def get(self, p, shape, dtype):
        out = np.empty(shape, dtype)
        assert self.rt.hipDeviceSynchronize() == 0
        if out.nbytes:
            assert self.rt.hipMemcpy(out.ctypes.data_as(C.c_void_p), C.c_void_p(p), out.nbytes, 2) == 0
        return out

    def close(self):
        self.hip.close()


class Cache:
    """A pool of one layer or more, and the sequences in it, with what they stand for on the host."""

    def __init__(self, dev, kv_type, page, kv_heads, head_size, lengths, seed=0, layers=1, extra_pages=3, layer=0):
        from llama2_rs import ops
        self.dev, self.kv_type, self.page, self.kv_heads, self.head_size, self.layer = dev, kv_type, page, kv_heads, head_size, layer
        rng = np.random.default_rng(seed)
        need = [-(-max(n, 0) // page) for n in lengths]
        self.lengths, self.n_pages = list(lengths), sum(need) + extra_pages
        order = rng.permutation(self.n_pages)
        self.max_pages = max(max(need), 1)
        self.table = np.full((len(lengths), self.max_pages), -1, np.int32)
        at = 0
        for i, m in enumerate(need):
            self.table[i, :m] = order[at:at + m]
            at += m
        self.pool = ops.KvPool(layers, self.n_pages, page, kv_heads, head_size, kv_type)
        self.k = self.v = None

    def batch(self, rows, lengths=None, first=0, behind=0, table=None, max_rows=None, max_length=None):
        """rows[i] last positions of sequence i, `first` rows in front of all and `behind` rows after them."""
        from llama2_rs import ops
        lengths = self.lengths if lengths is None else lengths
        starts = first + np.concatenate([[0], np.cumsum(rows)])
        table = self.table if table is None else table
        return ops.KvBatch(self.dev.put(starts.astype(np.int32)), self.dev.put(np.asarray(lengths, np.int32)), self.dev.put(table), len(rows),
                           table.shape[1], int(starts[-1]) + behind, max(rows) if max_rows is None else max_rows,
                           max(max(lengths), 0) if max_length is None else max_length)

    def fill(self, k, v, t=F32):
        """Writes all positions of all sequences: k, v [sum of lengths][kv heads][head size]."""
        self.k, self.v = held(rounded(k, t), self.kv_type), held(rounded(v, t), self.kv_type)
        b = self.batch(self.lengths)
        self.pool.write(self.layer, b, self.dev.put(to_type(k, t)), self.dev.put(to_type(v, t)), t)

    def rows_of(self, i):
        at = int(np.sum(self.lengths[:i]))
        return slice(at, at + self.lengths[i])

    def attend(self, q, rows, t, heads, window=0, sinks=0, scale=0.0, batch=None, stream=0, q_stride=0, out_stride=0, out=None, fill=7.0):
        """The operator's answer for q [rows][heads][head size] (float32, rounded to t here)."""
        b = batch if batch is not None else self.batch(rows)
        dq = self.dev.put(to_type(q, t))
        if out is None:
            out = self.dev.put(to_type(np.full(q.shape, fill, np.float32), t))
        n = self.pool.attention_workspace(b, heads, t, window, sinks)
        work = self.dev.put(np.full(max(n, 16), 0xFF, np.uint8))  # NaN wherever it is read before it is written
        self.pool.attention(self.layer, b, dq, out, heads, t, scale, window, sinks, work, n, q_stride, out_stride, stream)
        return from_type(self.dev.get(out, q.shape, {F32: np.float32, F16: np.float16, BF16: np.uint16}[t]), t)

    def check(self, got, q, rows, t, heads, window=0, sinks=0, scale=None, lengths=None, first=0, missing=()):
        """got against the formula, and rows outside of all sequences as they were (7).  missing: (sequence, page) that is not there."""
        scale = 1.0 / math.sqrt(self.head_size) if scale is None else scale
        lengths = self.lengths if lengths is None else lengths
        group = heads // self.kv_heads
        q = rounded(q, t)
        assert np.all(got[:first] == 7.0) and np.all(got[first + sum(rows):] == 7.0), "rows outside of the sequences"
        at = first
        for i, n in enumerate(rows):
            k, v = self.k[self.rows_of(i)][:max(lengths[i], 0)], self.v[self.rows_of(i)][:max(lengths[i], 0)]
            for j in range(n):
                pos = lengths[i] - n + j
                m = seen(pos, len(k), window, sinks)
                for s, page in missing:
                    if s == i:
                        m[page * self.page:(page + 1) * self.page] = False
                for h in range(heads):
                    want, size, most = attention_row(q[at, h], k[m][:, h // group], v[m][:, h // group], scale)
                    where = f"sequence {i} row {j} head {h}"
                    if not np.all(np.isfinite(want)):
                        assert np.array_equal(np.isnan(got[at, h]), np.isnan(want)), where
                        continue
                    bound = attention_bound(self.kv_type, t, size, most, int(m.sum()), self.head_size, want)
                    off = np.abs(got[at, h].astype(np.float64) - want)
                    assert np.all(off <= bound), (where, float(np.max(off / np.maximum(bound, 1e-300))), int(np.argmax(off / np.maximum(bound, 1e-300))))
                at += 1

    def close(self):
        self.pool.close()
