"""The key/value cache operators from their definitions, in 64 bits on the
host, and device copies of a cache for the tests of the kernels."""

from __future__ import annotations

import numpy as np

import awa_hip as A

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
HALF = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}  # half a step, relative to the value


def bf16(x):
    return A.bf16_bits_to_f32(A.f32_to_bf16_bits(np.asarray(x, np.float32)))


def as_type(x, dtype):
    return bf16(x) if dtype == "bf16" else np.asarray(x, np.float32)


def encode4(x):
    """Codes [.., D/2] and scale bytes [.., D/32] of x (64 bits)."""
    x = np.asarray(x, np.float64)
    g = x.reshape(*x.shape[:-1], x.shape[-1] // 32, 32)
    top = np.abs(g).max(-1, keepdims=True)
    fine = np.isfinite(top)
    m, e = np.frexp(np.where(fine, top, 1.0))
    e = np.where(top == 0, -126, np.maximum(e - 2 - (m <= 0.875), -126))
    y = np.abs(np.ldexp(np.where(fine, g, 0.0), -e))
    lower = np.clip(np.searchsorted(GRID, y, side="right") - 1, 0, 7)
    upper = np.minimum(lower + 1, 7)
    middle = (GRID[lower] + GRID[upper]) / 2
    up = (y > middle) | ((y == middle) & (upper % 2 == 0))
    code = np.where(up, upper, lower) + 8 * (np.signbit(g) & fine)
    code = code.reshape(x.shape).astype(np.uint8)
    byte = np.where(fine, e + 127, 255)[..., 0].astype(np.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), byte


def decode4(codes, byte):
    code = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], 2 * codes.shape[-1])
    v = np.where(code > 7, -1.0, 1.0) * GRID[code & 7]
    unit = np.where(byte == 255, np.nan, np.ldexp(1.0, byte.astype(np.int64) - 127))
    return (v.reshape(*byte.shape, 32) * unit[..., None]).reshape(v.shape)


def rotate(x, positions, rope_dim, axes=1, base=10000.0, halves=False, frequencies=None):
    """x [T][H][D], positions [T][axes]; angles in extended precision."""
    x = np.asarray(x, np.float64)
    pairs = rope_dim // axes // 2
    f = (np.asarray(frequencies, np.longdouble) if frequencies is not None
         else np.longdouble(base) ** (-np.arange(pairs, dtype=np.longdouble) / pairs))
    angle = (np.asarray(positions).astype(np.longdouble)[:, :, None] * f).reshape(len(x), -1)[:, None, :]
    cos, sin = np.cos(angle).astype(np.float64), np.sin(angle).astype(np.float64)
    out = x.copy()
    lo, hi = (slice(0, pairs), slice(pairs, rope_dim)) if halves else (slice(0, rope_dim, 2), slice(1, rope_dim, 2))
    out[..., lo] = x[..., lo] * cos - x[..., hi] * sin
    out[..., hi] = x[..., hi] * cos + x[..., lo] * sin
    return out


def visible(slot, length, window, sinks, block):
    """Truth values [length] of the keys that the row at `slot` sees."""
    k = np.arange(length)
    e = sinks + block * -(-(slot + 1 - sinks) // block)
    return (k < e) & ((window == 0) | (k >= e - window) | (k < sinks))


def attention(q, keys, values, length, window, sinks, block, scale, dtype, there=None):
    """q [n][H][D] at slots length - n .., keys and values [length][Hkv][D] ->
    the result and how far the kernels' arithmetic may be from it."""
    n, heads, dim = q.shape
    group = heads // keys.shape[1]
    out = np.zeros((n, heads, dim))
    bound = np.zeros((n, heads, dim))
    for j in range(n):
        see = visible(length - n + j, length, window, sinks, block)
        if there is not None:
            see &= there
        if not see.any():
            continue
        for h in range(heads):
            k, v = keys[see, h // group], values[see, h // group]
            qj = q[j, h].astype(np.float64)
            with np.errstate(invalid="ignore", over="ignore"):
                s = k @ qj * scale
                p = np.exp(s - s.max())
                w = p / p.sum()
                out[j, h] = w @ v
                # A weight is off by its score's error: an fp32 sum of dim
                # products, their scaling and the exponential (2^-22 and the
                # rounding of its argument); bf16 rows also round it once. The
                # quotient of two such sums, each of len(k) terms in fp32 with
                # at most 8 joins of parts.
                terms = scale * (np.abs(k) @ np.abs(qj)).max()
                e = (dim + 8) * 2.0 ** -24 * terms + 2.0 ** -22 + 2.0 ** -23 * np.abs(s - s.max()).max()
                e += (len(k) + 16) * 2.0 ** -24 + (HALF["bf16"] if dtype == "bf16" else 2.0 ** -23)
                bound[j, h] = 2 * e * (w @ np.abs(v)) + HALF[dtype] * 1.01 * np.abs(out[j, h])
    return out, bound


class Cache:
    """A cache on the host and its copy on the device."""

    def __init__(self, fmt, lengths, kv_heads=2, dim=128, page=16, seed=1, extra_pages=2, stride=0, width=None,
                 fill=None):
        rng = np.random.default_rng(seed)
        self.four, self.heads, self.dim, self.page = fmt == "4bit", kv_heads, dim, page
        self.lengths = np.asarray(lengths, np.int32)
        used = [max(0, -(-int(n) // page)) for n in lengths]
        self.width = width or max(1, max(used))
        self.stride = stride or self.width
        self.pages = sum(used) + extra_pages
        self.table = np.full((len(lengths), self.stride), -1, np.int32)
        order, at = rng.permutation(self.pages), 0
        for s, n in enumerate(used):
            self.table[s, :n] = order[at:at + n]
            at += n
        shape = (self.pages, kv_heads, page, dim)
        self.host = {}
        for name in ("k", "v"):
            x = rng.standard_normal(shape) if fill is None else np.full(shape, fill)
            if self.four:
                self.host[name], self.host[name + "_scale"] = encode4(x)
            else:
                self.host[name] = A.f32_to_bf16_bits(x.astype(np.float32))
        self.dev = {}
        self.status_buf = None

    def values(self, name):
        """[pages][heads][page][dim] in 64 bits."""
        if self.four:
            return decode4(self.host[name], self.host[name + "_scale"])
        return A.bf16_bits_to_f32(self.host[name]).astype(np.float64)

    def rows(self, name, s, length=None):
        """[length][heads][dim] of sequence s, and whether each slot's page is one."""
        length = int(self.lengths[s]) if length is None else length
        slot = np.arange(length)
        page = self.table[s, slot // self.page] if length else np.zeros(0, int)
        ok = (page >= 0) & (page < self.pages)
        at = np.where(ok, page, 0), slice(None), slot % self.page
        if self.four:
            return decode4(self.host[name][at], self.host[name + "_scale"][at]), ok
        return A.bf16_bits_to_f32(self.host[name][at]).astype(np.float64), ok

    def upload(self, spare=0):
        for name, x in {**self.host, "table": self.table, "lengths": self.lengths,
                        "status": np.zeros(1, np.int32)}.items():
            self.dev[name] = A.DeviceBuffer(max(16, x.nbytes))
            self.dev[name].upload(x)
        p = {n: b.ptr for n, b in self.dev.items()}
        self.desc = A.KvCache(A.KV_MXFP4 if self.four else A.KV_BF16, self.pages, self.page, self.heads, self.dim,
                              p["k"], p["v"], p["table"], len(self.lengths), self.width, p["lengths"],
                              k_scale=p.get("k_scale", 0), v_scale=p.get("v_scale", 0), status=p["status"],
                              table_stride=self.stride)
        return self.desc

    def download(self):
        """The device's pools."""
        return {n: self.dev[n].download(x.shape, x.dtype) for n, x in self.host.items()}

    def status(self):
        return int(self.dev["status"].download((1,), np.int32)[0])

    def set(self, **arrays):
        for name, x in arrays.items():
            x = np.asarray(x, np.int32)
            setattr(self, name, x)
            self.dev[name].upload(x)


class Rows:
    """Packed rows [T][H][D] on the device, each `lead` values into a row of
    `pitch` values, as a view of a wider projection is."""

    def __init__(self, x, dtype, pitch=0, lead=0):
        x = np.asarray(x, np.float32)
        self.shape, self.dtype, self.lead = x.shape, dtype, lead
        self.pitch = pitch or x.shape[1] * x.shape[2]
        self.size = 4 if dtype == "f32" else 2
        host = np.full((x.shape[0], self.pitch), 7.0, np.float32)
        host[:, lead:lead + x.shape[1] * x.shape[2]] = x.reshape(x.shape[0], -1)
        self.buf = A.DeviceBuffer(max(16, host.size * self.size))
        self.buf.upload(host if dtype == "f32" else A.f32_to_bf16_bits(host))
        self.blob = A.mat(self.buf.ptr + lead * self.size, x.shape[2], x.shape[1], x.shape[0], self.size, dims=3,
                          cstep=self.pitch)
        self.blob.buffer = self.buf  # a descriptor keeps its memory

    def read(self, whole=False):
        raw = self.buf.download((self.shape[0], self.pitch), np.float32 if self.dtype == "f32" else np.uint16)
        x = raw if self.dtype == "f32" else A.bf16_bits_to_f32(raw)
        return x if whole else x[:, self.lead:self.lead + self.shape[1] * self.shape[2]].reshape(self.shape)


def ints(x):
    x = np.ascontiguousarray(x, np.int32)
    b = A.DeviceBuffer(max(16, x.nbytes))
    b.upload(x)
    return b
