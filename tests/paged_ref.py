"""Plain float64 forms of the paged-cache operators in numpy, and device memory for their tests.

Device arrays are raw hipMalloc memory on the runtime that the library itself uses; bf16 travels as uint16 bits."""
import ctypes as C

import numpy as np

EPS = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}     # half a step, relative


def to_bits(a, dtype):
    """The device form of float values: nearest-even rounding."""
    a = np.ascontiguousarray(a, np.float32)
    if dtype == "float32":
        return a
    if dtype == "float16":
        return a.astype(np.float16)
    u = a.view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r)


def from_bits(b, dtype):
    if dtype == "bfloat16":
        return (b.astype(np.uint32) << 16).view(np.float32)
    return b.astype(np.float32)


def rounded(a, dtype):
    return from_bits(to_bits(a, dtype), dtype)


class Dev:
    """An array in device memory; .a is the DeviceArray that the calls take."""

    kinds = {"float32": np.float32, "bfloat16": np.uint16, "float16": np.float16, "int32": np.int32, "float64": np.float64, "uint8": np.uint8}

    def __init__(self, host, dtype):
        from hip_mem import hip
        from ptts_paged import DeviceArray
        host = np.ascontiguousarray(host, self.kinds[dtype])
        self.shape, self.dtype, self.nbytes = host.shape, dtype, host.nbytes
        p = C.c_void_p()
        assert hip().hipMalloc(C.byref(p), max(self.nbytes, 16)) == 0
        self.ptr = p.value
        if self.nbytes:
            assert hip().hipMemcpy(self.ptr, host.ctypes.data, self.nbytes, 1) == 0
        self.a = DeviceArray(self.ptr, host.shape, dtype) if dtype != "uint8" else None

    def view(self, offset, shape, strides):
        from ptts_paged import DeviceArray
        return DeviceArray(self.ptr + offset * np.dtype(self.kinds[self.dtype]).itemsize, shape, self.dtype, strides)

    def host(self):
        from hip_mem import hip
        out = np.empty(self.shape, self.kinds[self.dtype])
        assert hip().hipDeviceSynchronize() == 0
        if self.nbytes:
            assert hip().hipMemcpy(out.ctypes.data, self.ptr, self.nbytes, 2) == 0
        return out

    def put(self, host):
        from hip_mem import hip
        host = np.ascontiguousarray(host, self.kinds[self.dtype])
        assert host.shape == self.shape and hip().hipDeviceSynchronize() == 0
        if self.nbytes:
            assert hip().hipMemcpy(self.ptr, host.ctypes.data, self.nbytes, 1) == 0

    def __del__(self):
        try:
            from hip_mem import hip
            hip().hipFree(self.ptr)
        except Exception:
            pass


def floats(a, dtype):
    return Dev(to_bits(a, dtype), dtype)


def plan(cached, arriving, free, table, page, rows):
    """table, slot_map, positions, cu_rows, kv_len, counts; slot_map and positions start at -7 (left alone behind the last row)."""
    table = table.copy()
    n, width = table.shape
    slots, positions = np.full(rows, -7), np.full(rows, -7)
    cu, kv_len = [0], []
    picks = missing = no_page = 0
    for i in range(n):
        c, a = max(int(cached[i]), 0), max(int(arriving[i]), 0)
        have, end = min(-(-c // page), width), -(-(c + a) // page)
        fit = max(min(end, width), have)
        missing += end - fit if end > fit else 0
        for j in range(have, fit):
            if picks < len(free):
                table[i, j] = free[picks]
            else:
                table[i, j] = -1
                missing += 1
            picks += 1
        for t in range(a):
            pos, r = c + t, cu[-1] + t
            ok = pos // page < width and table[i, pos // page] >= 0
            no_page += (not ok)
            if r < rows:
                slots[r] = table[i, pos // page] * page + pos % page if ok else -1
                positions[r] = pos
        cu.append(cu[-1] + a)
        kv_len.append(c + a)
    return table, slots, positions, np.array(cu), np.array(kv_len), np.array([cu[-1], min(picks, len(free)), missing, no_page])


def rotate(x, positions, freq, interleaved, magnitude=1.0):
    """x [rows][heads][dim] float64."""
    rot, half = 2 * len(freq), len(freq)
    angle = positions.astype(np.float64)[:, None] * freq[None, :]
    c, s = np.cos(angle)[:, None] * magnitude, np.sin(angle)[:, None] * magnitude
    y = np.array(x, np.float64)
    a = x[..., 0:rot:2] if interleaved else x[..., :half]
    b = x[..., 1:rot:2] if interleaved else x[..., half:rot]
    ra, rb = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0:rot:2], y[..., 1:rot:2] = ra, rb
    else:
        y[..., :half], y[..., half:rot] = ra, rb
    return y


def attention(q, k_rows, v_rows, cu, kv_len, scale, window=0, sinks=0):
    """q [rows][heads][dim]; k_rows(i), v_rows(i): [kv_len[i]][kv_heads][dim].  Returns out, lse (NaN rows: in no request), the same
    sum over |v| and the largest scale * sum |q||k| of each row (what the tolerances are made of)."""
    rows, heads, dim = q.shape
    out, lse = np.full((rows, heads, dim), np.nan), np.full((rows, heads), np.nan)
    size, logit = np.zeros((rows, heads, dim)), np.zeros((rows, heads))
    for i in range(len(kv_len)):
        k, v = k_rows(i).astype(np.float64), v_rows(i).astype(np.float64)
        group = heads // k.shape[1]
        j = np.arange(kv_len[i])
        for r in range(cu[i], cu[i + 1]):
            p = kv_len[i] - (cu[i + 1] - r)
            see = j <= p
            if window > 0:
                see &= (j > p - window) | (j < sinks)
            for h in range(heads):
                if not see.any():
                    out[r, h], lse[r, h] = 0.0, -np.inf
                    continue
                ks, vs = k[see, h // group], v[see, h // group]
                with np.errstate(all="ignore"):
                    s = ks @ q[r, h].astype(np.float64) * scale
                    m = s.max()
                    w = np.exp(s - m)
                    out[r, h] = w @ vs / w.sum()
                    lse[r, h] = m + np.log(w.sum())
                    size[r, h] = w @ np.abs(vs) / w.sum()
                    logit[r, h] = (np.abs(ks) @ np.abs(q[r, h].astype(np.float64))).max() * scale
    return out, lse, size, logit


def attention_bounds(out, size, logit, lse, dtype, dim, keys):
    """Largest errors of a correct kernel.  A score is a sum of dim products in float32: off by at most (dim + 2) 2^-24 times the sum of
    magnitudes, and a weight's relative error is that of its exponent plus a few units of the exponential (2^-21).  Weights are rounded
    to the rows' type once before they meet the values, the sums run over `keys` terms in float32, numerator and denominator each carry the
    weight's error, and the result is rounded once."""
    u, f = EPS[dtype], 2.0 ** -24
    weight = (dim + 2) * f * logit + 2.0 ** -21 + keys * f
    return size * (u + 2.2 * weight[..., None]) + u * np.abs(out) + 1e-30, weight * 1.1 + 4 * f * np.abs(lse) + f
