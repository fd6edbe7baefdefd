"""Token operators on numpy arrays through the device C ABI, and their
definitions in 64 bits.

Tolerances follow from the arithmetic the header promises, worst case by
element: one rounding to FP16 of the output (2^-11 of it, or 2^-25 where FP16
is subnormal), FP32 sums of n terms (n 2^-24 of the terms' magnitudes), and in
attention the FP16 weights the matrix cores take (2^-11 of each weight, or
2^-25 of the largest where they are subnormal).
"""

import ctypes as C

import numpy as np

import mlvc_hip

LEVEL = {mlvc_hip.KV_E4M3: 448.0, mlvc_hip.KV_INT8: 127.0}


def f64(a):
    return np.asarray(a, np.float16).astype(np.float64)


def within(got, want, tol, what=""):
    """got within tol of want wherever want is finite, and as non-finite elsewhere."""
    got = np.asarray(got).astype(np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got)), f"{what}: non-finite outputs differ"
    off = np.abs(got - want)[fine] / np.broadcast_to(tol, want.shape)[fine]
    assert off.size == 0 or off.max() <= 1.0, f"{what}: {off.max():.3g} times the tolerance"


class Padded:
    """An FP16 tensor [tokens, heads, dim] inside wider rows, `shift` halves
    into its buffer; what is around it is `fill`."""

    def __init__(self, dev, a, extra=0, shift=0, fill=0x7E00):
        a = np.asarray(a, np.float16)
        self.shape, self.dev = a.shape, dev
        row = int(np.prod(a.shape[1:]))
        self.stride, self.shift = row + extra, shift
        buf = np.full(shift + max(a.shape[0], 1) * self.stride + 8, fill, np.uint16)
        rows = buf[shift:shift + a.shape[0] * self.stride].reshape(a.shape[0], self.stride)
        rows[:, :row] = a.reshape(a.shape[0], row).view(np.uint16)
        self.n, self.row, self.base = buf.size, row, dev.put(buf)
        self.at = self.base.value + 2 * shift

    def get(self):
        """The tensor, after checking that nothing around it changed from 0x7E00."""
        buf = self.dev.get(self.base, (self.n,), np.uint16)
        rows = buf[self.shift:self.shift + self.shape[0] * self.stride].reshape(self.shape[0], self.stride)
        assert (buf[:self.shift] == 0x7E00).all() and (rows[:, self.row:] == 0x7E00).all()
        return rows[:, :self.row].copy().view(np.float16).reshape(self.shape)


# ------------------------------------------------------------ norm and rotation

def rope64(x, w, eps, positions, freqs, interleaved, rot_scale):
    """(result, tolerance) of one tensor [tokens, heads, dim]."""
    x = f64(x)
    if w is not None:
        x = x / np.sqrt(np.mean(x * x, -1, keepdims=True) + eps) * f64(w)
    y, size = x.copy(), np.abs(x)
    half = len(freqs)
    if half:
        angle = np.mod(positions.astype(np.float64)[:, None] * freqs, 2 * np.pi)[:, None, :]
        c, s = rot_scale * np.cos(angle), rot_scale * np.sin(angle)
        i = np.arange(half) * (2 if interleaved else 1)
        j = i + (1 if interleaved else half)
        y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
        size[..., i] = size[..., j] = (np.abs(x[..., i]) + np.abs(x[..., j])) * max(rot_scale, 1)
    # Phase, sine and products: a few FP32 roundings of values up to `size`
    # (the FP64 phase of |p f| < 2^21 radians is 2^-31 of a turn off); the
    # norm's sum of dim squares: dim 2^-24 of itself.
    return y, np.abs(y) * 2.0 ** -11 + 2.0 ** -25 + size * (2.0 ** -20 + x.shape[-1] * 2.0 ** -24)


# ------------------------------------------------------------ cache

def stored64(x, kind):
    """What each row of the cache stands for."""
    x = f64(x)
    if kind == mlvc_hip.KV_F16:
        return x
    level = LEVEL[kind]
    top = np.abs(x).max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        scale = (top.astype(np.float32) / np.float32(level)).astype(np.float64)
        units = np.where(top > 0, x * level / np.where(top > 0, top, 1), 0.0)
        if kind == mlvc_hip.KV_INT8:
            back = np.round(units) * scale
        else:
            step = np.exp2(np.floor(np.log2(np.maximum(np.abs(units), 2.0 ** -6))) - 3)
            back = np.round(units / step) * step * scale
    return np.where(np.isfinite(top), back, np.nan)


class Cache:
    """A paged cache on the device, its memory filled with a byte (and scales with NaN) first."""

    def __init__(self, dev, kind, pages, page_size, heads, dim, fill=0x7F):
        self.dev, self.kind, self.page_size, self.heads, self.dim, self.pages = dev, kind, page_size, heads, dim, pages
        self.desc = mlvc_hip.KvCache(kind=kind, pages=pages, page_size=page_size, heads=heads, head_dim=dim)
        nbytes, scales = mlvc_hip.kv_cache_bytes(self.desc)
        assert nbytes == pages * page_size * heads * dim * (2 if kind == mlvc_hip.KV_F16 else 1)
        assert scales == (0 if kind == mlvc_hip.KV_F16 else 4 * pages * page_size * heads)
        self.desc.k, self.desc.v = (dev.put(np.full(nbytes, fill, np.uint8)) for _ in range(2))
        if scales:
            self.desc.k_scale, self.desc.v_scale = (dev.put(np.full(scales // 4, np.nan, np.float32)) for _ in range(2))

    def rows(self, k, v, slots):
        return mlvc_hip.KvRows(tokens=len(slots), k=k.at, v=v.at, k_stride=k.stride, v_stride=v.stride,
                               slots=self.dev.put(np.asarray(slots, np.int32)))

    def write(self, k, v, slots, extra=0, shift=0, stream=None):
        kp, vp = Padded(self.dev, k, extra, shift), Padded(self.dev, v, extra, shift)
        mlvc_hip.kv_write(self.desc, self.rows(kp, vp, slots), stream)

    def read(self, slots, extra=0, shift=0):
        shape = (len(slots), self.heads, self.dim)
        kp, vp = (Padded(self.dev, np.full(shape, np.nan, np.float16), extra, shift) for _ in range(2))
        mlvc_hip.kv_read(self.desc, self.rows(kp, vp, slots))
        return kp.get(), vp.get()


# ------------------------------------------------------------ attention

def attend64(q, k, v, scale, causal):
    """(result, tolerance): q [queries, q_heads, dim] on k, v [keys, kv_heads, dim] in 64 bits."""
    q, k, v = (np.asarray(t, np.float64) for t in (q, k, v))
    nq, heads, dim = q.shape
    nk, group = k.shape[0], heads // max(k.shape[1], 1)
    out, tol = np.zeros_like(q), np.full(q.shape, 2.0 ** -25)
    for h in range(heads):
        for i in range(nq):
            n = min(nk, max(0, nk - nq + i + 1)) if causal else nk
            if n == 0:
                continue
            kk, vv = k[:n, h // group], v[:n, h // group]
            with np.errstate(all="ignore"):
                s = kk @ q[i, h] * scale
                # FP32 products and sums of dim terms, then the exponent's own rounding.
                ds = (np.abs(kk) @ np.abs(q[i, h])) * abs(scale) * (dim + 4) * 2.0 ** -24 + np.abs(s) * 2.0 ** -22 + 2.0 ** -21
                p = np.exp(s - s.max())
                w = p / p.sum()
                o = w @ vv
                size = np.abs(vv)
                err = w * (2.0 ** -11 + 2 * ds) + 2.0 ** -25 / p.sum()
            out[i, h] = o
            # Each weight off by err moves the result by err |v - o|; sums of n terms in FP32.
            tol[i, h] += np.abs(o) * 2.0 ** -11 + err @ (size + np.abs(o)) + (n + 8) * 2.0 ** -24 * (w @ size)
    return out, tol


class Prompt:
    """Packed sequences on the device."""

    def __init__(self, dev, q, k, v, queries, keys, causal, scale, extra=0, shift=0, longest=None, starts=None):
        self.out = Padded(dev, np.full(q.shape, np.nan, np.float16), extra, shift)
        qp, kp, vp = (Padded(dev, t, extra, shift) for t in (q, k, v))
        sq, sk = starts or (np.concatenate([[0], np.cumsum(n)]) for n in (queries, keys))
        self.keep = (qp, kp, vp)
        self.desc = mlvc_hip.PromptAttention(
            sequences=len(queries), q_heads=q.shape[1], kv_heads=k.shape[1], head_dim=q.shape[2], q=qp.at, k=kp.at,
            v=vp.at, out=self.out.at, q_stride=qp.stride, k_stride=kp.stride, v_stride=vp.stride,
            out_stride=self.out.stride, q_starts=dev.put(np.asarray(sq, np.int32)),
            k_starts=dev.put(np.asarray(sk, np.int32)), q_tokens=q.shape[0], k_tokens=k.shape[0],
            longest_q=max(queries, default=0) if longest is None else longest, causal=int(causal), scale=scale)

    def run(self, stream=None):
        mlvc_hip.attention_prompt(self.desc, stream)
        return self.out.get()


class Token:
    """One query per stream on a cache."""

    def __init__(self, cache, q, table, lengths, scale, longest=None, extra=0, shift=0):
        dev = cache.dev
        self.cache, self.out = cache, Padded(dev, np.full(q.shape, np.nan, np.float16), extra, shift)
        self.q = Padded(dev, q, extra, shift)
        table = np.asarray(table, np.int32)
        self.lengths = dev.put(np.asarray(lengths, np.int32))
        self.desc = mlvc_hip.TokenAttention(
            cache=C.pointer(cache.desc), streams=q.shape[0], q_heads=q.shape[1], q=self.q.at, out=self.out.at,
            q_stride=self.q.stride, out_stride=self.out.stride, table=dev.put(table), table_stride=table.shape[1],
            lengths=self.lengths, longest=max(lengths, default=0) if longest is None else longest, scale=scale)
        need = mlvc_hip.attention_token_workspace_bytes(self.desc)
        if need:
            # NaN throughout, so that a partial that is read without having been written shows.
            self.desc.workspace = dev.put(np.full(need, 0xFF, np.uint8))
            self.desc.workspace_bytes = need

    def run(self, stream=None):
        mlvc_hip.attention_token(self.desc, stream)
        return self.out.get()
