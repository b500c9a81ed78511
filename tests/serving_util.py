"""Helpers of the serving-op tests: device copies of torch tensors (bf16 included) and 64-bit restatements."""
import math

import numpy as np
import torch

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def code(sg, name):
    return {"f32": sg.F32, "f16": sg.F16, "bf16": sg.BF16}[name]


def dev(sg, t):
    """Device copy of a CPU tensor."""
    t = t.contiguous()
    return sg.DeviceBuffer.from_numpy(t.view(torch.uint8).numpy().reshape(-1) if t.numel() else np.zeros(16, np.uint8))


def back(sg, buf, t):
    """The buffer's contents as a tensor like t."""
    n = t.numel() * t.element_size()
    return torch.from_numpy(buf.to_numpy(np.uint8, n).copy()).view(t.dtype).reshape(t.shape)


def i32(values):
    return torch.tensor(values, dtype=torch.int32)


def offsets(lengths):
    return i32(np.concatenate([[0], np.cumsum(lengths)]).tolist())


def half_ulp(dtype):
    """A rounding is off by at most this, relative to the value."""
    return torch.finfo(dtype).eps / 2


def attend64(q, k, v, scale):
    """Causal attention of one sequence in 64 bits: q [nq, H, D], k, v [nk, G, D].  Keys that a row does not see are left
    out (not multiplied by zero)."""
    nq, H, D = q.shape
    nk, G = k.shape[:2]
    out = torch.zeros(nq, H, D, dtype=torch.float64)
    if not nq or not nk:
        return out
    kk = k.double().repeat_interleave(H // G, 1)
    vv = v.double().repeat_interleave(H // G, 1)
    s = torch.einsum("ihd,jhd->hij", q.double(), kk) * scale
    seen = torch.arange(nk)[None] <= torch.arange(nq)[:, None] + (nk - nq)
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top)).masked_fill(~seen, 0.0)
    den = p.sum(-1, keepdim=True)
    p = p / torch.where(den == 0, torch.ones_like(den), den)
    finite = torch.isfinite(vv).all(-1).all(-1)
    out = torch.einsum("hij,jhd->ihd", p[:, :, finite], vv[finite])
    for j in torch.nonzero(~finite)[:, 0].tolist():
        rows = seen[:, j]
        out[rows] += torch.einsum("hi,hd->ihd", p[:, rows, j], vv[j])
    return out


def prompt_tolerance(q, k, v, scale, n, dtype, tensor_cores):
    """|error| of prompt attention, from the roundings: a score is a sum of D products (and a scaling), each operation off by
    2^-24 relative, 2^-23 where the tensor cores truncate, so it is off by ds <= (D + 4) 2^-23 scale sum_d |q_d k_d|; weights
    are exponentials of it (2^-21 for the exponential itself), numerator and denominator each carry it once; both are sums of
    n terms.  On the tensor cores every weight is rounded to the 16-bit type.  The output is rounded once."""
    D = q.shape[-1]
    finite = lambda t: t.double().abs()[torch.isfinite(t.double())]
    s1 = scale * D ** 0.5 * finite(q).max() * (finite(k).max() if k.numel() else 0) * D ** 0.5   # >= scale sum |q_d k_d|
    vmax = finite(v).max() if v.numel() else 0.0
    w = 2 * (D + 4) * 2.0 ** -23 * s1 + 2.0 ** -20 + 2 * n * 2.0 ** -23
    if tensor_cores:
        w = w + half_ulp(dtype)
    return float(vmax * w)


# ------------------------------------------------------------------------------------------------ 8-bit cache
def pitch(d):
    return (d + 31) // 32 * 32


class Cache64:
    """Plain restatement of the cache: integers per (block, head, token, element), one f32 scale per (block, head)."""

    def __init__(self, blocks, bt, heads, dim, rng=None):
        self.bt, self.heads, self.dim, self.blocks = bt, heads, dim, blocks
        shape = (blocks, heads, bt, dim)
        if rng is None:
            self.q = [np.zeros(shape, np.int8) for _ in range(2)]
            self.s = [np.zeros((blocks, heads), np.float32) for _ in range(2)]
        else:
            self.q = [rng.integers(-127, 128, shape).astype(np.int8) for _ in range(2)]
            self.s = [(0.01 + 0.02 * rng.random((blocks, heads))).astype(np.float32) for _ in range(2)]

    def bytes(self):
        """k, v, k_scales, v_scales in the library's layout."""
        p = pitch(self.dim)
        k = np.zeros((self.blocks, self.heads, self.bt, p), np.int8)
        k[..., :self.dim] = self.q[0]
        v = np.zeros((self.blocks, self.heads, self.bt // 16, p, 16), np.int8)
        v[..., :self.dim, :] = self.q[1].reshape(self.blocks, self.heads, self.bt // 16, 16, self.dim).swapaxes(-1, -2)
        return k, v, self.s[0], self.s[1]

    def from_bytes(self, k, v, ks, vs):
        """(integers, scales) of K and V from the library's layout."""
        p = pitch(self.dim)
        k = k.reshape(self.blocks, self.heads, self.bt, p)[..., :self.dim]
        v = v.reshape(self.blocks, self.heads, self.bt // 16, p, 16)[..., :self.dim, :].swapaxes(-1, -2)
        return [k, v.reshape(self.blocks, self.heads, self.bt, self.dim)], [ks.reshape(self.blocks, self.heads), vs.reshape(self.blocks, self.heads)]

    def append(self, table, rows, starts):
        """rows: per sequence (k, v) arrays [n, heads, dim]; written from places starts[s] on."""
        for s, kv in enumerate(rows):
            for which, x in enumerate(kv):
                x = np.asarray(x, np.float64)
                pos, end = starts[s], starts[s] + len(x)
                while pos < end:
                    b, a = table[s][pos // self.bt], pos % self.bt
                    n = min(self.bt - a, end - pos)
                    for h in range(self.heads):
                        new = x[pos - starts[s]: pos - starts[s] + n, h]
                        good = np.abs(new[np.isfinite(new)])
                        step = np.float32(np.float32(good.max() if good.size else 0.0) / np.float32(127))
                        if step < np.finfo(np.float32).tiny:
                            step = np.float32(0)
                        old = self.s[which][b, h]
                        if a:
                            step = max(step, old)
                            if step != old:
                                self.q[which][b, h, :a] = np.rint(self.q[which][b, h, :a].astype(np.float64) * float(old) / float(step))
                        q = np.zeros(new.shape)
                        if step > 0:
                            q = np.where(np.isfinite(new), np.rint(np.where(np.isfinite(new), new, 0) / float(step)), 0)
                            q = np.clip(q, -127, 127)
                            q[np.isposinf(new)], q[np.isneginf(new)] = 127, -127
                        self.q[which][b, h, a:a + n] = q
                        self.s[which][b, h] = step
                    pos += n

    def values(self, table_row, n, which):
        """The first n tokens of a sequence in 64 bits, [n, heads, dim]."""
        out = np.zeros((n, self.heads, self.dim))
        for t in range(n):
            b = table_row[t // self.bt]
            out[t] = self.q[which][b, :, t % self.bt].astype(np.float64) * self.s[which][b].astype(np.float64)[:, None]
        return out


class DeviceCache:
    def __init__(self, sg, c64):
        self.sg, self.c = sg, c64
        self.bufs = [sg.DeviceBuffer.from_numpy(a) for a in c64.bytes()]
        self.handle = sg.kv8_cache(*self.bufs, c64.blocks, c64.bt, c64.heads, c64.dim)

    def contents(self):
        c, p = self.c, pitch(self.c.dim)
        n = c.blocks * c.heads * c.bt * p
        raw = [b.to_numpy(np.int8, n) for b in self.bufs[:2]] + [b.to_numpy(np.float32, c.blocks * c.heads) for b in self.bufs[2:]]
        return c.from_bytes(*raw)


def make_table(lengths, bt, rng, extra=0, width=None, fill=-1):
    """A shuffled pool: table [n_seqs, width] int32 and the number of blocks (`extra` of them in no sequence)."""
    need = [(n + bt - 1) // bt for n in lengths]
    total = sum(need) + extra
    order = rng.permutation(max(total, 1))
    width = max(1, max(need)) if width is None else width
    t = np.full((len(lengths), width), fill, np.int32)
    at = 0
    for s, n in enumerate(need):
        t[s, :n] = order[at:at + n]
        at += n
    return t, max(total, 1)
