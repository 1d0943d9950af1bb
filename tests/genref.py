"""Plain 64-bit implementations of the generation operators, and device buffers of any element type."""
import math

import numpy as np
import torch

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CODE = {"fp32": 0, "bf16": 1, "fp16": 2}


class Buffers:
    """Registry buffers of one test, freed at its end; CPU torch tensors go in and out bit for bit."""

    def __init__(self, be):
        self.be, self.ids = be, []

    def new(self, floats):
        i = self.be.bufferAlloc(max(1, int(floats)))
        self.ids.append(i)
        return i

    def put(self, t, pad=0):
        raw = t.contiguous().reshape(-1).view(torch.uint8).numpy().tobytes()
        raw += b"\0" * (-len(raw) % 4)
        a = np.frombuffer(raw, np.float32)
        i = self.new(a.size + pad)
        if a.size:
            self.be.bufferUpload(i, a)
        return i

    def write(self, i, t):
        self.be.bufferUpload(i, np.frombuffer(t.contiguous().reshape(-1).view(torch.uint8).numpy().tobytes(), np.float32))

    def get(self, i, shape, dtype):
        n = int(np.prod(shape))
        size = torch.empty(0, dtype=dtype).element_size()
        a = self.be.bufferDownload(i, max(1, (n * size + 3) // 4))
        return torch.frombuffer(bytearray(a.tobytes()), dtype=dtype)[:n].reshape(tuple(shape)).clone()

    def close(self):
        for i in self.ids:
            self.be.bufferFree(i)
        self.ids = []


def rates(rot, base=10000.0, scaling=0, factor=1.0, original=1, slow=1.0, fast=32.0):
    """Radians a position of each pair, and the magnitude."""
    out = []
    if scaling == 2 and rot > 2:
        base = base * factor ** (rot / (rot - 2.0))
    for i in range(rot // 2):
        w = base ** (-2.0 * i / rot)
        if scaling == 1:
            w /= factor
        if scaling == 3:
            keep = min(1.0, max(0.0, (original * w / (2 * math.pi) - slow) / (fast - slow)))
            w = w * keep + w / factor * (1 - keep)
        out.append(w)
    return out, (0.1 * math.log(factor) + 1.0 if scaling == 3 else 1.0)


def rotate(x, pos, rot, interleaved, plan, sign=1.0):
    """x [rows, heads, dim] in fp64 turned at pos [rows]; and m (|a| + |b|) of each element's pair, for tolerances."""
    x = x.double()
    y, size = x.clone(), torch.zeros_like(x)
    w, m = plan
    for i in range(rot // 2):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)
        t = pos.double() * w[i]
        c, s = (m * torch.cos(t))[:, None], (sign * m * torch.sin(t))[:, None]
        y[..., a] = x[..., a] * c - x[..., b] * s
        y[..., b] = x[..., a] * s + x[..., b] * c
        size[..., a] = size[..., b] = m * (x[..., a].abs() + x[..., b].abs())
    return y, size


# Angle: the turn's fraction is rounded to fp32 (2^-26 turns = 9.4e-8 radians), its sine and cosine are off by
# 2 units of 2^-24 relative at most each (1.2e-7), the magnitude, two products and the sum round once each
# (4 * 6e-8): under 5e-7 of m (|a| + |b|).
ROTATION = 5e-7
# The 64-bit reference's own angle: pos * w rounds once (2^-53 of it) and w's power by a few 2^-53.
def far(pos):
    return 8 * 2.0 ** -53 * float(pos.abs().max() if pos.numel() else 0)


def half_step(y, dtype):
    """Half a step of dtype at y: subnormals keep the smallest normal's step."""
    f = torch.finfo(dtype)
    return torch.clamp(y.double().abs(), min=f.tiny) * (f.eps / 2)


def attend(q, k, v, start, length, pages, prefix_pages, prefix, scale, page):
    """fp64 attention; returns out, and the tolerance's sums: sum_i p_i |v_i|, max score error's base, keys, l."""
    rows, hq, d = q.shape
    hk = k.shape[1]
    g = hq // hk
    out = torch.full((rows, hq, d), float("nan"), dtype=torch.float64)
    mass, spread, small = torch.zeros_like(out), torch.zeros((rows, hq, 1), dtype=torch.float64), torch.zeros_like(out)
    for b in range(len(length)):
        n = start[b + 1] - start[b]
        for j in range(n):
            lim = max(0, length[b] - n + j + 1)
            where = [(prefix_pages[i // page], i % page) for i in range(prefix)]
            where += [(pages[b][i // page], i % page) for i in range(lim)]
            t = start[b] + j
            if not where:
                out[t] = 0
                continue
            pg, sl = torch.tensor(where).T
            for h in range(hk):
                kk, vv = k[pg, h, sl].double(), v[pg, h, sl].double()
                qq = q[t, h * g:(h + 1) * g].double()
                s = qq @ kk.T * scale
                p = torch.exp(s - s.max(1, keepdim=True).values)
                l = p.sum(1, keepdim=True)
                hs = slice(h * g, (h + 1) * g)
                out[t, hs] = p @ vv / l
                mass[t, hs] = p @ vv.abs() / l
                spread[t, hs, 0] = (qq.abs() @ kk.abs().T).max(1).values * abs(scale)
                small[t, hs] = len(where) * vv.abs().max() / l
    return out, mass, spread, small


def attend_tolerance(ref, d, dtype):
    """Weights are rounded to the type (half a step each, 2^-25 absolute below fp16's normals), scores are fp32 sums
    of d exact products (d 2^-24 of sum |q k|, twice for the maximum's own error), exponentials and the joins' sums 2^-20 together, the result rounds once."""
    out, mass, spread, small = ref
    f = torch.finfo(dtype)
    score = 2 * d * 2.0 ** -24 * spread
    t = mass * (f.eps / 2 + 2 * score + 2.0 ** -20) * 1.01
    if dtype == torch.float16:
        t = t + small * 2.0 ** -25
    return t + half_step(out, dtype)


def verify(p, q, draft, u, start, vocab):
    """tokens, accepted by the definition, sequence by sequence, in fp64 (q None: certain drafts)."""
    tokens, accepted = {}, []
    for b in range(len(start) - 1):
        n = start[b + 1] - start[b]
        if n == 0:
            accepted.append(0)
            continue
        a, k = 0, n - 1
        while a < k:
            r = start[b] + a
            d = int(draft[r])
            if not 0 <= d < vocab:
                break
            if not float(u[r]) * (1.0 if q is None else float(q[r, d])) < float(p[r, d]):
                break
            a += 1
        r = start[b] + a
        w = np.asarray(p[r, :vocab], np.float64).copy()
        if a < k:
            if q is None:
                if 0 <= int(draft[r]) < vocab:
                    w[int(draft[r])] = 0.0
            else:
                w = w - np.asarray(q[r, :vocab], np.float64)
        w = np.where(w > 0, w, 0.0)
        if not w.sum() > 0:
            w = np.asarray(p[r, :vocab], np.float64)
            w = np.where(w > 0, w, 0.0)
        c = np.cumsum(w)
        token = 0
        if c[-1] > 0:
            hit = np.nonzero((c > float(u[start[b] + k]) * c[-1]) & (w > 0))[0]
            token = int(hit[0]) if hit.size else int(np.nonzero(w > 0)[0][-1])
        for j in range(n):
            tokens[start[b] + j] = int(draft[start[b] + j]) if j < a else token if j == a else -1
        accepted.append(a)
    return tokens, accepted
