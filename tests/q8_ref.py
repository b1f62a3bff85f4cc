"""Plain 64-bit implementation of the 8-bit KV cache and the attention over it, and small helpers to build caches for
the tests.  A cache row is 128 e4m3 codes and one exponent byte x; value = code * 2^(x - 127)."""
import math

import numpy as np
import torch

D = 128
TORCH_DT = {4: torch.float16, 5: torch.bfloat16}


def e4m3_values():
    """The value of every code, NaN for 0x7F and 0xFF."""
    c = np.arange(256)
    s, e, m = np.where(c & 128, -1.0, 1.0), (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v = np.where((e == 15) & (m == 7), np.nan, v)
    return s * v


_VALUES = e4m3_values()
_POSITIVE = _VALUES[:127]                 # codes 0 .. 126, increasing


def quantise(x):
    """x float64 [..., 128] -> (codes uint8, exponent bytes uint8), to nearest with ties to the even code."""
    x = np.asarray(x, np.float64)
    bad = ~np.isfinite(x).all(-1)
    y = np.where(bad[..., None], 0.0, x)
    amax = np.abs(y).max(-1)
    e = np.full(amax.shape, -100)
    for cand in range(120, -101, -1):     # the smallest exponent that holds the row
        e = np.where(amax <= 448.0 * 2.0 ** cand, cand, e)
    z = np.abs(y) * 2.0 ** -e[..., None].astype(np.float64)
    hi = np.clip(np.searchsorted(_POSITIVE, z), 0, 126)
    lo = np.maximum(hi - 1, 0)
    dh, dl = _POSITIVE[hi] - z, z - _POSITIVE[lo]
    code = np.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(y), code + 128, code)
    code = np.where(bad[..., None], 0, code)
    return code.astype(np.uint8), np.where(bad, 255, e + 127).astype(np.uint8)


def values(codes, exps):
    """Codes [..., 128] and exponents -> float64 tensor on the codes' device; exponent 255 reads as NaN."""
    table = torch.from_numpy(_VALUES).to(codes.device)
    scale = torch.exp2(exps.double() - 127.0)
    scale = torch.where(exps == 255, torch.full_like(scale, math.nan), scale)
    return table[codes.long()] * scale[..., None]


def rotate_f32(x, table, neox):
    """x float32 [..., heads, 128], table float32 [..., 64, 2]: fp32 products, one sum or difference each."""
    x = np.asarray(x, np.float32)
    c, s = table[..., None, :, 0].astype(np.float32), table[..., None, :, 1].astype(np.float32)
    out = np.empty_like(x)
    a, b = (x[..., :64], x[..., 64:]) if neox else (x[..., 0::2], x[..., 1::2])
    oa, ob = a * c - b * s, a * s + b * c
    if neox:
        out[..., :64], out[..., 64:] = oa, ob
    else:
        out[..., 0::2], out[..., 1::2] = oa, ob
    return out


def rope_table(n, theta=1e6):
    inv = 1.0 / theta ** (np.arange(0, D, 2) / D)
    ang = np.arange(n)[:, None] * inv
    return np.stack([np.cos(ang), np.sin(ang)], -1).astype(np.float32)


class Cache:
    """An 8-bit cache on the GPU in one of the layouts: 'head' [batch][kvH][cap], 'token' [batch][cap][kvH] or pages
    of `page` positions.  Everything that is not written holds NaN codes and the exponent of a NaN row."""

    def __init__(self, ops, dt, batch, H, kvH, max_pos, layout="head", page=64, neox=False, seed=0, device="cuda", pad=0):
        self.layout, self.page, self.max_pos, self.batch, self.kvH, self.H = layout, page, max_pos, batch, kvH, H
        self.dt, self.dev = dt, device
        self.table = self.table_np = None
        cap = (max_pos + 15) // 16 * 16
        if layout == "paged":
            per = (max_pos + page - 1) // page
            n = batch * per + 3
            perm = np.random.default_rng(seed).permutation(n)[:batch * per].reshape(batch, per).astype(np.int32)
            self.table_np, self.table = perm, torch.from_numpy(perm).to(device)
            lead, cap = n, page
        else:
            lead = batch
        shape = (lead, cap, kvH, D) if layout == "token" else (lead, kvH, cap, D)
        self.k = torch.full(shape, 0x7F, dtype=torch.uint8, device=device)
        self.v = torch.full(shape, 0xFF, dtype=torch.uint8, device=device)
        self.kx = torch.full((lead, kvH, (cap + 15) // 16 * 16 + pad), 255, dtype=torch.uint8, device=device)
        self.vx = torch.full_like(self.kx, 255)
        self.desc = ops.make_desc(dt, batch, H, kvH, 1, cap, layout="token" if layout == "token" else "head", is_neox=neox)
        self.pages = ops.make_pages(self.table, page, kvH * page * D, lead) if layout == "paged" else None
        self.kv = ops.make_kv_q8(self.k, self.v, self.kx, self.vx, max_pos)

    def _slot(self, b, pos):
        if self.layout == "paged":
            return torch.from_numpy(self.table_np[b][pos // self.page]).long().to(self.dev), torch.from_numpy(pos % self.page).to(self.dev)
        p = torch.from_numpy(pos).to(self.dev)
        return torch.full_like(p, b), p

    def rows(self, b, pos):
        """(k, k_exp, v, v_exp) of positions pos (numpy) of sequence b, [n][kvH][...]."""
        o, p = self._slot(b, np.asarray(pos))
        if self.layout == "token":
            return self.k[o, p], self.kx[o, :, p], self.v[o, p], self.vx[o, :, p]
        return self.k[o, :, p], self.kx[o, :, p], self.v[o, :, p], self.vx[o, :, p]

    def put(self, b, pos, kc, kx, vc, vx):
        """Writes rows [n][kvH][...] at positions pos of sequence b."""
        o, p = self._slot(b, np.asarray(pos))
        t = [torch.from_numpy(np.ascontiguousarray(a)).to(self.dev) for a in (kc, kx, vc, vx)]
        if self.layout == "token":
            self.k[o, p], self.v[o, p] = t[0], t[2]
        else:
            self.k[o, :, p], self.v[o, :, p] = t[0], t[2]
        self.kx[o, :, p], self.vx[o, :, p] = t[1], t[3]

    def fill(self, lens, seed=1, spread=0.4):
        """Random rows at positions [0, lens[b]) of every sequence."""
        rng = np.random.default_rng(seed)
        for b, n in enumerate(lens):
            if n == 0:
                continue
            parts = []
            for _ in range(2):
                x = rng.standard_normal((n, self.kvH, D)) * np.exp(spread * rng.standard_normal((n, self.kvH, 1)))
                parts += list(quantise(x))
            self.put(b, np.arange(n), *parts)


def attention(cache, q, b, positions, window, n_sink, u):
    """64-bit attention of rows q [n][H][128] (16-bit tensor) of sequence b at `positions` (list), and the bound of
    its error that the derivation below gives; u: half a step of the output type.

    Bound, per output element o = sum_j w_j v_j with weights w_j = exp(s_j) / sum exp(s):
      - the result is rounded once: u |o|;
      - the weights enter the product as fp16, half a step 2^-11 each: 2^-11 A with A = sum_j w_j |v_j|;
      - a score is an fp32 sum of 128 exact products, computed by tensor cores that may cut instead of round:
        its error is at most 128 * 2^-23 * B with B = max_j sum_d |q_d k_jd| / sqrt(128); two more roundings and the
        hardware exponential (2^-21) join it.  Numerator and denominator carry it: 2 A (128 * 2^-23 B + 2^-20);
      - the two sums over n positions in fp32: 2 A n 2^-23.
    """
    H, kvH = cache.H, cache.kvH
    g = H // kvH
    n_pos = max(positions) + 1 if len(positions) else 0
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    tol = torch.full(q.shape, 2.0 ** -25, dtype=torch.float64, device=q.device)     # subnormal fp16 results
    if n_pos <= 0:
        return out, tol
    span = torch.arange(n_pos, device=q.device)
    pos = torch.tensor(positions, device=q.device)[:, None]
    seen = span <= pos
    if window:
        seen &= (span > pos - window) | (span < n_sink)
    used = seen.any(0)
    kc, kx, vc, vx = cache.rows(b, span[used].cpu().numpy())
    seen = seen[:, used]
    k, v = values(kc, kx), values(vc, vx)
    poison = torch.isnan(k).any(-1) | torch.isnan(v).any(-1)                        # [n][kvH]
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    alive = pos[:, 0] >= 0
    for h in range(H):
        kh, vh = k[:, h // g], v[:, h // g]
        qh = q[:, h].double()
        s = (qh @ kh.T) / math.sqrt(D)
        B = ((qh.abs() @ kh.abs().T) / math.sqrt(D)).masked_fill(~seen, 0.0).amax(-1, keepdim=True)
        w = torch.softmax(s.masked_fill(~seen, -math.inf), -1)
        w = torch.where(alive[:, None], w, torch.zeros_like(w))
        o, A = w @ vh, w @ vh.abs()
        hit = (seen & poison[None, :, h // g]).any(-1)
        o[hit] = math.nan
        out[:, h] = o
        tol[:, h] += u * o.abs() + A * (2.0 ** -11 + 2 * (128 * 2.0 ** -23 * B + 2.0 ** -20) + 2 * seen.sum(-1, keepdim=True) * 2.0 ** -23)
    return out, tol


def assert_close(got, want, tol, what=""):
    got = got.double()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), "%s: NaN in other places" % what
    off = ((got - want).abs() - tol).masked_fill(nan, -1.0)
    worst = int(off.argmax())
    assert float(off.max()) <= 0, "%s: off by %.3e where %.3e is allowed (element %d of %s, want %.5e)" % (
        what, float((got - want).abs().flatten()[worst]), float(tol.flatten()[worst]), worst, tuple(want.shape), float(want.flatten()[worst]))


def half_step(dt):
    return torch.finfo(TORCH_DT[dt]).eps / 2
