"""Steps over an 8-bit cache for the tests, and what the operators give for them: the append rounding by rounding on the CPU, the attention in float64."""
import math

import numpy as np
import torch

BLOCK, LARGEST, LEAST = 32, 448.0, -100


class Step:
    """Segments [(first position, tokens)] over pages handed out in any order. `tiles`: the listed tiles, by default all of them."""

    def __init__(self, segs, page=64, spare=2, seed=0, device="cuda", slots=None, tiles=None):
        from simplellminference_b200 import _lib
        rng = np.random.default_rng(seed)
        self.segs, self.page, self.device = segs, page, device
        need = [-(-(p + n) // page) for p, n in segs]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        table = np.full((len(segs), max(need + [1])), -1, np.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = order[at:at + n]
            at += n
        self.table_np = table
        lens = np.array([n for _, n in segs])
        start = np.concatenate([[0], np.cumsum(lens)[:-1]])
        slots = list(range(len(segs))) if slots is None else slots
        tiles = [(i, off) for i, (_, n) in enumerate(segs) for off in range(0, n, 32)] if tiles is None else tiles
        self.T = int(lens.sum())
        self.tok_pos_np = np.concatenate([np.arange(p, p + n) for p, n in segs])
        self.arrays = {"tok_slot": np.repeat(slots, lens), "tok_pos": self.tok_pos_np, "seg_start": start, "seg_len": lens, "seg_slot": slots,
                       "seg_pos0": [p for p, _ in segs], "qt_seg": [t[0] for t in tiles], "qt_off": [t[1] for t in tiles], "block_table": table}
        self.dev = {k: torch.tensor(np.asarray(v, dtype=np.int32), device=device) for k, v in self.arrays.items()}
        b = self.b = _lib.SeqBatch()
        b.T, b.nseg, b.n_qtiles, b.max_pages, b.page_len = self.T, len(segs), len(tiles), table.shape[1], page
        for k, v in self.dev.items():
            setattr(b, k, v.data_ptr())


def codes_of(x):
    """fp32 -> e4m3, nearest even (|x| <= 448; NaN stays)."""
    return x.float().to(torch.float8_e4m3fn)


def scale_for(amax):
    """The least power of two, 2^-100 at least, under which amax is at most 448."""
    out = torch.full_like(amax, 2.0 ** LEAST)
    for i, a in enumerate(amax.reshape(-1).tolist()):
        if a > 0:
            m, e = math.frexp(a / LARGEST)                      # double: exact enough to tell both sides of a border apart
            out.view(-1)[i] = 2.0 ** max(e if m > 0.5 else e - 1, LEAST)
    return out


def random_pool(step, kv_heads, width, seed, spread=1.0):
    """A pool with every row written, codes and scales as the append leaves them."""
    g = torch.Generator().manual_seed(seed)
    sub = step.page // BLOCK
    x = torch.randn(step.n_pages, kv_heads, sub, BLOCK, width, generator=g) * torch.exp(spread * torch.randn(step.n_pages, kv_heads, sub, 1, 1, generator=g))
    scale = scale_for(x.abs().amax((-1, -2)))
    return codes_of(x / scale[..., None, None]).view(step.n_pages, kv_heads, step.page, width).to(step.device), scale.to(step.device)


def turned(x, angles, n_freq, layout):
    """[T][heads][width] on the CPU, every product and sum rounded to fp32."""
    x, y = x.clone(), x.clone()
    c, s = angles[:, None, :n_freq, 0], angles[:, None, :n_freq, 1]
    ia = torch.arange(n_freq) * 2 if layout == 0 else torch.arange(n_freq)
    ib = ia + 1 if layout == 0 else ia + n_freq
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ib] * c + x[..., ia] * s
    return y


def append(step, pool, scale, x):
    """What the cache holds after the append of x [T][kv_heads][width] (CPU): codes as uint8, scales."""
    codes, scale, at = pool.cpu().view(torch.uint8).clone(), scale.cpu().clone(), 0
    for i, (p, n) in enumerate(step.segs):
        for lo in range(p // BLOCK * BLOCK, p + n, BLOCK):
            page, row = int(step.table_np[i, lo // step.page]), lo % step.page
            a, b = max(lo, p), min(lo + BLOCK, p + n)
            new = x[at + a - p:at + b - p].transpose(0, 1)
            size = torch.where(torch.isfinite(new), new.abs(), torch.zeros(()))
            sc = scale_for(size.amax((1, 2)))
            if a > lo:
                was = scale[page, :, row // BLOCK]
                sc = torch.maximum(sc, was)
                old = codes[page, :, row:row + a - lo].view(torch.float8_e4m3fn).float() * (was / sc)[:, None, None]
                codes[page, :, row:row + a - lo] = codes_of(old).view(torch.uint8)
            scale[page, :, row // BLOCK] = sc
            new = torch.where(torch.isfinite(new), new, torch.full((), math.nan))
            codes[page, :, row + a - lo:row + b - lo] = codes_of(new / sc[:, None, None]).view(torch.uint8)
        at += n
    return codes, scale


def cache_rows(step, pool, scale, i):
    """Segment i's positions as float64, [kv_heads][positions][width]."""
    p, n = step.segs[i]
    ids = torch.tensor(step.table_np[i, :-(-(p + n) // step.page)].astype(np.int64), device=pool.device)
    x = pool.view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() * scale[ids].double().repeat_interleave(BLOCK, -1)[..., None]
    return x.transpose(0, 1).flatten(1, 2)[:, :p + n]


def attention(step, q, kv, heads, scale, window=0, keep_first=0, softcap=0.0, slopes=None, chunk=0):
    """[T][heads * dv] in float64. A hidden key takes no part, whatever it holds."""
    out, at = [], 0
    for i, (p, n) in enumerate(step.segs):
        (k, v), group = kv[i], heads // kv[i][0].shape[0]
        qs = q[at:at + n].double().view(n, heads, -1).transpose(0, 1)
        s = qs @ k.repeat_interleave(group, 0).mT * scale
        if softcap:
            s = softcap * torch.tanh(s / softcap)
        mine, key = torch.arange(p, p + n, device=q.device)[:, None], torch.arange(p + n, device=q.device)
        if slopes is not None:
            s = s - slopes.double()[:, None, None] * (mine - key)
        seen = key <= mine
        if window:
            seen = seen & ((mine - key < window) | (key < keep_first))
        if chunk:
            seen = seen & (mine // chunk == key // chunk)
        w = torch.softmax(torch.where(seen, s, -math.inf), -1)
        vs = v.repeat_interleave(group, 0)
        bad = ~torch.isfinite(vs)
        o = w @ torch.where(bad, 0.0, vs)
        if bad.any():                                             # NaN where a visible row has it
            o = torch.where((seen.double() @ bad.double()) > 0, math.nan, o)
        out.append(o.transpose(0, 1).flatten(1))
        at += n
    return torch.cat(out)


def off(got, want):
    """Norm of the difference over the norm."""
    return float((got.double() - want).norm() / want.norm())
