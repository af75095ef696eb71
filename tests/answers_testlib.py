"""Steps whose requests share their first positions, and what the operators of many answers to one prompt give, in 64 bits."""
import math

import numpy as np
import torch


class SharedStep:
    """groups: [(shared positions, [(own positions, new tokens)])]. Pages are handed out in any order; a page that holds shared and own positions is every request's own copy."""

    def __init__(self, groups, heads, kv_heads, dk, dv=None, page=64, dtype=torch.bfloat16, seed=0, tiles=None, spread=0.4, tail=0, extra=2):
        from simplellminference_b200 import _lib
        dv = dv or dk
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.groups, self.page, self.heads, self.kv_heads, self.dk, self.dv, self.dtype = groups, page, heads, kv_heads, dk, dv, dtype
        self.segs = [(shared, shared + p, n) for shared, members in groups for p, n in members]
        rows, used = [], 0
        for shared, members in groups:
            common = list(range(used, used + shared // page))
            used += len(common)
            for p, n in members:
                need = -(-(shared + p + n) // page) - len(common)
                rows.append(common + list(range(used, used + need)))
                used += need
        self.n_pages = used + extra
        order = rng.permutation(self.n_pages)
        table = np.full((len(rows), max(len(r) for r in rows) + 1), -1, np.int32)
        for i, r in enumerate(rows):
            table[i, :len(r)] = order[r]
        self.table_np = table
        lens = np.array([n for _, _, n in self.segs])
        start = np.concatenate([[0], np.cumsum(lens)[:-1]])
        self.n_tokens = int(lens.sum())
        tiles = [(i, off) for i, (_, _, n) in enumerate(self.segs) for off in range(0, n, 32)] if tiles is None else tiles
        pos = np.concatenate([np.arange(p, p + n) for _, p, n in self.segs])
        starts = np.concatenate([[0], np.cumsum([len(m) for _, m in groups])])
        arrays = {"tok_slot": np.repeat(np.arange(len(lens)), lens), "tok_pos": pos, "seg_start": start, "seg_len": lens, "seg_slot": np.arange(len(lens)), "seg_pos0": [p for _, p, _ in self.segs],
                  "qt_seg": [t[0] for t in tiles], "qt_off": [t[1] for t in tiles], "block_table": table, "seg_tile0": np.zeros(len(lens))}
        self.dev = {k: torch.tensor(np.asarray(v, dtype=np.int32), device="cuda") for k, v in arrays.items()}
        self.group_start = torch.tensor(starts, dtype=torch.int32, device="cuda")
        self.group_len = torch.tensor([n for n, _ in groups], dtype=torch.int32, device="cuda")
        b = self.b = _lib.SeqBatch()
        b.T, b.nseg, b.n_qtiles, b.max_pages, b.page_len = self.n_tokens, len(lens), len(tiles), table.shape[1], page
        for k, v in self.dev.items():
            setattr(b, k, v.data_ptr())
        gain = torch.exp(spread * torch.randn(kv_heads, 1, dk, generator=g))
        self.k = (gain * torch.randn(self.n_pages, kv_heads, page, dk, generator=g)).to(dtype)
        self.v = torch.randn(self.n_pages, kv_heads, page, dv, generator=g).to(dtype)
        i = 0
        for shared, members in groups:
            first, whole, part = i, shared // page, shared % page
            for _ in members:
                if part and i > first:
                    for pool in (self.k, self.v):
                        pool[table[i, whole], :, :part] = pool[table[first, whole], :, :part]
                i += 1
        self.q = torch.randn(self.n_tokens + tail, heads * dk, generator=g)
        self.pos = pos

    def want(self, window=0, keep=0, cap=0.0, slopes=None, scale=None):
        """In float64, every request by itself over its own pages; positions that a table does not have are hidden."""
        scale = scale or self.dk ** -0.5
        per, out, at = self.heads // self.kv_heads, [], 0
        q = (self.q.to(self.dtype) if self.dtype == torch.bfloat16 else self.q).double()
        for i, (_, p, n) in enumerate(self.segs):
            ids = torch.tensor(self.table_np[i, :-(-(p + n) // self.page)], dtype=torch.long)
            have = ((ids >= 0) & (ids < self.n_pages)).repeat_interleave(self.page)[:p + n]
            k, v = (pool[ids.clamp(0, self.n_pages - 1)].double().transpose(0, 1).flatten(1, 2)[:, :p + n].repeat_interleave(per, 0) for pool in (self.k, self.v))
            z = q[at:at + n].view(n, self.heads, self.dk).transpose(0, 1) @ k.mT * scale
            if cap:
                z = cap * torch.tanh(z / cap)
            back = torch.arange(p, p + n)[:, None] - torch.arange(p + n)
            if slopes is not None:
                z = z - slopes.double()[:, None, None] * back
            seen = (back >= 0) & have
            if window:
                seen &= (back < window) | (torch.arange(p + n) < keep)
            w = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
            w = torch.where(seen.any(-1)[None, :, None], w, 0.0)
            v = torch.where(seen.any(0)[None, :, None], v, 0.0)                # a row that no token sees may hold anything
            if torch.isfinite(v).all():
                o = w @ v
            else:                                                             # only the rows a token sees count for it
                o = torch.stack([torch.where(seen[t][None, :, None], w[:, t, :, None] * v, 0.0).sum(1) for t in range(n)], 1)
            out.append(o.transpose(0, 1).flatten(1))
            at += n
        return torch.cat(out)

    def run(self, out=True, out16=False, ws=None, stream=None, scale=None, ldq=None, ldo=None, fill=7.0, slopes=None, groups=None, **opts):
        """(fp32 rows or None, bf16 rows or None); rows of no listed token keep `fill`."""
        from simplellminference_b200.config import BF16, F32
        from simplellminference_b200.seqops import Ops
        ops = Ops(BF16 if self.dtype == torch.bfloat16 else F32)
        rows = self.q.shape[0]
        ldq, ldo = ldq or self.heads * self.dk, ldo or self.heads * self.dv
        q = torch.full((rows, ldq), math.nan)
        q[:, :self.heads * self.dk] = self.q
        q, k, v = q.cuda(), self.k.cuda(), self.v.cuda()
        o = torch.full((rows, ldo), fill, device="cuda") if out else None
        o16 = torch.full((rows, self.heads * self.dv), fill, device="cuda", dtype=torch.bfloat16) if out16 else None
        start, length = groups or (self.group_start, self.group_len)
        need = ops.attention_shared_ws_bytes(self.b, length.numel(), self.heads, self.kv_heads, self.dk, self.dv)
        ws = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda") if ws is None else ws          # NaN in every float
        if slopes is not None:
            slopes = slopes.cuda()
        st = stream or torch.cuda.current_stream().cuda_stream
        ops.attention_shared(self.b, length.numel(), start, length, q.data_ptr(), ldq, self.heads, self.kv_heads, self.dk, self.dv, scale or self.dk ** -0.5, k, v, self.n_pages, ws, st, out=o,
                             ldo=ldo, out16=o16, opts=ops.attention_options(slopes=slopes, **opts) if opts or slopes is not None else None)
        torch.cuda.synchronize()
        ops._ck(ops.lib.sllm_status())
        return (None if o is None else o.cpu()), (None if o16 is None else o16.cpu())


def codes_of(x):
    """Codes and scales of rows, both quotients rounded to fp32 (numpy divides as IEEE says)."""
    x = x.float().numpy()
    scale = np.maximum(np.abs(x).max(-1) / np.float32(127), np.float32(2.0 ** -126))
    return torch.from_numpy(np.rint(x / scale[:, None]).astype(np.int8)), torch.from_numpy(scale)


def logprobs_of(x, token, top):
    """(log probability, rank, entropy, alternatives, their log probabilities) of rows of logits in float64; rows hold finite numbers and -infinity."""
    x = x.double()
    x = x - x.amax(-1, keepdim=True)                                          # (beside numbers of 1e38 the logarithm of the sum would be lost)
    logp = x - torch.logsumexp(x, -1, keepdim=True)
    p = logp.exp()
    entropy = -torch.special.xlogy(p, p).sum(-1)
    order = x.sort(dim=-1, descending=True, stable=True).indices
    rank = (order == token[:, None]).double().argmax(-1)
    return logp.gather(1, token[:, None])[:, 0], rank, entropy, order[:, :top], logp.gather(1, order[:, :top])
