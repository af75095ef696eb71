"""Many answers to one prompt, as cases that can be timed: attention of requests that share the first positions of their cache, products with weights and activations in 8-bit
integers, and the log probabilities by which answers are ranked. `listed` names one case per use, `draw` gives more of the same ranges.

Operators and their ranges:
  shared     Ops.attention_shared: groups of 1 .. 64 requests whose first 0 .. 8192 positions are the same, single tokens and portions of up to 311 behind up to 2000 positions of their own; heads of 64
             and 128, groups of 1 .. 8 query heads, caches in bf16 and fp32, windows, capped scores
  quantise   Ops.quantise_rows: 1 .. 16384 rows of 64 .. 16384 values in fp32 or bf16 to codes of 8 bits and a scale a row
  product    Ops.quantise_rows and Ops.linear8: 1 .. 2048 tokens, matrices of 64 .. 16384 rows and columns with a scale a row, with and without a bias
  logprob    Ops.token_logprobs: 1 .. 2048 rows of 500 .. 128256 logits: a given token's log probability and rank, the entropy, the 0 .. 20 most likely tokens

The scale of a row is max |x| / 127 (2^-126 at least), its codes are x / scale, rounded to fp32 and then to the nearest whole number (even ones where two are as near). With a cache in bf16
the queries are rounded to bf16.
"""
import math

import torch

own = False
DEV = "cuda"
LEAST = 2.0 ** -126


def listed():
    return [
        # four answers of a small model in fp32 throughout
        {"name": "shared_4_answers_f32", "op": "shared", "groups": "1500|" + owns(4, 90, 3, 1), "heads": 16, "kv_heads": 4, "dim": 64, "page": 32, "cache": "f32", "out": "f32", "window": 0, "keep": 0,
         "cap": 0.0},
        # eight answers to one prompt with TinyLlama's heads
        {"name": "shared_8_answers", "op": "shared", "groups": "2000|" + owns(8, 300, 5, 1), "heads": 32, "kv_heads": 4, "dim": 64, "page": 32, "cache": "bf16", "out": "f32", "window": 0, "keep": 0,
         "cap": 0.0},
        # a full batch of answers to a long prompt, Llama-3-8B-shaped heads
        {"name": "shared_64_answers", "op": "shared", "groups": "8000|" + owns(64, 400, 7, 1), "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "cache": "bf16", "out": "bf16", "window": 0, "keep": 0,
         "cap": 0.0},
        # a step of a server: questions taken in behind a common prompt, answers to another one, requests that share nothing
        {"name": "shared_mixed_step", "op": "shared", "groups": "4000|0+311,0+37,0+256,90+1,700+1;1031|" + owns(16, 500, 3, 1) + ";0|1500+1;0|311+1", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "cache": "bf16", "out": "f32", "window": 0, "keep": 0, "cap": 30.0},
        # the rows of one decoded token, the smallest call
        {"name": "quantise_1_token", "op": "quantise", "rows": 1, "k": 4096, "x": "f32"},
        # a matrix of a model taken over from bf16
        {"name": "quantise_matrix", "op": "quantise", "rows": 14336, "k": 4096, "x": "bf16"},
        # one token through a square projection
        {"name": "product_1_token", "op": "product", "T": 1, "n": 4096, "k": 4096, "x": "f32", "bias": False},
        # a full decoding batch through a wide projection: the weights are what it reads
        {"name": "product_64_tokens", "op": "product", "T": 64, "n": 14336, "k": 4096, "x": "f32", "bias": True},
        # prompts through the projection back
        {"name": "product_prompts", "op": "product", "T": 2000, "n": 4096, "k": 14336, "x": "bf16", "bias": False},
        # one drawn token, a vocabulary of 32000
        {"name": "logprob_1_row", "op": "logprob", "rows": 1, "n": 32000, "top": 5, "values": "f32"},
        # a full batch of drawn tokens over the vocabulary of Llama-3, with alternatives
        {"name": "logprob_64_rows", "op": "logprob", "rows": 64, "n": 128256, "top": 20, "values": "f32"},
        # a prompt's own tokens, logits as a product in bf16 leaves them: many are equal
        {"name": "logprob_prompt", "op": "logprob", "rows": 1000, "n": 128256, "top": 1, "values": "bf16"},
    ]


def owns(n, longest, step, new):
    """`n` requests of `new` tokens behind 0 .. longest - 1 positions of their own, as the text a case carries."""
    return ",".join("%d+%d" % ((i * i * step * 131 + i * 977) % longest, new) for i in range(n))


def split(case):
    """[(shared positions, [(own positions, new tokens)])]"""
    return [(int(g.split("|")[0]), [tuple(int(x) for x in s.split("+")) for s in g.split("|")[1].split(",")]) for g in case["groups"].split(";")]


def _joined(groups):
    return ";".join("%d|%s" % (n, ",".join("%d+%d" % s for s in segs)) for n, segs in groups)


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["shared", "shared", "product", "logprob", "quantise"])
    if op == "logprob":
        rows = _spread(rng, 1, 2048)
        return {"op": op, "rows": rows, "n": _spread(rng, 500, min(128256, max(501, 120_000_000 // rows))), "top": rng.choice([0, 1, 5, rng.randint(2, 20), 20]), "values": rng.choice(["f32", "bf16"])}
    if op == "quantise":
        k = _spread(rng, 64, 16384)
        return {"op": op, "rows": _spread(rng, 1, min(16384, max(2, 58_000_000 // k))), "k": k, "x": rng.choice(["f32", "bf16"])}
    if op == "product":
        case = {"op": op, "T": _spread(rng, 1, 2048), "n": _spread(rng, 64, 16384), "k": _spread(rng, 64, 16384), "x": rng.choice(["f32", "bf16"]), "bias": rng.random() < 0.5}
        while work(case)["flops"] > 230e9:
            big = max(("T", "n", "k"), key=lambda name: case[name])
            case[big] = case[big] // 2
        return case
    kv_heads, cache = rng.choice([1, 2, 4, 8]), rng.choice(["bf16", "bf16", "bf16", "f32"])
    groups = []
    for _ in range(rng.choice([1, 1, 2, 3])):
        members = _spread(rng, 1, 64 if cache == "bf16" else 16)
        portions = rng.random() < 0.4
        segs = [(rng.choice([0, _spread(rng, 1, 2000)]), _spread(rng, 2, 311) if portions and rng.random() < 0.3 else 1) for _ in range(members)]
        groups.append((rng.choice([0, _spread(rng, 1, 8192), _spread(rng, 1, 8192), _spread(rng, 1000, 8192)]), segs))
    window = rng.choice([0, 0, _spread(rng, 40, 4000)])
    case = {"op": op, "groups": "", "heads": kv_heads * rng.choice([1, 2, 3, 4, 8]), "kv_heads": kv_heads, "dim": rng.choice([64, 128]), "page": rng.choice([32, 64, 128]), "cache": cache,
            "out": rng.choice(["f32", "bf16"]), "window": window, "keep": rng.choice([0, 4]) if window else 0, "cap": rng.choice([0.0, 0.0, 30.0])}
    while True:
        case["groups"] = _joined(groups)
        w = work(case)
        if w["flops"] <= (16e9 if cache == "bf16" else 2e9) and w["bytes"] <= 300e6 and all(len(s) * max(p + n for p, n in s) * max(max(n for _, n in s) * case["heads"], kv_heads * case["dim"]) < 5e8
                                                                                           for _, s in groups):
            return case
        i = max(range(len(groups)), key=lambda j: sum(n for _, n in groups[j][1]) * (groups[j][0] + 500))       # the dearest group: its longest member goes, or its prefix is halved
        shared, segs = groups[i]
        if len(segs) > 1:
            segs.remove(max(segs, key=lambda s: (s[1], s[0])))
        groups[i] = (shared if len(segs) > 4 else shared * 3 // 4, segs if len(segs) > 1 else [(segs[0][0] // 2, max(1, segs[0][1] // 2))])


# ---------------------------------------------------------------------------------------------------------------------------
# What a program has in hand before the call
# ---------------------------------------------------------------------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    state = {"shared": _step, "quantise": _rows, "product": _matrix, "logprob": _logits}[case["op"]](case, g)
    state["case"] = case
    if own:
        _plan(state)
    return state


def _step(case, g):
    """The index arrays of a step whose groups share the pages of their first positions; a page that holds shared and own positions is every request's own copy."""
    groups, page, heads, kv_heads, dim = split(case), case["page"], case["heads"], case["kv_heads"], case["dim"]
    segs = [(shared, shared + p, n) for shared, members in groups for p, n in members]
    widest = max(-(-(p + n) // page) for _, p, n in segs)
    table, copies, used = torch.full((len(segs), widest), -1, dtype=torch.int32), [], 0
    i = 0
    for shared, members in groups:
        whole = shared // page
        common = list(range(used, used + whole))
        used += whole
        first = i
        for p, n in members:
            need = -(-(shared + p + n) // page) - whole
            table[i, :whole + need] = torch.tensor(common + list(range(used, used + need)), dtype=torch.int32)
            used += need
            if shared % page and i > first:
                copies.append((first, i, whole, shared % page))
            i += 1
    pages = used + 2
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    table = torch.where(table.to(DEV) >= 0, order[table.to(DEV).long().clamp_min(0)], -1).contiguous()
    lens = torch.tensor([n for _, _, n in segs])
    first = torch.cumsum(lens, 0) - lens
    slot = torch.repeat_interleave(torch.arange(len(segs)), lens)
    pos = torch.arange(int(lens.sum())) - first[slot] + torch.tensor([p for _, p, _ in segs])[slot]
    tiles = [(i, off) for i, (_, _, n) in enumerate(segs) for off in range(0, n, 32)]
    tiles.sort(key=lambda t: -(segs[t[0]][1] + t[1]))
    counts = [-(-n // 32) for _, _, n in segs]
    starts = torch.cumsum(torch.tensor([0] + [len(m) for _, m in groups]), 0).tolist()
    st = {"groups": groups, "segs": segs, "table": table, "tok_slot": _ints(slot.tolist()), "tok_pos": _ints(pos.tolist()), "seg_start": _ints(first.tolist()), "seg_len": _ints(lens.tolist()),
          "seg_slot": _ints(list(range(len(segs)))), "seg_pos0": _ints([p for _, p, _ in segs]), "qt_seg": _ints([t[0] for t in tiles]), "qt_off": _ints([t[1] for t in tiles]),
          "seg_tile0": _ints([sum(counts[:i]) for i in range(len(segs))]), "starts": starts, "group_start": _ints(starts), "group_len": _ints([n for n, _ in groups])}
    dtype = torch.bfloat16 if case["cache"] == "bf16" else torch.float32
    for name in ("k", "v"):
        # keys have channels that are larger than others, all the time; values do not
        gain = torch.exp(0.5 * torch.randn(kv_heads, 1, dim, generator=g, device=DEV)) if name == "k" else 1.0
        pool = (gain * torch.randn(pages, kv_heads, page, dim, generator=g, device=DEV)).to(dtype)
        for a, b, at, rows in copies:
            pool[table[b, at].long(), :, :rows] = pool[table[a, at].long(), :, :rows]
        st[name + "_pool"] = pool
    T = pos.numel()
    st["q"] = torch.randn(T, heads * dim, generator=g, device=DEV)
    st["out"] = torch.empty(T, heads * dim, device=DEV, dtype=torch.float32 if case["out"] == "f32" else torch.bfloat16)
    return st


def _activations(rows, k, kind, g):
    """Rows of different sizes, with a few channels that are larger than the others."""
    x = torch.randn(rows, k, generator=g, device=DEV) * torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=DEV))
    x[:, torch.randint(0, k, (max(1, k // 500),), generator=g, device=DEV)] *= 8.0
    return x if kind == "f32" else x.bfloat16()


def _wide(k):
    return -(-k // 16) * 16                                               # bytes from one row of codes to the next


def _rows(case, g):
    rows, k = case["rows"], case["k"]
    return {"x": _activations(rows, k, case["x"], g), "codes": torch.zeros(rows, _wide(k), dtype=torch.int8, device=DEV), "scale": torch.zeros(rows, device=DEV)}


def _matrix(case, g):
    T, n, k = case["T"], case["n"], case["k"]
    w = torch.zeros(n, _wide(k), dtype=torch.int8, device=DEV)
    w[:, :k] = (36.0 * torch.randn(n, k, generator=g, device=DEV)).round_().clamp_(-127, 127).to(torch.int8)
    return {"x": _activations(T, k, case["x"], g), "codes": torch.zeros(T, _wide(k), dtype=torch.int8, device=DEV), "scale": torch.zeros(T, device=DEV), "w": w,
            "w_scale": (0.5 + torch.rand(n, generator=g, device=DEV)) / (36.0 * math.sqrt(k)), "bias": torch.randn(n, generator=g, device=DEV) if case["bias"] else None,
            "out": torch.empty(T, n, device=DEV)}


def _logits(case, g):
    """Logits as a language model leaves them: a bell of unlikely tokens, some likely ones, a few banned; and a token for every row, mostly a likely one."""
    rows, n, top = case["rows"], case["n"], case["top"]
    x = 2.5 * torch.randn(rows, n, generator=g, device=DEV)
    likely = torch.randint(0, n, (rows, 24), generator=g, device=DEV)
    x.scatter_reduce_(1, likely, 9.0 + 3.0 * torch.randn(rows, 24, generator=g, device=DEV), "amax")      # the same place twice: the larger, whichever comes first
    if case["values"] == "bf16":
        x = x.bfloat16().float()
    token = torch.where(torch.arange(rows, device=DEV) % 4 == 3, torch.randint(0, n, (rows,), generator=g, device=DEV), likely[:, 0])
    banned = torch.randint(0, n, (rows, 8), generator=g, device=DEV)
    x.scatter_(1, torch.where(banned == token[:, None], (banned + 1) % n, banned), -math.inf)             # not the token itself
    state = {"logits": x, "token": token.to(torch.int32), "logprob": torch.empty(rows, device=DEV), "entropy": torch.empty(rows, device=DEV),
             "rank": torch.empty(rows, dtype=torch.int32, device=DEV)}
    if top:
        state |= {"top_idx": torch.empty(rows, top, dtype=torch.int32, device=DEV), "top_logprob": torch.empty(rows, top, device=DEV)}
    return state


def _plan(state):
    """What such a program keeps from call to call: the launchers, the step's description, the workspace of the attention."""
    from simplellminference_b200 import _lib
    from simplellminference_b200.config import BF16, F32
    from simplellminference_b200.seqops import Ops
    case = state["case"]
    ops = state["ops"] = Ops(F32 if case.get("cache") == "f32" else BF16)
    if case["op"] != "shared":
        return
    b = _lib.SeqBatch()
    b.T, b.nseg, b.n_qtiles = state["tok_pos"].numel(), len(state["segs"]), state["qt_seg"].numel()
    for name in ("tok_slot", "tok_pos", "seg_start", "seg_len", "seg_slot", "seg_pos0", "qt_seg", "qt_off", "seg_tile0"):
        setattr(b, name, state[name].data_ptr())
    b.block_table, b.max_pages, b.page_len = state["table"].data_ptr(), state["table"].shape[1], case["page"]
    state["batch"] = b
    need = ops.attention_shared_ws_bytes(b, len(state["groups"]), case["heads"], case["kv_heads"], case["dim"], case["dim"])
    state["ws"] = torch.zeros(need, dtype=torch.uint8, device=DEV)
    state["opts"] = ops.attention_options(window=case["window"], keep_first=case["keep"], softcap=case["cap"]) if case["window"] or case["cap"] else None


# ---------------------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------------------
def run(state):
    return {"shared": _attend, "quantise": _quantise, "product": _product, "logprob": _logprob}[state["case"]["op"]](state)


def _attend(s):
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if own:
        f32 = case["out"] == "f32"
        s["ops"].attention_shared(s["batch"], len(s["groups"]), s["group_start"], s["group_len"], s["q"].data_ptr(), heads * dim, heads, kv_heads, dim, dim, dim ** -0.5, s["k_pool"], s["v_pool"], s["k_pool"].shape[0],
                                  s["ws"], torch.cuda.current_stream().cuda_stream, out=s["out"] if f32 else None, ldo=heads * dim, out16=None if f32 else s["out"], opts=s["opts"])
        return s["out"]
    q = s["q"] if case["cache"] == "f32" else s["q"].bfloat16().float()
    per = heads // kv_heads
    at = 0
    for gi, (shared, members) in enumerate(s["groups"]):
        i0, i1 = s["starts"][gi], s["starts"][gi + 1]
        count = sum(n for _, n in members)
        mine = q[at:at + count].view(count, kv_heads, per, dim)
        pos = s["tok_pos"][at:at + count].long()
        # the shared positions once for all tokens of the group: [head][token][query head of it][position]
        k, v = (_cached(s, name, i0, 1, 0, shared)[0] for name in ("k", "v"))
        before = torch.einsum("tgpd,gjd->gtpj", mine, k)
        before = _scores(before, case, pos[:, None] - torch.arange(shared, device=DEV), shared)
        # the positions behind them: a padded batch
        seg = s["tok_slot"][at:at + count].long() - i0
        own_rows = max(p + n for p, n in members)
        ks, vs = (_cached(s, name, i0, i1 - i0, shared, shared + own_rows) for name in ("k", "v"))
        rows = max(n for _, n in members)
        where = (seg, pos - s["seg_pos0"][i0:i1].long()[seg])
        padded = torch.zeros(i1 - i0, rows, kv_heads, per, dim, device=DEV)
        padded[where] = mine
        behind = torch.einsum("srgpd,sgjd->srgpj", padded, ks)[where].transpose(0, 1)
        behind = _scores(behind, case, pos[:, None] - shared - torch.arange(own_rows, device=DEV), shared, shared)
        score = torch.cat([before, behind], -1)
        score -= score.amax(-1, keepdim=True)
        weight = score.exp_()
        weight /= weight.sum(-1, keepdim=True)
        out = torch.einsum("gtpj,gjd->tgpd", weight[..., :shared], v)
        padded = torch.zeros(i1 - i0, rows, kv_heads, per, own_rows, device=DEV)
        padded[where] = weight[..., shared:].transpose(0, 1)
        out += torch.einsum("srgpj,sgjd->srgpd", padded, vs)[where]
        s["out"][at:at + count] = out.reshape(count, heads * dim)
        at += count
    return s["out"]


def _scores(score, case, back, shared, first=0):
    """Scaled, capped, and hidden where the key is behind the token or the window: [head][token][query head of it][position]; `back` [token][position]."""
    score = score * case["dim"] ** -0.5
    if case["cap"]:
        score = case["cap"] * torch.tanh(score / case["cap"])
    seen = back >= 0
    if case["window"]:
        key = first + torch.arange(back.shape[1], device=DEV)
        seen &= (back < case["window"]) | (key < case["keep"])
    return score.masked_fill(~seen[None, :, None], -math.inf)


def _cached(s, name, first, count, lo, hi):
    """Positions lo .. hi - 1 of `count` segments in fp32, zeros where a sequence has none: [segment][head][position][column]."""
    pool, page = s[name + "_pool"], s["case"]["page"]
    pages = s["table"].long()[first:first + count, lo // page:-(-hi // page)]
    x = pool[pages.clamp_min(0)].float().transpose(1, 2).flatten(2, 3)
    have = s["seg_pos0"][first:first + count].long() + s["seg_len"][first:first + count].long()
    at = lo // page * page + torch.arange(x.shape[2], device=DEV)
    x = x * (at < have[:, None])[:, None, :, None]
    return torch.nn.functional.pad(x, (0, 0, 0, max(0, hi - lo // page * page - x.shape[2])))[:, :, lo - lo // page * page:][:, :, :hi - lo]


def _codes(x):
    x = x.float()
    scale = (x.abs().amax(-1) / torch.full((), 127.0, device=DEV)).clamp_min(LEAST)           # (a Python number would be multiplied by as its inverse, another rounding)
    return torch.round(x / scale[:, None]), scale


def _quantise(s):
    x = s["x"]
    rows, k = x.shape
    if own:
        s["ops"].quantise_rows(x.data_ptr(), x.dtype == torch.bfloat16, k, s["codes"].data_ptr(), s["codes"].shape[1], s["scale"], rows, k, torch.cuda.current_stream().cuda_stream)
    else:
        codes, scale = _codes(x)
        s["codes"][:, :k] = codes.to(torch.int8)
        s["scale"].copy_(scale)
    return {"codes": s["codes"], "scale": s["scale"]}


def _product(s):
    x, w = s["x"], s["w"]
    (T, k), n = x.shape, w.shape[0]
    if own:
        st = torch.cuda.current_stream().cuda_stream
        s["ops"].quantise_rows(x.data_ptr(), x.dtype == torch.bfloat16, k, s["codes"].data_ptr(), s["codes"].shape[1], s["scale"], T, k, st)
        s["ops"].linear8(s["codes"].data_ptr(), s["codes"].shape[1], s["scale"], w, w.shape[1], s["w_scale"], s["bias"], s["out"].data_ptr(), n, T, n, k, st)
        return s["out"]
    codes, scale = _codes(x)
    out = (codes @ w[:, :k].float().T) * scale[:, None] * s["w_scale"]
    s["out"].copy_(out if s["bias"] is None else out + s["bias"])
    return s["out"]


def _logprob(s):
    x, token, top = s["logits"], s["token"], s["case"]["top"]
    rows, n = x.shape
    if own:
        s["ops"].token_logprobs(x.data_ptr(), n, rows, n, token, torch.cuda.current_stream().cuda_stream, logprob=s["logprob"], entropy=s["entropy"], rank=s["rank"], top=top,
                                top_idx=s.get("top_idx"), top_logprob=s.get("top_logprob"))
        return {name: s[name] for name in ("logprob", "entropy", "rank", "top_idx", "top_logprob") if name in s}
    z = x - x.amax(-1, keepdim=True)
    weight = z.exp()
    total = weight.sum(-1, keepdim=True)
    z -= total.log()                                                     # the log probabilities
    mine = x.gather(1, token.long()[:, None])
    s["logprob"].copy_(z.gather(1, token.long()[:, None])[:, 0])
    s["entropy"].copy_(-(weight / total * torch.where(weight > 0, z, 0.0)).sum(-1))
    s["rank"].copy_(((x > mine) | ((x == mine) & (torch.arange(n, device=DEV) < token[:, None]))).sum(-1))
    out = {name: s[name] for name in ("logprob", "entropy", "rank")}
    if top:
        order = x.sort(dim=-1, descending=True, stable=True).indices[:, :top]                    # of equal ones the first comes first
        s["top_idx"].copy_(order)
        s["top_logprob"].copy_(z.gather(1, order))
        out |= {"top_idx": s["top_idx"], "top_logprob": s["top_logprob"]}
    return out


# ---------------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------------
def _visible(case):
    """Keys that have to be read (those that a query sees, shared ones once), and pairs of a query and a key that it sees."""
    w, keep = case["window"] or 1 << 30, case["keep"]
    keys = pairs = 0
    for shared, members in split(case):
        oldest = min(max(0, shared + p - w + 1) for p, _ in members)                         # of the shared ones
        keys += max(0, shared - oldest) + min(keep, oldest, shared)
        for p, n in members:
            lo = max(0, shared + p - w + 1)
            keys += shared + p + n - max(lo, shared) + max(0, min(keep, lo) - shared)
            for i in range(shared + p, shared + p + n):
                back = max(0, i - w + 1)
                pairs += i + 1 - back + min(keep, back)
    return keys, pairs


def work(case):
    if case["op"] == "logprob":
        values = case["rows"] * case["n"]
        return {"bytes": 4.0 * values + case["rows"] * (16.0 + 8.0 * case["top"]), "flops": 5.0 * values}
    if case["op"] == "quantise":
        values = case["rows"] * case["k"]
        return {"bytes": values * ((4.0 if case["x"] == "f32" else 2.0) + 1.0) + 4.0 * case["rows"], "flops": 3.0 * values}
    if case["op"] == "product":
        T, n, k = case["T"], case["n"], case["k"]
        return {"bytes": T * k * (4.0 if case["x"] == "f32" else 2.0) + float(n) * k + 4.0 * T * n + n * (8.0 if case["bias"] else 4.0), "flops": 2.0 * T * n * k}
    T = sum(n for _, members in split(case) for _, n in members)
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    keys, pairs = _visible(case)
    return {"bytes": 2.0 * keys * kv_heads * dim * (2.0 if case["cache"] == "bf16" else 4.0) + T * heads * dim * (4.0 + (4.0 if case["out"] == "f32" else 2.0)), "flops": 4.0 * pairs * heads * dim}


# ---------------------------------------------------------------------------------------------------------------------------
# The same in 64 bits, request by request and row by row
# ---------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] == "product" and case["T"] * case["n"] * case["k"] > 300e9:
        return None
    s = prepare(case, seed)
    return {"shared": _exact_attend, "quantise": _exact_quantise, "product": _exact_product, "logprob": _exact_logprob}[case["op"]](s)


def _exact_attend(s):
    """Every request by itself, over its own pages."""
    case = s["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out, at = [], 0
    for i, (_, p, n) in enumerate(s["segs"]):
        ids = s["table"][i, :-(-(p + n) // page)].long()
        k, v = (s[name + "_pool"][ids].double().transpose(0, 1).flatten(1, 2)[:, :p + n].repeat_interleave(heads // kv_heads, 0) for name in ("k", "v"))
        q = s["q"][at:at + n]
        q = (q.bfloat16() if case["cache"] == "bf16" else q).double().view(n, heads, dim).transpose(0, 1)
        z = q @ k.mT / math.sqrt(dim)
        if case["cap"]:
            z = case["cap"] * torch.tanh(z / case["cap"])
        far = torch.arange(p, p + n, device=DEV)[:, None] - torch.arange(p + n, device=DEV)
        hidden = far < 0
        if case["window"]:
            hidden |= (far >= case["window"]) & (torch.arange(p + n, device=DEV) >= case["keep"])
        out.append((torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ v).transpose(0, 1).flatten(1))
        at += n
    return torch.cat(out)


def _exact_codes(x):
    """Codes and scales, the two quotients rounded to fp32 as the definition says."""
    x = x.double()
    scale = torch.maximum((x.abs().max(-1).values / 127).float().double(), torch.tensor(LEAST, dtype=torch.float64, device=DEV))
    quotient = (x / scale[:, None]).float().double()
    low = torch.floor(quotient)
    rest = quotient - low
    return low + ((rest > 0.5) | ((rest == 0.5) & (low % 2 == 1))).double(), scale


def _exact_quantise(s):
    k = s["x"].shape[1]
    codes = torch.zeros(s["codes"].shape, dtype=torch.int8, device=DEV)
    q, scale = _exact_codes(s["x"])
    codes[:, :k] = q.to(torch.int8)
    return {"codes": codes, "scale": scale}


def _exact_product(s):
    k = s["x"].shape[1]
    codes, scale = _exact_codes(s["x"])
    w = s["w"][:, :k].double() * s["w_scale"].double()[:, None]
    out = torch.empty(s["out"].shape, dtype=torch.float64, device=DEV)
    for i in range(0, codes.shape[0], 256):
        out[i:i + 256] = (codes[i:i + 256] * scale[i:i + 256, None]) @ w.mT
        if s["bias"] is not None:
            out[i:i + 256] += s["bias"].double()
    return out


def _exact_logprob(s):
    top, got = s["case"]["top"], {"logprob": [], "entropy": [], "rank": [], "top_idx": [], "top_logprob": []}
    for i in range(s["logits"].shape[0]):
        x, t = s["logits"][i].double(), int(s["token"][i])
        logp = x - torch.logsumexp(x, 0)
        p = logp.exp()
        before = x > x[t]
        got["logprob"].append(logp[t])
        got["entropy"].append(-torch.special.xlogy(p, p).sum())
        got["rank"].append(before.sum() + (x[:t] == x[t]).sum())
        if top:
            border = torch.topk(x, top).values[-1]
            at = (x >= border).nonzero()[:, 0]                                            # ascending, so that a stable sort leaves the first of equals in front
            at = at[x[at].sort(descending=True, stable=True).indices][:top]
            got["top_idx"].append(at.to(torch.int32))
            got["top_logprob"].append(logp[at])
    got = {name: torch.stack(v) for name, v in got.items() if v}
    got["rank"] = got["rank"].to(torch.int32)
    return got
