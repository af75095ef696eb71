"""A serving step over an 8-bit key/value cache, as cases that can be timed: keys and values appended to the paged cache with the rotation on the way, attention
over that cache, and the draw of the next tokens from given random numbers. `listed` names one case per use, `draw` gives more of the same ranges.

Operators and their ranges:
  append   Ops.rotary_kv8: queries and keys turned, keys and values into the cache as e4m3 with a power of two as scale for each block of 32 positions and head;
           1 .. 64 segments, single tokens and portions of up to 4096, heads of 64 and 128, both pairings
  attend   Ops.attention8: 1 .. 64 requests of up to 8192 positions decoding, portions of prompts of up to 2048 tokens, both together; heads of 64 and 128, groups of 1 .. 8,
           results in fp32 or bf16, windows, capped scores
  sample   Ops.sample_rows: 1 .. 64 rows of 500 .. 128256 logits, every row with its own temperature, top-k, top-p, min-p and random number

A cache pool is [pages][kv_heads][page_len][width] in e4m3, its scales are [pages][kv_heads][page_len / 32] in fp32: a value is code * scale. The scale of a block is the
smallest power of two (2^-100 at least) under which the block's largest magnitude is at most 448; a block that grows takes the larger of its old scale and that of the new
rows, and its older rows move to it.
"""
import math

import torch

own = False
DEV = "cuda"
BLOCK = 32
LARGEST = 448.0
LEAST_EXPONENT = -100


def listed():
    return [
        # one request of a Llama-3-8B-shaped model decoding: the smallest call
        {"name": "append_1_token", "op": "append", "segs": "4000+1", "heads": 32, "kv_heads": 8, "dim": 128, "layout": 1, "page": 64},
        # a full decoding batch of the same model, every request somewhere in a block
        {"name": "append_64_requests", "op": "append", "segs": requests(64, 8191, 3, 1), "heads": 32, "kv_heads": 8, "dim": 128, "layout": 1, "page": 64},
        # prompts of the same model, taken in together
        {"name": "append_prompts", "op": "append", "segs": "0+2048,1000+1500,37+311,0+37", "heads": 32, "kv_heads": 8, "dim": 128, "layout": 1, "page": 64},
        # portions beside decoding requests with TinyLlama's heads, neighbouring dimensions paired
        {"name": "append_mixed_step", "op": "append", "segs": "0+256,512+256,777+131,90+1,1500+1,31+1,32+1,2000+17", "heads": 32, "kv_heads": 4, "dim": 64, "layout": 0, "page": 32},
        # a long conversation of one user
        {"name": "decode_1_request", "op": "attend", "segs": "7999+1", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "out": "f32", "window": 0, "keep": 0, "cap": 0.0},
        # eight requests of unequal length decoding together
        {"name": "decode_8_requests", "op": "attend", "segs": "7999+1,310+1,2047+1,1024+1,4089+1,76+1,1499+1,5999+1", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64,
         "out": "f32", "window": 0, "keep": 0, "cap": 0.0},
        # a full batch: the cache is what such a step reads
        {"name": "decode_64_requests", "op": "attend", "segs": requests(64, 8191, 5, 1), "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "out": "bf16", "window": 0, "keep": 0,
         "cap": 0.0},
        # TinyLlama's heads behind a sliding window that keeps the first positions
        {"name": "decode_window", "op": "attend", "segs": "1999+1,700+1,130+1,0+1,64+1", "heads": 32, "kv_heads": 4, "dim": 64, "page": 32, "out": "bf16", "window": 500, "keep": 4,
         "cap": 0.0},
        # prompts taken in together, one of them behind an earlier context
        {"name": "attend_prompts", "op": "attend", "segs": "0+2048,700+1300,0+311,4000+37", "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "out": "bf16", "window": 0, "keep": 0,
         "cap": 0.0},
        # a step of a server: a portion of a long prompt beside decoding requests, capped scores, results for a projection in fp32
        {"name": "attend_mixed_step", "op": "attend", "segs": "6000+256," + requests(12, 4000, 7, 1), "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "out": "f32", "window": 0,
         "keep": 0, "cap": 30.0},
        # one user's next token, a vocabulary of 32000
        {"name": "sample_1_row", "op": "sample", "rows": 1, "n": 32000, "kind": "k_p"},
        # a full batch over the vocabulary of Llama-3, every request with settings of its own
        {"name": "sample_64_rows", "op": "sample", "rows": 64, "n": 128256, "kind": "mixed"},
    ]


def requests(n, longest, step, new):
    """`n` segments of `new` tokens behind contexts spread over 0 .. longest - 1, as the text a case carries."""
    return ",".join("%d+%d" % ((i * i * step * 131 + i * 977) % longest, new) for i in range(n))


def split(case):
    return [tuple(int(x) for x in s.split("+")) for s in case["segs"].split(",")]


def _spread(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample"])
    if op == "sample":
        return {"op": op, "rows": _spread(rng, 1, 64), "n": _spread(rng, 500, 128256), "kind": rng.choice(["k_p", "mixed", "p", "min_p", "plain"])}
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8])
    case = {"op": op, "heads": kv_heads * rng.choice([1, 2, 3, 4, 8]), "kv_heads": kv_heads, "dim": dim, "page": rng.choice([32, 64, 128])}
    shape = rng.choice(["decode", "prompts", "mixed"])
    segs = []
    if shape != "prompts":
        segs += [(rng.randrange(_spread(rng, 1, 8191)), 1) for _ in range(_spread(rng, 1, 64 if shape == "decode" else 16))]
    if shape != "decode":
        segs += [(rng.choice([0, rng.randrange(4096)]), _spread(rng, 2, 2048 if op == "attend" else 4096)) for _ in range(rng.randint(1, 3))]
    rng.shuffle(segs)
    if op == "append":
        case["layout"] = rng.choice([0, 1])
    else:
        window = rng.choice([0, 0, _spread(rng, 40, 2000)])
        case |= {"out": rng.choice(["f32", "bf16"]), "window": window, "keep": rng.choice([0, 4]) if window else 0, "cap": rng.choice([0.0, 0.0, 30.0])}
    case["segs"] = ",".join("%d+%d" % s for s in segs)
    while _beyond(case):                                                 # the longest portion, or context, is halved
        segs = split(case)
        i = max(range(len(segs)), key=lambda j: (segs[j][1], segs[j][0]))
        segs[i] = (segs[i][0] // 2, max(1, segs[i][1] // 2))
        case["segs"] = ",".join("%d+%d" % s for s in segs)
    return case


def _beyond(case):
    """Whether a case costs more than the largest listed ones, or its padded batch, which the plain form holds at once, takes more room."""
    w, segs = work(case), split(case)
    if case["op"] == "append":
        return w["bytes"] > 160e6
    rows, context = max(n for _, n in segs), max(p + n for p, n in segs)
    return w["flops"] > 60e9 or w["bytes"] > 500e6 or len(segs) * case["heads"] * rows * context > 1e9 or len(segs) * case["kv_heads"] * context * case["dim"] > 0.55e9


# ---------------------------------------------------------------------------------------------------------------------------
# What a program has in hand before the call
# ---------------------------------------------------------------------------------------------------------------------------
def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _codes(x):
    """[..., BLOCK, width] fp32 -> e4m3 codes and the scale of each block."""
    amax = x.double().abs().amax((-1, -2))
    scale = torch.exp2(torch.ceil(torch.log2(amax / LARGEST)).clamp_min(LEAST_EXPONENT))
    return (x.double() / scale[..., None, None]).float().to(torch.float8_e4m3fn), scale.float()


def _step(case, g):
    """The index arrays of a step over pages handed out in any order, and pools filled with what earlier steps have left."""
    segs, page = split(case), case["page"]
    need = [-(-(p + n) // page) for p, n in segs]
    pages, widest = sum(need) + 2, max(need)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    starts = torch.cumsum(torch.tensor([0] + need[:-1]), 0).tolist()
    table = torch.full((len(segs), widest), -1, dtype=torch.int32, device=DEV)
    for i, (at, n) in enumerate(zip(starts, need)):
        table[i, :n] = order[at:at + n]
    tiles = [(i, off) for i, (_, n) in enumerate(segs) for off in range(0, n, BLOCK)]
    tiles.sort(key=lambda t: -(segs[t[0]][0] + t[1]))
    lens = torch.tensor([n for _, n in segs])
    first = torch.cumsum(lens, 0) - lens
    slot = torch.repeat_interleave(torch.arange(len(segs)), lens)
    pos = torch.arange(int(lens.sum())) - first[slot] + torch.tensor([p for p, _ in segs])[slot]
    counts = [-(-n // BLOCK) for _, n in segs]
    st = {"segs": segs, "table": table, "n_pages": pages, "tok_slot": _ints(slot.tolist()), "tok_pos": _ints(pos.tolist()), "seg_start": _ints(first.tolist()),
          "seg_len": _ints(lens.tolist()), "seg_slot": _ints(list(range(len(segs)))), "seg_pos0": _ints([p for p, _ in segs]), "qt_seg": _ints([t[0] for t in tiles]),
          "qt_off": _ints([t[1] for t in tiles]), "seg_tile0": _ints([sum(counts[:i]) for i in range(len(segs))])}
    for name in ("k", "v"):
        # keys have channels that are larger than others, all the time; values do not
        gain = torch.exp(0.7 * torch.randn(case["kv_heads"], 1, 1, case["dim"], generator=g, device=DEV)) if name == "k" else 1.0
        x = gain * torch.randn(pages, case["kv_heads"], page // BLOCK, BLOCK, case["dim"], generator=g, device=DEV)
        codes, scale = _codes(x)
        st[name + "_pool"], st[name + "_scale"] = codes.view(pages, case["kv_heads"], page, case["dim"]), scale
        if name == "k":
            st["gain"] = gain.reshape(1, case["kv_heads"], case["dim"])
    return st


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    if case["op"] == "sample":
        state = _logits(case, g)
    else:
        state = _step(case, g)
        T, heads, kv_heads, dim = state["tok_pos"].numel(), case["heads"], case["kv_heads"], case["dim"]
        if case["op"] == "append":
            # one row of queries, keys and values as a fused projection leaves it
            state["qkv"] = torch.randn(T, heads + 2 * kv_heads, dim, generator=g, device=DEV)
            state["qkv"][:, heads:heads + kv_heads] *= state["gain"]
            freq = 500000.0 ** (-torch.arange(dim // 2, dtype=torch.float64, device=DEV) * 2 / dim)
            turn = state["tok_pos"].double()[:, None] * freq
            state["angles"] = torch.stack([torch.cos(turn), torch.sin(turn)], -1).float().contiguous()
            state["q_out"] = torch.empty(T, heads * dim, device=DEV)
        else:
            state["q"] = torch.randn(T, heads * dim, generator=g, device=DEV)
            state["out"] = torch.empty(T, heads * dim, device=DEV, dtype=torch.float32 if case["out"] == "f32" else torch.bfloat16)
    state["case"] = case
    if own:
        _plan(state)
    return state


def _logits(case, g):
    """Logits as a language model leaves them: a bell of unlikely tokens, some likely ones, a few banned; and every row's settings."""
    rows, n, kind = case["rows"], case["n"], case["kind"]
    x = 2.5 * torch.randn(rows, n, generator=g, device=DEV)
    likely = torch.randint(0, n, (rows, 24), generator=g, device=DEV)
    x.scatter_reduce_(1, likely, 9.0 + 3.0 * torch.randn(rows, 24, generator=g, device=DEV), "amax")      # the same place twice: the larger, whichever comes first
    x.scatter_(1, torch.randint(0, n, (rows, 8), generator=g, device=DEV), -math.inf)
    r = torch.rand(rows, 5, generator=g, device=DEV)
    one = torch.ones(rows, device=DEV)
    which = torch.arange(rows, device=DEV) % 5 if kind == "mixed" else torch.full((rows,), {"k_p": 0, "p": 1, "min_p": 2, "plain": 3}[kind], device=DEV)
    temperature = torch.where(which == 4, 0 * one, 0.6 + 0.9 * r[:, 0])                        # 0: the largest logit
    top_k = torch.where(which == 0, (20 + 80 * r[:, 1]).floor(), 0 * one).to(torch.int32)      # 0: all
    top_p = torch.where((which == 0) | (which == 1), 0.85 + 0.14 * r[:, 2], one)               # 1: all
    min_p = torch.where(which == 2, 0.02 + 0.1 * r[:, 3], 0 * one)                             # 0: all
    return {"logits": x, "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p, "u": r[:, 4].contiguous(),
            "idx": torch.empty(rows, dtype=torch.int32, device=DEV), "prob": torch.empty(rows, device=DEV)}


def _plan(state):
    """What such a program keeps from call to call: the launchers, the step's description, the workspace of the attention."""
    from simplellminference_b200 import _lib
    from simplellminference_b200.config import BF16
    from simplellminference_b200.seqops import Ops
    case, ops = state["case"], Ops(BF16)
    state["ops"] = ops
    if case["op"] == "sample":
        return
    b = _lib.SeqBatch()
    b.T, b.nseg, b.n_qtiles = state["tok_pos"].numel(), len(state["segs"]), state["qt_seg"].numel()
    for name in ("tok_slot", "tok_pos", "seg_start", "seg_len", "seg_slot", "seg_pos0", "qt_seg", "qt_off", "seg_tile0"):
        setattr(b, name, state[name].data_ptr())
    b.block_table, b.max_pages, b.page_len = state["table"].data_ptr(), state["table"].shape[1], case["page"]
    state["batch"] = b
    if case["op"] == "attend":
        need = ops.attention8_ws_bytes(b, case["heads"], case["kv_heads"], case["dim"], case["dim"])
        state["ws"] = torch.zeros(need, dtype=torch.uint8, device=DEV)
        state["opts"] = ops.attention_options(window=case["window"], keep_first=case["keep"], softcap=case["cap"]) if case["window"] or case["cap"] else None


# ---------------------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------------------
def run(state):
    return {"append": _append, "attend": _attend, "sample": _sample}[state["case"]["op"]](state)


def _append(s):
    case = s["case"]
    heads, kv_heads, dim, layout = case["heads"], case["kv_heads"], case["dim"], case["layout"]
    if own:
        row, at = (heads + 2 * kv_heads) * dim, s["qkv"].data_ptr()
        s["ops"].rotary_kv8(s["batch"], at, row, heads, dim, at + 4 * heads * dim, row, kv_heads, at + 4 * (heads + kv_heads) * dim, row, dim, s["angles"], dim // 2, layout,
                            s["q_out"].data_ptr(), heads * dim, s["k_pool"], s["k_scale"], s["v_pool"], s["v_scale"], s["n_pages"], torch.cuda.current_stream().cuda_stream)
    else:
        s["q_out"].copy_(_turned(s["qkv"][:, :heads], s["angles"], layout).flatten(1))
        _store(s, "k", _turned(s["qkv"][:, heads:heads + kv_heads], s["angles"], layout))
        _store(s, "v", s["qkv"][:, heads + kv_heads:])
    return {"q": s["q_out"], "k": s["k_pool"], "k_scale": s["k_scale"], "v": s["v_pool"], "v_scale": s["v_scale"]}


def _turned(x, angles, layout):
    """Pairs (2i, 2i + 1) with layout 0, (i, i + half) with layout 1, turned by their angle."""
    half = x.shape[-1] // 2
    a, b = (x[..., 0::2], x[..., 1::2]) if layout == 0 else (x[..., :half], x[..., half:])
    c, s = angles[:, None, :, 0], angles[:, None, :, 1]
    return torch.stack([a * c - b * s, b * c + a * s], -1).flatten(-2) if layout == 0 else torch.cat([a * c - b * s, b * c + a * s], -1)


def _scale_for(amax):
    """The smallest power of two under which amax is at most 448."""
    m, e = torch.frexp(amax / LARGEST)                                   # m in [0.5, 1): a power of two itself where m is 0.5
    e = torch.where(amax > 0, torch.where(m > 0.5, e, e - 1), LEAST_EXPONENT)
    return torch.exp2(e.double().clamp_min(LEAST_EXPONENT)).float()


def _store(s, name, x):
    pool, scale = s[name + "_pool"], s[name + "_scale"]
    page, sub = s["case"]["page"], s["case"]["page"] // BLOCK
    tok_slot, tok_pos, seg_slot, pos0 = (s[n].long() for n in ("tok_slot", "tok_pos", "seg_slot", "seg_pos0"))
    kv_heads, dim = pool.shape[1], pool.shape[3]
    codes = pool.view(torch.uint8).view(-1, kv_heads, sub, BLOCK, dim).transpose(1, 2)                 # [pages][blocks of a page][head][row][column]
    scales = scale.transpose(1, 2)
    at = (s["table"].long()[tok_slot, tok_pos // page], tok_pos % page // BLOCK)
    old_at = (s["table"].long()[seg_slot, pos0 // page], pos0 % page // BLOCK)
    fresh = torch.zeros(codes.shape[0] * sub, kv_heads, device=DEV)
    fresh.index_reduce_(0, at[0] * sub + at[1], x.abs().amax(-1), "amax")
    new = _scale_for(fresh).view(codes.shape[0], sub, kv_heads)
    before = scales[old_at]                                              # a segment's first block may hold earlier rows
    has_old = (pos0 % BLOCK > 0)[:, None]
    first = torch.where(has_old, torch.maximum(before, new[old_at]), new[old_at])
    moved = (codes[old_at].view(torch.float8_e4m3fn).float() * (before / first)[..., None, None]).to(torch.float8_e4m3fn).view(torch.uint8)
    earlier = torch.arange(BLOCK, device=DEV) < (pos0 % BLOCK)[:, None]
    codes[old_at] = torch.where(earlier[:, None, :, None], moved, codes[old_at])
    new[old_at] = first
    scales[at] = new[at]
    codes[at[0], at[1], :, tok_pos % BLOCK] = (x / new[at][..., None]).to(torch.float8_e4m3fn).view(torch.uint8)


def _attend(s):
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    if own:
        f32 = case["out"] == "f32"
        s["ops"].attention8(s["batch"], s["q"].data_ptr(), heads * dim, heads, kv_heads, dim, dim, dim ** -0.5, s["k_pool"], s["k_scale"], s["v_pool"], s["v_scale"], s["n_pages"],
                            s["ws"], torch.cuda.current_stream().cuda_stream, out=s["out"] if f32 else None, ldo=heads * dim, out16=None if f32 else s["out"], opts=s["opts"])
        return s["out"]
    nseg, group = len(s["segs"]), heads // kv_heads
    lens, pos0, slot = s["seg_len"].long(), s["seg_pos0"].long(), s["tok_slot"].long()
    rows, context = max(n for _, n in s["segs"]), max(p + n for p, n in s["segs"])
    at = (slot, s["tok_pos"].long() - pos0[slot])
    q = torch.zeros(nseg, rows, heads, dim, device=DEV)                                # a padded batch
    q[at] = s["q"].view(-1, heads, dim)
    q = q.view(nseg, rows, kv_heads, group, dim).permute(0, 2, 3, 1, 4).reshape(nseg, kv_heads, group * rows, dim)
    k, v = (_padded(s, name, context) for name in ("k", "v"))                          # [segment][head][position][column]
    score = torch.matmul(q, k.transpose(2, 3)).view(nseg, kv_heads, group, rows, context)
    score *= dim ** -0.5
    if case["cap"]:
        score = torch.tanh_(score.div_(case["cap"])).mul_(case["cap"])
    mine = pos0[:, None, None] + torch.arange(rows, device=DEV)[:, None]
    key = torch.arange(context, device=DEV)
    seen = key <= mine
    if case["window"]:
        seen &= (mine - key < case["window"]) | (key < case["keep"])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    score -= score.amax(-1, keepdim=True)
    score.exp_()
    score /= score.sum(-1, keepdim=True)
    out = torch.matmul(score.view(nseg, kv_heads, group * rows, context), v)
    out = out.view(nseg, kv_heads, group, rows, dim).permute(0, 3, 1, 2, 4).reshape(nseg, rows, heads * dim)
    s["out"].copy_(out[at])
    return s["out"]


def _padded(s, name, context):
    """The cache as numbers, a row of positions for each segment; zeros where a sequence has none."""
    pool, scale, page = s[name + "_pool"], s[name + "_scale"], s["case"]["page"]
    pages = s["table"].long()[s["seg_slot"].long()].clamp_min(0)
    x = pool.view(torch.uint8)[pages].view(torch.float8_e4m3fn).float()                # [segment][page][head][row][column]
    x = x.view(*x.shape[:3], page // BLOCK, BLOCK, -1) * scale[pages][..., None, None]
    x = x.flatten(3, 4).transpose(1, 2).flatten(2, 3)[:, :, :context]
    last = (s["seg_pos0"] + s["seg_len"]).long()
    return x * (torch.arange(x.shape[2], device=DEV) < last[:, None])[:, None, :, None]


def _sample(s):
    x, rows, n = s["logits"], *s["logits"].shape
    if own:
        s["ops"].sample_rows(x.data_ptr(), n, rows, n, s["temperature"], s["top_k"], s["top_p"], s["min_p"], s["u"], s["idx"], torch.cuda.current_stream().cuda_stream, prob=s["prob"])
        return {"idx": s["idx"], "prob": s["prob"]}
    # in 64 bits: a draw lies next to one of as many borders as there are candidates
    greedy = s["temperature"] <= 0
    temperature = torch.where(greedy, 1.0, s["temperature"]).double()[:, None]
    ranked = x.sort(-1, descending=True).values
    top = ranked[:, :1]
    weight = torch.exp((ranked.double() - top) / temperature)
    k = torch.where(s["top_k"] <= 0, n, s["top_k"]).clamp_max(n).long()
    kth = ranked.gather(1, k[:, None] - 1)                               # equal logits are in or out together
    weight = weight * (ranked >= kth)
    mass = weight.cumsum(-1)
    p = torch.where((s["top_p"] <= 0) | (s["top_p"] >= 1), 1.0, s["top_p"]).double()[:, None]
    cut = torch.where(p < 1, ranked.gather(1, (mass < p * mass[:, -1:]).sum(-1, keepdim=True).clamp_max(n - 1)), kth)
    weight = torch.exp((x.double() - top) / temperature)
    weight = weight * ((x >= kth) & (x >= cut) & (weight >= s["min_p"].double()[:, None]))
    running = weight.cumsum(-1)
    total = running[:, -1:]
    idx = (running <= s["u"].double()[:, None] * total).sum(-1, keepdim=True).clamp_max(n - 1)
    first = torch.where(x == top, torch.arange(n, device=DEV), n).amin(-1)
    s["idx"].copy_(torch.where(greedy, first, idx[:, 0]))
    s["prob"].copy_(torch.where(greedy, 1.0, (weight.gather(1, idx) / total)[:, 0]))
    return {"idx": s["idx"], "prob": s["prob"]}


# ---------------------------------------------------------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------------
def _visible(case):
    """Keys that each segment has to read (those that one of its queries sees), and pairs of a query and a key that it sees."""
    w, keep = case["window"] or 1 << 30, case["keep"]
    keys = pairs = 0
    for p, n in split(case):
        oldest = max(0, p - w + 1)
        keys += p + n - oldest + min(keep, oldest)
        for i in range(p, p + n):
            back = max(0, i - w + 1)
            pairs += i + 1 - back + min(keep, back)
    return keys, pairs


def work(case):
    if case["op"] == "sample":
        values = case["rows"] * case["n"]
        return {"bytes": 4.0 * values + 28.0 * case["rows"], "flops": 4.0 * values}
    segs, heads, kv_heads, dim = split(case), case["heads"], case["kv_heads"], case["dim"]
    T = sum(n for _, n in segs)
    if case["op"] == "append":
        blocks = sum((p + n - 1) // BLOCK - p // BLOCK + 1 for p, n in segs)
        return {"bytes": 4.0 * T * ((2 * heads + 2 * kv_heads) * dim + dim) + 2.0 * T * kv_heads * dim + 8.0 * blocks * kv_heads, "flops": T * (3.0 * (heads + kv_heads) + 2 * kv_heads) * dim}
    keys, pairs = _visible(case)
    return {"bytes": 2.0 * keys * kv_heads * (dim + 4.0 / BLOCK) + T * heads * dim * (4.0 + (4.0 if case["out"] == "f32" else 2.0)), "flops": 4.0 * pairs * heads * dim}


# ---------------------------------------------------------------------------------------------------------------------------
# The same in 64 bits, segment by segment and row by row
# ---------------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s)


def _e4m3(x):
    """Rounded to the nearest of the numbers with three bits behind the point (ties to even) down to steps of 2^-9."""
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -20))).clamp_min(-6)
    step = torch.exp2(e - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    case = s["case"]
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    x = s["qkv"].double()
    angle = torch.complex(s["angles"][..., 0].double(), s["angles"][..., 1].double())[:, None]
    if case["layout"] == 0:
        z = torch.view_as_complex(x[:, :heads + kv_heads].unflatten(-1, (-1, 2)).contiguous()) * angle
        turned = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(*x[:, :heads + kv_heads].chunk(2, -1)) * angle
        turned = torch.cat([z.real, z.imag], -1)
    got = {"q": turned[:, :heads].flatten(1)}
    for name, new in (("k", turned[:, heads:]), ("v", x[:, heads + kv_heads:])):
        pool, scale = s[name + "_pool"].double(), s[name + "_scale"].double()
        at = 0
        for i, (p, n) in enumerate(s["segs"]):
            for lo in range(p // BLOCK * BLOCK, p + n, BLOCK):
                page, row = int(s["table"][i, lo // case["page"]]), lo % case["page"]
                a, b = max(lo, p), min(lo + BLOCK, p + n)
                rows = new[at + a - p:at + b - p].transpose(0, 1)
                sc = torch.exp2(torch.ceil(torch.log2(rows.abs().amax((1, 2)) / LARGEST)).clamp_min(LEAST_EXPONENT))
                if a > lo:
                    was = scale[page, :, row // BLOCK]
                    sc = torch.maximum(sc, was)
                    pool[page, :, row:row + a - lo] = _e4m3(pool[page, :, row:row + a - lo] * (was / sc)[:, None, None])
                scale[page, :, row // BLOCK] = sc
                pool[page, :, row + a - lo:row + b - lo] = _e4m3(rows / sc[:, None, None])
            at += n
        got[name], got[name + "_scale"] = pool, scale
    return {k: got[k] for k in ("q", "k", "k_scale", "v", "v_scale")}


def _exact_attend(s):
    case = s["case"]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    out, at = [], 0
    for i, (p, n) in enumerate(s["segs"]):
        ids = s["table"][i, :-(-(p + n) // page)].long()
        kv = []
        for name in ("k", "v"):
            x = s[name + "_pool"].view(torch.uint8)[ids].view(torch.float8_e4m3fn).double() * s[name + "_scale"][ids].double().repeat_interleave(BLOCK, -1)[..., None]
            kv.append(x.transpose(0, 1).flatten(1, 2)[:, :p + n].repeat_interleave(heads // kv_heads, 0))
        q = s["q"][at:at + n].double().view(n, heads, dim).transpose(0, 1)
        z = q @ kv[0].mT / math.sqrt(dim)
        if case["cap"]:
            z = case["cap"] * torch.tanh(z / case["cap"])
        far = torch.arange(p, p + n, device=DEV)[:, None] - torch.arange(p + n, device=DEV)
        hidden = far < 0
        if case["window"]:
            hidden |= (far >= case["window"]) & (torch.arange(p + n, device=DEV) >= case["keep"])
        w = torch.softmax(z.masked_fill(hidden, -math.inf), -1)
        out.append((w @ kv[1]).transpose(0, 1).flatten(1))
        at += n
    return torch.cat(out)


def _exact_sample(s):
    idx, prob = [], []
    for i in range(s["logits"].shape[0]):
        x = s["logits"][i].double()
        t, k, p, m, u = (float(s[name][i]) for name in ("temperature", "top_k", "top_p", "min_p", "u"))
        if t <= 0:
            idx.append(int((x == x.max()).nonzero()[0]))
            prob.append(1.0)
            continue
        alive = x > -math.inf
        if 0 < k < x.numel():
            alive = alive & (x >= torch.topk(x, int(k)).values[-1])
        w = torch.softmax(torch.where(alive, x, -math.inf) / t, -1)
        if 0 < p < 1:
            values = x[alive].unique().flip(0)                           # distinct ones, the largest first
            at = values.numel() - 1 - torch.searchsorted(values.flip(0), x[alive])
            mass = torch.zeros(values.numel(), dtype=torch.float64, device=DEV).index_add_(0, at, w[alive])
            alive = alive & (x >= values[int((mass.cumsum(0) < p).sum().clamp_max(values.numel() - 1))])
        if m > 0:
            alive = alive & (w >= m * w.max())
        w = torch.where(alive, w, 0.0) / w[alive].sum()
        idx.append(min(int((w.cumsum(0) <= u).sum()), x.numel() - 1))
        prob.append(float(w[idx[-1]]))
    return {"idx": torch.tensor(idx, dtype=torch.int32), "prob": torch.tensor(prob, dtype=torch.float64)}
