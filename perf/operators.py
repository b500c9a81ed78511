"""Measured cases of the serving operators: prompt attention over packed sequences, the 8-bit key/value cache (write, read
back, attention of one query token per sequence) and the rules between logits and the next token.

``run`` computes a case in its plain form (elementary torch operations in f32, rounded once at the end) or, where ``own``
is true, through the library's entry points.  ``exact`` is the definition in 64 bits, written apart from the plain form.

The cache lies in memory as the library defines it: K [blocks, heads, block tokens, pitch] and
V [blocks, heads, block tokens / 16, pitch, 16] int8 with one f32 scale per (block, head); pitch is head_dim rounded up
to a multiple of 32.
"""
import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the 110M f32 model: a batch of ordinary prompts, one of a single token
        {"name": "prompt_f32_d64", "op": "prompt", "dtype": "f32", "heads": 12, "kv_heads": 12, "dim": 64, "q": "1024,333,1,64", "before": "0,0,0,0"},
        # the 3B model's head size, which is not a power of two, in f32
        {"name": "prompt_f32_d100", "op": "prompt", "dtype": "f32", "heads": 32, "kv_heads": 32, "dim": 100, "q": "777,1200", "before": "0,0"},
        # 1B-style grouped heads in f16: many short prompts, one empty, two that continue a cached prefix
        {"name": "prompt_f16_d64_short", "op": "prompt", "dtype": "f16", "heads": 32, "kv_heads": 8, "dim": 64,
         "q": "17,250,1,96,0,511,33,64,128,129,7,300,450,12,88,200,31,5,409,77,65,2,144,260", "before": "0,0,0,0,0,0,0,640,0,0,0,0,1024,0,0,0,0,0,0,0,0,0,0,0"},
        # long prompts, bf16
        {"name": "prompt_bf16_d128_long", "op": "prompt", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "q": "8192,1000,4500", "before": "0,0,0"},
        # a batch of prompts into an empty cache, and the rows read back
        {"name": "append_prompt_bf16_d128", "op": "append", "dtype": "bf16", "kv_heads": 8, "dim": 128, "block": 64, "new": "4096,2500,1203,393", "before": "0,0,0,0"},
        # one token for each of many running sequences, f32
        {"name": "append_token_f32_d64", "op": "append", "dtype": "f32", "kv_heads": 8, "dim": 64, "block": 32,
         "new": ",".join(["1"] * 48), "before": ",".join(str((i * 173) % 2048) for i in range(48))},
        # one running sequence, ordinary context: latency
        {"name": "cache_f32_d64_one", "op": "cache", "dtype": "f32", "heads": 32, "kv_heads": 8, "dim": 64, "block": 32, "lengths": "1024"},
        # the 3B model's heads, a small ragged batch with one sequence that has nothing yet
        {"name": "cache_f32_d100_batch", "op": "cache", "dtype": "f32", "heads": 32, "kv_heads": 32, "dim": 100, "block": 16, "lengths": "2048,1,700,0,1999,33,1500,512"},
        # one very long context
        {"name": "cache_bf16_d128_long", "op": "cache", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "block": 64, "lengths": "131072"},
        # a full serving batch of ragged contexts
        {"name": "cache_bf16_d128_batch", "op": "cache", "dtype": "bf16", "heads": 32, "kv_heads": 8, "dim": 128, "block": 64,
         "lengths": ",".join(str(97 + (i * 2657) % 8000) for i in range(64))},
        # one row of the models' vocabulary with its history and a grammar's mask
        {"name": "logits_one", "op": "logits", "dtype": "f32", "rows": 1, "vocab": 32000, "history": 1024, "biases": 16, "mask": True},
        # a serving batch over a large vocabulary
        {"name": "logits_batch", "op": "logits", "dtype": "f32", "rows": 200, "vocab": 128256, "history": 2000, "biases": 100, "mask": True},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 8, 8])
    rep = rng.choice([1, 2, 4, 4, 5, 8])
    return kv * rep, kv


def draw(rng):
    op = rng.choice(["prompt", "prompt", "append", "cache", "cache", "logits"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    dim = rng.choice([64, 64, 100, 128, 128])
    heads, kv = _heads(rng)
    if op == "prompt":
        longest = _log(rng, 2, 2048 if dtype == "f32" or dim == 100 else 8192)
        n = rng.randint(1, max(1, min(24, 16384 // longest)))
        q = [longest] + [rng.randint(0, longest) for _ in range(n - 1)]
        before = [rng.choice([0, 0, 0, rng.randint(1, longest)]) for _ in q]
        while n * heads * max(q) * max(a + b for a, b in zip(q, before)) > 3 * 32 * 8192 ** 2:      # no more than the largest listed batch
            q, before = [-(-a // 2) for a in q], [b // 2 for b in before]
        return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv, "dim": dim, "q": ",".join(map(str, q)), "before": ",".join(map(str, before))}
    if op == "append":
        longest = _log(rng, 1, 4096)
        n = rng.randint(1, max(1, min(64, 8192 // longest)))
        new = [longest] + [rng.randint(0, longest) for _ in range(n - 1)]
        before = [rng.choice([0, rng.randint(0, 2048)]) for _ in new]
        return {"op": op, "dtype": dtype, "kv_heads": kv, "dim": dim, "block": rng.choice([16, 32, 64, 128]), "new": ",".join(map(str, new)), "before": ",".join(map(str, before))}
    if op == "cache":
        longest = _log(rng, 16, 65536)
        n = rng.randint(1, max(1, min(64, 131072 // longest)))
        lengths = [longest] + [rng.randint(0, longest) for _ in range(n - 1)]
        return {"op": op, "dtype": dtype, "heads": heads, "kv_heads": kv, "dim": dim, "block": rng.choice([16, 32, 64, 128]), "lengths": ",".join(map(str, lengths))}
    rows = _log(rng, 1, 200)
    return {"op": op, "dtype": dtype, "rows": rows, "vocab": rng.choice([32000, rng.randint(1000, 128256), 128256]), "history": _log(rng, 1, 4096),
            "biases": rng.choice([0, rng.randint(1, 300)]), "mask": rng.random() < 0.5}


def _numbers(text):
    return [int(t) for t in text.split(",")]


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return out


def _pitch(dim):
    return (dim + 31) // 32 * 32


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    make = {"prompt": _prepare_prompt, "append": _prepare_append, "cache": _prepare_cache, "logits": _prepare_logits}
    s = make[case["op"]](case, g, random.Random(seed))
    s["op"], s["dtype"] = case["op"], TYPES[case["dtype"]]
    return s


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _prepare_prompt(case, g, rng):
    t = TYPES[case["dtype"]]
    q, before = _numbers(case["q"]), _numbers(case["before"])
    k = [a + b for a, b in zip(q, before)]
    H, G, D = case["heads"], case["kv_heads"], case["dim"]
    r = lambda n, h: torch.randn(n, h, D, generator=g, device=DEV)
    qt, kt, vt = r(sum(q), H) * 1.5, r(sum(k), G), r(sum(k), G)
    return {"q": qt.to(t), "k": kt.to(t), "v": vt.to(t), "out": torch.zeros(sum(q), H, D, dtype=t, device=DEV),
            "q_off": _ints(_offsets(q)), "k_off": _ints(_offsets(k)), "n": len(q), "max_q": max(q), "max_k": max(k), "scale": 1.0 / math.sqrt(D)}


def _empty_cache(blocks, G, D, bt):
    P = _pitch(D)
    z = lambda *shape: torch.zeros(*shape, dtype=torch.int8, device=DEV)
    f = lambda: torch.zeros(blocks, G, device=DEV)
    return {"k8": z(blocks, G, bt, P), "v8": z(blocks, G, bt // 16, P, 16), "ks": f(), "vs": f()}


def _table(lengths, bt, g):
    """Blocks of each sequence in a shuffled pool, as a pool looks after some hours of serving; unused entries are -1."""
    need = [(n + bt - 1) // bt for n in lengths]
    total, width = max(1, sum(need)), max(1, max(need))
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    at = torch.arange(width, device=DEV)
    start = torch.tensor(_offsets(need)[:-1], device=DEV)
    used = at[None] < torch.tensor(need, device=DEV)[:, None]
    return torch.where(used, order[(start[:, None] + at).clamp(max=total - 1)], torch.full_like(order[:1], -1)).contiguous(), total


def _fill(c, g, D):
    """Contents of a running cache: normally distributed values, scales that differ from block to block."""
    for p, s in (("k8", "ks"), ("v8", "vs")):
        c[p].copy_((torch.randn(c[p].shape, generator=g, device=DEV) * 40).round().clamp(-127, 127))
        c[s].copy_(0.015 + 0.015 * torch.rand(c[s].shape, generator=g, device=DEV))
    if _pitch(D) != D:
        c["k8"][..., D:] = 0
        c["v8"][..., D:, :] = 0


def _prepare_append(case, g, rng):
    t = TYPES[case["dtype"]]
    new, before = _numbers(case["new"]), _numbers(case["before"])
    G, D, bt = case["kv_heads"], case["dim"], case["block"]
    table, blocks = _table([a + b for a, b in zip(new, before)], bt, g)
    c = _empty_cache(blocks, G, D, bt)
    _fill(c, g, D)
    begin = [b // bt * bt if a else b for a, b in zip(new, before)]        # the blocks that change are read back whole
    back = [b + a - s for a, b, s in zip(new, before, begin)]
    r = lambda: torch.randn(sum(new), G, D, generator=g, device=DEV).to(t)
    o = lambda: torch.zeros(sum(back), G, D, dtype=t, device=DEV)
    return {**c, "table": table, "k": r(), "v": r(), "k_back": o(), "v_back": o(), "off": _ints(_offsets(new)), "start": _ints(before),
            "back_off": _ints(_offsets(back)), "begin": _ints(begin), "n": len(new), "bt": bt, "dim": D}


def _prepare_cache(case, g, rng):
    t = TYPES[case["dtype"]]
    lengths = _numbers(case["lengths"])
    H, G, D, bt = case["heads"], case["kv_heads"], case["dim"], case["block"]
    table, blocks = _table(lengths, bt, g)
    c = _empty_cache(blocks, G, D, bt)
    _fill(c, g, D)
    q = torch.randn(len(lengths), H, D, generator=g, device=DEV) * 1.5
    return {**c, "table": table, "q": q.to(t), "out": torch.zeros(len(lengths), H, D, dtype=t, device=DEV), "lengths": _ints(lengths),
            "max_len": max(lengths), "n": len(lengths), "bt": bt, "dim": D, "scale": 1.0 / math.sqrt(D)}


def _prepare_logits(case, g, rng):
    R, V, n, b = case["rows"], case["vocab"], case["history"], case["biases"]
    t = TYPES[case["dtype"]]
    lens = [max(0, n - rng.randint(0, n // 2)) for _ in range(R)]          # rows at different places of their texts
    total = sum(lens)
    history = (torch.rand(max(1, total), generator=g, device=DEV).square() * V).to(torch.int32).clamp(max=V - 1)   # frequent tokens repeat
    b = min(b, V)
    bias_ids = torch.rand(R, V, generator=g, device=DEV).topk(b, dim=1).indices.to(torch.int32).reshape(-1) if b else _ints([0])
    u = lambda lo, hi: lo + (hi - lo) * torch.rand(R, generator=g, device=DEV)
    words = (V + 31) // 32
    mask = torch.randint(-2 ** 31, 2 ** 31, (R, words), generator=g, device=DEV, dtype=torch.int64).to(torch.int32) if case["mask"] else None
    return {"logits": (torch.randn(R, V, generator=g, device=DEV) * 4).to(t), "out": torch.zeros(R, V, dtype=t, device=DEV),
            "best": torch.zeros(R, dtype=torch.int32, device=DEV), "history": history, "off": _ints(_offsets(lens)), "n_history": total,
            "rep": u(1.0, 1.5), "freq": u(0.0, 0.5), "pres": u(0.0, 0.5), "bias_ids": bias_ids,
            "bias": torch.randn(max(1, R * b), generator=g, device=DEV) * 2, "bias_off": _ints([i * b for i in range(R + 1)]), "n_bias": R * b, "mask": mask}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    if own:
        return _own(state)
    return {"prompt": _plain_prompt, "append": _plain_append, "cache": _plain_cache, "logits": _plain_logits}[state["op"]](state)


def _handle(s):
    """The cache's handle, as a program keeps it."""
    import simplang_b200 as sg
    if "handle" not in s:
        nb, G, bt, _ = s["k8"].shape
        s["handle"] = sg.kv8_cache(s["k8"].data_ptr(), s["v8"].data_ptr(), s["ks"].data_ptr(), s["vs"].data_ptr(), nb, bt, G, s["dim"])
    return s["handle"]


def _own(s):
    import simplang_b200 as sg
    t = {torch.float32: sg.F32, torch.float16: sg.F16, torch.bfloat16: sg.BF16}[s["dtype"]]
    if s["op"] == "prompt":
        q, k = s["q"], s["k"]
        sg.attn_prompt(q.data_ptr(), k.data_ptr(), s["v"].data_ptr(), s["out"].data_ptr(), s["q_off"].data_ptr(), s["k_off"].data_ptr(), s["n"],
                       q.shape[0], k.shape[0], q.shape[1], k.shape[1], q.shape[2], scale=s["scale"], dtype=t)
        return s["out"]
    if s["op"] == "append":
        c, width = _handle(s), s["table"].shape[1]
        sg.kv8_append(c, s["table"].data_ptr(), width, s["k"].data_ptr(), s["v"].data_ptr(), s["off"].data_ptr(), s["start"].data_ptr(), s["n"], s["k"].shape[0], dtype=t)
        sg.kv8_read(c, s["table"].data_ptr(), width, s["k_back"].data_ptr(), s["v_back"].data_ptr(), s["back_off"].data_ptr(), s["begin"].data_ptr(), s["n"],
                    s["k_back"].shape[0], dtype=t)
        return {"k": s["k_back"], "v": s["v_back"], "k_scales": s["ks"], "v_scales": s["vs"]}
    if s["op"] == "cache":
        sg.attn_kv8(_handle(s), s["table"].data_ptr(), s["table"].shape[1], s["q"].data_ptr(), s["out"].data_ptr(), s["lengths"].data_ptr(), s["n"], s["max_len"],
                    s["q"].shape[1], scale=s["scale"], dtype=t)
        return s["out"]
    if "rules" not in s:
        s["rules"] = sg.logits_rules(tokens=s["history"].data_ptr(), token_offsets=s["off"].data_ptr(), n_tokens=s["n_history"], repetition=s["rep"].data_ptr(),
                                     frequency=s["freq"].data_ptr(), presence=s["pres"].data_ptr(), bias_tokens=s["bias_ids"].data_ptr(),
                                     bias_values=s["bias"].data_ptr(), bias_offsets=s["bias_off"].data_ptr(), n_bias=s["n_bias"],
                                     allowed=None if s["mask"] is None else s["mask"].data_ptr(), allowed_stride=0 if s["mask"] is None else s["mask"].shape[1])
    R, V = s["logits"].shape
    sg.logits_process(s["logits"].data_ptr(), s["out"].data_ptr(), R, V, s["rules"], argmax=s["best"].data_ptr(), dtype=t)
    return {"logits": s["out"], "token": s["best"]}


def _rows_of(off, total):
    """(sequence, place in it) of each packed row."""
    at = torch.arange(total, device=DEV)
    seq = (torch.searchsorted(off, at.to(off.dtype), right=True) - 1).clamp(min=0)
    return seq, at - off[seq]


def _padded(x, off, longest):
    """Packed rows [total, heads, dim] as f32 [sequences, longest, heads, dim], zeros behind each sequence."""
    at = torch.arange(longest, device=DEV)
    there = at[None] < (off[1:] - off[:-1])[:, None]
    rows = torch.where(there, off[:-1, None] + at, torch.zeros_like(at))
    return x[rows].float() * there[:, :, None, None]


def _attend(q, k, v, visible, scale):
    """q [B, G, rep, Lq, D], k and v [B, G, Lk, D], visible [B, Lq, Lk] -> [B, G, rep, Lq, D]; a row that sees nothing is zero."""
    B, G, rep, Lq, D = q.shape
    s = torch.matmul((q * scale).reshape(B, G, rep * Lq, D), k.transpose(-1, -2)).view(B, G, rep, Lq, -1)
    s.masked_fill_(~visible[:, None, None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, G, rep * Lq, -1), v).view(B, G, rep, Lq, D)
    return o / torch.where(total > 0, total, torch.ones_like(total))


def _plain_prompt(s):
    total, H, D = s["q"].shape
    G = s["k"].shape[1]
    q_off, k_off = s["q_off"], s["k_off"]
    q = _padded(s["q"], q_off, s["max_q"]).view(s["n"], s["max_q"], G, H // G, D).permute(0, 2, 3, 1, 4)
    k, v = (_padded(s[x], k_off, s["max_k"]).transpose(1, 2) for x in "kv")
    nq, nk = q_off[1:] - q_off[:-1], k_off[1:] - k_off[:-1]
    i, j = torch.arange(s["max_q"], device=DEV), torch.arange(s["max_k"], device=DEV)
    visible = (j[None, None] <= i[None, :, None] + (nk - nq)[:, None, None]) & (j[None, None] < nk[:, None, None])
    o = _attend(q, k, v, visible, s["scale"]).permute(0, 3, 1, 2, 4).reshape(s["n"], s["max_q"], H, D)
    seq, place = _rows_of(q_off, total)
    return o[seq, place].to(s["dtype"])


def _dequantised(s, table):
    """K and V of the tables' blocks as f32 [sequences, tokens, heads, dim]; a place without a block holds zeros."""
    there = (table >= 0)[:, :, None, None, None]
    b = table.clamp(min=0).long()
    k = (s["k8"][b].float() * s["ks"][b][..., None, None] * there).permute(0, 1, 3, 2, 4)          # [n, w, bt, G, P]
    v = (s["v8"][b].float() * s["vs"][b][..., None, None, None] * there[..., None])                 # [n, w, G, bt / 16, P, 16]
    v = v.permute(0, 1, 3, 5, 2, 4)
    n, w, bt, G, P = k.shape
    return k.reshape(n, w * bt, G, P)[..., :s["dim"]], v.reshape(n, w * bt, G, P)[..., :s["dim"]]


def _plain_cache(s):
    n, H, D = s["q"].shape
    k, v = _dequantised(s, s["table"])
    G = k.shape[2]
    q = s["q"].float().view(n, G, H // G, 1, D)
    visible = torch.arange(k.shape[1], device=DEV)[None, None] < s["lengths"][:, None, None]
    return _attend(q, k.transpose(1, 2), v.transpose(1, 2), visible, s["scale"]).reshape(n, H, D).to(s["dtype"])


def _step(top):
    """max|x| / 127 correctly rounded to f32 (the quotient in 64 bits rounds to the same number)."""
    return (top.double() / 127).float()


def _nearest(x, step):
    """x / step to the nearest whole number, halves to even; in 64 bits, where no quotient is taken for a half that is none."""
    step = step.double()
    q = torch.where(step > 0, x.double() / torch.where(step > 0, step, torch.ones_like(step)), torch.zeros_like(step))
    return q.round().clamp(-127, 127).to(torch.int8)


def _plain_append(s):
    total, G, D = s["k"].shape
    bt, n = s["bt"], s["n"]
    seq, place = _rows_of(s["off"], total)
    pos = s["start"][seq] + place
    block = s["table"][seq, pos // bt].long()
    # the block in which each sequence goes on, where it holds tokens already and gets more
    count = s["off"][1:] - s["off"][:-1]
    goes_on = (s["start"] % bt > 0) & (count > 0)
    open_block = s["table"].gather(1, (s["start"] // bt).long().clamp(max=s["table"].shape[1] - 1)[:, None])[:, 0].long().clamp(min=0)
    held = (torch.arange(bt, device=DEV)[None] < (s["start"] % bt)[:, None]) & goes_on[:, None]      # [n, bt]
    hh = torch.arange(G, device=DEV)
    for x, c8, cs in ((s["k"], "k8", "ks"), (s["v"], "v8", "vs")):
        x = x.float()
        nb = s[cs].shape[0]
        old = s[cs].clone()
        top = torch.zeros(nb, G, device=DEV).scatter_reduce_(0, block[:, None].expand(-1, G), x.abs().amax(-1), "amax")
        touched = torch.zeros(nb, dtype=torch.bool, device=DEV).index_fill_(0, block, True)
        keeps = torch.zeros(nb, device=DEV).index_add_(0, open_block, goes_on.float()) > 0
        new = torch.where(touched[:, None], torch.maximum(_step(top), torch.where(keeps[:, None], old, torch.zeros_like(old))), old)
        s[cs].copy_(new)
        c = s[c8]
        # tokens that the block holds, to the new step
        a, b = old[open_block], new[open_block]                                                     # [n, G]
        if c8 == "k8":
            was = c[open_block]                                                                     # [n, G, bt, P]
            again = _nearest(was.double() * a[:, :, None, None].double(), b[:, :, None, None])
            pick = held[:, None, :, None]
        else:
            was = c[open_block]                                                                     # [n, G, bt / 16, P, 16]
            again = _nearest(was.double() * a[:, :, None, None, None].double(), b[:, :, None, None, None])
            pick = held.view(n, 1, bt // 16, 1, 16)
        change = torch.where(pick, again.to(torch.int16) - was.to(torch.int16), torch.zeros_like(was, dtype=torch.int16))
        c.index_add_(0, open_block, change.to(torch.int8))                                          # modulo 256: again - was added to was
        # the new tokens
        q = _nearest(x, new[block][..., None])                                                      # [total, G, D]
        at = pos % bt
        if c8 == "k8":
            c[block[:, None], hh[None], at[:, None], :D] = q
        else:
            c[block[:, None], hh[None], (at // 16)[:, None], :D, (at % 16)[:, None]] = q
    k, v = _dequantised(s, s["table"])
    seq, place = _rows_of(s["back_off"], s["k_back"].shape[0])
    pos = (s["begin"][seq] + place).long()
    return {"k": k[seq, pos].to(s["dtype"]), "v": v[seq, pos].to(s["dtype"]), "k_scales": s["ks"], "v_scales": s["vs"]}


def _plain_logits(s):
    R, V = s["logits"].shape
    x = s["logits"].float()
    seq, _ = _rows_of(s["off"], s["n_history"])
    ids = s["history"][:s["n_history"]].long()
    count = torch.zeros(R * V, device=DEV).index_add_(0, seq * V + ids, torch.ones(ids.shape, device=DEV)).view(R, V)
    seen = count > 0
    rep, freq, pres = (s[w][:, None] for w in ("rep", "freq", "pres"))
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - (freq * count + torch.where(seen, pres, torch.zeros_like(pres)))
    if s["n_bias"]:
        row = torch.arange(s["n_bias"], device=DEV) // (s["n_bias"] // R)
        x.view(-1).index_add_(0, row * V + s["bias_ids"].long(), s["bias"])
    if s["mask"] is not None:
        at = torch.arange(V, device=DEV)
        x.masked_fill_(((s["mask"][:, at // 32] >> (at % 32)) & 1) == 0, float("-inf"))
    out = x.to(s["dtype"])
    top = out.amax(-1, keepdim=True)
    at = torch.where(out == top, torch.arange(V, device=DEV), V).amin(-1)
    return {"logits": out, "token": torch.where(torch.isinf(top[:, 0]), -torch.ones_like(at), at).to(torch.int32)}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    if case["op"] == "prompt":
        q, before = _numbers(case["q"]), _numbers(case["before"])
        H, G, D = case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(n * b + n * (n + 1) // 2 for n, b in zip(q, before))
        return {"bytes": size * D * (2 * H * sum(q) + 2 * G * (sum(q) + sum(before))), "flops": 4 * D * H * pairs}
    if case["op"] == "append":
        new, before = _numbers(case["new"]), _numbers(case["before"])
        G, D, bt = case["kv_heads"], case["dim"], case["block"]
        back = sum(n + b % bt if n else 0 for n, b in zip(new, before))
        blocks = sum((n + b % bt + bt - 1) // bt if n else 0 for n, b in zip(new, before))
        # rows in, their bytes and scales out; then those blocks' bytes and scales in, their rows out
        return {"bytes": 2 * G * (D * (sum(new) * (size + 1) + back * (size + 1)) + 8 * blocks), "flops": 4 * G * D * (sum(new) + back)}
    if case["op"] == "cache":
        lengths = _numbers(case["lengths"])
        H, G, D, bt = case["heads"], case["kv_heads"], case["dim"], case["block"]
        blocks = sum((n + bt - 1) // bt for n in lengths)
        return {"bytes": 2 * G * (D * sum(lengths) + 4 * blocks) + 4 * blocks + 2 * size * H * D * len(lengths), "flops": 4 * H * D * sum(lengths)}
    R, V = case["rows"], case["vocab"]
    return {"bytes": R * (2 * size * V + (V // 8 if case["mask"] else 0) + 3 * case["history"] + 8 * case["biases"] + 16), "flops": 6 * R * V}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def _softmax_rows(scores, v):
    """softmax(scores) . v in 64 bits; rows of -inf give zeros."""
    top = scores.max(-1, keepdim=True).values
    e = torch.where(torch.isinf(top), torch.zeros_like(scores), torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top)))
    den = e.sum(-1, keepdim=True)
    return (e / torch.where(den == 0, torch.ones_like(den), den)) @ v


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "prompt":
        return _exact_prompt(case, s)
    if case["op"] == "append":
        return _exact_append(case, s)
    if case["op"] == "cache":
        return _exact_cache(case, s)
    return _exact_logits(case, s)


def _exact_prompt(case, s):
    H, G = case["heads"], case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    q0 = k0 = 0
    for n, b in zip(_numbers(case["q"]), _numbers(case["before"])):
        m = n + b
        if n:
            hidden = torch.ones(n, m, dtype=torch.bool, device=DEV).triu(1 + m - n)
            for h in range(H):
                k, v = (s[x][k0:k0 + m, h // (H // G)].double() for x in "kv")
                sc = (s["q"][q0:q0 + n, h].double() @ k.T) * s["scale"]
                out[q0:q0 + n, h] = _softmax_rows(sc.masked_fill_(hidden, float("-inf")), v)
        q0, k0 = q0 + n, k0 + m
    return out


def _block_values(s, b):
    """K and V of one block as 64-bit [tokens, heads, dim]."""
    G, bt, P = s["k8"].shape[1:]
    k = s["k8"][b].double().permute(1, 0, 2) * s["ks"][b].double()[None, :, None]
    v = s["v8"][b].double().permute(1, 3, 0, 2).reshape(bt, G, P) * s["vs"][b].double()[None, :, None]
    return k[..., :s["dim"]], v[..., :s["dim"]]


def _exact_cache(case, s):
    H, G, bt = case["heads"], case["kv_heads"], case["block"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    P, D = _pitch(case["dim"]), case["dim"]
    for i, n in enumerate(_numbers(case["lengths"])):
        if not n:
            continue
        b = s["table"][i, :(n + bt - 1) // bt].long()
        for g in range(G):
            k = (s["k8"][b, g].double() * s["ks"][b, g].double()[:, None, None]).reshape(-1, P)[:n, :D]
            v = (s["v8"][b, g].double() * s["vs"][b, g].double()[:, None, None, None]).transpose(2, 3).reshape(-1, P)[:n, :D]
            h = slice(g * (H // G), (g + 1) * (H // G))
            out[i, h] = _softmax_rows((s["q"][i, h].double() @ k.T) * s["scale"], v)
    return out


def _exact_append(case, s):
    G, D, bt = case["kv_heads"], case["dim"], case["block"]
    new, before = _numbers(case["new"]), _numbers(case["before"])
    ks, vs = s["ks"].double().clone(), s["vs"].double().clone()
    back_k, back_v = [], []
    if sum((n + bt - 1) // bt + 1 for n in new) > 2500:
        return None
    table, row = s["table"].tolist(), 0
    for i, (n, b0) in enumerate(zip(new, before)):
        done = 0
        while done < n:
            pos = b0 + done
            blk, at = table[i][pos // bt], pos % bt
            take = min(bt - at, n - done)
            held = _block_values(s, blk)
            for x, scales, h, back in ((s["k"], ks, held[0], back_k), (s["v"], vs, held[1], back_v)):
                fresh = x[row + done:row + done + take].double()                                   # [take, G, D]
                step = (fresh.abs().amax((0, 2)) / 127).float().double()
                if at:
                    step = torch.maximum(step, scales[blk])
                scales[blk] = step
                whole = torch.cat([h[:at], fresh])
                back.append(torch.round(whole / step[None, :, None]).clamp(-127, 127) * step[None, :, None])
            done += take
        row += n
    empty = torch.zeros(0, G, D, dtype=torch.float64, device=DEV)
    return {"k": torch.cat(back_k or [empty]), "v": torch.cat(back_v or [empty]), "k_scales": ks, "v_scales": vs}


def _exact_logits(case, s):
    R, V = s["logits"].shape
    x = s["logits"].double()
    off, boff = s["off"].tolist(), s["bias_off"].tolist()
    bits = torch.arange(32, device=DEV)
    for r in range(R):
        n = torch.bincount(s["history"][off[r]:off[r + 1]].long(), minlength=V).double()
        rep, f, p = (s[w][r].double() for w in ("rep", "freq", "pres"))
        y = x[r]
        hit = n > 0
        y = torch.where(hit & (y > 0), y / rep, torch.where(hit, y * rep, y)) - f * n - p * hit
        if s["n_bias"]:
            y[s["bias_ids"][boff[r]:boff[r + 1]].long()] += s["bias"][boff[r]:boff[r + 1]].double()
        if s["mask"] is not None:
            allowed = ((s["mask"][r][:, None] >> bits) & 1).reshape(-1)[:V].bool()
            y = torch.where(allowed, y, torch.full_like(y, float("-inf")))
        x[r] = y
    return {"logits": x, "token": None}
