"""What a pass through the attention operators of a serving loop costs: block tables and slot maps built from request
lengths, keys and values stored into a paged cache, attention over whole packed prompts, and attention of new tokens
(a chunk of a prompt, or one token each) over the paged cache.

`listed()` holds the cases, `draw(rng)` gives more of the same ranges, `prepare` makes a case's inputs on the GPU,
`run` is one pass -- in elementary torch operations, or, where `own` is set, through hodu_amd.ffi -- and `exact` is the
same from the definition in 64 bits.  The lengths of a case's sequences come from the case itself (its "lengths" number);
a seed shuffles them, draws the values and the order of the cache's pages.
"""
import math
import random

import torch

own = False

TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "f8e4m3": torch.float8_e4m3fn}
BYTES = {"bf16": 2, "f16": 2, "f8e4m3": 1}
F8_MAX = 448.0


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the table update in front of every decode step of a small batch: pure latency
        dict(name="plan_decode", op="plan", batch=8, longest=2048, added=1, page=16, lengths=1),
        # a scheduler tick that admits many prompts at once, ragged, onto a large pool
        dict(name="plan_prompts", op="plan", batch=512, longest=2048, added=2048, page=16, lengths=2),
        # one decode step's keys and values of a small batch
        dict(name="store_decode", op="store", tokens=8, kv_heads=8, heads=32, dim=128, dtype="bf16", cache="bf16", page=16),
        # a batch of prompts stored as 8-bit floats, rows read in place out of a joint q-k-v projection
        dict(name="store_prompts_f8", op="store", tokens=16384, kv_heads=8, heads=32, dim=128, dtype="bf16", cache="f8e4m3", page=64),
        # a handful of very short prompts (a chat's first words): the smallest attention call
        dict(name="prompt_short", op="prompt", batch=4, longest=61, heads=8, kv_heads=2, dim=64, dtype="f16", causal=True, lengths=3),
        # an ordinary admitted batch: sixteen prompts of up to 2048 tokens, none of them of the same length
        dict(name="prompt_packed", op="prompt", batch=16, longest=2048, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True, lengths=4),
        # one long document
        dict(name="prompt_long", op="prompt", batch=1, longest=8192, heads=32, kv_heads=8, dim=128, dtype="bf16", causal=True, lengths=0),
        # a chunk of each of four long prompts over what is cached of them already
        dict(name="chunk_512", op="paged", batch=4, longest=8192, added=512, heads=32, kv_heads=8, dim=128, dtype="bf16", cache="bf16", page=16, lengths=5),
        # chunks and single tokens in one step, the way a scheduler mixes them
        dict(name="chunk_mixed", op="paged", batch=24, longest=2048, added=-256, heads=32, kv_heads=32, dim=64, dtype="f16", cache="f16", page=32, lengths=6),
        # one user's next token: latency, with too few rows to fill the card
        dict(name="decode_one", op="paged", batch=1, longest=1999, added=1, heads=32, kv_heads=8, dim=128, dtype="bf16", cache="bf16", page=16, lengths=0),
        # a full decode batch over long contexts: the cache's bytes
        dict(name="decode_batch", op="paged", batch=64, longest=8192, added=1, heads=32, kv_heads=8, dim=128, dtype="bf16", cache="bf16", page=64, lengths=7),
        # the same need with the cache held in 8 bits
        dict(name="decode_batch_f8", op="paged", batch=48, longest=16384, added=1, heads=64, kv_heads=8, dim=128, dtype="bf16", cache="f8e4m3", page=32, lengths=8),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


MOST_FLOPS = 4.0 * 32 * 128 * (8192 * 8193 / 2)   # prompt_long: no drawn case computes more
MOST_BYTES = 1.44e9                               # decode_batch: or reads more


def draw(rng):
    while True:
        op = rng.choice(["plan", "store", "prompt", "prompt", "paged", "paged", "paged"])
        lengths = rng.randrange(1, 1 << 30)
        if op == "plan":
            case = dict(op=op, batch=_log(rng, 1, 512), longest=_log(rng, 16, 4096), added=rng.choice([1, 1, 64, 512, 2048]),
                        page=rng.choice([1, 16, 24, 32, 64, 128, 256]), lengths=lengths)
        else:
            dim, dtype = rng.choice([64, 128]), rng.choice(["bf16", "f16"])
            kv_heads = rng.choice([1, 2, 4, 8, 8, 16])
            heads = kv_heads * rng.choice([1, 2, 4, 5, 7, 8])
            page = rng.choice([1, 8, 16, 16, 24, 32, 64, 128, 256])
            cache = rng.choice([dtype, dtype, "f8e4m3"])
            if op == "store":
                case = dict(op=op, tokens=_log(rng, 1, 16384), kv_heads=kv_heads, heads=heads, dim=dim, dtype=dtype, cache=cache, page=page)
            elif op == "prompt":
                case = dict(op=op, batch=_log(rng, 1, 64), longest=_log(rng, 1, 8192), heads=heads, kv_heads=kv_heads, dim=dim,
                            dtype=dtype, causal=rng.random() < 0.8, lengths=lengths)
            else:
                longest = _log(rng, 2, 16384)
                added = rng.choice([1, 1, 1, rng.randrange(2, 17), _log(rng, 2, 1024), -_log(rng, 2, 512)])
                added = max(-longest, min(longest, added))
                case = dict(op=op, batch=_log(rng, 1, 64), longest=longest, added=added, heads=heads, kv_heads=kv_heads, dim=dim,
                            dtype=dtype, cache=cache, page=page, lengths=lengths)
        w = work(case)
        padded = 0.0  # what the plain form spends on sequences padded to the longest
        if op in ("prompt", "paged"):
            new, total = _lengths(case)
            padded = 4.0 * case["batch"] * case["heads"] * max(max(new), 1) * max(total)
        if w["flops"] <= MOST_FLOPS and w["bytes"] <= MOST_BYTES and padded <= 4.0 * 32 * 8192 * 8192:
            return case


def _lengths(case):
    """(new tokens, tokens in all) of the case's sequences, in the order of seed 0."""
    r, b, longest = random.Random(case["lengths"]), case["batch"], case["longest"]
    total = [longest if case["lengths"] == 0 else r.randint(max(1, longest // 3), longest) for _ in range(b)]
    total[0] = longest
    if case["op"] == "prompt":
        return total, total
    a = case["added"]
    if a < 0:  # half of them single tokens, half of them chunks
        new = [1 if i % 2 else r.randint(1, -a) for i in range(b)]
    else:
        new = [a] * b
    new = [min(n, t) for n, t in zip(new, total)]
    return new, total


def _shuffled(case, seed):
    new, total = _lengths(case)
    order = list(range(len(total)))
    random.Random(seed).shuffle(order)
    return [new[i] for i in order], [total[i] for i in order]


def work(case):
    if case["op"] == "plan":
        new, total = _lengths(case)
        pages = [-(-t // case["page"]) for t in total]
        taken = sum(p - (-(-(t - n) // case["page"])) for p, t, n in zip(pages, total, new))
        # lengths in and out, the new tokens' slots, the pages taken off the list and entered; the tables' old entries are
        # read where a request's new tokens begin inside a page
        return {"bytes": 4.0 * (4 * case["batch"] + sum(new) + 2 * taken), "flops": 0.0}
    if case["op"] == "store":
        one = 2.0 * case["tokens"] * case["kv_heads"] * case["dim"]
        return {"bytes": one * (BYTES[case["dtype"]] + BYTES[case["cache"]]) + 4.0 * case["tokens"], "flops": 0.0}
    new, total = _lengths(case)
    causal = case["op"] == "paged" or case["causal"]
    pairs = sum(n * t - (n * (n - 1) / 2 if causal else 0) for n, t in zip(new, total))
    rows = 2.0 * sum(new) * case["heads"] * case["dim"] * BYTES[case["dtype"]]  # q in, the result out
    kv = 2.0 * sum(total) * case["kv_heads"] * case["dim"] * BYTES[case.get("cache", case["dtype"])]
    return {"bytes": rows + kv + 8.0 * case["batch"], "flops": 4.0 * pairs * case["heads"] * case["dim"]}


# ---- inputs ---------------------------------------------------------------------------------------------------------
def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _offsets(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _normal(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(TORCH[dtype])


def _cache(gen, case, pages):
    """keys or values of `pages` pages, [pages, page, kv_heads, dim], in pieces: 8 bits hold values / scale"""
    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    out = torch.empty(shape, device="cuda", dtype=TORCH[case["cache"]])
    step = max(1, (1 << 26) // max(1, out[0].numel()))
    for i in range(0, pages, step):
        x = torch.randn((min(step, pages - i), *shape[1:]), generator=gen, device="cuda", dtype=torch.float32)
        out[i:i + step] = (x * 16.0 if case["cache"] == "f8e4m3" else x).to(out.dtype)
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed + 1)
    s = {"case": case}
    if case["op"] == "plan":
        new, total = _shuffled(case, seed)
        page, b = case["page"], case["batch"]
        width = -(-max(case["longest"], 1) // page)
        held = [-(-(t - n) // page) for n, t in zip(new, total)]
        need = sum(-(-t // page) for t in total)
        order = list(range(need + 64))  # the pool: some pages are held already, the others are on the free list
        host.shuffle(order)
        at, table = 0, [[-1] * width for _ in range(b)]
        for i, h in enumerate(held):
            table[i][:h] = order[at:at + h]
            at += h
        s.update(cached=_ints([t - n for n, t in zip(new, total)]), added=_ints(new), free=_ints(order[at:]), table=_ints(table),
                 lens=_ints([0] * b), offsets=_ints([0] * (b + 1)), slots=_ints([0] * sum(new)), used=_ints([0, 0]))
        return s
    dim, hq, hkv, dt = case["dim"], case["heads"], case["kv_heads"], case["dtype"]
    if case["op"] == "store":
        t, page = case["tokens"], case["page"]
        pages = -(-t // page) + 4
        rows = _normal(gen, (t, hq + 2 * hkv, dim), dt)  # the joint projection's output: q, k and v of a token side by side
        s.update(k=rows[:, hq:hq + hkv], v=rows[:, hq + hkv:], k_cache=_cache(gen, case, pages), v_cache=_cache(gen, case, pages))
        order = torch.randperm(pages, generator=gen, device="cuda")[:-(-t // page)]
        i = torch.arange(t, device="cuda")
        s["slots"] = (order[i // page] * page + i % page).to(torch.int32)
        scales = torch.linspace(0.0625, 0.125, hkv, device="cuda")
        s["k_scale"], s["v_scale"] = (scales, scales * 0.5) if case["cache"] == "f8e4m3" else (None, None)
        return s
    new, total = _shuffled(case, seed)
    s.update(q=_normal(gen, (sum(new), hq, dim), dt), offsets=_ints(_offsets(new)), longest=max(total), most_new=max(new),
             out=torch.empty((sum(new), hq, dim), device="cuda", dtype=TORCH[dt]), scale=torch.tensor(dim ** -0.5, dtype=TORCH[dt]))
    if case["op"] == "prompt":
        s.update(k=_normal(gen, (sum(total), hkv, dim), dt), v=_normal(gen, (sum(total), hkv, dim), dt))
        return s
    page = case["page"]
    count = [-(-t // page) for t in total]
    order = list(range(sum(count) + 8))
    host.shuffle(order)
    at, width = 0, -(-case["longest"] // page)
    table = []
    for n in count:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    s.update(k_cache=_cache(gen, case, len(order)), v_cache=_cache(gen, case, len(order)), table=_ints(table), lens=_ints(total))
    scales = torch.linspace(0.0625, 0.125, hkv, device="cuda")
    s["k_scale"], s["v_scale"] = (scales * 0.5, scales) if case["cache"] == "f8e4m3" else (None, None)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _plain_plan(s):
    page, slots = s["case"]["page"], s["slots"]
    cached, added = s["cached"].long(), s["added"].long()
    lens = cached + added
    offsets = torch.cat([torch.zeros_like(lens[:1]), torch.cumsum(added, 0)])
    held, need = (cached + page - 1) // page, (lens + page - 1) // page
    first = torch.cumsum(need - held, 0) - (need - held)  # where a request's share of the free list begins
    col = torch.arange(s["table"].shape[1], device=lens.device)[None, :]
    fresh = (col >= held[:, None]) & (col < need[:, None])
    at = torch.where(fresh, first[:, None] + col - held[:, None], 0)
    table = torch.where(fresh, s["free"][at], s["table"])
    t = torch.arange(slots.shape[0], device=lens.device)
    row = torch.searchsorted(offsets[1:], t, right=True)
    pos = cached[row] + t - offsets[row]
    slots = table[row, pos // page].long() * page + pos % page
    used = torch.stack([(need - held).sum(), torch.zeros_like(lens[0])])
    return {"table": table, "lens": lens.int(), "offsets": offsets.int(), "slots": slots.int(), "used": used.int()}


def _plain_store(s):
    out = {}
    for name in ("k", "v"):
        x, cache, scale = s[name].float(), s[name + "_cache"], s[name + "_scale"]
        if scale is not None:
            x = (x / scale[None, :, None]).clamp(-F8_MAX, F8_MAX)
        flat = cache.view(torch.uint8 if scale is not None else torch.int16).view(-1, *cache.shape[2:])
        flat[s["slots"].long()] = x.to(cache.dtype).view(flat.dtype)
        out[name] = cache
    return out


def _attend(q, k, v, keep, scale):
    """q [B, Sq, Hq, D], k and v [B, Sk, Hkv, D] in 32 bits, keep [B, Sq, Sk]: softmax(q k^T * scale) v over the kept keys, 0
    for a row that keeps none"""
    b, sq, hq, d = q.shape
    hkv, g = k.shape[2], hq // k.shape[2]
    q = q.view(b, sq, hkv, g, d).permute(0, 2, 3, 1, 4).reshape(b * hkv, g * sq, d)
    k = k.permute(0, 2, 3, 1).reshape(b * hkv, d, -1).contiguous()
    v = v.permute(0, 2, 1, 3).reshape(b * hkv, -1, d).contiguous()
    s = torch.bmm(q, k).view(b, hkv, g, sq, -1).mul_(scale)
    s.masked_fill_(~keep[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(torch.isinf(m), 0.0, m)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.bmm(s.view(b * hkv, g * sq, -1), v).view(b, hkv, g, sq, d) / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(b, sq, hq, d)


def _padded_rows(s):
    """where row i of every sequence stands among the packed ones, and whether it is there: [B, longest]"""
    at, n = s["offsets"][:-1].long(), s["offsets"].diff().long()
    i = torch.arange(s["most_new"], device=at.device)
    there = i[None] < n[:, None]
    return torch.where(there, at[:, None] + i[None], 0), there, i


def _plain_prompt(s):
    rows, there, i = _padded_rows(s)
    keep = there[:, None, :] & there[:, :, None]
    if s["case"]["causal"]:
        keep = keep & (i[None, :, None] >= i[None, None, :])
    o = _attend(s["q"][rows].float(), s["k"][rows].float(), s["v"][rows].float(), keep, s["scale"].float().item())
    s["out"][rows[there]] = o[there].to(s["out"].dtype)
    return s["out"]


def _plain_paged(s):
    rows, there, i = _padded_rows(s)
    page, lens = s["case"]["page"], s["lens"].long()
    j = torch.arange(s["longest"], device=lens.device)
    written = j[None] < lens[:, None]
    slot = torch.where(written, s["table"][:, j // page].long() * page + j % page, 0)

    def gathered(cache, scale):
        x = cache.view(torch.uint8 if scale is not None else cache.dtype).view(-1, *cache.shape[2:])[slot].view(cache.dtype).float()
        return x if scale is None else x * scale[None, None, :, None]

    last = (lens - s["offsets"].diff().long())[:, None] + i[None]  # the last key that a row attends
    keep = there[:, :, None] & written[:, None, :] & (j[None, None, :] <= last[:, :, None])
    o = _attend(s["q"][rows].float(), gathered(s["k_cache"], s["k_scale"]), gathered(s["v_cache"], s["v_scale"]), keep,
                s["scale"].float().item())
    s["out"][rows[there]] = o[there].to(s["out"].dtype)
    return s["out"]


# ---- the framework's operators ----------------------------------------------------------------------------------------
_context = None


def _own(s):
    global _context
    from hodu_amd import ffi

    if _context is None:
        _context = ffi.Context(0)
        # the operands are torch's: the calls are in order with its work on them, before and after (handed over once, as by a
        # program that stays on the stream it begins with)
        _context.set_stream(torch.cuda.current_stream())
    c, case, of = _context, s["case"], ffi.DeviceView.of
    if case["op"] == "plan":
        c.paged_plan(of(s["cached"]), of(s["added"]), of(s["free"]), of(s["table"]), of(s["lens"]), of(s["offsets"]), of(s["slots"]),
                     of(s["used"]), ffi.paged_plan_md(case["batch"], case["page"], s["table"].shape[1], s["free"].shape[0], s["slots"].shape[0]))
        return {"table": s["table"], "lens": s["lens"], "offsets": s["offsets"], "slots": s["slots"], "used": s["used"]}
    scales = {} if s.get("k_scale") is None else {"k_scale": of(s["k_scale"]), "v_scale": of(s["v_scale"])}
    if case["op"] == "store":
        k, v, kc = s["k"], s["v"], s["k_cache"]
        md = ffi.paged_store_md(case["tokens"], case["kv_heads"], case["dim"], kc.shape[0], case["page"],
                                k_strides=k.stride()[:2], v_strides=v.stride()[:2], k_cache_strides=kc.stride()[:3],
                                v_cache_strides=s["v_cache"].stride()[:3])
        c.paged_store(case["dtype"], of(k), of(v), of(kc), of(s["v_cache"]), of(s["slots"]), md, cache_dt=case["cache"], **scales)
        return {"k": s["k_cache"], "v": s["v_cache"]}
    q, scale = s["q"], s["scale"].view(torch.int16).numpy()
    if case["op"] == "prompt":
        k, v = s["k"], s["v"]
        md = ffi.varlen_md(case["batch"], q.shape[0], k.shape[0], case["heads"], case["kv_heads"], case["dim"],
                           q_strides=q.stride()[:2], k_strides=k.stride()[:2], v_strides=v.stride()[:2])
        offsets = of(s["offsets"])
        c.attention_varlen(case["dtype"], of(q), of(k), of(v), of(s["out"]), offsets, offsets, md, scale, causal=case["causal"])
        return s["out"]
    kc, vc = s["k_cache"], s["v_cache"]
    md = ffi.paged_attention_md(case["batch"], q.shape[0], case["heads"], case["kv_heads"], case["dim"], kc.shape[0], case["page"],
                                s["table"].shape[1], q_strides=q.stride()[:2], k_cache_strides=kc.stride()[:3],
                                v_cache_strides=vc.stride()[:3])
    c.attention_paged(case["dtype"], of(q), of(kc), of(vc), of(s["out"]), of(s["offsets"]), of(s["table"]), of(s["lens"]), md, scale,
                      cache_dt=case["cache"], **scales)
    return s["out"]


def run(state):
    if own:
        return _own(state)
    return {"plan": _plain_plan, "store": _plain_store, "prompt": _plain_prompt, "paged": _plain_paged}[state["case"]["op"]](state)


# ---- from the definition, in 64 bits ------------------------------------------------------------------------------------
def _one_sequence(q, k, v, scale, shift):
    """q [n, Hq, D], k and v [m, Hkv, D] in 64 bits; row i attends keys 0 .. i + shift (all of them where shift is None)"""
    n, hq, _ = q.shape
    out, g = torch.zeros_like(q), hq // k.shape[1]
    if not n or not k.shape[0]:
        return out
    hide = None
    if shift is not None:
        hide = torch.ones(n, k.shape[0], dtype=torch.bool, device=q.device).triu(shift + 1)
    for h in range(hq):
        for i in range(0, n, 2048):
            a = (q[i:i + 2048, h] @ k[:, h // g].t().contiguous()) * scale
            if hide is not None:
                a.masked_fill_(hide[i:i + 2048], -math.inf)
            out[i:i + 2048, h] = torch.nan_to_num(torch.softmax(a, -1)) @ v[:, h // g].contiguous()
    return out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "plan":
        return None  # whole numbers
    if case["op"] == "store":
        out = {}
        for name in ("k", "v"):
            whole = s[name + "_cache"].double()
            x = s[name].double()
            if case["cache"] == "f8e4m3":
                x = torch.clamp(x / s[name + "_scale"].double()[:, None], -F8_MAX, F8_MAX)
            slots = s["slots"].long()
            whole[slots // case["page"], slots % case["page"]] = x
            out[name] = whole
        return out
    scale, at = s["scale"].double().item(), s["offsets"].tolist()
    parts = []
    if sum(_lengths(case)[0]) * case["heads"] == 0:
        return s["out"].double()
    for b in range(case["batch"]):
        q = s["q"][at[b]:at[b + 1]].double()
        if case["op"] == "prompt":
            k, v, shift = s["k"][at[b]:at[b + 1]].double(), s["v"][at[b]:at[b + 1]].double(), 0 if case["causal"] else None
        else:
            n = int(s["lens"][b])
            pages = s["table"][b, :-(-n // case["page"])].long()
            k, v = (s[c].view(torch.uint8 if case["cache"] == "f8e4m3" else s[c].dtype)[pages].view(s[c].dtype).double().flatten(0, 1)[:n]
                    for c in ("k_cache", "v_cache"))
            if case["cache"] == "f8e4m3":
                k, v = k * s["k_scale"].double()[:, None], v * s["v_scale"].double()[:, None]
            shift = n - q.shape[0]
        parts.append(_one_sequence(q, k, v, scale, shift))
    return torch.cat(parts)
