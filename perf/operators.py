"""Measured cases of the operators that serve a paged K/V cache chunk by chunk.

  attend   attention of a chunk of new tokens over the pages (every sequence brings one token or many)
  rope     rotary positions: half and interleaved layouts, part of the head, one position per token
  extend   rotate a chunk's queries and keys and write its keys and values into the pages
  weights  accumulate each cached slot's attention weight (the sums that eviction goes by)
  evict    keep each head's heaviest slots up to a budget and close the gaps

With ``own`` false ``run`` computes an operator in plain torch, in 32 bits, rounded once;
with ``own`` true it calls the framework's kernels.  All sequences are ragged: sequence b
brings the tokens [q_start[b], q_start[b + 1]) and lens[b] counts its cached slots with
those tokens included, so token i of its n sits in slot lens[b] - n + i.
"""
import random

import torch

own = False
D = 128  # head size of the cache


# ------------------------------------------------------------------ cases
def listed():
    return [
        # four short conversations, one new token each, small pages: latency alone
        dict(name="attend 4 tokens", op="attend", B=4, hq=32, hkv=8, page=16, ctx_lo=37, ctx_hi=1023, new_lo=1, new_hi=1,
             long=0, causal=True, lse=False, ragged=1),
        # the benchmark's decode batch: 64 sequences of 1024 to 32768 cached tokens
        dict(name="attend 64 tokens long", op="attend", B=64, hq=32, hkv=8, page=128, ctx_lo=1024, ctx_hi=32768, new_lo=1,
             new_hi=1, long=0, causal=True, lse=False, ragged=2),
        # a server's mixed step: one prompt chunk of 512 beside 31 sequences of one to five tokens, weights wanted
        dict(name="attend mixed step", op="attend", B=32, hq=32, hkv=8, page=64, ctx_lo=1, ctx_hi=4001, new_lo=1, new_hi=5,
             long=512, causal=True, lse=True, ragged=3),
        # the last 2048 tokens of a 32768-token prompt: tensor-bound
        dict(name="attend prompt tail", op="attend", B=1, hq=32, hkv=8, page=128, ctx_lo=30720, ctx_hi=30720, new_lo=2048,
             new_hi=2048, long=0, causal=True, lse=False, ragged=4),
        # the queries of one decode step of four sequences
        dict(name="rope 4 tokens", op="rope", T=4, heads=32, dim=128, rot=128, rows=8192, interleaved=False, inverse=False,
             f32=False),
        # the gradient through a partly rotated, interleaved layout over a long odd batch, in 32 bits
        dict(name="rope gradient 8191", op="rope", T=8191, heads=40, dim=128, rot=64, rows=32768, interleaved=True,
             inverse=True, f32=True),
        # one decode step of 64 sequences
        dict(name="extend 64 tokens", op="extend", B=64, hq=32, hkv=8, page=128, ctx_lo=0, ctx_hi=1024, new_lo=1, new_hi=1,
             long=0, rot=128, interleaved=False, ragged=5),
        # prompts of about 1000 tokens each, 8192 in all, into small pages
        dict(name="extend prompts", op="extend", B=8, hq=32, hkv=8, page=16, ctx_lo=0, ctx_hi=777, new_lo=900, new_hi=1148,
             long=0, rot=128, interleaved=False, ragged=6),
        # after a decode step: 64 sequences, one query each
        dict(name="weights 64 tokens", op="weights", B=64, hq=32, hkv=8, page=128, ctx_lo=128, ctx_hi=8191, new_lo=1, new_hi=1,
             long=0, causal=True, ragged=7),
        # after a prompt chunk of 1024 over 8192 slots
        dict(name="weights chunk", op="weights", B=1, hq=32, hkv=8, page=128, ctx_lo=7168, ctx_hi=7168, new_lo=1024,
             new_hi=1024, long=0, causal=True, ragged=8),
        # a small cache is cut to half
        dict(name="evict 4 short", op="evict", B=4, hkv=8, page=64, ctx_lo=1100, ctx_hi=2048, budget=1024, recent=128, sink=4,
             ragged=9),
        # sixteen long sequences are cut to 16384 slots
        dict(name="evict 16 long", op="evict", B=16, hkv=8, page=128, ctx_lo=20000, ctx_hi=32768, budget=16384, recent=256,
             sink=4, ragged=10),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    op = rng.choice(["attend", "attend", "attend", "rope", "extend", "weights", "evict"])
    ragged = rng.randrange(100, 1 << 20)
    hq, hkv = rng.choice([(32, 8), (32, 8), (32, 8), (16, 4), (8, 2), (4, 1), (8, 8), (32, 4), (24, 8)])
    page = rng.choice([16, 48, 64, 128, 256])
    if op == "rope":
        dim = rng.choice([64, 80, 128, 256])
        rot = dim if rng.random() < 0.5 else rng.choice([dim // 4, dim // 2])
        T = _spread(rng, 4, 8191)
        return dict(op=op, T=T, heads=rng.choice([1, 8, 32, 40]), dim=dim, rot=rot, rows=32768,
                    interleaved=rng.random() < 0.5, inverse=rng.random() < 0.3, f32=rng.random() < 0.3, ragged=ragged)
    if op == "evict":
        hi = _spread(rng, 256, 32768)
        B = max(1, min(_spread(rng, 1, 32), 524288 // hi))
        budget = rng.randint(max(64, hi // 4), hi)
        return dict(op=op, B=B, hkv=hkv, page=page, ctx_lo=max(1, hi // 2), ctx_hi=hi, budget=budget,
                    recent=rng.randint(0, budget // 4), sink=rng.randint(0, 8), ragged=ragged)
    if op == "extend":
        T = _spread(rng, 4, 8192)
        B = _spread(rng, 1, min(64, T))
        new = T // B
        return dict(op=op, B=B, hq=hq, hkv=hkv, page=page, ctx_lo=0, ctx_hi=1024, new_lo=max(1, new // 2), new_hi=new, long=0,
                    rot=rng.choice([32, 64, 128, 128]), interleaved=rng.random() < 0.4, ragged=ragged)
    new = _spread(rng, 1, 2048) if rng.random() < 0.6 else 1
    ctx = _spread(rng, 16, 32768 if op == "attend" else 8192)
    B = _spread(rng, 1, 64)
    B = max(1, min(B, 2048 // new, int(2.0e9 / (32.0 * new * (ctx + new)))))
    long = 0 if new > 8 or rng.random() < 0.6 else _spread(rng, 16, 512)
    if long:
        ctx = min(ctx, 4096)
        B = min(B, 32)
    case = dict(op=op, B=B, hq=hq, hkv=hkv, page=page, ctx_lo=rng.randint(0, ctx), ctx_hi=ctx, new_lo=max(1, new // 2), new_hi=new,
                long=long, causal=rng.random() < 0.85, ragged=ragged)
    if op == "attend":
        case["lse"] = rng.random() < 0.4
    return case


def _lengths(case):
    """New tokens and earlier slots of every sequence: the case's own, whatever the seed."""
    r = random.Random(case["ragged"])
    new = [r.randint(case["new_lo"], case["new_hi"]) for _ in range(case["B"])] if "new_lo" in case else [0] * case["B"]
    old = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["B"])]
    if case.get("long"):
        new[case["B"] // 2] = case["long"]
    return new, old


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    s = dict(case)
    if case["op"] == "rope":
        s["x"] = normal(case["T"], case["heads"], case["dim"], dtype=torch.float32 if case["f32"] else torch.bfloat16)
        s["positions"] = torch.randint(0, case["rows"], (case["T"],), generator=gen, device="cuda", dtype=torch.int32)
        s["cos"], s["sin"] = _table(case["rows"], case["rot"])
        s["out"] = torch.empty_like(s["x"])
        return s
    new, old = _lengths(case)
    B, hkv, page = case["B"], case["hkv"], case["page"]
    lens = [a + b for a, b in zip(new, old)]
    s["max_new"], s["cap_pages"] = max(new), -(-max(lens + [1]) // page)
    s["cap"] = s["cap_pages"] * page
    # every sequence's pages lie scattered over the pool; entries past its length name no page
    need = [-(-x // page) for x in lens]
    pool = sum(need) + 2
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    at = [sum(need[:b]) for b in range(B)]
    lp = torch.arange(s["cap_pages"], device="cuda")[None]
    need_t, at_t = ints(need)[:, None], ints(at)[:, None]
    s["table"] = torch.where(lp < need_t, order[(at_t + lp).clamp(max=pool - 1).long()], -1).to(torch.int32)
    s["lens"] = ints(lens)
    s["q_start"] = ints([sum(new[:b]) for b in range(B + 1)])
    s["tokens"] = sum(new)
    s["k_pages"] = normal(pool, hkv, page, D)
    s["v_pages"] = normal(pool, hkv, page, D)
    if case["op"] == "evict":
        slots = torch.arange(s["cap"], device="cuda", dtype=torch.int32)
        # weights decay by a power law in no order, as attention mass does; many slots were never looked at
        u = torch.rand(B, hkv, s["cap"], generator=gen, device="cuda")
        s["acc"] = torch.where(u < 0.1, 0.0, (u + 1e-3) ** -1.5)
        s["slot_pos"] = slots.expand(B, hkv, -1).contiguous()
        s["next_pos"] = s["lens"].clone()
        s["acc_out"], s["pos_out"] = torch.zeros_like(s["acc"]), torch.zeros_like(s["slot_pos"])
        s["lens_out"] = torch.zeros_like(s["lens"])
        return s
    T, hq = s["tokens"], case["hq"]
    # queries, keys and values lie in one row per token, as a fused projection leaves them
    s["qkv"] = normal(T, hq + 2 * hkv, D)
    s["qkv"][:, :hq] *= 1.5  # scores with a spread as trained heads have it
    s["q"], s["k"], s["v"] = s["qkv"][:, :hq], s["qkv"][:, hq:hq + hkv], s["qkv"][:, hq + hkv:]
    if case["op"] == "extend":
        s["cos"], s["sin"] = _table(max(lens) + 1, case["rot"])
        s["positions"] = torch.cat([torch.arange(a, a + n, dtype=torch.int32, device="cuda") for a, n in zip(old, new)])
        s["q_out"] = torch.empty(T, hq, D, dtype=torch.bfloat16, device="cuda")
        s["slot_pos"] = torch.zeros(B, hkv, s["cap"], dtype=torch.int32, device="cuda")
        return s
    s["scale"] = D ** -0.5
    if case["op"] == "attend":
        s["out"] = torch.empty(T, hq, D, dtype=torch.bfloat16, device="cuda")
        s["lse_out"] = torch.empty(T, hq, device="cuda") if case["lse"] else None
        return s
    s["lse"] = _attend(s)[1]
    s["acc"] = torch.rand(B, hkv, s["cap"], generator=gen, device="cuda") * 4
    s["acc_out"] = torch.zeros_like(s["acc"])
    return s


def _table(rows, rot):
    """cos and sin of position x frequency, [rows][rot / 2] in 32 bits."""
    inv = 500000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64, device="cuda") / rot)
    angle = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None] * inv
    return angle.cos().float(), angle.sin().float()


# ------------------------------------------------------------------ plain forms
def _rotate(x, cos, sin, positions, interleaved, inverse):
    rot = 2 * cos.shape[1]
    c, n = cos[positions.long()][:, None], sin[positions.long()][:, None] * (-1.0 if inverse else 1.0)
    y, x = x.clone(), x.float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    p, r = a * c - b * n, b * c + a * n
    y[..., :rot] = (torch.stack((p, r), -1).flatten(-2) if interleaved else torch.cat((p, r), -1)).to(y.dtype)
    return y


def _rows(s):
    """Of every token: its sequence, its place among that sequence's new tokens and its slot."""
    t = torch.arange(s["tokens"], device="cuda", dtype=torch.int32)
    b = torch.searchsorted(s["q_start"][1:].contiguous(), t, right=True)
    i = t - s["q_start"][b]
    return b, i, s["lens"][b] - (s["q_start"][b + 1] - s["q_start"][b]) + i


def _dense(s, pages):
    """The pages as [B][Hkv][slots][128], zero past each sequence's length."""
    x = pages[s["table"].clamp(min=0).long()].permute(0, 2, 1, 3, 4).reshape(s["B"], s["hkv"], s["cap"], D)
    there = torch.arange(s["cap"], device="cuda")[None] < s["lens"][:, None]
    return torch.where(there[:, None, :, None], x, 0).float()


def _scores(s):
    """Scaled scores [B][Hkv][group x new tokens][slots], -inf where a slot is not seen, and what puts rows back."""
    b, i, slot = _rows(s)
    n, group = s["max_new"], s["hq"] // s["hkv"]
    q = torch.zeros(s["B"], n, s["hq"], D, device="cuda")
    q[b, i.long()] = s["q"].float()
    q = q.reshape(s["B"], n, s["hkv"], group, D).permute(0, 2, 3, 1, 4).reshape(s["B"], s["hkv"], group * n, D)
    last = torch.full((s["B"], n), -1, dtype=torch.int32, device="cuda")
    last[b, i.long()] = slot if s["causal"] else s["lens"][b] - 1
    x = torch.matmul(q, _dense(s, s["k_pages"]).transpose(2, 3)).mul_(s["scale"])
    seen = torch.arange(s["cap"], device="cuda") <= last[:, None, :, None]
    x.view(s["B"], s["hkv"] * group, n, s["cap"]).masked_fill_(~seen, -torch.inf)

    def back(y):  # [B][Hkv][group x new][w] -> [T][Hq][w]
        y = y.view(s["B"], s["hkv"], group, n, -1).permute(0, 3, 1, 2, 4).reshape(s["B"], n, s["hq"], -1)
        return y[b, i.long()]

    return x, back


def _attend(s):
    x, back = _scores(s)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(top.clamp(min=-3e38)).exp_()
    total = x.sum(-1, keepdim=True)
    out = torch.matmul(x, _dense(s, s["v_pages"])) / torch.where(total > 0, total, 1.0)
    return back(out).to(torch.bfloat16), back(top + total.log())[..., 0].contiguous()


def _extend(s):
    b, _, slot = _rows(s)
    page = s["table"][b, (slot // s["page"]).long()].long()
    at = (slot % s["page"]).long()
    q = _rotate(s["q"], s["cos"], s["sin"], s["positions"], s["interleaved"], False)
    s["k_pages"][page, :, at] = _rotate(s["k"], s["cos"], s["sin"], s["positions"], s["interleaved"], False)
    s["v_pages"][page, :, at] = s["v"]
    s["slot_pos"][b, :, slot.long()] = s["positions"][:, None]
    return q, s["k_pages"], s["v_pages"], s["slot_pos"]


def _weights(s):
    x, _ = _scores(s)
    b, i, _ = _rows(s)
    n, group = s["max_new"], s["hq"] // s["hkv"]
    lse = torch.full((s["B"], n, s["hq"]), torch.inf, device="cuda")
    lse[b, i.long()] = torch.where(s["lse"] == -torch.inf, torch.inf, s["lse"])
    lse = lse.view(s["B"], n, s["hkv"], group).permute(0, 2, 3, 1).reshape(s["B"], s["hkv"], group * n, 1)
    added = x.sub_(lse).exp_().sum(2)
    slots = torch.arange(s["cap"], device="cuda")[None, None]
    first_new = (s["lens"] - (s["q_start"][1:] - s["q_start"][:-1]))[:, None, None]
    total = torch.where(slots < first_new, s["acc"], 0.0) + added
    s["acc_out"].copy_(torch.where(slots < s["lens"][:, None, None], total, s["acc_out"]))
    return s["acc_out"]


def _evict(s):
    lens, slots = s["lens"][:, None, None], torch.arange(s["cap"], device="cuda")[None, None]
    live = slots < lens
    held = (s["slot_pos"] < s["sink"]) | (s["slot_pos"] >= s["next_pos"][:, None, None] - s["recent"])
    key = torch.where(live, torch.where(held, torch.inf, s["acc"]), -torch.inf)
    order = key.sort(dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(live.expand_as(key)).scatter_(-1, order[..., :s["budget"]], True) & live
    left = torch.clamp(lens, max=s["budget"])
    # the i-th slot below the new length that goes takes the i-th kept slot above it
    hole, mover = ~kept & (slots < left), kept & (slots >= left)
    src = mover.nonzero()
    dst = hole.nonzero()
    for name in ("k_pages", "v_pages"):
        rows = s[name][s["table"][src[:, 0], src[:, 2] // s["page"]].long(), src[:, 1], src[:, 2] % s["page"]]
        s[name][s["table"][dst[:, 0], dst[:, 2] // s["page"]].long(), dst[:, 1], dst[:, 2] % s["page"]] = rows
    for name, out in (("acc", "acc_out"), ("slot_pos", "pos_out")):
        x = s[name].clone()
        x[dst[:, 0], dst[:, 1], dst[:, 2]] = s[name][src[:, 0], src[:, 1], src[:, 2]]
        s[out].copy_(torch.where(slots < left, x, s[out]))
    s["lens_out"].copy_(left[:, 0, 0])
    return s["k_pages"], s["v_pages"], s["acc_out"], s["pos_out"], s["lens_out"]


def run(s):
    if own:
        return _run_own(s)
    if s["op"] == "rope":
        return s["out"].copy_(_rotate(s["x"], s["cos"], s["sin"], s["positions"], s["interleaved"], s["inverse"]))
    if s["op"] == "attend":
        out, lse = _attend(s)
        return (out, lse) if s["lse"] else out
    return {"extend": _extend, "weights": _weights, "evict": _evict}[s["op"]](s)


def _run_own(s):
    from llama3_8b_attention_optimize_b200 import kernels
    if s["op"] == "rope":
        return kernels.rope_positions(s["x"], s["positions"], s["cos"], s["sin"], interleaved=s["interleaved"],
                                      inverse=s["inverse"], out=s["out"])
    if s["op"] == "attend":
        out = kernels.attend_chunk(s["q"], s["k_pages"], s["v_pages"], s["table"], s["q_start"], s["lens"], causal=s["causal"],
                                   scale=s["scale"], max_q_len=s["max_new"], out=s["out"], lse=s["lse_out"])
        return (out, s["lse_out"]) if s["lse"] else out
    if s["op"] == "extend":
        kernels.kv_extend(s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["q_start"], s["lens"], s["positions"],
                          s["cos"], s["sin"], q=s["q"], q_out=s["q_out"], interleaved=s["interleaved"], slot_pos=s["slot_pos"])
        return s["q_out"], s["k_pages"], s["v_pages"], s["slot_pos"]
    if s["op"] == "weights":
        return kernels.attn_weight_sums(s["q"], s["k_pages"], s["table"], s["q_start"], s["lens"], s["lse"], s["acc"],
                                        causal=s["causal"], scale=s["scale"], max_q_len=s["max_new"], acc_out=s["acc_out"])
    kernels.kv_evict(s["k_pages"], s["v_pages"], s["table"], s["lens"], s["acc"], s["slot_pos"], s["next_pos"], s["budget"],
                     recent=s["recent"], sink=s["sink"], acc_out=s["acc_out"], slot_pos_out=s["pos_out"],
                     lens_out=s["lens_out"])
    return s["k_pages"], s["v_pages"], s["acc_out"], s["pos_out"], s["lens_out"]


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "rope":
        n = case["T"] * case["heads"]
        # read and write each value, one position and one table row a token; 3 operations a rotated value
        return {"bytes": n * case["dim"] * (8 if case["f32"] else 4) + case["T"] * (4 + 4 * case["rot"]),
                "flops": 3 * n * case["rot"]}
    new, old = _lengths(case)
    hkv, row = case["hkv"], D * 2
    if op == "evict":
        lens = [a for a in old]
        cut = [n for n in lens if n > case["budget"]]
        # every slot's weight and position are read, the kept ones written; about the share of the kept rows that
        # lies above the new length moves (read and written, keys and values)
        moved = sum((n - case["budget"]) * case["budget"] / n for n in cut)
        return {"bytes": hkv * (8 * sum(lens) + 8 * sum(min(n, case["budget"]) for n in lens) + 4 * row * moved),
                "flops": hkv * sum(lens)}
    T, hq = sum(new), case["hq"]
    if op == "extend":
        return {"bytes": T * (2 * (hq + 2 * hkv) * row + 4 + 4 * case["rot"] + 4 * hkv), "flops": 3 * T * (hq + hkv) * case["rot"]}
    pairs = sum(n * a + (n * (n + 1) // 2 if case["causal"] else n * n) for n, a in zip(new, old))
    if op == "attend":
        return {"bytes": 2 * T * hq * row + 2 * hkv * row * sum(n + a for n, a in zip(new, old)) + 4 * T * hq * case["lse"],
                "flops": 4 * D * hq * pairs}
    return {"bytes": T * hq * (row + 4) + hkv * (row + 8) * sum(n + a for n, a in zip(new, old)), "flops": 2 * D * hq * pairs}


# ------------------------------------------------------------------ the operators in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "rope":
        return _exact_rotate(s["x"], s)
    new, old = _lengths(case)
    hkv, page = case["hkv"], case["page"]
    if case["op"] == "extend":
        k, v, pos = s["k_pages"].to(f), s["v_pages"].to(f), s["slot_pos"]
        kr, t = _exact_rotate(s["k"], s), 0
        for b, (n, a) in enumerate(zip(new, old)):
            slot = torch.arange(a, a + n, device="cuda")
            pages = s["table"][b].long()[slot // page]
            k[pages, :, slot % page] = kr[t:t + n]
            v[pages, :, slot % page] = s["v"][t:t + n].to(f)
            pos[b, :, a:a + n] = s["positions"][t:t + n]
            t += n
        return _exact_rotate(s["q"], s), k, v, pos
    if case["op"] == "evict":
        return _exact_evict(s, old)
    hq = case["hq"]
    g, t = hq // hkv, 0
    out, lse = torch.zeros(s["tokens"], hq, D, dtype=f, device="cuda"), torch.full((s["tokens"], hq), -torch.inf, dtype=f, device="cuda")
    acc = torch.zeros(case["B"], hkv, s["cap"], dtype=f, device="cuda")
    for b, (n, a) in enumerate(zip(new, old)):
        L = n + a
        pages = s["table"][b, :-(-L // page)].long()
        slot = torch.arange(L, device="cuda")
        unseen = slot[None] > (torch.arange(a, L, device="cuda")[:, None] if case["causal"] else L)
        for h in range(hkv):
            k = s["k_pages"][pages, h].reshape(-1, D)[:L].to(f)
            q = s["q"][t:t + n, h * g:(h + 1) * g].to(f).transpose(0, 1)
            x = (q @ k.T * D ** -0.5).masked_fill(unseen, -torch.inf)
            if case["op"] == "weights":
                kept = s["acc"][b, h, :L].to(f).masked_fill(slot >= a, 0.0)
                acc[b, h, :L] = kept + (x - s["lse"][t:t + n, h * g:(h + 1) * g].to(f).T[..., None]).exp().sum((0, 1))
                continue
            norm = x.logsumexp(-1)
            lse[t:t + n, h * g:(h + 1) * g] = norm.T
            v = s["v_pages"][pages, h].reshape(-1, D)[:L].to(f)
            out[t:t + n, h * g:(h + 1) * g] = ((x - norm[..., None]).exp() @ v).transpose(0, 1)
        t += n
    if case["op"] == "weights":
        return acc
    return (out, lse) if case["lse"] else out


def _exact_rotate(x, s):
    y = x.to(torch.float64)
    rot = s["rot"]
    c, n = (w.to(torch.float64)[s["positions"].long()][:, None] for w in (s["cos"], s["sin"]))
    z = torch.complex(c, -n if s.get("inverse") else n)
    pairs = y[..., :rot].unflatten(-1, (-1, 2)) if s["interleaved"] else y[..., :rot].unflatten(-1, (2, -1)).transpose(-1, -2)
    turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * z)
    turned = turned if s["interleaved"] else turned.transpose(-1, -2)
    return torch.cat((turned.flatten(-2), y[..., rot:]), -1)


def _exact_evict(s, lens):
    f = torch.float64
    k, v = s["k_pages"].to(f), s["v_pages"].to(f)
    acc_out, pos_out = s["acc_out"].to(f), s["pos_out"].clone()
    for b, n in enumerate(lens):
        left = min(n, s["budget"])
        slot = torch.arange(n, device="cuda")
        pages, at = s["table"][b].long()[slot // s["page"]], slot % s["page"]
        for h in range(s["hkv"]):
            pos = s["slot_pos"][b, h, :n]
            rank = s["acc"][b, h, :n].to(f)
            rank[(pos < s["sink"]) | (pos >= n - s["recent"])] = torch.inf
            keep = torch.sort(-rank, stable=True).indices[:left].sort().values
            stay, move = keep[keep < left], keep[keep >= left]
            free = torch.ones(left, dtype=torch.bool, device="cuda")
            free[stay] = False
            to = free.nonzero()[:, 0]
            frm = torch.arange(left, device="cuda")
            frm[to] = move
            k[pages[to], h, at[to]] = k[pages[move], h, at[move]]
            v[pages[to], h, at[to]] = v[pages[move], h, at[move]]
            acc_out[b, h, :left] = s["acc"][b, h].to(f)[frm]
            pos_out[b, h, :left] = s["slot_pos"][b, h][frm]
    left = s["lens"].clamp(max=s["budget"])
    return k, v, acc_out, pos_out, left
