"""Cases that measure the KV-cache operators of the attention layers.

Four entry points on one cache descriptor, each measured alone:

  rope     rotary positions of a strided [tokens, heads, D] tensor
  append   rotary positions of new q and k, with k and v rounded into their
           f16 cache rows
  attn     attention of one new token per sequence over a prefix that the
           whole batch shares and the sequences' own cached tokens, with or
           without the accumulation of each cached token's attention weight
  evict    shrinking every sequence's cache to a budget by those weights

With ``own`` false, ``run`` computes the operator in elementary torch
operations; with ``own`` true it makes the library's calls.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
D = 128                                    # head_dim of the attention entries
DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# --------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------
def listed():
    return [
        # a prompt's q and k heads together, as one bf16 projection leaves them: half layout, half of the head
        dict(name="rope_prompt_bf16", op="rope", tokens=4096, heads=48, dim=128, rope=64, layout="half", dtype="bf16",
             gap=1024, scale=1.0, ext=0.0, first=0, back=False),
        # a long prompt far beyond the trained length: interleaved, whole head, YaRN scaling, fp32
        dict(name="rope_long_f32", op="rope", tokens=8192, heads=40, dim=128, rope=128, layout="interleaved",
             dtype="f32", gap=0, scale=0.125, ext=1.0, first=120000, back=False),
        # one decode step of 64 sequences: q rotated, k rotated and cached, v cached
        dict(name="append_step64", op="append", seqs=64, per_seq=1, ctx=512, kv=8, group=5, rope=64, layout="half",
             dtype="f32", scale=1.0, ext=0.0),
        # four prompts written into their caches (an odd length)
        dict(name="append_prompts_f16", op="append", seqs=4, per_seq=1999, ctx=2048, kv=8, group=4, rope=128,
             layout="interleaved", dtype="f16", scale=0.25, ext=0.0),
        # a single chat after a short system prompt: latency
        dict(name="attn_one", op="attn", seqs=1, prefix=512, ctx=256, lo=100, hi=100, kv=8, group=5, scored=False,
             decay=1.0),
        # a small batch, odd prefix, ragged turns
        dict(name="attn_b16_ragged", op="attn", seqs=16, prefix=2085, ctx=800, lo=1, hi=777, kv=8, group=4,
             scored=True, decay=1.0),
        # the usual serving batch: a long shared document, short own turns
        dict(name="attn_b64_shared8k", op="attn", seqs=64, prefix=8192, ctx=512, lo=130, hi=500, kv=8, group=5,
             scored=False, decay=1.0),
        # the largest batch: the shared part is bound by the tensor cores
        dict(name="attn_b256_shared8k", op="attn", seqs=256, prefix=8192, ctx=256, lo=60, hi=256, kv=8, group=5,
             scored=False, decay=1.0),
        # a few sequences over a very long shared document
        dict(name="attn_b8_shared128k", op="attn", seqs=8, prefix=131072, ctx=256, lo=17, hi=201, kv=8, group=4,
             scored=False, decay=1.0),
        # no shared part, full own caches, weights accumulated for the eviction
        dict(name="attn_b64_own4k_scored", op="attn", seqs=64, prefix=0, ctx=4096, lo=4096, hi=4096, kv=8, group=5,
             scored=True, decay=0.98),
        # one sequence over its budget by a few tokens: latency
        dict(name="evict_one", op="evict", seqs=1, ctx=1152, lo=1100, hi=1100, kv=8, budget=1024, sink=4, recent=64),
        # a ragged batch, some sequences below the budget
        dict(name="evict_b64_4k", op="evict", seqs=64, ctx=4352, lo=3900, hi=4352, kv=8, budget=4096, sink=4,
             recent=256),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "attn", "attn", "evict"])
    if op == "rope":
        dim = rng.choice([64, 80, 128, 128, 256])
        heads = rng.choice([1, 8, 32, 40, 48])
        top = max(1, min(16384, 8192 * 40 * 128 // (heads * dim)))
        scale = rng.choice([1.0, 1.0, 0.25, 0.125])
        return dict(op=op, tokens=_log_int(rng, 1, top), heads=heads, dim=dim,
                    rope=rng.choice([dim, dim // 2, dim // 4]), layout=rng.choice(["half", "interleaved"]),
                    dtype=rng.choice(["f32", "f16", "bf16"]), gap=rng.choice([0, 128, 1024]), scale=scale,
                    ext=rng.choice([0.0, 1.0]) if scale < 1.0 else 0.0, first=_log_int(rng, 1, 500000),
                    back=rng.random() < 0.25)
    kv = rng.choice([1, 2, 4, 8, 8])
    if op == "append":
        one = rng.random() < 0.5
        scale = rng.choice([1.0, 0.25])
        per = 1 if one else _log_int(rng, 2, 2000)
        return dict(op=op, seqs=_log_int(rng, 1, 256 if one else 4), per_seq=per, ctx=per + _log_int(rng, 1, 100),
                    kv=kv, group=rng.choice([1, 4, 5, 8]), rope=rng.choice([32, 64, 128]),
                    layout=rng.choice(["half", "interleaved"]), dtype=rng.choice(["f32", "f16", "bf16"]), scale=scale,
                    ext=rng.choice([0.0, 1.0]) if scale < 1.0 else 0.0)
    if op == "attn":
        group = rng.choice([1, 2, 3, 4, 5, 6, 7, 8, 16])
        seqs = _log_int(rng, 1, 256)
        rows = seqs * kv * group                       # q heads of the whole batch
        # the shared and the own part each up to half of the largest listed ones
        prefix = rng.choice([0, 1]) and _log_int(rng, 1, max(1, min(65536, 5120 * 8192 // rows)))
        ctx = _log_int(rng, 1, max(1, min(8192, 64 * 8 * 2048 // (seqs * kv))))
        hi = rng.randint(0 if prefix else 1, ctx)
        return dict(op=op, seqs=seqs, prefix=prefix, ctx=ctx, lo=rng.choice([0, hi // 2, hi]), hi=hi, kv=kv,
                    group=group, scored=rng.random() < 0.5, decay=rng.choice([0.0, 0.98, 1.0]))
    ctx = _log_int(rng, 64, 32768)
    budget = rng.randint(ctx // 2, ctx - 1)
    sink = rng.choice([0, 4])
    return dict(op=op, seqs=_log_int(rng, 1, max(1, min(64, 64 * 4352 // ctx))), ctx=ctx, lo=rng.randint(0, ctx),
                hi=ctx, kv=kv, budget=budget, sink=sink, recent=rng.randint(0, (budget - sink) // 2))


def _lens(case):
    """Evenly spread lengths lo..hi, so that the work is known from the case."""
    n, lo, hi = case["seqs"], case["lo"], case["hi"]
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def work(case):
    op = case["op"]
    if op == "rope":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2.0 * n * case["dim"] * SIZE[case["dtype"]] + 4 * case["tokens"],
                "flops": 3.0 * n * case["rope"]}
    if op == "append":
        t, hk, hq = case["seqs"] * case["per_seq"], case["kv"], case["kv"] * case["group"]
        e = SIZE[case["dtype"]]
        # q read and written, k and v read, their f16 rows written; position, sequence, slot
        return {"bytes": t * (2.0 * hq * D * e + 2 * hk * D * e + 2 * hk * D * 2 + 12),
                "flops": 3.0 * t * (hq + hk) * case["rope"]}
    if op == "attn":
        own_t, b, hq = sum(_lens(case)), case["seqs"], case["kv"] * case["group"]
        toks = case["prefix"] + own_t                   # cached tokens read once each
        return {"bytes": toks * case["kv"] * D * 4.0 + 8.0 * b * hq * D + (8.0 * own_t * case["kv"] if case["scored"]
                                                                          else 0.0),
                "flops": 4.0 * hq * D * (b * case["prefix"] + own_t)}
    tail = [max(0, n - case["budget"]) for n in _lens(case)]
    # moved rows: the protected newest, and of the others about the share that is kept
    moved = sum(min(t, case["recent"]) + max(0, t - case["recent"]) * case["budget"] / case["ctx"] for t in tail)
    return {"bytes": case["kv"] * (8.0 * sum(n for n, t in zip(_lens(case), tail) if t) + moved * (2 * 2 * D * 2 + 16)),
            "flops": float(case["kv"] * sum(_lens(case)) + 1)}


# --------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------
def _rope_case(case, dim):
    """The rotary parameters of a case: base 10^7 unscaled, 10^6 scaled; trained on 16384 positions."""
    return dict(layout=case["layout"], head_dim=dim, rope_dim=case["rope"], theta=1e7 if case["scale"] == 1.0 else 1e6,
                freq_scale=case["scale"], ext_factor=case["ext"], attn_factor=1.0, beta_fast=32.0, beta_slow=1.0,
                n_ctx_orig=16384)


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device=DEV, dtype=torch.float32 if dtype == torch.bfloat16 else dtype
                           ).to(dtype)

    st = dict(case=case)
    op = case["op"]
    if op == "rope":
        dt = DT[case["dtype"]]
        row = case["heads"] * case["dim"] + case["gap"]          # a slice of a wider projection
        st["wide"] = normal(case["tokens"], row, dtype=dt)
        st["x"] = st["wide"][:, :case["heads"] * case["dim"]].view(case["tokens"], case["heads"], case["dim"])
        st["pos"] = torch.arange(case["tokens"], device=DEV, dtype=torch.int32) + case["first"]
        st["out"] = torch.empty(case["tokens"], case["heads"], case["dim"], device=DEV, dtype=dt)
        st["rope"] = _rope_case(case, case["dim"])
        return st
    b, hk, ctx = case["seqs"], case["kv"], case["ctx"]
    if op == "append":
        t, hq, dt = b * case["per_seq"], hk * case["group"], DT[case["dtype"]]
        st["proj"] = normal(t, (hq + 2 * hk) * D, dtype=dt)      # q | k | v, one row a token
        st["q"] = st["proj"][:, :hq * D].view(t, hq, D)
        st["k"] = st["proj"][:, hq * D:(hq + hk) * D].view(t, hk, D)
        st["v"] = st["proj"][:, (hq + hk) * D:].view(t, hk, D)
        seq = torch.arange(b, device=DEV, dtype=torch.int32)
        start = torch.randint(0, ctx - case["per_seq"] + 1, (b,), generator=g, device=DEV, dtype=torch.int32)
        step = torch.arange(case["per_seq"], device=DEV, dtype=torch.int32)
        st["seq"] = seq[:, None].expand(b, case["per_seq"]).reshape(-1).contiguous()
        st["slot"] = (start[:, None] + step[None]).reshape(-1).contiguous()
        st["pos"] = st["slot"] + 40000
        st["k_cache"] = torch.zeros(b, ctx, hk, D, device=DEV, dtype=torch.float16)
        st["v_cache"] = torch.zeros(b, ctx, hk, D, device=DEV, dtype=torch.float16)
        st["len"] = (start + case["per_seq"]).to(torch.int32)
        st["weight"] = torch.rand(b, hk, ctx, generator=g, device=DEV)
        st["slot_pos"] = torch.full((b, hk, ctx), -1, device=DEV, dtype=torch.int32)
        st["out"] = torch.empty(t, hq, D, device=DEV, dtype=dt)
        st["rope"] = _rope_case(case, D)
        return st
    lens = torch.tensor(_lens(case), device=DEV, dtype=torch.int32)
    lens = lens[torch.randperm(b, generator=g, device=DEV)].contiguous()
    st["k_cache"] = normal(b, ctx, hk, D, dtype=torch.float16)   # slots past a length hold what was there before
    st["v_cache"] = normal(b, ctx, hk, D, dtype=torch.float16)
    if op == "attn":
        hq, p = hk * case["group"], case["prefix"]
        st["q"] = 1.5 * normal(b, hq, D)
        st["k_prefix"] = normal(p, hk, D, dtype=torch.float16) if p else None
        st["v_prefix"] = normal(p, hk, D, dtype=torch.float16) if p else None
        st["len"] = lens
        st["weight"] = torch.rand(b, hk, ctx, generator=g, device=DEV) if case["scored"] else None
        st["out"] = torch.empty(b, hq, D, device=DEV)
        return st
    # weights as they accumulate: a few large, many small, the slots of tokens just appended still zero;
    # positions as earlier evictions leave them: sinks in front, the newest at the end, the rest shuffled
    sink, recent = case["sink"], case["recent"]
    w = torch.rand(b, hk, ctx, generator=g, device=DEV).pow(6) * 8.0
    w = torch.where(torch.rand(b, hk, ctx, generator=g, device=DEV) < 0.02, torch.zeros_like(w), w)
    idx = torch.arange(ctx, device=DEV)
    n = lens[:, None, None].long()
    key = torch.rand(b, hk, ctx, generator=g, device=DEV)
    key = torch.where(idx < sink, idx * 1e-5 - 1.0, torch.where(idx >= n - recent, idx * 1e-5 + 1.0, key))
    at = key.argsort(dim=2).argsort(dim=2)
    st["slot_pos0"] = (at + (at >= sink) * 777).to(torch.int32).contiguous()
    st["weight0"], st["len0"] = w, lens
    st["pos"] = lens - 1 + 777
    st["weight"], st["slot_pos"], st["len"] = torch.empty_like(w), torch.empty_like(st["slot_pos0"]), lens.clone()
    return st


# --------------------------------------------------------------------------
# one pass
# --------------------------------------------------------------------------
def run(st):
    return {"rope": _run_rope, "append": _run_append, "attn": _run_attn, "evict": _run_evict}[st["case"]["op"]](st)


def _handles(st):
    """The library's descriptors over the state's tensors, built once, as a serving program keeps them."""
    if "handles" not in st:
        from leaninfer_b200 import ops
        rope = ops.Rope(**st["rope"]) if "rope" in st else None
        cache = None
        if "k_cache" in st:
            cache = ops.KVCache(st["k_cache"], st["v_cache"], st["len"], k_prefix=st.get("k_prefix"),
                                v_prefix=st.get("v_prefix"), weight=st.get("weight"), slot_pos=st.get("slot_pos"))
        st["handles"] = (ops, rope, cache)
    return st["handles"]


def _angles(rope, pos):
    """cos and sin of every (token, pair), scaled by the magnitude: [tokens, rope_dim / 2], from 64-bit angles."""
    d, base, scale = rope["rope_dim"], rope["theta"], rope["freq_scale"]
    i = torch.arange(d // 2, device=pos.device, dtype=torch.float64)
    freq = base ** (-2.0 * i / d)
    mag = rope["attn_factor"]
    coef = torch.full_like(freq, scale)
    if rope["ext_factor"] != 0.0:
        def dim_of(turns):
            return d * math.log(rope["n_ctx_orig"] / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(0.0, math.floor(dim_of(rope["beta_fast"]))), min(d - 1.0, math.ceil(dim_of(rope["beta_slow"])))
        keep = (1.0 - ((i - lo) / max(0.001, hi - lo)).clamp(0.0, 1.0)) * rope["ext_factor"]
        coef = scale * (1.0 - keep) + keep
        mag = mag * (1.0 + 0.1 * math.log(1.0 / scale))
    a = pos.double()[:, None] * (freq * coef)
    return (a.cos() * mag).float(), (a.sin() * mag).float()


def _rotate(x, rope, pos, back=False):
    """fp32 rotation of [tokens, heads, D]."""
    x = x.float()
    cos, sin = (t[:, None] for t in _angles(rope, pos))
    if back:
        sin = -sin
    d = rope["rope_dim"]
    if rope["layout"] == "half":
        a, b = x[..., :d // 2], x[..., d // 2:d]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., d:]], -1)
    a, b = x[..., 0:d:2], x[..., 1:d:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., d:]], -1)


def _run_rope(st):
    if own:
        ops, rope, _ = _handles(st)
        return ops.rope(rope, st["x"], st["pos"], out=st["out"], transpose=st["case"]["back"])
    return _rotate(st["x"], st["rope"], st["pos"], st["case"]["back"]).to(st["x"].dtype)


def _run_append(st):
    if own:
        _, rope, cache = _handles(st)
        q = cache.append(st["k"], st["v"], st["pos"], q=st["q"], rope=rope, seq=st["seq"], slot=st["slot"],
                         q_out=st["out"])
    else:
        q = _rotate(st["q"], st["rope"], st["pos"]).to(st["q"].dtype)
        seq, slot = st["seq"].long(), st["slot"].long()
        st["k_cache"][seq, slot] = _rotate(st["k"], st["rope"], st["pos"]).half()
        st["v_cache"][seq, slot] = st["v"].float().half()
        st["weight"][seq, :, slot] = 0.0
        st["slot_pos"][seq, :, slot] = st["pos"][:, None].expand(-1, st["case"]["kv"])
    return dict(q=q, k_cache=st["k_cache"], v_cache=st["v_cache"], weight=st["weight"], slot_pos=st["slot_pos"])


def _run_attn(st):
    case = st["case"]
    if own:
        _, _, cache = _handles(st)
        o = cache.decode(st["q"], scale=D ** -0.5, decay=case["decay"], out=st["out"])
    else:
        b, hk, gr, ctx, p = case["seqs"], case["kv"], case["group"], case["ctx"], case["prefix"]
        q = (st["q"] * D ** -0.5).view(b, hk, gr, D)
        valid = torch.arange(ctx, device=DEV) < st["len"][:, None]                       # [b, ctx]
        s = q @ st["k_cache"].float().permute(0, 2, 3, 1)                                # [b, hk, gr, ctx]
        s = s.masked_fill(~valid[:, None, None], float("-inf"))
        m = s.amax(-1, keepdim=True)
        if p:
            qp = q.transpose(0, 1).reshape(hk, b * gr, D)
            sp = (qp @ st["k_prefix"].float().permute(1, 2, 0)).view(hk, b, gr, p).transpose(0, 1)
            m = torch.maximum(m, sp.amax(-1, keepdim=True))
        m = torch.where(m.isinf(), torch.zeros_like(m), m)                               # a row without tokens
        e = (s - m).exp()
        tot = e.sum(-1, keepdim=True)
        v = st["v_cache"].float().masked_fill(~valid[:, :, None, None], 0.0)
        o = e @ v.permute(0, 2, 1, 3)
        if p:
            ep = (sp - m).exp()
            tot = tot + ep.sum(-1, keepdim=True)
            epj = ep.transpose(0, 1).reshape(hk, b * gr, p)
            o = o + (epj @ st["v_prefix"].float().permute(1, 0, 2)).view(hk, b, gr, D).transpose(0, 1)
        tot = torch.where(tot == 0, torch.ones_like(tot), tot)
        o = (o / tot).reshape(b, hk * gr, D)
        if case["scored"]:
            w = st["weight"]
            w.copy_(torch.where(valid[:, None], case["decay"] * w + (e / tot).sum(2), w))
    return dict(o=o, weight=st["weight"]) if case["scored"] else o


def _run_evict(st):
    case = st["case"]
    # the step before the eviction leaves new weights, positions and lengths: each pass begins from the same ones
    st["weight"].copy_(st["weight0"])
    st["slot_pos"].copy_(st["slot_pos0"])
    st["len"].copy_(st["len0"])
    if own:
        _, _, cache = _handles(st)
        cache.evict(st["pos"], case["budget"], n_sink=case["sink"], n_recent=case["recent"])
    else:
        b, hk, ctx, budget = case["seqs"], case["kv"], case["ctx"], case["budget"]
        w, sp, n = st["weight"], st["slot_pos"], st["len"].long()[:, None, None]
        idx = torch.arange(ctx, device=DEV).expand(b, hk, ctx)
        valid = idx < n
        safe = (sp < case["sink"]) | (sp > st["pos"][:, None, None] - case["recent"])
        key = torch.where(w > 0, w, torch.zeros_like(w))
        key = torch.where(safe, torch.full_like(key, float("inf")), key)
        key = torch.where(valid, key, torch.full_like(key, -1.0))
        order = key.sort(dim=2, descending=True, stable=True).indices
        rank = torch.empty_like(order).scatter_(2, order, idx)
        new = n.clamp(max=budget)
        keep = rank < new
        hole, src = ~keep & (idx < new), keep & (idx >= new)
        most = min(budget, ctx - budget)                      # moves a (sequence, head) can need
        # the r-th freed slot and the r-th kept row behind the budget, ascending; where there is none: slot 0 onto itself
        def ranked(mask):
            r = torch.where(mask, mask.cumsum(2) - 1, torch.full_like(idx, most))
            return torch.zeros(b, hk, most + 1, device=DEV, dtype=torch.long).scatter_(2, r, idx)[..., :most]
        moves = hole.sum(2, keepdim=True) > torch.arange(most, device=DEV)
        dst, frm = (torch.where(moves, ranked(x), torch.zeros_like(moves, dtype=torch.long)) for x in (hole, src))
        # slot 0 may be filled by a move as well: those that do nothing write its new row
        at0 = torch.where(moves & (dst == 0), frm, torch.zeros_like(frm)).amax(2, keepdim=True)
        frm = torch.where(moves, frm, at0.expand_as(frm))
        bi, hi = torch.arange(b, device=DEV)[:, None, None], torch.arange(hk, device=DEV)[None, :, None]
        kc, vc = st["k_cache"], st["v_cache"]
        kc[bi, dst, hi], vc[bi, dst, hi] = kc[bi, frm, hi], vc[bi, frm, hi]
        w[bi, hi, dst], sp[bi, hi, dst] = w[bi, hi, frm], sp[bi, hi, frm]
        st["len"].copy_(new.view(-1))
    return dict(k_cache=st["k_cache"], v_cache=st["v_cache"], weight=st["weight"], slot_pos=st["slot_pos"],
                len=st["len"])


# --------------------------------------------------------------------------
# the definitions, in 64 bits
# --------------------------------------------------------------------------
def _exact_rope(x, rope, pos, back=False):
    """Rotation as a complex product, pair by pair."""
    d, base = rope["rope_dim"], float(rope["theta"])
    y = x.double().clone()
    sign = -1.0 if back else 1.0
    for i in range(d // 2):
        f = math.exp(-2.0 * i / d * math.log(base))
        mag, c = rope["attn_factor"], rope["freq_scale"]
        if rope["ext_factor"] != 0.0:
            lo, hi = (d * math.log(rope["n_ctx_orig"] / (t * 2 * math.pi)) / (2 * math.log(base))
                      for t in (rope["beta_fast"], rope["beta_slow"]))
            lo, hi = max(0, math.floor(lo)), min(d - 1, math.ceil(hi))
            r = rope["ext_factor"] * (1 - min(1.0, max(0.0, (i - lo) / max(0.001, hi - lo))))
            c = c * (1 - r) + r
            mag = mag * (1 + 0.1 * math.log(1 / rope["freq_scale"]))
        u, v = (i, i + d // 2) if rope["layout"] == "half" else (2 * i, 2 * i + 1)
        z = torch.complex(x[..., u].double(), x[..., v].double())
        z = z * torch.polar(torch.full_like(pos, 1, dtype=torch.float64) * mag, sign * pos.double() * f * c)[:, None]
        y[..., u], y[..., v] = z.real, z.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "rope":
        return _exact_rope(st["x"], st["rope"], st["pos"], case["back"])
    if op == "append":
        kc, vc, w = st["k_cache"].double(), st["v_cache"].double(), st["weight"].double()
        k = _exact_rope(st["k"], st["rope"], st["pos"])
        at = st["seq"].long() * case["ctx"] + st["slot"].long()
        kc.view(-1, case["kv"], D)[at] = k
        vc.view(-1, case["kv"], D)[at] = st["v"].double()
        for j in range(case["kv"]):
            w[st["seq"].long(), j, st["slot"].long()] = 0.0
        return dict(q=_exact_rope(st["q"], st["rope"], st["pos"]), k_cache=kc, v_cache=vc, weight=w, slot_pos=None)
    if op == "attn":
        o = torch.zeros(case["seqs"], case["kv"] * case["group"], D, device=DEV, dtype=torch.float64)
        w = st["weight"].double() if case["scored"] else None
        lens = st["len"].tolist()
        for j in range(case["kv"]):
            hs = slice(j * case["group"], (j + 1) * case["group"])
            kp, vp = ((t[:, j].double() for t in (st["k_prefix"], st["v_prefix"])) if case["prefix"] else (None, None))
            for i, n in enumerate(lens):
                k, v = st["k_cache"][i, :n, j].double(), st["v_cache"][i, :n, j].double()
                if case["prefix"]:
                    k, v = torch.cat([kp, k]), torch.cat([vp, v])
                if k.shape[0]:
                    s = st["q"][i, hs].double() @ k.T / math.sqrt(D)
                    pr = (s - s.logsumexp(-1, keepdim=True)).exp()
                    o[i, hs] = pr @ v
                    if case["scored"] and n:
                        w[i, j, :n] = case["decay"] * w[i, j, :n] + pr[:, case["prefix"]:].sum(0)
        return dict(o=o, weight=w) if case["scored"] else o
    kc, vc = st["k_cache"], st["v_cache"]
    w, sp, lens, budget = st["weight0"].double(), st["slot_pos0"], st["len0"].tolist(), case["budget"]
    for i, n in enumerate(lens):
        for j in range(case["kv"]):
            if n <= budget:
                continue
            free = (sp[i, j, :n] < case["sink"]) | (sp[i, j, :n] > int(st["pos"][i]) - case["recent"])
            score = torch.where(free, math.inf, w[i, j, :n].clamp(min=0.0))
            cut = score.sort(descending=True).values[budget - 1]
            kept = score > cut
            ties = (score == cut).nonzero().view(-1)[:budget - int(kept.sum())]
            kept[ties] = True
            dst, frm = (~kept[:budget]).nonzero().view(-1), budget + kept[budget:].nonzero().view(-1)
            for t in (kc[i, :, j], vc[i, :, j], w[i, j], sp[i, j]):
                t[dst] = t[frm]
    return dict(k_cache=kc, v_cache=vc, weight=w, slot_pos=None, len=None)
