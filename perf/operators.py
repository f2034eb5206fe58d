"""What is measured of the bounded KV cache: the store of normalised and rotated keys, the attention that accumulates the weight every
cached position draws, and the eviction by that weight.  `own` False: plain torch; True: the framework's entry points (llm_amd.ops).

Layouts: q [seq, head, token, d] for the attention and [seq, token, head, d] before it; caches [seq, kv head, slot, row]."""
import math

import torch

own = False

F32, F16, Q8_0, Q4_0, BF16 = 0, 1, 8, 2, 30            # ggml type ids
NAMES = {"f16": F16, "bf16": BF16, "q8_0": Q8_0, "q4_0": Q4_0}
EPS = 1e-6
DECAY = 0.95                                          # of the mass with every step


def listed():
    return [
        # a decode step of one sequence, heads of an 8B model: latency only
        _store("store_step_f16", 1, 1, 32, 8, 128, 2048, "f16"),
        # a decode step of 16 sequences, heads of a 70B model, q8_0 cache, every head into a slot of its own
        _store("store_16_seqs_q8_0", 16, 1, 64, 8, 128, 512, "q8_0"),
        # an odd prompt, small heads, adjacent pairs rotated, half of each head only
        _store("store_prompt_1111_bf16", 1, 1111, 24, 4, 96, 1200, "bf16", n_dims=48, mode=0, base=10000.0),
        # a long prompt far into its context, heads of a 70B model
        _store("store_prompt_8192_f16", 1, 8192, 64, 8, 128, 8192, "f16", start=100000),
        # decode against a short cache: latency only
        _attend("attend_step_512_f16", 1, 1, 512, 32, 8, 128, "f16"),
        # decode against a long cache, heads of a 70B model
        _attend("attend_step_32768_f16", 1, 1, 32768, 64, 8, 128, "f16"),
        # 8 sequences of different lengths, q8_0 cache
        _attend("attend_8_seqs_4099_q8_0", 8, 1, 4099, 32, 8, 128, "q8_0"),
        # a speculative step of 5 tokens, q4_0 cache
        _attend("attend_5_tokens_8192_q4_0", 1, 5, 8192, 32, 8, 128, "q4_0"),
        # the last 64 tokens of a long prompt score its positions
        _observe("observe_window_16384_f16", 1, 64, 16384, 32, 8, 128, "f16"),
        # a whole prompt of odd length scores itself, causal
        _observe("observe_prompt_2047_bf16", 1, 2047, 2047, 32, 8, 128, "bf16"),
        # 16 sequences at their budget: the one slot each head gives to the next token
        _evict("evict_step_2049", 16, 2049, 2048, 8, 128, "f16", False),
        # a long prompt's cache reduced to an eighth
        _evict("evict_prompt_32768_f16", 1, 32768, 4096, 8, 128, "f16", True),
    ]


def _store(name, seqs, n, heads, kv_heads, d, slots, kv, n_dims=None, mode=2, base=1000000.0, start=1000):
    return dict(name=name, op="store", seqs=seqs, n=n, heads=heads, kv_heads=kv_heads, d=d, slots=slots, kv=kv, n_dims=n_dims or d, mode=mode, base=base, start=start)


def _attend(name, seqs, n, n_kv, heads, kv_heads, d, kv):
    return dict(name=name, op="attend", seqs=seqs, n=n, n_kv=n_kv, heads=heads, kv_heads=kv_heads, d=d, kv=kv)


def _observe(name, seqs, n, n_kv, heads, kv_heads, d, kv):
    return dict(name=name, op="observe", seqs=seqs, n=n, n_kv=n_kv, heads=heads, kv_heads=kv_heads, d=d, kv=kv)


def _evict(name, seqs, n_kv, n_keep, kv_heads, d, kv, gather):
    return dict(name=name, op="evict", seqs=seqs, n_kv=n_kv, n_keep=n_keep, kv_heads=kv_heads, d=d, kv=kv, gather=gather)


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 6, 8])
    op = rng.choice(["store", "attend", "attend", "observe", "evict"])
    d = rng.choice([64, 128, 128, 96, 256]) if op != "store" else rng.choice([64, 80, 96, 128, 128, 256])
    kv = rng.choice(["f16", "bf16", "q8_0", "q4_0"])
    if op == "store":
        kv = "f16" if d % 32 and kv == "q8_0" or kv == "q4_0" else kv
        seqs, n = rng.choice([(1, log(1, 4096)), (1, log(1, 4096)), (log(2, 24), 1)])
        c = _store("", seqs, n, heads, kv_heads, d, n + log(1, 500), kv, mode=rng.choice([0, 2, 2]), base=rng.choice([1e4, 5e5, 1e6]), start=log(1, 120000))
        c["n_dims"] = rng.choice([d, d, d // 2 // 8 * 8])
    elif op == "attend":
        seqs = rng.choice([1, 1, log(2, 12)])
        c = _attend("", seqs, rng.choice([1, 1, 1, 2, 3, 4, 5, 6, 7, 8]), log(1, 32768 // seqs), heads, kv_heads, d, kv)
    elif op == "observe":
        n_kv = log(2, 16384)
        n = min(n_kv, log(1, max(1, min(2047, 2 ** 20 // n_kv))))
        c = _observe("", 1, n, n_kv, heads, kv_heads, d, kv)
    else:
        n_kv = log(2, 32768)
        seqs, gather = rng.choice([(1, True), (log(2, 8), False), (log(2, 4), True)])
        c = _evict("", seqs, n_kv, max(1, int(n_kv * rng.uniform(0.05, 1.0))), kv_heads, d, kv, gather)
    c.pop("name")
    return c


def _lengths(c):
    """Slots in use of every sequence: the first is full, the others shorter."""
    return [max(1, c["n_kv"] - i * c["n_kv"] // (2 * c["seqs"])) for i in range(c["seqs"])]


def _recent(c):
    """Of the kept slots a quarter for the newest positions and at most 4 for the first ones."""
    return c["n_keep"] // 4, min(4, c["n_keep"] - c["n_keep"] // 4)


# ---- inputs -------------------------------------------------------------------------------------------------------------------------

def _cache(shape, kv, g, scale=1.0):
    """Random rows [.., d] in the cache's own format: float values, or ggml blocks of 32 as bytes."""
    x = torch.randn(shape, device="cuda", generator=g)
    if scale != 1.0:
        x = x * scale
    if kv in ("f16", "bf16"):
        return x.to(torch.float16 if kv == "f16" else torch.bfloat16)
    return _blocks(x, kv)


def _blocks(x, kv):
    """f32 values -> blocks of 32: q8_0 (f16 scale, 32 int8) or q4_0 (f16 scale, 16 bytes of low and high nibbles)."""
    b = x.float().reshape(*x.shape[:-1], -1, 32)
    if kv == "q8_0":
        d = b.abs().amax(-1, keepdim=True) / 127.0
        t = b * torch.where(d > 0, 1.0 / d, torch.zeros_like(d))
        q = torch.trunc(t + torch.copysign(torch.full_like(t, 0.5), t)).to(torch.int8).view(torch.uint8)
    else:
        at = b.abs().argmax(-1, keepdim=True)
        d = b.gather(-1, at) / -8.0
        t = torch.where(d != 0, b * (1.0 / d), torch.zeros_like(b))
        u = torch.clamp(torch.trunc(t + 8.5), max=15.0).to(torch.uint8)
        q = u[..., :16] | (u[..., 16:] << 4)
    return torch.cat([d.to(torch.float16).view(torch.uint8), q], -1).reshape(*x.shape[:-1], -1)


def _values(rows, kv, to=torch.float32):
    """The values that a cache's rows stand for."""
    if kv in ("f16", "bf16"):
        return rows.to(to)
    size = 34 if kv == "q8_0" else 18
    b = rows.reshape(*rows.shape[:-1], -1, size)
    d = b[..., :2].contiguous().view(torch.float16).to(to)
    q = b[..., 2:].contiguous()
    q = q.view(torch.int8).to(to) if kv == "q8_0" else torch.cat([q & 15, q >> 4], -1).to(to) - 8.0
    return (d * q).reshape(*rows.shape[:-1], -1)


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "store":
        S, n, H, HK, d = c["seqs"], c["n"], c["heads"], c["kv_heads"], c["d"]
        s["q"] = torch.randn((S, n, H, d), device="cuda", generator=g) * 3.0
        s["k"] = torch.randn((S, n, HK, d), device="cuda", generator=g) * 3.0
        s["v"] = torch.randn((S, n, HK, d), device="cuda", generator=g)
        s["q_norm"] = 1.0 + 0.3 * torch.randn(d, device="cuda", generator=g)
        s["k_norm"] = 1.0 + 0.3 * torch.randn(d, device="cuda", generator=g)
        s["pos"] = (torch.arange(n, device="cuda", dtype=torch.int32) + c["start"]).expand(S, n).contiguous()
        # a free slot for every token: one after the other for a prompt, anywhere (the slot each head evicted) for a step
        first = torch.randint(0, c["slots"] - n + 1, (S, HK, 1), device="cuda", generator=g) if n == 1 else torch.zeros((S, HK, 1), device="cuda", dtype=torch.int64)
        s["rows"] = (first + torch.arange(n, device="cuda")).to(torch.int32)
        s["k_cache"] = _cache((S, HK, c["slots"], d), c["kv"], g)
        s["v_cache"] = _cache((S, HK, c["slots"], d), c["kv"], g)
        s["slot_pos"] = torch.arange(c["slots"], device="cuda", dtype=torch.int32).expand(S, HK, -1).contiguous()
        s["slot_mass"] = torch.rand((S, HK, c["slots"]), device="cuda", generator=g)
    elif c["op"] in ("attend", "observe"):
        S, n, H, HK, d, n_kv = c["seqs"], c["n"], c["heads"], c["kv_heads"], c["d"], c["n_kv"]
        s["q"] = torch.randn((S, H, n, d), device="cuda", generator=g) * 1.5
        s["k"] = _cache((S, HK, n_kv, d), c["kv"], g)
        if c["op"] == "attend":
            s["v"] = _cache((S, HK, n_kv, d), c["kv"], g)
        # the last n tokens of every sequence, each sees what is before it; slots behind the sequence are masked
        j, i = torch.arange(n_kv, device="cuda"), torch.arange(n, device="cuda")
        L = torch.tensor(_lengths(c), device="cuda")
        seen = j[None, None, :] < torch.clamp(L[:, None, None] - (n - 1 - i)[None, :, None], min=1)
        s["mask"] = torch.where(seen, 0.0, float("-inf")).to(torch.float16).contiguous()
        if c["op"] == "attend":                          # what some earlier steps of the same size left
            s["mass"] = torch.rand((S, HK, n_kv), device="cuda", generator=g) ** 4 * (8.0 * n * (H // HK) / n_kv)
        s["scale"] = 1.0 / math.sqrt(d)
    else:
        S, HK, d, n_kv = c["seqs"], c["kv_heads"], c["d"], c["n_kv"]
        L = _lengths(c)
        s["n_used"] = torch.tensor(L, device="cuda", dtype=torch.int32)
        s["n_past"] = torch.tensor([2 * n for n in L], device="cuda", dtype=torch.int32)
        mass = torch.rand((S, HK, n_kv), device="cuda", generator=g) ** 6 * 20.0
        s["mass"] = torch.where(torch.rand((S, HK, n_kv), device="cuda", generator=g) < 0.05, torch.zeros_like(mass), mass)   # never looked at
        # positions survive earlier evictions in any order: distinct, below n_past
        r = torch.rand((S, HK, n_kv), device="cuda", generator=g)
        used = torch.arange(n_kv, device="cuda")[None, None, :] < s["n_used"][:, None, None]
        rank = torch.where(used, r, torch.full_like(r, 2.0)).argsort(-1).argsort(-1)
        s["slot_pos"] = (2 * rank + (r > 0.5)).to(torch.int32)
        if c["gather"]:
            s["k"] = _cache((S, HK, n_kv, d), c["kv"], g)
            s["v"] = _cache((S, HK, n_kv, d), c["kv"], g)
            s["k_out"] = torch.zeros((S, HK, c["n_keep"], s["k"].shape[-1]), dtype=s["k"].dtype, device="cuda")
            s["v_out"] = torch.zeros_like(s["k_out"])
    return s


# ---- one pass -----------------------------------------------------------------------------------------------------------------------

def run(state):
    s, c = state, state["case"]
    if own:
        return _own(s, c)
    return {"store": _plain_store, "attend": _plain_attend, "observe": _plain_observe, "evict": _plain_evict}[c["op"]](s, c)


def _own(s, c):
    from llm_amd import ops

    t = NAMES[c["kv"]]
    if c["op"] == "store":
        q = ops.qk_norm_rope(s["q"], s["k"], s["v"], s["q_norm"], s["k_norm"], EPS, s["pos"], s["k_cache"], s["v_cache"], t, rows=s["rows"],
                             slot_pos=s["slot_pos"], slot_mass=s["slot_mass"], n_dims=c["n_dims"], mode=c["mode"], freq_base=c["base"])
        k, v = s["k_cache"], s["v_cache"]
        if c["kv"] == "q8_0":
            shape = (c["seqs"], c["kv_heads"], c["slots"], c["d"])
            k, v = (ops.dequantize(t, x, math.prod(shape)).view(shape).to(torch.float16) for x in (k, v))
        return {"q": q, "k": k, "v": v, "slot_pos": s["slot_pos"], "slot_mass": s["slot_mass"]}
    if c["op"] == "attend":
        dst, mass = ops.flash_attn_ext_mass(s["q"], s["k"], s["v"], s["mask"], t, s["scale"], mass=s["mass"], decay=DECAY)
        return {"dst": dst, "mass": mass}
    if c["op"] == "observe":
        return {"mass": ops.attn_mass(s["q"], s["k"], s["mask"], t, s["scale"])}
    recent, sink = _recent(c)
    if not c["gather"]:
        kept, evicted = ops.kv_evict(s["mass"], s["slot_pos"], s["n_past"], c["n_keep"], n_sink=sink, n_recent=recent, n_used=s["n_used"])
        return {"kept": kept, "evicted": evicted}
    kept, evicted, mass, pos = ops.kv_evict(s["mass"], s["slot_pos"], s["n_past"], c["n_keep"], n_sink=sink, n_recent=recent, n_used=s["n_used"],
                                            k=s["k"], v=s["v"], type_kv=t, d=c["d"], k_out=s["k_out"], v_out=s["v_out"])
    return {"kept": kept, "evicted": evicted, "mass": mass, "slot_pos": pos, "k": s["k_out"], "v": s["v_out"]}




def _plain_norm(x, w):
    x = x.float()
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w


def _plain_rotate(x, cos, sin, n_dims, mode):
    """x [seq, token, head, d]; pairs (2i, 2i + 1) in mode 0, (i, i + n_dims / 2) in mode 2; features past n_dims stay."""
    r = x[..., :n_dims]
    a, b = (r[..., 0::2], r[..., 1::2]) if mode == 0 else (r[..., : n_dims // 2], r[..., n_dims // 2:])
    y, z = a * cos - b * sin, a * sin + b * cos
    y = torch.stack([y, z], -1).flatten(-2) if mode == 0 else torch.cat([y, z], -1)
    return torch.cat([y, x[..., n_dims:]], -1)


def _plain_store(s, c):
    freq = c["base"] ** (-2.0 * torch.arange(c["n_dims"] // 2, device="cuda", dtype=torch.float64) / c["n_dims"])
    angle = s["pos"].double()[:, :, None, None] * freq          # far positions: in 64 bits
    cos, sin = angle.cos().float(), angle.sin().float()
    q = _plain_rotate(_plain_norm(s["q"], s["q_norm"]), cos, sin, c["n_dims"], c["mode"])
    k = _plain_rotate(_plain_norm(s["k"], s["k_norm"]), cos, sin, c["n_dims"], c["mode"])
    rows = s["rows"].long()
    at = (torch.arange(c["seqs"], device="cuda")[:, None, None], torch.arange(c["kv_heads"], device="cuda")[None, :, None], rows)
    for cache, x in ((s["k_cache"], k), (s["v_cache"], s["v"])):
        x = x.transpose(1, 2)
        cache[at] = x.to(cache.dtype) if c["kv"] != "q8_0" else _blocks(x, "q8_0")
    s["slot_pos"][at] = s["pos"][:, None, :].expand(-1, c["kv_heads"], -1)
    s["slot_mass"][at] = 0.0
    k, v = s["k_cache"], s["v_cache"]
    if c["kv"] == "q8_0":
        k, v = _values(k, "q8_0").to(torch.float16), _values(v, "q8_0").to(torch.float16)
    return {"q": q.transpose(1, 2).contiguous(), "k": k, "v": v, "slot_pos": s["slot_pos"], "slot_mass": s["slot_mass"]}


def _plain_weights(s, c):
    """exp(logits - max) [seq, kv head, group, token, slot] and their sums; rows that see nothing have none."""
    S, n, H, HK, d, n_kv = c["seqs"], c["n"], c["heads"], c["kv_heads"], c["d"], c["n_kv"]
    k = _values(s["k"], c["kv"])
    x = torch.matmul(s["q"].reshape(S, HK, H // HK * n, d), k.transpose(-1, -2)).reshape(S, HK, H // HK, n, n_kv)
    x = x * s["scale"] + s["mask"].float()[:, None, None]
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == float("-inf"), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p, torch.where(total > 0, 1.0 / total, torch.zeros_like(total))


def _plain_attend(s, c):
    S, n, H, HK, d, n_kv = c["seqs"], c["n"], c["heads"], c["kv_heads"], c["d"], c["n_kv"]
    p, r = _plain_weights(s, c)
    o = torch.matmul(p.reshape(S, HK, H // HK * n, n_kv), _values(s["v"], c["kv"])).reshape(S, HK, H // HK, n, d) * r
    return {"dst": o.reshape(S, H, n, d).transpose(1, 2).contiguous(), "mass": DECAY * s["mass"] + (p * r).sum((2, 3))}


def _plain_observe(s, c):
    p, r = _plain_weights(s, c)
    return {"mass": (p * r).sum((2, 3))}


def _plain_evict(s, c):
    S, HK, n_kv, n_keep = c["seqs"], c["kv_heads"], c["n_kv"], c["n_keep"]
    recent, sink = _recent(c)
    j = torch.arange(n_kv, device="cuda")
    used = j[None, None, :] < s["n_used"][:, None, None]
    safe = (s["slot_pos"] < sink) | (s["slot_pos"] >= s["n_past"][:, None, None] - recent)
    key = torch.where(safe, torch.full_like(s["mass"], float("inf")), s["mass"]).double()
    key = torch.where(used, key, torch.full_like(key, float("-inf")))
    order = key.sort(dim=-1, descending=True, stable=True).indices       # equal masses: the lower slot first
    n = torch.clamp(s["n_used"], max=n_keep)[:, None, None]
    slot = torch.arange(n_kv, device="cuda")[None, None, :]
    keep = torch.zeros((S, HK, n_kv), dtype=torch.bool, device="cuda").scatter_(-1, order, (slot < n).expand(S, HK, -1))
    kept = _ascending(keep, n_keep)
    evicted = _ascending(used & ~keep, max(0, n_kv - n_keep))
    if not c["gather"]:
        return {"kept": kept, "evicted": evicted}
    there = kept >= 0
    at = kept.long().clamp(min=0)
    mass = torch.where(there, s["mass"].gather(-1, at), torch.zeros((), device="cuda"))
    pos = torch.where(there, s["slot_pos"].gather(-1, at), torch.full((), -1, dtype=torch.int32, device="cuda"))
    seq, head = torch.arange(S, device="cuda")[:, None, None], torch.arange(HK, device="cuda")[None, :, None]
    for x, y in ((s["k"], s["k_out"]), (s["v"], s["v_out"])):
        y.copy_(torch.where(there[..., None], x[seq, head, at], y))
    return {"kept": kept, "evicted": evicted, "mass": mass, "slot_pos": pos, "k": s["k_out"], "v": s["v_out"]}


def _ascending(chosen, n):
    """The chosen slots of every row in ascending order, n of them, -1 behind the last."""
    n_kv = chosen.shape[-1]
    j = torch.arange(n_kv, device=chosen.device)
    x = torch.where(chosen, j, torch.full_like(j, n_kv)).sort(-1).values[..., :n]
    x = torch.cat([x, x.new_full((*x.shape[:-1], max(0, n - n_kv)), n_kv)], -1)
    return torch.where(x < n_kv, x, torch.full_like(x, -1)).to(torch.int32)


# ---- what a pass cannot do without --------------------------------------------------------------------------------------------------

def _row_bytes(c):
    return c["d"] * {"f16": 2, "bf16": 2, "q8_0": 34 / 32, "q4_0": 18 / 32}[c["kv"]]


def work(case):
    c = case
    if c["op"] == "store":
        tokens = c["seqs"] * c["n"]
        values = tokens * (c["heads"] + c["kv_heads"]) * c["d"]
        return {"bytes": 4 * values + 4 * tokens * c["kv_heads"] * c["d"] + 4 * tokens * c["heads"] * c["d"] + tokens * c["kv_heads"] * (2 * _row_bytes(c) + 12),
                "flops": 10 * values}
    if c["op"] in ("attend", "observe"):
        rows = sum(_lengths(c))
        # every query sees what is before it: of a prompt's own square that is half
        pairs = sum(sum(max(1, L - (c["n"] - 1 - i)) for i in range(c["n"])) for L in _lengths(c)) * c["heads"]
        q = 4 * c["seqs"] * c["heads"] * c["n"] * c["d"]
        mass = (8 if c["op"] == "attend" else 4) * c["seqs"] * c["kv_heads"] * c["n_kv"]
        mask = 2 * c["seqs"] * c["n"] * c["n_kv"]
        kv = rows * c["kv_heads"] * _row_bytes(c)
        if c["op"] == "attend":
            return {"bytes": 2 * kv + 2 * q + mass + mask, "flops": 4 * pairs * c["d"]}
        return {"bytes": kv + q + mass + mask, "flops": 2 * pairs * c["d"]}
    moved = sum(min(L, c["n_keep"]) for L in _lengths(c)) * c["kv_heads"]
    bytes_ = 8 * c["kv_heads"] * sum(_lengths(c)) + 4 * c["seqs"] * c["kv_heads"] * max(c["n_kv"], c["n_keep"])
    return {"bytes": bytes_ + (moved * (4 * _row_bytes(c) + 16) if c["gather"] else 0), "flops": 2 * c["kv_heads"] * sum(_lengths(c))}


# ---- the definition in 64 bits ------------------------------------------------------------------------------------------------------

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "store":
        return _exact_store(c, s)
    if c["op"] == "evict":
        return _exact_evict(c, s)
    S, n, H, HK, d, n_kv = c["seqs"], c["n"], c["heads"], c["kv_heads"], c["d"], c["n_kv"]
    k = _values(s["k"], c["kv"], torch.float64)
    mass = s["mass"].double() * DECAY if c["op"] == "attend" else torch.zeros((S, HK, n_kv), dtype=torch.float64, device="cuda")
    dst = torch.zeros((S, n, H, d), dtype=torch.float64, device="cuda")
    for b in range(S):
        for h in range(H):
            hk = h // (H // HK)
            logits = s["q"][b, h].double() @ k[b, hk].T.contiguous() / math.sqrt(d) + s["mask"][b].double()
            p = torch.softmax(logits, -1)
            p = torch.where(torch.isnan(p), torch.zeros_like(p), p)
            mass[b, hk] += p.sum(0)
            if c["op"] == "attend":
                dst[b, :, h] = p @ _values(s["v"][b, hk], c["kv"], torch.float64)
    return {"dst": dst, "mass": mass} if c["op"] == "attend" else {"mass": mass}


def _exact_store(c, s):
    half = c["n_dims"] // 2
    out = {}
    for name in ("q", "k"):
        x = s[name].double()
        x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / c["d"] + EPS) * s[name + "_norm"].double()
        for i in range(half):
            a, b = (2 * i, 2 * i + 1) if c["mode"] == 0 else (i, i + half)
            t = s["pos"].double()[:, :, None] / c["base"] ** (2.0 * i / c["n_dims"])
            x[..., a], x[..., b] = x[..., a] * torch.cos(t) - x[..., b] * torch.sin(t), x[..., a] * torch.sin(t) + x[..., b] * torch.cos(t)
        out[name] = x.transpose(1, 2)
    rows = s["rows"].long()
    got = {"q": out["q"].contiguous()}
    for name, x in (("k", out["k"]), ("v", s["v"].double().transpose(1, 2))):
        if c["kv"] == "q8_0":                                           # 32 values share a scale, kept in f16
            b = x.reshape(*x.shape[:-1], -1, 32)
            top = b.abs().amax(-1, keepdim=True) / 127
            q = torch.where(top > 0, torch.floor(b.abs() / top + 0.5) * b.sign(), torch.zeros_like(b))
            x = (q * top.half().double()).reshape(x.shape)
        held = _values(s[name + "_cache"], c["kv"], torch.float64)
        got[name] = held.scatter(2, rows[..., None].expand(-1, -1, -1, c["d"]), x)
    got["slot_pos"] = None
    got["slot_mass"] = s["slot_mass"].double().scatter(2, rows, 0.0)
    return got


def _exact_evict(c, s):
    if not c["gather"]:
        return None
    recent, sink = _recent(c)
    mass, pos = torch.zeros((c["seqs"], c["kv_heads"], c["n_keep"]), dtype=torch.float64, device="cuda"), None
    rows = {x: torch.zeros(s[x + "_out"].shape, dtype=torch.float64, device="cuda") for x in ("k", "v")}
    held, used, past, at = s["mass"].tolist(), s["n_used"].tolist(), s["n_past"].tolist(), s["slot_pos"].tolist()
    for b in range(c["seqs"]):
        for h in range(c["kv_heads"]):
            safe = lambda j: at[b][h][j] < sink or at[b][h][j] >= past[b] - recent  # noqa: E731
            best = sorted(range(used[b]), key=lambda j: (0 if safe(j) else 1, 0.0 if safe(j) else -held[b][h][j], j))[: c["n_keep"]]
            i = torch.tensor(sorted(best), device="cuda")
            mass[b, h, : len(best)] = s["mass"][b, h, i].double()
            for x in rows:
                rows[x][b, h, : len(best)] = s[x][b, h, i].double()
    whole = c["kv"] in ("q8_0", "q4_0")
    return {"kept": None, "evicted": None, "mass": mass, "slot_pos": pos, "k": None if whole else rows["k"], "v": None if whole else rows["v"]}
