"""The operators around the delta of a decode step, as cases with sizes.

* ``append``  q, k and v of a step's tokens are rotated by position (after the LoRA deltas were added, where there
              are any); q is written out, k and v go to their slots of a paged cache.
* ``attend``  one query token per request over a paged cache; groups of neighbouring requests (those of one adapter)
              share a prefix, whose keys come before a request's own.
* ``int4``    ``y = x W^T (+ add)`` with 4-bit codes, a scale and optionally a zero point per group of columns.

What has a size or a length follows from the case, values follow from the seed.  A cache holds old values
wherever no request's keys are, as in a server that has run for a while.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # one token of one request with its deltas: latency only
        dict(name="append-1", op="append", dtype="fp16", tokens=1, heads=32, kv=32, dim=128, rot=128, page=16, deltas=True,
             fused=False, interleaved=False, padded=0),
        # a full decode batch, grouped-query, q/k/v as parts of one product's rows, with deltas
        dict(name="append-256-gqa", op="append", dtype="bf16", tokens=256, heads=64, kv=8, dim=128, rot=128, page=64,
             deltas=True, fused=True, interleaved=False, padded=0),
        # the prompts of a prefill batch, padded to a bucket, adjacent-pair rotation of half a head, a slot per token
        # instead of pages (the token table of the reference)
        dict(name="append-8191-padded", op="append", dtype="fp16", tokens=8191, heads=40, kv=40, dim=128, rot=64, page=1,
             deltas=False, fused=True, interleaved=True, padded=333),
        # a single user's decode step
        dict(name="attend-1", op="attend", dtype="fp16", requests=1, heads=32, kv=32, dim=128, page=16, longest=311, groups=0,
             loose=1, prefix=0, lse=False),
        # an ordinary decode batch of ragged lengths, nothing shared
        dict(name="attend-32-paged", op="attend", dtype="fp16", requests=32, heads=32, kv=32, dim=128, page=16, longest=2048,
             groups=0, loose=32, prefix=0, lse=False),
        # one long system prompt under a full batch, grouped-query
        dict(name="attend-64-prefix8192", op="attend", dtype="bf16", requests=64, heads=64, kv=8, dim=128, page=64, longest=512,
             groups=1, loose=0, prefix=8192, lse=False),
        # adapters with prompts of their own, odd lengths, some requests without any
        dict(name="attend-93-7groups", op="attend", dtype="fp16", requests=93, heads=40, kv=40, dim=128, page=16, longest=333,
             groups=7, loose=5, prefix=1999, lse=True),
        # the largest: a document that 256 requests ask about
        dict(name="attend-256-prefix16384", op="attend", dtype="bf16", requests=256, heads=64, kv=8, dim=128, page=128,
             longest=1024, groups=1, loose=0, prefix=16384, lse=False),
        # one projection of one token
        dict(name="int4-1", op="int4", dtype="fp16", tokens=1, inner=4096, outer=4096, group=128, zeros=False, add=False, f32=False),
        # a narrow k/v projection, small groups with zero points, an odd batch
        dict(name="int4-7-kv", op="int4", dtype="bf16", tokens=7, inner=8192, outer=1024, group=32, zeros=True, add=False, f32=False),
        # the vocabulary of a single token, fp32 logits
        dict(name="int4-1-vocab", op="int4", dtype="bf16", tokens=1, inner=8192, outer=32000, group=64, zeros=True, add=False, f32=True),
        # a decode batch's output projection, added to the residual
        dict(name="int4-64-o", op="int4", dtype="bf16", tokens=64, inner=8192, outer=8192, group=128, zeros=False, add=True, f32=False),
    ]


# ---- drawn cases -----------------------------------------------------------------------------------
def _log_int(rng, lo, hi):
    return min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5))))))


def draw(rng):
    most = {op: [max(work(c)[k] for c in listed() if c["op"] == op) for k in ("bytes", "flops")]
            for op in ("append", "attend", "int4")}
    while True:
        c = _draw_one(rng)
        w = work(c)
        if w["bytes"] <= most[c["op"]][0] and w["flops"] <= most[c["op"]][1] and _plain_bytes(c) <= 6e9:
            return c


def _draw_one(rng):
    op = rng.choice(["append", "attend", "attend", "int4"])
    c = dict(op=op, dtype=rng.choice(["fp16", "bf16"]))
    if op == "int4":
        c["group"] = rng.choice([32, 64, 128])
        c.update(tokens=_log_int(rng, 1, 64), inner=c["group"] * _log_int(rng, 1024 // c["group"], 8192 // c["group"]),
                 outer=_log_int(rng, 256, 32000), zeros=rng.random() < 0.5, add=rng.random() < 0.3, f32=rng.random() < 0.2)
        return c
    c["heads"], c["kv"] = rng.choice([(32, 32), (40, 40), (64, 8), (32, 8), (8, 1), (5, 5), (24, 2)])
    c["dim"] = rng.choice([64, 128, 128])
    c["page"] = rng.choice([1, 16, 16, 32, 64, 128])
    if op == "append":
        c["tokens"] = _log_int(rng, 1, 8192)
        c.update(rot=rng.choice([c["dim"], c["dim"], c["dim"] // 2]), deltas=rng.random() < 0.5, fused=rng.random() < 0.5,
                 interleaved=rng.random() < 0.3, padded=rng.choice([0, c["tokens"] // 10]))
        return c
    c.update(requests=_log_int(rng, 1, 256), longest=_log_int(rng, 1, 4096), lse=rng.random() < 0.5)
    c["groups"] = rng.choice([0, 1, 1, min(c["requests"], _log_int(rng, 1, 12))])
    c["prefix"] = _log_int(rng, 64, 32768) if c["groups"] else 0
    c["loose"] = rng.randint(0, c["requests"] // 4) if c["groups"] else c["requests"]
    if c["groups"] > c["requests"] - c["loose"]:
        c["loose"] = 0
    return c


def _plain_bytes(c):
    """What the plain form keeps at a time."""
    if c["op"] == "int4":
        return 12 * c["inner"] * c["outer"]
    if c["op"] == "append":
        return 12 * c["tokens"] * (c["heads"] + 2 * c["kv"]) * c["dim"]
    _, starts, plens = _lengths(c)
    most = int(np.diff(starts).max()) if c["groups"] else 0
    own_keys = c["requests"] * c["longest"] * (8 * c["kv"] * c["dim"] + 8 * c["heads"])
    return own_keys + c["groups"] * c["prefix"] * (8 * c["kv"] * c["dim"] + 8 * most * c["heads"])


def _lengths(c):
    """Own keys of each request, first request of each group (and the last one's end), keys of each group's prefix."""
    b, g = c["requests"], c["groups"]
    rng = np.random.default_rng([b, g, c["longest"], c["prefix"]])
    lens = rng.integers(max(1, c["longest"] // 4), c["longest"] + 1, b)
    lens[:1] = c["longest"]
    if g == 0:
        return lens, np.zeros(1, np.int64), np.zeros(0, np.int64)
    plens = rng.integers(max(1, c["prefix"] // 4), c["prefix"] + 1, g)
    plens[-1:] = c["prefix"]
    sizes = 1 + rng.multinomial(b - c["loose"] - g, rng.dirichlet(np.full(g, 2.0)))
    return lens, np.concatenate([[0], np.cumsum(sizes)]), plens


def work(c):
    """Every input once, every output once; of a cache the keys that are attended to, or the slots that are written."""
    if c["op"] == "append":
        t = c["tokens"] - c["padded"]
        row = (c["heads"] + 2 * c["kv"]) * c["dim"]
        table = 4 * c["rot"] * min(t, _positions(c))
        return {"bytes": t * row * 2 * (3 if c["deltas"] else 2) + table + 12 * c["tokens"],
                "flops": t * (3 * (c["heads"] + c["kv"]) * c["rot"] + (row if c["deltas"] else 0))}
    if c["op"] == "int4":
        n, k, t = c["outer"], c["inner"], c["tokens"]
        y = 4 if c["f32"] else 2
        return {"bytes": n * k // 2 + n * (k // c["group"]) * (3 if c["zeros"] else 2) + 2 * t * k + t * n * (2 * y if c["add"] else y),
                "flops": 2 * t * n * k}
    lens, starts, plens = _lengths(c)
    keys = int(lens.sum()) + int(plens.sum())
    seen = int(lens.sum()) + int((np.diff(starts) * plens).sum())
    pages = sum(-(-int(n) // c["page"]) for n in (*lens, *plens))
    return {"bytes": keys * c["kv"] * c["dim"] * 4 + c["requests"] * c["heads"] * (4 * c["dim"] + (4 if c["lse"] else 0)) + 4 * pages
            + 4 * (c["requests"] + 2 * c["groups"]),
            "flops": 4 * c["dim"] * c["heads"] * seen}


# ---- states ----------------------------------------------------------------------------------------
def _positions(c):
    """Rows of the rotation tables: a long context for decode tokens, as long as the batch for prompts."""
    return 32768 if c["tokens"] <= 512 else 8192


def _normal(g, *shape, dtype, std=1.0):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    return {"append": _prepare_append, "attend": _prepare_attend, "int4": _prepare_int4}[case["op"]](case, g, dt)


def _prepare_append(c, g, dt):
    t, hq, hk, d, rot = c["tokens"], c["heads"], c["kv"], c["dim"], c["rot"]
    if c["fused"]:
        qkv = _normal(g, t, (hq + 2 * hk) * d, dtype=dt)
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv.split([hq * d, hk * d, hk * d], 1))
    else:
        q, k, v = (_normal(g, t, h, d, dtype=dt) for h in (hq, hk, hk))
    pages = -(-(t + t // 4 + 64) // c["page"])
    n_pos = _positions(c)
    angle = torch.arange(n_pos, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    slots = torch.randperm(pages * c["page"], generator=g, device="cuda")[:t].to(torch.int32)
    if t > 512:                                  # prompts: positions count up, a prompt's tokens lie in neighbouring slots
        positions = torch.arange(t, device="cuda") % (n_pos // 8)
        slots = slots.sort().values
    else:
        positions = torch.randint(0, n_pos, (t,), generator=g, device="cuda")
    if c["padded"]:                              # rows behind the last prompt have no slot
        slots[t - c["padded"]:] = -1
    s = dict(case=c, q=q, k=k, v=v, positions=positions, slots=slots, cos=angle.cos().float(), sin=angle.sin().float(),
             q_out=torch.zeros(t, hq, d, dtype=dt, device="cuda"),
             k_cache=_normal(g, pages, c["page"], hk, d, dtype=dt), v_cache=_normal(g, pages, c["page"], hk, d, dtype=dt),
             dq=None, dk=None, dv=None)
    if c["deltas"]:
        s["dq"], s["dk"], s["dv"] = (_normal(g, t, h, d, dtype=dt, std=0.25) for h in (hq, hk, hk))
    return s


def _prepare_attend(c, g, dt):
    b, hq, hk, d, page = c["requests"], c["heads"], c["kv"], c["dim"], c["page"]
    lens, starts, plens = _lengths(c)
    n_own, n_pre = -(-lens // page), -(-plens // page)
    total = int(n_own.sum() + n_pre.sum())
    pages = total + total // 8 + 1
    order = torch.randperm(pages, generator=g, device="cuda")[:total].to(torch.int32)

    def table(counts, first):
        width = int(counts.max()) if len(counts) else 0
        at = first + np.concatenate([[0], np.cumsum(counts)])[:-1]
        index = at[:, None] + np.minimum(np.arange(width), np.maximum(counts[:, None] - 1, 0))
        filled = order[torch.from_numpy(index).cuda()]
        return torch.where(torch.from_numpy(np.arange(width) < counts[:, None]).cuda(), filled, 0)

    def i32(a):
        return torch.from_numpy(np.asarray(a, np.int32)).cuda()

    s = dict(case=c, q=_normal(g, b, hq, d, dtype=dt, std=2.0), out=torch.zeros(b, hq, d, dtype=dt, device="cuda"),
             k_cache=_normal(g, pages, page, hk, d, dtype=dt), v_cache=_normal(g, pages, page, hk, d, dtype=dt),
             block_table=table(n_own, 0), lens=i32(lens), prefix_table=None, prefix_lens=None, group_starts=None,
             lse=torch.zeros(b, hq, device="cuda") if c["lse"] else None, largest=0)
    if c["groups"]:
        s.update(prefix_table=table(n_pre, int(n_own.sum())), prefix_lens=i32(plens), group_starts=i32(starts),
                 largest=int(np.diff(starts).max()))
    return s


def _prepare_int4(c, g, dt):
    t, k, n, group = c["tokens"], c["inner"], c["outer"], c["group"]
    s = dict(case=c, x=_normal(g, t, k, dtype=dt), y=torch.zeros(t, n, dtype=torch.float32 if c["f32"] else dt, device="cuda"),
             codes=torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8),
             scales=(_normal(g, n, k // group, dtype=torch.float32).abs() * 0.1 + 0.1).mul_(k ** -0.5).to(dt), zeros=None, add=None)
    if c["zeros"]:
        s["zeros"] = torch.randint(4, 12, (n, k // group), generator=g, device="cuda", dtype=torch.uint8)
    if c["add"]:
        s["add"] = _normal(g, t, n, dtype=s["y"].dtype)
    return s


# ---- one pass --------------------------------------------------------------------------------------
def run(s):
    return {"append": _run_append, "attend": _run_attend, "int4": _run_int4}[s["case"]["op"]](s)


def _run_append(s):
    c = s["case"]
    if own:
        import ae296_b200
        ae296_b200.append_kv(s["q_out"], s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], s["positions"], s["slots"], s["cos"],
                             s["sin"], s["dq"], s["dk"], s["dv"], interleaved=c["interleaved"])
        return s["q_out"], s["k_cache"], s["v_cache"]
    live = s["slots"] >= 0
    slots = s["slots"].long()
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    rot = c["rot"]

    def summed(x, dx):
        return x.float() if dx is None else x.float() + dx.float()

    def rotated(x):
        a, rest = x[..., :rot], x[..., rot:]
        if c["interleaved"]:
            x0, x1 = a[..., 0::2], a[..., 1::2]
            turned = torch.stack([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1).flatten(-2)
        else:
            x0, x1 = a[..., :rot // 2], a[..., rot // 2:]
            turned = torch.cat([x0 * cos - x1 * sin, x1 * cos + x0 * sin], -1)
        return torch.cat([turned, rest], -1).to(s["q"].dtype)

    s["q_out"].copy_(torch.where(live[:, None, None], rotated(summed(s["q"], s["dq"])), s["q_out"]))
    pages, page, hk, d = s["k_cache"].shape
    for cache, new in ((s["k_cache"], rotated(summed(s["k"], s["dk"]))), (s["v_cache"], summed(s["v"], s["dv"]).to(s["v"].dtype))):
        flat = torch.cat([cache.view(pages * page, hk, d), cache.new_zeros(1, hk, d)])   # the last row takes what has no slot
        flat[torch.where(live, slots, pages * page)] = new
        cache.copy_(flat[:-1].view_as(cache))
    return s["q_out"], s["k_cache"], s["v_cache"]


def _run_attend(s):
    c = s["case"]
    if own:
        import ae296_b200
        ae296_b200.prefix_attention(s["out"], s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["lens"], s["prefix_table"],
                                    s["prefix_lens"], s["group_starts"], lse=s["lse"])
        return (s["out"],) if s["lse"] is None else (s["out"], s["lse"])
    b, hq, hk, d, page = c["requests"], c["heads"], c["kv"], c["dim"], c["page"]
    per = hq // hk
    scale = d ** -0.5

    def keys(table, cache):                                        # [rows, kv heads, keys, dim]
        return cache[table.long()].flatten(1, 2).transpose(1, 2).float()

    def scores(q, table, lens):                                    # q [rows, kv heads, x, dim]
        s_ = q @ keys(table, s["k_cache"]).transpose(-1, -2) * scale
        return s_.masked_fill(torch.arange(s_.shape[-1], device="cuda") >= lens[:, None, None, None], -math.inf)

    def exps(s_, m):
        return torch.exp(s_ - torch.where(m == -math.inf, 0.0, m)[..., None])

    q = s["q"].float().view(b, hk, per, d)
    mine = scores(q, s["block_table"], s["lens"])
    m = mine.amax(-1)
    if c["groups"]:
        starts, most = s["group_starts"].long(), s["largest"]
        row = starts[:-1, None] + torch.arange(most, device="cuda")                      # [groups, most]
        there = row < starts[1:, None]
        row = torch.where(there, row, 0)
        shared = scores(q[row].transpose(1, 2).reshape(c["groups"], hk, most * per, d), s["prefix_table"], s["prefix_lens"])
        m_shared = shared.amax(-1).view(c["groups"], hk, most, per).transpose(1, 2)
        m = m.index_put((row[there],), torch.maximum(m[row[there]], m_shared[there]))
        e = exps(shared, m[row].transpose(1, 2).reshape(c["groups"], hk, most * per))
    p = exps(mine, m)
    total, o = p.sum(-1), p @ keys(s["block_table"], s["v_cache"])
    if c["groups"]:
        o_shared = (e @ keys(s["prefix_table"], s["v_cache"])).view(c["groups"], hk, most, per, d).transpose(1, 2)
        l_shared = e.sum(-1).view(c["groups"], hk, most, per).transpose(1, 2)
        o.index_put_((row[there],), o_shared[there], accumulate=True)
        total.index_put_((row[there],), l_shared[there], accumulate=True)
    s["out"].copy_((o / torch.where(total == 0, 1.0, total)[..., None]).view(b, hq, d))
    if s["lse"] is None:
        return (s["out"],)
    s["lse"].copy_((m + torch.log(total)).view(b, hq))
    return s["out"], s["lse"]


def _run_int4(s):
    c = s["case"]
    if own:
        import ae296_b200
        ae296_b200.int4_linear(s["y"], s["x"], s["codes"], s["scales"], s["zeros"], add=s["add"])
        return s["y"]
    q = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).view(c["outer"], -1, c["group"]).float()
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[..., None]
    w = ((q - zero) * s["scales"].float()[..., None]).view(c["outer"], c["inner"])
    y = s["x"].float() @ w.t()
    s["y"].copy_(y if s["add"] is None else y + s["add"].float())
    return s["y"]


# ---- the same in 64 bits, from the definitions -------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "int4": _exact_int4}[case["op"]](case, s)


def _exact_append(c, s):
    rot, pair = c["rot"], torch.arange(c["rot"] // 2, device="cuda")
    first = 2 * pair if c["interleaved"] else pair
    second = first + 1 if c["interleaved"] else pair + rot // 2
    live = (s["slots"] >= 0).nonzero()[:, 0]
    turn = torch.complex(s["cos"].double(), s["sin"].double())[s["positions"][live]][:, None]

    def whole(x, dx, turned):
        x = x[live].double() + (0.0 if dx is None else dx[live].double())
        if turned:
            z = torch.complex(x[..., first], x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
        return x

    q_out = s["q_out"].double()
    q_out[live] = whole(s["q"], s["dq"], True)
    at = s["slots"][live].long()
    caches = []
    for cache, x, dx, turned in ((s["k_cache"], s["k"], s["dk"], True), (s["v_cache"], s["v"], s["dv"], False)):
        new = cache.double()
        new[at // c["page"], at % c["page"]] = whole(x, dx, turned)
        caches.append(new)
    return q_out, caches[0], caches[1]


def _exact_attend(c, s):
    page, per = c["page"], c["heads"] // c["kv"]
    lens, starts, plens = _lengths(c)
    out = torch.zeros(c["requests"], c["heads"], c["dim"], dtype=torch.float64, device="cuda")
    lse = torch.full((c["requests"], c["heads"]), -math.inf, dtype=torch.float64, device="cuda")

    def load(table, n):
        at = torch.arange(int(n), device="cuda")
        where = table[at // page].long(), at % page
        return [x[where].double().permute(1, 0, 2) for x in (s["k_cache"], s["v_cache"])]         # [kv heads, n, dim]

    group, shared = -1, None
    for r in range(c["requests"]):
        k, v = load(s["block_table"][r], lens[r])
        g = int(np.searchsorted(starts, r, side="right")) - 1 if c["groups"] else -1
        if 0 <= g < c["groups"]:
            if g != group:
                group, shared = g, load(s["prefix_table"][g], plens[g])
            k, v = torch.cat([shared[0], k], 1), torch.cat([shared[1], v], 1)
        z = torch.einsum("hpd,hnd->hpn", s["q"][r].double().view(c["kv"], per, -1), k) / math.sqrt(c["dim"])
        out[r] = torch.einsum("hpn,hnd->hpd", torch.softmax(z, -1), v).reshape(c["heads"], -1)
        lse[r] = torch.logsumexp(z, -1).reshape(-1)
    return (out, lse) if c["lse"] else (out,)


def _exact_int4(c, s):
    w = torch.empty(c["outer"], c["inner"], dtype=torch.float64, device="cuda")
    w[:, 0::2] = (s["codes"] % 16).double()
    w[:, 1::2] = torch.div(s["codes"], 16, rounding_mode="floor").double()
    w -= 8.0 if s["zeros"] is None else s["zeros"].double().repeat_interleave(c["group"], 1)
    w *= s["scales"].double().repeat_interleave(c["group"], 1)
    y = s["x"].double() @ w.T
    return y if s["add"] is None else y + s["add"].double()
