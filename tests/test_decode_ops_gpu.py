"""GPU: append, attention and 4-bit products against the float64 oracle.

Tolerances, derived: ``h = eps / 2`` of the 16-bit type is the relative error of one rounding, ``u = 2^-24`` that of fp32
(sums inside the tensor cores are cut instead of rounded: ``2 u`` an addition).

* append: one rounding of the result, three fp32 roundings of terms no larger than |x0| + |x1| before it.
* attention: a weight's relative error is that of its exponent, (D + 4) additions and roundings of terms that sum to at most
  ``scale |q|.|k|``, plus that of the exponential (2 ulp) and of the split in two 16-bit halves (h^2); the quotient doubles it.  Where a
  prefix is shared the weight may be one 16-bit number: h.  Additions of n terms into the running sums: 2 u n.  All of
  it scales the softmax average of |v|.
* int4: products are exact, K + groups + 16 additions of terms that sum to sum |w x|.
"""
import numpy as np
import pytest
import torch

import ae296_b200 as L
from ae296_b200 import decode
from oracle import decode_oracle as O

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def half_step(dt):
    return torch.finfo(dt).eps / 2


def tiny(dt):
    return 2.0 ** -25 if dt == torch.float16 else 0.0           # half of the smallest step


def f64(t):
    return t.detach().double().cpu().numpy()


def randn(g, *shape, dtype, std=1.0):
    return (torch.randn(*shape, generator=g) * std).to(dtype).cuda()


def within(got, want, tol, what=""):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size}, worst {np.abs(got - want)[bad].max()} at {np.argwhere(bad)[0]}"


# ---- append --------------------------------------------------------------------------------------
def append_case(seed, T, hq, hk, d, rot, page, dtype, deltas=True, n_pos=700, fused=False, tables=torch.float32, itype=torch.int32, head_major=False):
    g = torch.Generator().manual_seed(seed)
    dt = TYPES[dtype]
    if fused:
        qkv = randn(g, T, (hq + 2 * hk) * d + 8, dtype=dt)
        q, k, v = (x.unflatten(1, (-1, d)) for x in qkv[:, :-8].split([hq * d, hk * d, hk * d], 1))
    else:
        q, k, v = (randn(g, T, h, d, dtype=dt) for h in (hq, hk, hk))
    pages = -(-(T + 5) // page) + 1
    shape = (pages, hk, page, d) if head_major else (pages, page, hk, d)
    kc, vc = (torch.full(shape, float("nan"), dtype=dt, device="cuda") for _ in range(2))
    if head_major:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    ang = torch.arange(n_pos, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    slots = torch.randperm(pages * page, generator=g)[:T].to(itype).cuda()
    pos = torch.randint(0, n_pos, (T,), generator=g).to(itype).cuda()
    pos[-1] = n_pos - 1
    pos[0] = 0
    s = dict(q_out=torch.full_like(q.contiguous(), 7.0), q=q, k=k, v=v, k_cache=kc, v_cache=vc, positions=pos, slots=slots,
             cos=ang.cos().to(tables).cuda(), sin=ang.sin().to(tables).cuda())
    if deltas:
        s.update(dq=randn(g, T, hq, d, dtype=dt, std=0.3), dk=randn(g, T, hk, d, dtype=dt, std=0.3), dv=randn(g, T, hk, d, dtype=dt, std=0.3))
    return s


def check_append(s, interleaved=False, before=None):
    """Runs the op and compares q_out and the caches; what has no slot must keep its bits."""
    host = {n: f64(t) if t.is_floating_point() else t.cpu().numpy() for n, t in (before or s).items()}
    want = O.append(**host, interleaved=interleaved)
    L.append_kv(**s, interleaved=interleaved)
    torch.cuda.synchronize()
    dt = s["q"].dtype
    size = max(float(np.abs(host[n]).max()) + float(np.abs(host.get("d" + n, np.zeros(1))).max()) for n in "qkv")
    for name, w in zip(("q_out", "k_cache", "v_cache"), want):
        got = f64(s[name])
        untouched = (w == host[name]) | np.isnan(w)
        assert (np.isnan(got) == np.isnan(w)).all(), name
        tol = half_step(dt) * np.abs(w) + 6 * U * 2 * size + tiny(dt)
        tol[untouched] = 0.0 if name != "q_out" else tol[untouched]
        keep = ~np.isnan(w)
        within(got[keep], w[keep], tol[keep], name)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("T,hq,hk,d,rot,page", [
    (1, 32, 32, 128, 128, 16), (1, 1, 1, 64, 64, 1), (3, 64, 8, 128, 128, 64), (37, 5, 5, 128, 64, 16), (130, 8, 1, 64, 32, 128),
    (65, 24, 2, 96, 96, 48), (9, 3, 3, 80, 80, 7), (21, 4, 2, 36, 20, 5), (5, 2, 1, 2, 2, 3), (4, 16, 16, 256, 128, 16), (2, 1, 1, 512, 512, 2)])
def test_append_values(T, hq, hk, d, rot, page, dtype):
    for i, (inter, fused, deltas) in enumerate([(False, False, True), (True, True, False)]):
        check_append(append_case(11 * T + i, T, hq, hk, d, rot, page, dtype, deltas, fused=fused), inter)


@pytest.mark.parametrize("kw", [dict(tables="own"), dict(itype=torch.int64), dict(head_major=True), dict(fused=True, deltas=False)])
def test_append_forms(kw):
    if kw.get("tables"):
        kw = dict(kw, tables=torch.bfloat16)
    check_append(append_case(5, 45, 8, 2, 128, 128, 16, "bf16", **kw))
    check_append(append_case(6, 45, 8, 2, 64, 32, 16, "bf16", **kw), True)


def test_append_of_single_deltas_and_in_place():
    s = append_case(7, 19, 8, 2, 128, 128, 16, "fp16")
    check_append({n: t for n, t in s.items() if n not in ("dq", "dv")})
    s = append_case(8, 19, 8, 2, 128, 128, 16, "fp16", fused=True)
    before = {n: t.clone() for n, t in s.items()}
    s["q_out"], before["q_out"] = s["q"], before["q"]
    check_append(s, before=before)


def test_append_misaligned_views():
    s = append_case(9, 13, 4, 2, 64, 64, 16, "fp16", deltas=False)
    for n in ("q", "k", "v"):                                     # rows that start at odd elements
        t = s[n]
        wide = torch.empty(t.shape[0], t[0].numel() + 3, dtype=t.dtype, device="cuda")
        s[n] = wide[:, 1:1 + t[0].numel()].unflatten(1, tuple(t.shape[1:])).copy_(t)
        assert s[n].data_ptr() % 16 != 0
    check_append(s)


def test_append_leaves_padding_and_bad_rows_alone_and_reports_them():
    s = append_case(10, 40, 8, 2, 128, 128, 16, "bf16")
    slots = s["slots"]
    cap = s["k_cache"].shape[0] * 16
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    slots[[0, 7, 39]] = -1
    slots[3] = -2 ** 31
    check_append(dict(s))
    L.append_kv(**s, status=word)
    assert int(word) == 0
    assert (s["q_out"][[0, 3, 7, 39]] == 7).all()
    for name, value, bit in (("slots", cap, decode.BAD_SLOT), ("slots", 2 ** 31 - 1, decode.BAD_SLOT), ("positions", -1, decode.BAD_POSITION),
                             ("positions", 700, decode.BAD_POSITION)):
        c = append_case(10, 40, 8, 2, 128, 128, 16, "bf16")
        c[name][5] = value
        word.zero_()
        L.append_kv(**c, status=word)
        assert int(word) == bit
        check_append(c)
        assert (c["q_out"][5] == 7).all()
    c = append_case(10, 40, 8, 2, 128, 128, 16, "bf16", itype=torch.int64)
    c["slots"][4] = 2 ** 40
    check_append(c)


def test_append_of_nothing():
    s = append_case(1, 4, 8, 2, 128, 128, 16, "bf16")
    none = {n: t[:0] if n in ("q_out", "q", "k", "v", "dq", "dk", "dv", "positions", "slots") else t for n, t in s.items()}
    L.append_kv(**none)
    assert torch.isnan(s["k_cache"]).all()


# ---- attention -----------------------------------------------------------------------------------
def attend_case(seed, B, hq, hk, d, page, dtype, lens, starts=None, plens=None, std=1.5, spare=3, fill=float("nan"), head_major=False):
    """Pages in random order; wherever no request's keys are, the caches hold `fill`."""
    g = torch.Generator().manual_seed(seed)
    dt = TYPES[dtype]
    lens, plens = np.asarray(lens), np.asarray(plens if plens is not None else [], np.int64)
    counts = [-(-lens // page), -(-plens // page)]
    total = int(counts[0].sum() + counts[1].sum())
    shape = (total + spare, hk, page, d) if head_major else (total + spare, page, hk, d)
    kc, vc = (torch.full(shape, fill, dtype=dt, device="cuda") for _ in range(2))
    if head_major:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    order = torch.randperm(total + spare, generator=g)[:total].int()
    at, tables = 0, []
    for ns, cs in ((lens, counts[0]), (plens, counts[1])):
        table = torch.full((len(ns), max([int(c) for c in cs], default=0) + 1), -7, dtype=torch.int32)   # -7 behind the last page
        for i, (n, c) in enumerate(zip(ns, cs)):
            table[i, :c] = order[at:at + c]
            keys = torch.arange(int(n))
            where = table[i].long()[keys // page].cuda(), (keys % page).cuda()
            kc[where] = randn(g, int(n), hk, d, dtype=dt)
            vc[where] = randn(g, int(n), hk, d, dtype=dt) + 0.25
            at += int(c)
        tables.append(table.cuda())
    s = dict(out=torch.full((B, hq, d), 9.0, dtype=dt, device="cuda"), q=randn(g, B, hq, d, dtype=dt, std=std), k_cache=kc, v_cache=vc,
             block_table=tables[0], lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    if starts is not None:
        s.update(prefix_table=tables[1], prefix_lens=torch.tensor(plens, dtype=torch.int32, device="cuda"),
                 group_starts=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    return s


def check_attend(s, scale=None, expect_status=0, oracle=None):
    want, lse, weighted = oracle if oracle is not None else attend_oracle(s, scale)
    got_lse = torch.full(tuple(s["q"].shape[:2]), 5.0, device="cuda")
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    L.prefix_attention(**s, scale=scale, lse=got_lse, status=word)
    torch.cuda.synchronize()
    assert int(word) == expect_status
    dt, d = s["q"].dtype, s["q"].shape[2]
    sc = d ** -0.5 if scale is None else abs(scale)
    kmax = float(torch.nan_to_num(s["k_cache"].float()).norm(dim=-1).max())
    zmax = sc * float(s["q"].float().norm(dim=-1).max()) * kmax
    n = int(s["lens"].clamp(min=0).max()) + (int(s["prefix_lens"].max()) if "prefix_lens" in s and s["prefix_lens"].numel() else 0)
    h = half_step(dt)
    weight = (d + 4) * 2 * U * zmax + 4 * U + h * h + (h if "prefix_lens" in s else 0.0)
    within(f64(s["out"]), want, h * np.abs(want) + weighted * (2 * weight + 2 * U * n) + tiny(dt), "out")
    empty = np.isinf(lse)
    got = f64(got_lse)
    assert (got[empty] == -np.inf).all() and (f64(s["out"])[empty] == 0).all()
    within(got[~empty], lse[~empty], (d + 4) * 2 * U * zmax + (n + 4) * 2 * U + 2 * U * np.abs(lse[~empty]), "lse")


def attend_oracle(s, scale=None):
    kc, vc = f64(s["k_cache"]), f64(s["v_cache"])
    pre = ("prefix_table", "prefix_lens", "group_starts")
    return O.attention(f64(s["q"]), kc, vc, s["block_table"].cpu().numpy(), s["lens"].cpu().numpy(),
                       *(s[n].cpu().numpy() if n in s else None for n in pre), scale=scale)


HEADS = [(8, 8), (16, 2), (8, 1), (24, 2), (20, 1), (5, 5)]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 1), (128, 64), (64, 256)])
@pytest.mark.parametrize("hq,hk", HEADS)
def test_attention_own_keys(hq, hk, d, page, dtype):
    check_attend(attend_case(hq + d + page, 7, hq, hk, d, page, dtype, [1, 0, 15, 16, 17, 333, 64]))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,page", [(128, 16), (64, 2), (128, 128), (64, 32)])
@pytest.mark.parametrize("hq,hk", HEADS)
def test_attention_shared_prefixes(hq, hk, d, page, dtype):
    """Groups of one, several and no requests, prefixes of no key, one key and more, requests before and behind the groups, without own keys."""
    check_attend(attend_case(hq + d + page, 12, hq, hk, d, page, dtype, [5, 0, 33, 0, 1, 17, 64, 3, 0, 0, 20, 2],
                             starts=[1, 2, 2, 7, 8, 10], plens=[70, 40, 257, 0, 1]))


@pytest.mark.parametrize("hq,hk,B,plen", [(16, 2, 33, 1000), (8, 8, 70, 515), (64, 8, 40, 129), (8, 1, 150, 2049), (4, 4, 129, 128)])
@pytest.mark.parametrize("d,dtype", [(128, "bf16"), (64, "fp16")])
def test_attention_large_groups(hq, hk, B, plen, d, dtype):
    lens = np.random.default_rng(B).integers(0, 40, B)
    check_attend(attend_case(B, B, hq, hk, d, 16, dtype, lens, starts=[0, B - 3, B - 1], plens=[plen, 64]))


@pytest.mark.parametrize("B,hq,hk,starts,plens", [
    (93, 40, 40, [0, 18, 40, 57, 93], [1999, 130, 700, 128]),      # more parts of a few blocks, some of one, than SMs
    (160, 32, 8, [0, 20, 160], [300, 1100]),                       # tiles of one stream's rows, of both and of a rest
    (64, 64, 64, [0, 20, 40, 64], [1, 129, 257]),                  # one block per item: the second stream has none
    (70, 16, 2, [0, 35, 70], [4000, 5000])])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_attention_large_groups_of_many_items(B, hq, hk, starts, plens, dtype):
    check_attend(attend_case(B, B, hq, hk, 128, 16, dtype, np.arange(B) % 7, starts=starts, plens=plens))
    check_attend(attend_case(B, B, hq, hk, 64, 1, dtype, np.arange(B) % 5, starts=starts, plens=plens))


def test_attention_one_long_request_is_split():
    check_attend(attend_case(3, 1, 8, 1, 128, 16, "bf16", [20011]))
    check_attend(attend_case(4, 2, 4, 4, 64, 1, "fp16", [9001, 1]))


def test_attention_scales_and_large_scores():
    """Scores far from zero, of one sign and of both; a scale of zero and a negative one."""
    for std, scale in ((30.0, None), (1.0, 0.0), (2.0, -0.3)):
        check_attend(attend_case(6, 40, 8, 2, 64, 16, "fp16", [1] * 40, starts=[0, 39], plens=[700], std=std), scale=scale)
        check_attend(attend_case(5, 5, 8, 2, 64, 16, "bf16", [100, 3, 65, 1, 0], starts=[0, 3], plens=[300], std=std), scale=scale)


def test_attention_strided_operands():
    s = attend_case(6, 5, 16, 4, 128, 16, "fp16", [100, 3, 65, 1, 0], starts=[1, 4], plens=[90], head_major=True)
    qkv = torch.zeros(5, 24, 128, dtype=torch.float16, device="cuda")
    qkv[:, :16] = s["q"]
    out = torch.full((5, 16, 136), 9.0, dtype=torch.float16, device="cuda")
    s.update(q=qkv[:, :16], out=out[:, :, :128])
    check_attend(s)
    assert (out[:, :, 128:] == 9).all()


def test_attention_infinities_behind_the_lengths():
    for fill in (float("inf"), -float("inf")):
        check_attend(attend_case(7, 6, 8, 2, 128, 64, "bf16", [100, 3, 65, 1, 0, 64], starts=[0, 2, 5], plens=[90, 127], fill=fill))


def test_attention_passes_nan_and_infinity_of_real_keys_on():
    s = attend_case(8, 3, 8, 2, 128, 16, "fp16", [40, 40, 40], fill=0.0)
    page = int(s["block_table"][1, 1])
    s["v_cache"][page, 3, 1, 5] = float("nan")
    s["k_cache"][int(s["block_table"][2, 0]), 0, 0, 0] = float("nan")
    L.prefix_attention(**s)
    out = s["out"].float()
    assert torch.isfinite(out[0]).all() and torch.isnan(out[1, 4:, 5]).all() and torch.isfinite(out[1, :4]).all()
    assert torch.isnan(out[2, :4]).all() and torch.isfinite(out[2, 4:]).all()


def test_attention_leaves_bad_pages_lengths_and_groups_out_and_reports_them():
    def case():
        return attend_case(9, 6, 8, 2, 128, 16, "bf16", [100, 30, 65, 1, 0, 64], starts=[0, 2, 5], plens=[90, 127], fill=0.0)

    wide = attend_case(9, 40, 8, 2, 128, 16, "bf16", [3] * 40, starts=[0, 39], plens=[700], fill=0.0)
    wide["prefix_table"][0, 3], wide["prefix_table"][0, 20] = 10 ** 6, -1
    check_attend(wide, expect_status=decode.BAD_PAGE)
    for name, where, value in (("block_table", (0, 2), -1), ("block_table", (2, 0), 10 ** 6), ("prefix_table", (1, 3), -2 ** 31 + 1)):
        s = case()
        s[name][where] = value
        check_attend(s, expect_status=decode.BAD_PAGE)
    s = case()
    s["lens"][1], s["prefix_lens"][0] = -5, -1
    good = dict(s, lens=s["lens"].clamp(min=0), prefix_lens=s["prefix_lens"].clamp(min=0))
    check_attend(s, expect_status=decode.BAD_LENGTH, oracle=attend_oracle(good))
    s = case()
    s["block_table"] = s["block_table"][:, :3]                    # requests 0, 2 and 5 are longer than their rows
    check_attend(s, expect_status=decode.BAD_LENGTH, oracle=attend_oracle(dict(s, lens=s["lens"].clamp(max=48))))
    for starts in ([2, 0, 5], [0, 2, 7], [-1, 2, 5], [0, 9, 5]):
        s = case()
        s["group_starts"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
        plain = {n: t for n, t in s.items() if n not in ("prefix_table", "prefix_lens", "group_starts")}
        check_attend(s, expect_status=decode.BAD_GROUPS, oracle=attend_oracle(plain))


@pytest.mark.parametrize("value", [-2 ** 31, -1, "behind", 2 ** 31 - 1])
@pytest.mark.parametrize("B,starts,plens", [(6, [0, 2, 5], [90, 127]), (40, [0, 39], [700])])        # groups of at most and of more than 32 rows
def test_attention_leaves_every_page_that_does_not_exist_out(B, starts, plens, value):
    """First, last and middle page of a row, of a request's own table and of a group's; the lowest number there is means nothing else."""
    for name, where in (("block_table", (1, 0)), ("prefix_table", (0, 0)), ("prefix_table", (0, 3)), ("prefix_table", (0, (plens[0] - 1) // 16))):
        s = attend_case(9, B, 8, 2, 128, 16, "bf16", [21] * B, starts=starts, plens=plens, fill=0.0)
        s[name][where] = s["k_cache"].shape[0] if value == "behind" else value
        check_attend(s, expect_status=decode.BAD_PAGE)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 1)])
def test_attention_of_small_groups_has_the_weights_in_full(d, page, dtype):
    """Groups of at most 32 rows, like own keys, take each weight as two 16-bit numbers: its error is that of the exponent, of the exponential and
    h^2, not h.  Values around zero leave many outputs so small that their own rounding hides nothing."""
    s = attend_case(13, 24, 8, 2, d, page, dtype, [1, 0, 2, 5] * 6, starts=[0, 8, 12, 13, 21], plens=[40, 17, 33, 24], std=0.3)
    s["v_cache"] -= 0.25
    want, lse, weighted = attend_oracle(s)
    L.prefix_attention(**s)
    dt, h = s["q"].dtype, half_step(s["q"].dtype)
    zmax = d ** -0.5 * float(s["q"].float().norm(dim=-1).max()) * float(torch.nan_to_num(s["k_cache"].float()).norm(dim=-1).max())
    weight = (d + 4) * 2 * U * zmax + 4 * U + h * h
    within(f64(s["out"]), want, h * np.abs(want) + weighted * (2 * weight + 2 * U * 45) + tiny(dt), "out")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("B,starts,plens", [(7, [0, 2, 7], [90, 127]), (60, [0, 37, 59], [300, 129])])       # groups of at most and of more than 32 rows
def test_attention_no_bit_depends_on_what_lies_behind_the_lengths(B, starts, plens, dtype):
    outs = []
    for fill in (0.0, float("nan"), float("inf"), -float("inf"), 60000.0):
        s = attend_case(14, B, 8, 2, 128, 64, dtype, [(7 * i) % 70 for i in range(B)], starts=starts, plens=plens, fill=fill)
        lse = torch.empty(B, 8, device="cuda")
        L.prefix_attention(**s, lse=lse)
        outs.append((s["out"], lse))
    for out, lse in outs[1:]:
        assert torch.equal(out, outs[0][0]) and torch.equal(lse, outs[0][1])


def test_attention_without_pages_and_without_requests():
    s = attend_case(10, 4, 8, 2, 64, 16, "fp16", [0, 0, 0, 0], starts=[0, 2], plens=[40])
    s["block_table"] = s["block_table"][:, :0]
    check_attend(s)
    none = dict(s, out=s["out"][:0], q=s["q"][:0], block_table=s["block_table"][:0], lens=s["lens"][:0],
                group_starts=torch.zeros(2, dtype=torch.int32, device="cuda"))
    L.prefix_attention(**none)


def test_attention_most_requests_and_groups():
    B, G = 4096, 2048
    rng = np.random.default_rng(1)
    lens, plens = rng.integers(0, 4, B), rng.integers(0, 6, G)
    starts = np.sort(rng.integers(0, B + 1, G + 1))
    check_attend(attend_case(11, B, 2, 1, 64, 4, "bf16", lens, starts=starts, plens=plens))


def test_cache_beyond_32_bit_offsets():
    """Pages whose elements lie more than 2^31 (and 2^32) elements behind the cache's start."""
    hk, d, page = 8, 128, 64
    pages = (2 ** 32 + 2 ** 24) // (hk * d * page)
    big = torch.empty(pages, page, hk, d, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator().manual_seed(1)
    k_pages, v_pages = [pages - 1, pages // 2 + 9], [pages - 2, pages // 2 + 8]
    k, v = (randn(g, 100, hk, d, dtype=torch.bfloat16) for _ in range(2))
    one = torch.ones(1, d // 2, device="cuda")
    q = randn(g, 100, hk, d, dtype=torch.bfloat16)
    kc, vc = big[1:], big[:-1]                                    # the same memory, a page apart: v's pages are k's neighbours
    slots = (torch.tensor(k_pages, device="cuda")[:, None] * page + torch.arange(page, device="cuda") - page).flatten()[:100]
    L.append_kv(q.clone(), q, k, v, kc, vc, torch.zeros_like(slots), slots, one, torch.zeros_like(one))
    table = torch.tensor([k_pages], device="cuda", dtype=torch.int32) - 1
    out = torch.empty(1, hk, d, dtype=torch.bfloat16, device="cuda")
    L.prefix_attention(out, q[:1], kc, vc, table, torch.tensor([100], dtype=torch.int32, device="cuda"))
    small = torch.stack([k[:64], torch.cat([k[64:], k[:28]])]), torch.stack([v[:64], torch.cat([v[64:], v[:28]])])
    want, _, weighted = O.attention(f64(q[:1]), f64(small[0]), f64(small[1]), np.array([[0, 1]]), [100])
    assert torch.equal(kc[k_pages[0] - 1], k[:64]) and torch.equal(vc[k_pages[1] - 1, :36], v[64:])
    within(f64(out), want, half_step(torch.bfloat16) * np.abs(want) + weighted * 1e-4)


# ---- 4-bit products --------------------------------------------------------------------------------
def int4_case(seed, T, K, N, group, dtype, zeros=True, add=False, f32=False):
    g = torch.Generator().manual_seed(seed)
    dt = TYPES[dtype]
    s = dict(y=torch.full((T, N), 9.0, dtype=torch.float32 if f32 else dt, device="cuda"), x=randn(g, T, K, dtype=dt),
             codes=torch.randint(0, 256, (N, K // 2), generator=g, dtype=torch.uint8).cuda(),
             scales=((torch.rand(N, K // group, generator=g) - 0.3) * K ** -0.5).to(dt).cuda())
    if zeros:
        s["zeros"] = torch.randint(0, 16, (N, K // group), generator=g, dtype=torch.uint8).cuda()
    if add:
        s["add"] = randn(g, T, N, dtype=s["y"].dtype)
    return s


def check_int4(s):
    w = O.int4_weights(s["codes"].cpu().numpy(), f64(s["scales"]), s["zeros"].cpu().numpy() if "zeros" in s else None)
    x, base = f64(s["x"]), f64(s["add"]) if "add" in s else 0.0
    want = x @ w.T + base
    sums = np.abs(x) @ np.abs(w).T + np.abs(base)
    L.int4_linear(**s)
    torch.cuda.synchronize()
    dt = s["y"].dtype
    h, t = (U, 0.0) if dt == torch.float32 else (half_step(dt), tiny(dt))
    steps = x.shape[1] + s["scales"].shape[1] + 16
    within(f64(s["y"]), want, h * np.abs(want) + 2 * U * steps * sums + t, "y")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T,K,N", [(1, 1024, 1024), (1, 128, 1), (2, 384, 17), (7, 8192, 96), (8, 640, 130), (9, 1152, 31), (16, 256, 64),
                                   (17, 2048, 200), (33, 128, 16), (64, 1024, 515), (65, 512, 40), (200, 256, 33)])
def test_int4_values(T, K, N, group, dtype):
    i = T + N + group
    check_int4(int4_case(i, T, K, N, group, dtype, zeros=i % 2 == 0, add=i % 3 == 0, f32=i % 5 == 0))


@pytest.mark.parametrize("K", [32, 64, 96, 160, 992])
def test_int4_inner_sizes_that_no_step_divides(K):
    for T in (1, 12, 40):
        check_int4(int4_case(K, T, K, 50, 32, "fp16"))


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 129])
def test_int4_token_counts_around_the_tiles(T, group):
    check_int4(int4_case(T, T, 512, 136, group, "bf16"))


@pytest.mark.parametrize("T,K,N", [(1, 49152, 9), (1, 49184, 9), (2, 24576, 33), (2, 25600, 33), (4, 12288, 130), (3, 13312, 130), (1, 1024, 9001), (3, 2080, 5000)])
def test_int4_few_tokens_of_long_rows_and_of_many(T, K, N):
    check_int4(int4_case(K + N, T, K, N, 32, "bf16", add=True))


@pytest.mark.parametrize("T", [1, 3, 12, 40])
@pytest.mark.parametrize("K,group", [(1152, 32), (1152, 128), (1088, 64), (2048, 32), (512, 128)])
def test_int4_factors_at_odd_addresses(T, K, group):
    """Scales two bytes and zeros one byte behind a boundary, and rows of them that no word divides."""
    s = int4_case(K + T, T, K, 140, group, "fp16")
    for name in ("scales", "zeros"):
        room = torch.full((s[name].numel() + 9,), 3, dtype=s[name].dtype, device="cuda")
        s[name] = room[1:-8].view(s[name].shape).copy_(s[name])
        assert s[name].data_ptr() % 4 != 0
    check_int4(s)


@pytest.mark.parametrize("T", [1, 9])
def test_int4_scales_at_the_ends_of_their_type(T):
    for dtype, sizes in (("fp16", (2.0 ** -24, 65504.0)), ("bf16", (2.0 ** -126, 2.0 ** 127))):
        s = int4_case(11, T, 256, 64, 64, dtype, f32=True)
        for size in sizes:
            s["scales"].fill_(size)
            s["x"].copy_(randn(torch.Generator().manual_seed(5), T, 256, dtype=TYPES[dtype], std=2.0 ** -4 if size < 1 else 2.0 ** -14))
            check_int4(s)


@pytest.mark.parametrize("T", [1, 5, 8, 9, 33])
@pytest.mark.parametrize("K,group", [(5120, 128), (5120, 64), (6656, 128), (6656, 32)])
def test_int4_parts_that_begin_inside_a_word_of_factors(T, K, group):
    check_int4(int4_case(K + T, T, K, 40, group, "bf16"))


def test_int4_strided_rows_and_add_in_place():
    s = int4_case(3, 5, 512, 100, 64, "bf16", add=True)
    wide, out = torch.zeros(5, 600, dtype=torch.bfloat16, device="cuda"), torch.full((5, 131), 4.0, dtype=torch.bfloat16, device="cuda")
    wide[:, 8:520] = s["x"]
    out[:, 7:107] = s["add"]
    base = s["add"].clone()
    s.update(x=wide[:, 8:520], y=out[:, 7:107], add=out[:, 7:107])
    w = O.int4_weights(s["codes"].cpu().numpy(), f64(s["scales"]), s["zeros"].cpu().numpy())
    want = f64(s["x"]) @ w.T + f64(base)
    L.int4_linear(**s)
    within(f64(s["y"]), want, half_step(torch.bfloat16) * np.abs(want) + 1e-5 * (np.abs(f64(s["x"])) @ np.abs(w).T))
    assert (out[:, :7] == 4).all() and (out[:, 107:] == 4).all()


def test_int4_every_code_and_zero_is_exact():
    """x = 1, one code per group against every zero point: sums of whole numbers, exact in fp32 and compared as such."""
    for dt in TYPES.values():
        codes = torch.arange(16, dtype=torch.uint8).repeat_interleave(16)
        zeros = torch.arange(16, dtype=torch.uint8).repeat(16)[:, None].cuda()
        y = torch.empty(1, 256, dtype=torch.float32, device="cuda")
        L.int4_linear(y, torch.ones(1, 32, dtype=dt, device="cuda"), (codes * 17)[:, None].expand(256, 16).contiguous().cuda(),
                      torch.ones(256, 1, dtype=dt, device="cuda"), zeros)
        assert torch.equal(y[0].cpu(), 32.0 * (codes.float() - zeros[:, 0].cpu().float()))


def test_int4_infinite_and_nan_inputs_stay_in_their_token():
    s = int4_case(4, 9, 256, 40, 64, "bf16")
    s["x"][3, 5], s["x"][8, 200] = float("inf"), float("nan")
    L.int4_linear(**s)
    assert torch.isfinite(s["y"][[0, 1, 2, 4, 5, 6, 7]]).all()
    assert torch.isnan(s["y"][8]).all() and not torch.isfinite(s["y"][3]).any()


@pytest.mark.parametrize("T", [1, 2, 3, 8, 9, 33, 64])
def test_int4_leaves_a_status_word_alone(T):
    """Nothing but an expired wait writes to it; what other calls have set stays."""
    s = int4_case(T, T, 512, 200, 64, "bf16")
    for value in (0, decode.BAD_PAGE):
        word = torch.full((1,), value, dtype=torch.int32, device="cuda")
        check_int4(dict(s, status=word))
        assert int(word) == value


# ---- together --------------------------------------------------------------------------------------
class Layer:
    """A decode layer's attention block with 4-bit projections and deltas; every stage's output is kept."""

    def __init__(self, seed, B, hq, hk, d, dtype, lens, starts, plens):
        g = torch.Generator().manual_seed(seed)
        self.dt, self.h, self.hq, self.hk, self.d = TYPES[dtype], 512, hq, hk, d
        out = (hq + 2 * hk) * d
        self.qkv_w, self.o_w = int4_case(seed, B, self.h, out, 64, dtype), int4_case(seed + 1, B, hq * d, self.h, 128, dtype)
        self.pools = []
        for n in (hq * d, hk * d, hk * d):
            p = L.AdapterPool.empty(4, 1, self.h, n, np.full(4, 16), np.full(4, 2.0), dtype=self.dt)
            for w, std in ((p.wa, self.h ** -0.5), (p.wb, 0.25)):       # the same weights for the same seed
                w.copy_(torch.randn(w.numel(), generator=g).mul_(std).view(w.shape))
            self.pools.append(p)
        self.x = self.qkv_w["x"]
        self.ids = torch.randint(0, 4, (B,), generator=g).int().cuda()
        self.batch = L.LoraBatch(B, 4, self.h, 3)
        self.cache = attend_case(seed, B, hq, hk, d, 16, dtype, lens, starts, plens, fill=0.0)
        ang = torch.arange(4096, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
        self.cos, self.sin = ang.cos().float().cuda(), ang.sin().float().cuda()
        group = torch.zeros(B, dtype=torch.int32)
        for i in range(len(starts) - 1):
            group[starts[i]:starts[i + 1]] = plens[i]
        c = self.cache
        last = (c["lens"] - 1).long()
        self.slots = c["block_table"].gather(1, (last // 16)[:, None])[:, 0].long() * 16 + last % 16
        self.positions = group.cuda().long() + last
        self.qkv = torch.empty(B, out, dtype=self.dt, device="cuda")
        self.deltas = [torch.empty(B, n, dtype=self.dt, device="cuda") for n in (hq * d, hk * d, hk * d)]
        self.q = torch.empty(B, hq, d, dtype=self.dt, device="cuda")
        self.y = torch.empty(B, self.h, dtype=self.dt, device="cuda")

    def step(self):
        L.int4_linear(self.qkv, self.x, self.qkv_w["codes"], self.qkv_w["scales"], self.qkv_w["zeros"])
        self.batch.set_ids(self.ids, self.pools[0])
        self.batch.apply([(self.x, y, p) for y, p in zip(self.deltas, self.pools)], 0, flags=128)
        self.parts = q, k, v = [t.unflatten(1, (-1, self.d)) for t in self.qkv.split([d.shape[1] for d in self.deltas], 1)]
        self.dparts = [t.unflatten(1, (-1, self.d)) for t in self.deltas]
        c = self.cache
        L.append_kv(self.q, q, k, v, c["k_cache"], c["v_cache"], self.positions, self.slots, self.cos, self.sin, *self.dparts)
        L.prefix_attention(**dict(c, q=self.q))
        L.int4_linear(self.y, c["out"].flatten(1), self.o_w["codes"], self.o_w["scales"], self.o_w["zeros"], add=self.x)

    def outputs(self):
        return [t.clone() for t in (self.qkv, *self.deltas, self.q, self.cache["k_cache"], self.cache["v_cache"], self.cache["out"], self.y)]


def make_layer(seed=21, dtype="bf16"):
    return Layer(seed, 9, 8, 2, 64, dtype, [5, 33, 1, 17, 64, 3, 48, 20, 2], [0, 4, 7], [70, 129])


def test_a_layer_step_stage_by_stage():
    a = make_layer()
    before = {n: t.clone() for n, t in a.cache.items()}
    a.step()
    torch.cuda.synchronize()
    check_int4(dict(a.qkv_w, y=a.qkv.clone(), x=a.x))
    host = [f64(t) for t in (torch.zeros_like(a.q), *a.parts, before["k_cache"], before["v_cache"])]
    want = O.append(*host, a.positions.cpu().numpy(), a.slots.cpu().numpy(), f64(a.cos), f64(a.sin), *(f64(t) for t in a.dparts))
    for got, w in zip((a.q, a.cache["k_cache"], a.cache["v_cache"]), want):
        within(f64(got), w, half_step(a.dt) * np.abs(w) + 1e-5)
    check_attend(dict(a.cache, q=a.q, out=torch.empty_like(a.q)))
    check_int4(dict(a.o_w, x=a.cache["out"].flatten(1), y=a.y.clone(), add=a.x))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_the_layer_object_appends_its_deltas(dtype):
    """append_one_layer is the three deltas and the append, from whatever stream and in a captured graph."""
    dt, H, T, D = TYPES[dtype], 512, 12, 64
    torch.manual_seed(9)
    obj = L.Lora_GPU({"n_layers": 2, "batch_size": 16, "lora_rank": 16, "hidden_dim": H, "tp_degree": 1, "max_prefill_batch_size": 2}, dtype=dt)
    for pool in (obj.q_down, obj.q_up, obj.k_down, obj.k_up, obj.v_down, obj.v_up):
        pool.copy_(torch.randn_like(pool) * 0.1)
    s = append_case(61, T, H // D, H // D, D, D, 16, dtype, deltas=False)
    for c in (s["k_cache"], s["v_cache"]):
        c.zero_()
    x = randn(torch.Generator().manual_seed(62), T, H, dtype=dt)
    obj.set_indices(torch.randint(0, 16, (T,), device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
    d = [f(x, 1).view(T, -1, D).clone() for f in (obj.invoke_one_layer_q, obj.invoke_one_layer_k, obj.invoke_one_layer_v)]
    assert all(t.abs().max() > 0 for t in d)
    outs = ("q_out", "k_cache", "v_cache")
    check_append(dict(s, dq=d[0], dk=d[1], dv=d[2]))
    want = [s[n].clone() for n in outs]
    rest = [s[n] for n in ("q_out", "q", "k", "v", "k_cache", "v_cache", "positions", "slots", "cos", "sin")]

    def check():
        torch.cuda.synchronize()
        for n, w in zip(outs, want):
            assert torch.equal(s[n], w)
            s[n].zero_()

    for n in outs:
        s[n].zero_()
    obj.append_one_layer(x, 1, *rest)
    check()
    with torch.cuda.stream(torch.cuda.Stream()):
        obj.append_one_layer(x, 1, *rest)
    check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        obj.append_one_layer(x, 1, *rest)
    graph.replay()
    check()
    with pytest.raises(ValueError, match="q must be"):
        obj.append_one_layer(x, 1, s["q_out"], s["q"][:, :4], *rest[2:])
    with pytest.raises(ValueError, match="k must be"):
        obj.append_one_layer(x[:5], 1, s["q_out"], s["q"][:5], *rest[2:])


def test_a_captured_step_follows_its_inputs_and_eager_calls_between_replays():
    a, b = make_layer(), make_layer()
    a.step(), b.step()                                          # both caches hold this step's keys
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    other = make_layer(33, "fp16")
    for step in range(3):
        for m in (a, b):                                        # another token: one key more, other slots, other inputs
            m.x.copy_(randn(torch.Generator().manual_seed(step), *m.x.shape, dtype=m.dt))
            m.ids.copy_((m.ids + 1) % 4)
            grow = (m.cache["lens"] % 16 != 0).int()            # while the page has room
            m.cache["lens"] += grow
            m.slots += grow.long()
            m.positions += grow.long()
        graph.replay()
        other.step()
        b.step()
        torch.cuda.synchronize()
        for x, y in zip(a.outputs(), b.outputs()):
            assert torch.equal(x, y)


def test_steps_on_two_streams_at_once():
    want = []
    for seed in (41, 42):
        m = make_layer(seed)
        m.step()
        torch.cuda.synchronize()
        want.append(m.outputs())
    models = [make_layer(41), make_layer(42)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for m, s in zip(models, streams):
            with torch.cuda.stream(s):
                m.step()
    torch.cuda.synchronize()
    for m, w in zip(models, want):
        for x, y in zip(m.outputs(), w):
            assert torch.equal(x, y)


# ---- together, with groups of more than 32 rows: both attention kernels have work in every call -----------------
def make_wide_layer(seed=51, dtype="bf16"):
    """Groups of 160 and 420 rows (two streams of rows, two tiles) and of 20, and 20 requests in none."""
    lens = 1 + np.random.default_rng(seed).integers(0, 40, 170)
    return Layer(seed, 170, 8, 2, 64, dtype, lens, [0, 40, 45, 150], [300, 40, 515])


def one_token_more(m, step):
    m.x.copy_(randn(torch.Generator().manual_seed(step), *m.x.shape, dtype=m.dt))
    m.ids.copy_((m.ids + 1) % 4)
    grow = (m.cache["lens"] % 16 != 0).int()                    # while the page has room
    m.cache["lens"] += grow
    m.slots += grow.long()
    m.positions += grow.long()


def test_a_layer_step_of_large_groups_stage_by_stage():
    for dtype in TYPES:
        a = make_wide_layer(dtype=dtype)
        a.step()
        torch.cuda.synchronize()
        got = a.cache["out"].clone()
        check_attend(dict(a.cache, q=a.q, out=torch.empty_like(a.q)))
        out = torch.empty_like(a.q)
        L.prefix_attention(**dict(a.cache, q=a.q, out=out))
        assert torch.equal(got, out)
        check_int4(dict(a.o_w, x=got.flatten(1), y=a.y.clone(), add=a.x))


def test_steps_of_large_groups_follow_what_was_written_just_before():
    """Steps enqueued one behind the other, lengths, slots, queries and keys all written by the call before: as with a wait between."""
    a, b = make_wide_layer(), make_wide_layer()
    got, want = [], []
    torch.cuda.synchronize()
    for step in range(8):
        one_token_more(a, step)
        a.step()
        got.append(a.outputs())
    torch.cuda.synchronize()
    for step in range(8):
        one_token_more(b, step)
        torch.cuda.synchronize()
        b.step()
        torch.cuda.synchronize()
        want.append(b.outputs())
    for x, y in zip(got, want):
        for s, t in zip(x, y):
            assert torch.equal(s, t)


def test_a_captured_step_of_large_groups_follows_its_inputs():
    a, b = make_wide_layer(), make_wide_layer()
    a.step(), b.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    other = make_wide_layer(52, "fp16")
    for step in range(3):
        for m in (a, b):
            one_token_more(m, step)
        graph.replay()
        other.step()
        b.step()
        torch.cuda.synchronize()
        for x, y in zip(a.outputs(), b.outputs()):
            assert torch.equal(x, y)


def test_steps_of_large_groups_on_two_streams_at_once():
    want = []
    for seed in (53, 54):
        m = make_wide_layer(seed)
        m.step()
        torch.cuda.synchronize()
        want.append(m.outputs())
    models, streams = [make_wide_layer(53), make_wide_layer(54)], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(20):
        for m, s in zip(models, streams):
            with torch.cuda.stream(s):
                m.step()
    torch.cuda.synchronize()
    for m, w in zip(models, want):
        for x, y in zip(m.outputs(), w):
            assert torch.equal(x, y)
