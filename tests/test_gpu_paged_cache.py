"""The operators over a paged cache in 16, 8 or 4 bits against plain forms in 64 bits
(paged_util): per-head norms with the rotation and the append, the quantised append
bit for bit against its rule, the read-back, and attention of decode steps, prompt
chunks and drafted trees, at the lengths, pages and masks where a kernel can go wrong."""
import itertools
import math
import random

import pytest
import torch

import mlx_server_runtime_b200 as mxq
from mlx_server_runtime_b200 import attention as A, core, qwen2

import paged_util as P

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(*shape, device="cuda", generator=g)


def quantized_pool(x, gs, bits):
    """A pool's QuantizedKV from its 16-bit form, by quantize()."""
    pages, page, hkv, hd = x.shape
    w, s, b = mxq.quantize(x.reshape(-1, hd), gs, bits)
    return A.QuantizedKV(w.reshape(pages, page, hkv, -1), s.reshape(pages, page, hkv, -1),
                         b.reshape(pages, page, hkv, -1), gs, bits)


def pool_values(c):
    """[rows, hkv, hd] in 64 bits of what a pool stands for (rounded to its type)."""
    if not isinstance(c, A.QuantizedKV):
        return c.flatten(0, 1).double()
    v = P.values(c.codes, c.scales, c.biases, c.group_size, c.bits).flatten(0, 1)
    return v.to(torch.float32).to(c.dtype).double()


# ---------------------------------------------------------------------------- append

@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("hq,hkv,hd,T", [(28, 4, 128, 9), (8, 2, 64, 5), (1, 1, 128, 1),
                                         (3, 1, 64, 2), (64, 8, 128, 300), (28, 4, 128, 2500)])
@pytest.mark.parametrize("qn,kn", [(True, True), (True, False), (False, True)])
def test_append_norms(t, hq, hkv, hd, T, qn, kn):
    if T > 9 and (t is HF or not (qn and kn)):
        pytest.skip("large sizes once")
    g = _gen(hq * T + hd)
    page, pages = 16, T // 16 + 3
    qkv = _randn(g, T, (hq + 2 * hkv) * hd).to(t)
    wq, wk = (1 + 0.3 * _randn(g, hd)).to(t), (1 + 0.3 * _randn(g, hd)).to(t)
    positions = torch.randint(0, 1 << 20, (T,), device="cuda", generator=g, dtype=torch.int32)
    positions[0] = 0
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:T].to(torch.int32)
    if T > 2:
        slots[1], slots[2] = -1, pages * page      # neither is a row of the pool
    kc = torch.full((pages, page, hkv, hd), 7.0, dtype=t, device="cuda")
    vc = kc.clone()
    base, eps = 1e6, 1e-6
    q = A.rope_kv_append(qkv, positions, slots, kc, vc, hq, hkv, hd, base,
                         q_norm=wq if qn else None, k_norm=wk if kn else None, eps=eps)
    x = qkv.reshape(T, -1, hd)
    for got, part, w in ((q, x[:, :hq], wq if qn else None),
                         (None, x[:, hq:hq + hkv], wk if kn else None)):
        ref, mag = P.rotate(part, w, positions, base, eps)
        ok = torch.ones(T, dtype=torch.bool, device="cuda")
        if got is None:
            ok = (slots >= 0) & (slots < pages * page)
            got = kc.flatten(0, 1)[slots.long().clamp(0, pages * page - 1)]
        d = (got.double() - ref).abs()
        assert bool((d <= P.rotate_bound(ref, mag, t))[ok].all()), float(d[ok].max())
    live = (slots >= 0) & (slots < pages * page)
    assert torch.equal(vc.flatten(0, 1)[slots[live].long()], x[live][:, hq + hkv:])
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[slots[live].long()] = False
    assert bool((kc.flatten(0, 1)[rest] == 7).all()) and bool((vc.flatten(0, 1)[rest] == 7).all())


@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hd,gs", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("T,norms", [(1, True), (37, False), (600, True)])
def test_append_quantised_is_the_rule_on_the_rows(t, bits, hd, gs, T, norms):
    """Codes, scales and biases of the written rows are the rule's on the rows the 16-bit
    form writes, bit for bit (constant groups, zero rows, outliers and groups whose ends
    have one magnitude among them); the queries are the same, and rows without a slot keep
    what they held."""
    hq, hkv, page = 7, 1 if T == 37 else 3, 8
    hq = hq * hkv
    g = _gen(T + gs + bits)
    pages = T // page + 2
    qkv = _randn(g, T, (hq + 2 * hkv) * hd)
    qkv[0] = 0.0
    if T > 3:
        qkv[1] = 2.5
        qkv[2, ::17] *= 300.0
    if T > 30:   # values and keys whose groups reach as far up as down
        qkv[20:30, 0::gs] = 3.25
        qkv[20:30, 5::gs] = -3.25
        qkv[20:30] = qkv[20:30].clamp(-3.25, 3.25)
    qkv = qkv.to(t)
    w = (1 + 0.3 * _randn(g, hd)).to(t) if norms else None
    positions = torch.randint(0, 5000, (T,), device="cuda", generator=g, dtype=torch.int32)
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:T].to(torch.int32)
    if T > 9:
        slots[5] = -1
    plain = [torch.zeros(pages, page, hkv, hd, dtype=t, device="cuda") for _ in range(2)]
    ones = torch.ones(hd, dtype=t, device="cuda")
    kq, vq = (A.QuantizedKV.zeros(pages, page, hkv, hd, gs, bits, t) for _ in range(2))
    for c in (kq, vq):
        c.codes.view(torch.int32).fill_(0x5a5a5a5a)
        c.scales.fill_(3)
        c.biases.fill_(-2)
    q = A.rope_kv_append(qkv, positions, slots, kq, vq, hq, hkv, hd, 1e4, q_norm=w, k_norm=w)
    if norms:
        q16 = A.rope_kv_append(qkv, positions, slots, *plain, hq, hkv, hd, 1e4, q_norm=w, k_norm=w)
        assert torch.equal(q, q16)
    else:   # (a norm of the queries alone leaves the keys as they are here)
        A.rope_kv_append(qkv, positions, slots, *plain, hq, hkv, hd, 1e4, q_norm=ones)
    live = slots[slots >= 0].long()
    rest = torch.ones(pages * page, dtype=torch.bool, device="cuda")
    rest[live] = False
    for c16, c in zip(plain, (kq, vq)):
        rows = c16.flatten(0, 1)[live]
        words, scales, biases = (x.cuda() for x in P.quantized(rows, gs, bits))
        got = [c.codes.view(torch.int32), c.scales.view(torch.int16), c.biases.view(torch.int16)]
        got = [x.flatten(0, 1)[live] for x in got]
        assert torch.equal(got[0], words)
        assert torch.equal(got[1], scales.view(torch.int16))
        assert torch.equal(got[2], biases.view(torch.int16))
        assert bool((c.scales.flatten(0, 1)[rest] == 3).all())
        assert bool((c.biases.flatten(0, 1)[rest] == -2).all())
        assert bool((c.codes.view(torch.int32).flatten(0, 1)[rest] == 0x5a5a5a5a).all())


def test_append_row_stride_and_empty():
    hq, hkv, hd, t = 7, 1, 128, BF
    g = _gen(3)
    wide = _randn(g, 6, (hq + 2 * hkv) * hd + 64).to(t)
    qkv = wide[:, 64:]
    positions = torch.arange(6, dtype=torch.int32, device="cuda")
    w = torch.ones(hd, dtype=t, device="cuda")
    caches = [[torch.zeros(2, 8, hkv, hd, dtype=t, device="cuda") for _ in range(2)]
              for _ in range(2)]
    qa = A.rope_kv_append(qkv, positions, positions, *caches[0], hq, hkv, hd, q_norm=w, k_norm=w)
    qb = A.rope_kv_append(qkv.contiguous(), positions, positions, *caches[1], hq, hkv, hd,
                          q_norm=w, k_norm=w)
    assert torch.equal(qa, qb) and torch.equal(caches[0][0], caches[1][0])
    none = positions[:0]
    q = A.rope_kv_append(qkv[:0], none, none, *caches[0], hq, hkv, hd, q_norm=w, k_norm=w)
    assert q.shape == (0, hq, hd)
    k, v = A.kv_cache_read(*caches[0], none)
    assert k.shape == v.shape == (0, hkv, hd)


# ---------------------------------------------------------------------------- read back

@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("bits,hd,gs", [(4, 64, 32), (4, 128, 64), (8, 64, 64), (8, 128, 128),
                                        (8, 128, 32), (4, 128, 128), (16, 128, 0), (16, 64, 0)])
def test_read_back(t, bits, hd, gs):
    g = _gen(bits + hd)
    pages, page, hkv = 5, 32, 3
    if bits == 16:
        kc, vc = (_randn(g, pages, page, hkv, hd).to(t) for _ in range(2))
    else:
        kc, vc = (quantized_pool(_randn(g, pages, page, hkv, hd).to(t), gs, bits)
                  for _ in range(2))
        # every code against scales and biases of all signs and sizes
        kc.codes.view(torch.int32).copy_(torch.randint(-2 ** 31, 2 ** 31, kc.codes.shape,
                                                       device="cuda", generator=g))
        kc.scales.copy_(_randn(g, *kc.scales.shape) * torch.exp(3 * _randn(g, *kc.scales.shape)))
    slots = torch.tensor([0, 159, 160, -1, 7, 7, 2 ** 31 - 1, -2 ** 31] + list(range(3, 150, 2)),
                         dtype=torch.int32, device="cuda")
    k, v = A.kv_cache_read(kc, vc, slots)
    bad = (slots < 0) | (slots >= pages * page)
    at = slots.long().clamp(0, pages * page - 1)
    for got, c in ((k, kc), (v, vc)):
        assert got.dtype == t and got.shape == (len(slots), hkv, hd)
        assert not bool(got[bad].any())
        if bits == 16:
            assert torch.equal(got[~bad], c.flatten(0, 1)[at][~bad])
        else:
            ref = P.values(c.codes, c.scales, c.biases, gs, bits).flatten(0, 1)[at][~bad]
            near = (got[~bad].double() - ref).abs() <= P.half_step(ref, t)
            if t is HF:   # 65504 plus half a step and beyond rounds to infinity
                near |= (ref.abs() >= 65520) & (got[~bad].double() == torch.sign(ref) * math.inf)
            assert bool(near.all())


# ---------------------------------------------------------------------------- attention

def _problem(seed, t, bits, gs, hq, hkv, hd, page, lens, news, tree=False, stale=True):
    """Random pools over shuffled pages, with NaN in every row no sequence holds."""
    g = _gen(seed)
    r = random.Random(seed)
    blocks = [-(-L // page) for L in lens]
    pages = sum(blocks) + 3
    perm = list(range(pages))
    r.shuffle(perm)
    width = max(1, max(blocks)) + 1
    rows, at = [], 0
    for nb in blocks:
        rows.append(perm[at:at + nb] + [perm[-1]] * (width - nb))
        at += nb
    k16 = (_randn(g, pages, page, hkv, hd) * torch.exp(0.5 * _randn(g, hd))).to(t)
    v16 = _randn(g, pages, page, hkv, hd).to(t)
    kc, vc = (k16, v16) if bits == 16 else (quantized_pool(x, gs, bits) for x in (k16, v16))
    kd, vd = pool_values(kc), pool_values(vc)
    if stale:
        held = torch.zeros(pages * page, dtype=torch.bool)
        for b, L in enumerate(lens):
            for j in range(L):
                held[rows[b][j // page] * page + j % page] = True
        for c in (kc, vc):
            for x in ([c] if bits == 16 else [c.scales, c.biases]):
                x.flatten(0, 1)[~held.cuda()] = float("nan")
    cu = [0] + list(itertools.accumulate(news))
    q = (_randn(g, cu[-1], hq, hd) * 1.5).to(t)
    masks = None
    if tree:
        masks = A.tree_masks([[r.randint(max(-1, i - 4), i - 1) for i in range(n)] for n in news],
                             "cpu").tolist()
    return dict(q=q, cu=cu, kc=kc, vc=vc, kd=kd, vd=vd, lens=lens, masks=masks, scale=hd ** -0.5,
                table={"page": page, "pages": pages, "rows": rows}, t=t, news=news)


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _run(p, how, max_kv=None):
    bt, lens = _i32(p["table"]["rows"]), _i32(p["lens"])
    max_kv = max(p["lens"]) if max_kv is None else max_kv
    if how == "decode":
        return A.paged_attention_decode(p["q"], p["kc"], p["vc"], bt, lens, max_kv, p["scale"])
    cu, mq = _i32(p["cu"]), max(p["news"])
    if how == "tree":
        m = torch.tensor(p["masks"], dtype=torch.int64, device="cuda")
        return A.paged_attention_tree(p["q"], cu, mq, p["kc"], p["vc"], bt, lens, max_kv, m,
                                      p["scale"])
    return A.paged_attention_prefill(p["q"], cu, mq, p["kc"], p["vc"], bt, lens, p["scale"])


def _check(p, got):
    ref, tol = P.attention(p["q"], p["cu"], p["kd"], p["vd"], p["table"], p["lens"], p["scale"],
                           p["masks"], p["t"])
    d = (got.double() - ref).abs()
    assert bool(torch.isfinite(got).all())
    worst = float((d / tol.clamp_min(1e-30)).max())
    assert bool((d <= tol).all()), f"error up to {worst:.2f} of the bound"


CACHES = [(4, 32), (4, 64), (4, 128), (8, 32), (8, 64), (8, 128)]
HEADS = [(28, 4, 128), (8, 2, 64), (4, 4, 128), (8, 1, 128), (3, 3, 64), (10, 2, 64)]


@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("bits,gs", CACHES)
@pytest.mark.parametrize("hq,hkv,hd", HEADS[:4])
@pytest.mark.parametrize("page", [8, 16, 32])
def test_decode(t, bits, gs, hq, hkv, hd, page):
    if gs > hd:
        pytest.skip("a group is at most a row")
    lens = [1, 17, 0, 64, 65, 300, 7, 129]
    p = _problem(hq + page + bits, t, bits, gs, hq, hkv, hd, page, lens, [1] * len(lens))
    _check(p, _run(p, "decode"))


@pytest.mark.parametrize("bits,gs", [(4, 64), (8, 32)])
@pytest.mark.parametrize("lens", [[1], [2], [8], [9], [63], [4000, 1, 5000], [64] * 70,
                                  [3, 0, 0, 0, 11] * 60])
def test_decode_lengths(bits, gs, lens):
    p = _problem(len(lens), BF, bits, gs, 28, 4, 128, 16, lens, [1] * len(lens))
    _check(p, _run(p, "decode"))
    # a looser bound on the lengths shares the work out differently
    _check(p, _run(p, "decode", max_kv=(max(lens) + 15) // 16 * 16))


@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("bits,gs", [(16, 0), (4, 64), (8, 32), (8, 64)])
@pytest.mark.parametrize("hq,hkv,hd", HEADS)
@pytest.mark.parametrize("news", [[1, 3, 8, 5], [33, 64, 1, 17], [0, 2, 0, 40]])
def test_tree(t, bits, gs, hq, hkv, hd, news):
    lens = [news[0] + 300, news[1], news[2] + 1, news[3] + 64 - news[3] % 16]
    p = _problem(sum(news) + hq, t, bits, gs, hq, hkv, hd, 16, lens, news, tree=True)
    _check(p, _run(p, "tree"))


@pytest.mark.parametrize("bits,gs", [(16, 0), (4, 64)])
def test_tree_long_and_wide(bits, gs):
    news = [64, 64, 31, 1, 0]
    lens = [4100, 64, 2000, 777, 5]
    p = _problem(bits, BF, bits, gs, 28, 4, 128, 16, lens, news, tree=True)
    _check(p, _run(p, "tree"))


@pytest.mark.parametrize("bits,gs,page", [(16, 0, 8), (8, 64, 32), (4, 32, 16)])
def test_tree_rows_that_see_nothing(bits, gs, page):
    """No context and an empty mask: zeros. Bit 63, bits past the tree, and masks that are
    no tree at all are taken as they stand."""
    news, lens = [64, 3, 10], [64, 3, 30]
    p = _problem(5, BF, bits, gs, 8, 2, 64, page, lens, news, tree=True)
    r = random.Random(1)
    m = [r.getrandbits(64) for _ in range(sum(news))]
    m[0], m[65], m[5] = 0, 0xfff8 << 48 | 0xff8, (1 << 64) - 1
    p["masks"] = [x - (1 << 64) if x >> 63 else x for x in m]
    got = _run(p, "tree")
    assert not bool(got[0].any()) and not bool(got[65].any())
    _check(p, got)


@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("bits,gs", [(4, 64), (8, 32), (8, 128)])
@pytest.mark.parametrize("hq,hkv,hd", [(28, 4, 128), (8, 2, 64), (5, 5, 64)])
def test_prefill(t, bits, gs, hq, hkv, hd):
    if gs > hd:
        pytest.skip("a group is at most a row")
    news, lens = [64, 100, 1, 0, 200, 130], [64, 333, 77, 5, 200, 131]
    p = _problem(hq + bits, t, bits, gs, hq, hkv, hd, 16, lens, news)
    _check(p, _run(p, "prefill"))


def test_prefill_long():
    news, lens = [700, 513], [1500, 513]
    p = _problem(9, BF, 4, 64, 28, 4, 128, 16, lens, news)
    _check(p, _run(p, "prefill"))


@pytest.mark.parametrize("how,bits", [("decode", 4), ("tree", 16), ("tree", 8), ("prefill", 8)])
def test_bad_pages_are_left_out(how, bits):
    lens = [100, 40, 200]
    news = [1] * 3 if how == "decode" else [20, 5, 30]
    p = _problem(4, BF, bits, 64, 8, 2, 64, 16, lens, news, tree=how == "tree")
    rows = [list(r) for r in p["table"]["rows"]]
    rows[0][2], rows[1][0], rows[2][5], rows[2][12] = -1, p["table"]["pages"], 2 ** 31 - 1, -2 ** 31
    p["table"] = dict(p["table"], rows=rows)
    _check(p, _run(p, how))


@pytest.mark.parametrize("how,bits", [("tree", 16), ("tree", 4), ("prefill", 4)])
def test_rows_behind_the_last_sequence(how, bits):
    """A padded batch: rows of q behind cu_q[-1] hold NaN and come out as zeros."""
    news, lens = [7, 30], [90, 30]
    p = _problem(6, BF, bits, 64, 7, 1, 128, 16, lens, news, tree=how == "tree")
    want = _run(p, how)
    pad = torch.full((11, 7, 128), float("nan"), dtype=BF, device="cuda")
    p2 = dict(p, q=torch.cat([p["q"], pad]),
              masks=None if p["masks"] is None else p["masks"] + [-1] * 11)
    got = _run(p2, how)
    assert torch.equal(got[:37], want) and not bool(got[37:].any())


def test_nothing_but_padding():
    """No sequence, or none with a token: every row is behind the last and comes out zero."""
    p = _problem(7, BF, 4, 64, 7, 1, 128, 16, [30], [3], tree=True)
    m = torch.zeros(3, dtype=torch.int64, device="cuda")
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    out = A.paged_attention_tree(p["q"], _i32([0]), 4, p["kc"], p["vc"], none.reshape(0, 2), none,
                                 0, m, 0.1)
    assert out.shape == p["q"].shape and not bool(out.any())
    bt = _i32(p["table"]["rows"])
    for cu, max_q in (([0, 0], 0), ([0, 0], 4)):
        out = A.paged_attention_tree(p["q"], _i32(cu), max_q, p["kc"], p["vc"], bt, _i32([30]), 30,
                                     m, 0.1)
        assert not bool(out.any())
    out = A.paged_attention_decode(p["q"][:0], p["kc"], p["vc"], none.reshape(0, 2), none, 0, 0.1)
    assert out.shape == (0, 7, 128)
    # sequences without a key, and no key anywhere
    out = A.paged_attention_tree(p["q"], _i32([0, 3]), 3, p["kc"], p["vc"], bt, _i32([0]), 0, m,
                                 0.1)
    assert not bool(out.any())


@pytest.mark.parametrize("bits", [16, 4])
def test_sequences_in_groups(bits):
    """More expanded keys than are held at once: the sequences are taken group by group."""
    news, lens = [20, 0, 5, 33, 1], [4000, 3, 2500, 33, 700]
    p = _problem(13, BF, bits, 64, 8, 2, 128, 16, lens, news)
    bound = 300_000          # keys a sequence could have: 614 MB of them, so two groups and more
    width = bound // 16
    rows = [r + [0] * (width - len(r)) for r in p["table"]["rows"]]
    p["table"] = dict(p["table"], rows=rows)
    got = (_run(p, "prefill") if bits != 16 else
           A.paged_attention_tree(p["q"], _i32(p["cu"]), 33, p["kc"], p["vc"], _i32(rows),
                                  _i32(lens), bound,
                                  A.tree_masks([list(range(-1, n - 1)) for n in news]), p["scale"]))
    _check(p, got)


def test_lengths_past_their_bounds_stay_in_bounds():
    """Device-side lengths and offsets that break the contract are cut to it."""
    p = _problem(8, BF, 4, 64, 8, 2, 64, 16, [50, 20], [4, 3], tree=True)
    bt = _i32(p["table"]["rows"])
    m = torch.tensor(p["masks"], dtype=torch.int64, device="cuda")
    for cu, lens in (([0, 4, 2 ** 31 - 1], [50, 20]), ([-5, 4, 2], [-7, 20]),
                     ([0, 4, 7], [2 ** 31 - 1, 20]), ([6, 2, 7], [1, 1])):
        out = A.paged_attention_tree(p["q"], _i32(cu), 4, p["kc"], p["vc"], bt, _i32(lens), 50, m,
                                     0.125)
        assert out.shape == p["q"].shape
    torch.cuda.synchronize()


@pytest.mark.parametrize("how,bits", [("decode", 8), ("tree", 4), ("tree", 16), ("prefill", 8)])
def test_large_scores_and_equal_keys(how, bits):
    """Scores far apart (one key takes all), equal scores, and a scale of zero."""
    news = [1] * 3 if how == "decode" else [50, 3, 64]
    p = _problem(10, HF, bits, 64, 8, 2, 64, 16, [200, 77, 64], news, tree=how == "tree")
    for scale in (0.0, 4.0, -0.3):
        p["scale"] = scale
        _check(p, _run(p, how))


def test_rising_scores():
    """The largest score grows tile after tile, so what is summed so far is rescaled again
    and again."""
    for how, bits in (("decode", 8), ("tree", 16), ("prefill", 4)):
        news = [1] if how == "decode" else [40]
        p = _problem(12, BF, bits, 64, 8, 2, 64, 16, [1500], news, tree=how == "tree")
        t = torch.linspace(0, 1, p["table"]["pages"] * 16, device="cuda")
        order = torch.zeros(p["table"]["pages"] * 16, device="cuda")
        rows = [p["table"]["rows"][0][j // 16] * 16 + j % 16 for j in range(1500)]
        order[rows] = t[:1500]
        k = (p["q"][0, 0].float() * order[:, None, None]).to(BF).expand(-1, 2, -1)
        k = k.reshape(p["table"]["pages"], 16, 2, 64).contiguous()
        p["kc"] = k if bits == 16 else quantized_pool(k, 64, bits)
        p["kd"] = pool_values(p["kc"])
        p["scale"] = 8.0
        _check(p, _run(p, how))


@pytest.mark.parametrize("bits,rows", [(16, 5 << 20), (4, 18 << 20)])
def test_offsets_past_32_bits(bits, rows):
    """Rows more than 2^32 bytes into their pools give what rows at the front give."""
    hq, hkv, hd, page, T = 8, 4, 128, 16, 200
    g = _gen(61)
    qkv = _randn(g, T, (hq + 2 * hkv) * hd).to(BF)
    pos = _i32(list(range(T)))

    def pool():
        shape = (rows // page, page, hkv)
        if bits == 16:
            return torch.empty(*shape, hd, dtype=BF, device="cuda")
        codes = torch.empty(*shape, hd * bits // 32, dtype=torch.int32, device="cuda")
        assert codes.numel() * 4 > 1 << 32
        return A.QuantizedKV(codes, *(torch.empty(*shape, hd // 64, dtype=BF, device="cuda")
                                      for _ in range(2)), 64, bits)

    k, v = pool(), pool()
    blocks = -(-T // page)
    outs = []
    for first in (0, rows // page - blocks):
        slots = _i32([first * page + i for i in range(T)])
        bt = _i32([[first + j for j in range(blocks)]])
        q = A.rope_kv_append(qkv, pos, slots, k, v, hq, hkv, hd, 1e6, q_norm=None,
                             k_norm=torch.ones(hd, dtype=BF, device="cuda"))
        outs.append([*A.kv_cache_read(k, v, slots)])
        for n in (1, 40):  # few rows of a kv head, and many
            m = A.tree_masks([list(range(-1, n - 1))])
            outs[-1].append(A.paged_attention_tree(q[T - n:], _i32([0, n]), n, k, v, bt, _i32([T]),
                                                   T, m, hd ** -0.5))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(a.any())


def test_same_result_every_time():
    p = _problem(11, BF, 4, 64, 28, 4, 128, 16, [3000, 50, 900], [1] * 3)
    first = _run(p, "decode")
    for _ in range(20):
        assert torch.equal(_run(p, "decode"), first)


# ---------------------------------------------------------------------------- as they are used

def test_streams_and_graphs():
    """Calls on another stream, and two captured graphs replayed at once on two streams,
    give what the eager calls give."""
    ps = [_problem(20 + i, BF, 4, 64, 28, 4, 128, 16, [2500, 700 + 100 * i, 64], [1] * 3)
          for i in range(2)]
    want = [_run(p, "decode") for p in ps]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _run(ps[0], "decode")
    torch.cuda.synchronize()
    assert torch.equal(got, want[0])
    # static inputs for the captures
    graphs, outs = [], []
    for p in ps:
        bt, lens = _i32(p["table"]["rows"]), _i32(p["lens"])
        with torch.cuda.stream(side):
            A.paged_attention_decode(p["q"], p["kc"], p["vc"], bt, lens, 2500, p["scale"])
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(A.paged_attention_decode(p["q"], p["kc"], p["vc"], bt, lens, 2500,
                                                 p["scale"]))
        graphs.append((g, bt, lens))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(20):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for st, (g, _, _) in zip(streams, graphs):
            with torch.cuda.stream(st):
                for _ in range(3):
                    g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


@pytest.mark.parametrize("bits,how", [(4, "tree"), (16, "tree"), (8, "prefill")])
def test_many_rows_at_once_and_in_graphs(bits, how):
    """The calls of several launches and a large workspace: two of them at once on two
    streams, eager and as captured graphs, give what each gives alone."""
    ps = [_problem(40 + i, BF, bits, 64, 28, 4, 128, 16, [1900 - 300 * i, 77, 640], [31, 9 + i, 64],
                   tree=how == "tree") for i in range(2)]
    devs = [[_i32(p["table"]["rows"]), _i32(p["lens"]), _i32(p["cu"]),
             torch.tensor(p["masks"] or [0], dtype=torch.int64, device="cuda")] for p in ps]

    def call(p, d):
        bt, lens, cu, m = d
        if how == "tree":
            return A.paged_attention_tree(p["q"], cu, 64, p["kc"], p["vc"], bt, lens,
                                          max(p["lens"]), m, p["scale"])
        return A.paged_attention_prefill(p["q"], cu, 64, p["kc"], p["vc"], bt, lens, p["scale"])

    want = [call(p, d) for p, d in zip(ps, devs)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ps]
    got = []
    for _ in range(5):
        for st, p, d in zip(streams, ps, devs):
            with torch.cuda.stream(st):
                got.append(call(p, d))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 2])
    graphs, outs = [], []
    for st, p, d in zip(streams, ps, devs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            outs.append(call(p, d))
        graphs.append(g)
    for _ in range(10):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_overlapped_launches(bits):
    """With launch overlap every launch waits for what it reads and for what it writes over:
    steps that append, attend (one row, a tree) and read back on the rows of the step before
    give what they give without."""
    hq, hkv, hd, page, n, steps = 28, 4, 128, 16, 24, 8
    g = _gen(51)
    qkv = _randn(g, steps, n, (hq + 2 * hkv) * hd).to(BF)
    w = (1 + 0.2 * _randn(g, hd)).to(BF)
    masks = A.tree_masks([[-1] + [i // 2 for i in range(n - 1)]])

    def run():
        cache = A.PagedKVCache(1, hkv, hd, 64, page, bits=bits)
        k, v = cache.keys[0], cache.values[0]
        bt = cache.allocate([1000], generator=torch.Generator().manual_seed(3))
        slots = cache.slots(bt, [range(1000)])
        args = []
        for i in range(steps):  # (every step's tokens lie over half of the last one's)
            at = 600 + i * n // 2
            args.append((_i32(list(range(at, at + n))), slots[at:at + n].contiguous(),
                         _i32([at + n]), _i32([0, n])))
        torch.cuda.synchronize()
        outs = []
        for i, (pos, sl, lens, cu) in enumerate(args):
            q = A.rope_kv_append(qkv[i], pos, sl, k, v, hq, hkv, hd, 1e6, w, w)
            outs.append(A.paged_attention_tree(q, cu, n, k, v, bt, lens, 1000, masks, hd ** -0.5))
            one = _i32([0, 1])
            outs.append(A.paged_attention_tree(q[-1:], one, 1, k, v, bt, lens, 1000, masks[:1],
                                               hd ** -0.5))
            outs += A.kv_cache_read(k, v, sl)
        torch.cuda.synchronize()
        return outs

    want = run()
    for _ in range(3):
        with mxq.launch_overlap(True):
            got = run()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


CFG = dict(hidden_size=896, intermediate_size=1536, num_attention_heads=7, num_key_value_heads=1,
           num_hidden_layers=2, vocab_size=640, rope_theta=1e6, qk_norm=True)


def _decoder(bits, launch=False, cfg=CFG, B=3, max_len=160):
    c = qwen2.Qwen2Config(**cfg)
    model = qwen2.Qwen2ForCausalLM(c, seed=3, norm_jitter=0.1, bias_std=0.5)
    cache = A.PagedKVCache(c.num_hidden_layers, c.num_key_value_heads, c.head_dim, num_pages=64,
                           bits=bits, group_size=64)
    return model, cache, qwen2.GreedyDecoder(model, cache, B, max_len=max_len,
                                             page_generator=torch.Generator().manual_seed(4))


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_decoder_over_each_cache(bits):
    """Prefill and decode steps of a model with head norms over a cache of each width, and
    the captured step replayed: the graph's tokens are the eager steps'."""
    lengths = [5, 37, 130]
    ids = torch.randint(0, 640, (sum(lengths),), generator=torch.Generator().manual_seed(1),
                        dtype=torch.int32)
    runs = []
    for graph in (False, True):
        model, cache, dec = _decoder(bits)
        out = [dec.prefill(ids, lengths)]
        if graph:
            dec.capture()
            out.append(dec.ids.clone())
            for _ in range(4):
                dec.replay()
                out.append(dec.ids.clone())
        else:
            for _ in range(5):
                dec.step()
                out.append(dec.ids.clone())
        torch.cuda.synchronize()
        runs.append(torch.stack(out).cpu())
        dec.close()
    assert torch.equal(*runs)


def test_drafted_tree_equals_steps():
    """Append a tree of drafted tokens and attend: each token's row is what a decode step
    over its own path (context, ancestors, itself) gives, for each width of cache. The
    append, read-back and attention run together as a serving step does."""
    hq, hkv, hd, page, ctx = 7, 1, 128, 16, 75
    parents = [-1, 0, 0, 1, 3, 2, -1, 6]
    n = len(parents)
    g = _gen(31)
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    qkv = _randn(g, ctx + n, (hq + 2 * hkv) * hd).to(BF)
    w = (1 + 0.2 * _randn(g, hd)).to(BF)
    positions = _i32(list(range(ctx)) + [ctx + d for d in depth])
    for bits in (16, 8, 4):
        cache = A.PagedKVCache(1, hkv, hd, 32, page, bits=bits)
        k, v = cache.keys[0], cache.values[0]
        bt = cache.allocate([ctx + n], generator=torch.Generator().manual_seed(2))
        slots = cache.slots(bt, [range(ctx + n)])
        q = A.rope_kv_append(qkv, positions, slots, k, v, hq, hkv, hd, 1e6, q_norm=w, k_norm=w)
        tree = A.paged_attention_tree(q[ctx:], _i32([0, n]), n, k, v, bt, _i32([ctx + n]), ctx + n,
                                      A.tree_masks([parents]), hd ** -0.5)
        kd, vd = A.kv_cache_read(k, v, slots)
        for i in range(n):
            path, j = [], i
            while j >= 0:
                path.append(ctx + j)
                j = parents[j]
            rows = list(range(ctx)) + sorted(path)
            ref, tol = P.attention(q[ctx + i:ctx + i + 1], [0, 1], kd[rows].double(),
                                   vd[rows].double(),
                                   {"page": len(rows), "pages": 1, "rows": [[0]]}, [len(rows)],
                                   hd ** -0.5, None, BF)
            assert bool(((tree[i:i + 1].double() - ref).abs() <= tol).all())
