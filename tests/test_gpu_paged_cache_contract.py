"""The paged-cache operators against 64-bit forms where the other tests of them do not go:
values that are not finite, the cache's quantisation beside quantize()'s, calls of nine to
sixteen rows, every page size under the tensor-memory accelerator, batches of hundreds of
sequences, block tables far wider than the sequences, and a model's attention layer over a
quantised cache."""
import math

import pytest
import torch

import mlx_server_runtime_b200 as mxq
from mlx_server_runtime_b200 import attention as A, core, qwen2

import paged_util as P
import test_gpu_paged_cache as base

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


# ---------------------------------------------------------------------------- not finite

@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("bits,hd,gs", [(4, 64, 32), (4, 128, 64), (8, 64, 64), (8, 128, 128),
                                        (8, 128, 32), (4, 128, 128)])
@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("norms", [True, False])
def test_append_of_values_that_are_not_finite(t, bits, hd, gs, value, norms):
    """A group that holds a NaN or an infinity reads back as NaN, all of it, and every other
    group as it does without."""
    hq, hkv, T, page = 4, 2, 6, 8
    g = base._gen(bits + hd + gs)
    clean = base._randn(g, T, (hq + 2 * hkv) * hd).to(t)
    qkv = clean.clone()
    k_at, v_at = hq * hd, (hq + hkv) * hd
    hit = [(1, 0, 3), (2, 1, hd - 1), (4, 1, hd // 2)]     # token, head, element
    for tok, h, e in hit:
        qkv[tok, k_at + h * hd + e] = value
        qkv[tok, v_at + h * hd + e] = value
    w = torch.ones(hd, dtype=t, device="cuda") if norms else None
    ids = base._i32(list(range(T)))
    outs = []
    for x in (clean, qkv):
        kc, vc = (A.QuantizedKV.zeros(2, page, hkv, hd, gs, bits, t) for _ in range(2))
        A.rope_kv_append(x, ids + 3, ids, kc, vc, hq, hkv, hd, 1e4, q_norm=w, k_norm=w)
        outs.append(A.kv_cache_read(kc, vc, ids))
    lost_k = torch.zeros(T, hkv, hd, dtype=torch.bool, device="cuda")
    lost_v = lost_k.clone()
    for tok, h, e in hit:
        lost_v[tok, h, e // gs * gs:(e // gs + 1) * gs] = True
        if norms:          # (the mean of squares is none of the head's values' any more)
            lost_k[tok, h] = True
        else:              # the element and the one it is rotated with
            for x in (e, (e + hd // 2) % hd):
                lost_k[tok, h, x // gs * gs:(x // gs + 1) * gs] = True
    if norms and math.isinf(value):
        # an infinite mean of squares makes zeros of the finite elements and a NaN of the
        # infinite one, so only the groups of its pair are lost
        lost_k[:] = False
        for tok, h, e in hit:
            for x in (e, (e + hd // 2) % hd):
                lost_k[tok, h, x // gs * gs:(x // gs + 1) * gs] = True
    for want, got, lost in zip(outs[0], outs[1], (lost_k, lost_v)):
        assert bool(torch.isnan(got[lost]).all())
        same = ~lost
        if lost is lost_k and norms and math.isinf(value):
            for tok, h, _ in hit:      # (the rest of those heads is zeros: checked apart)
                rest = got[tok, h][~lost[tok, h]]
                assert not bool(rest.any())
                same[tok, h] = False
        assert torch.equal(got[same], want[same])


@pytest.mark.parametrize("how,bits,hd", [("decode", 4, 128), ("decode", 8, 64), ("tree", 16, 128),
                                         ("tree", 16, 64), ("tree", 4, 128), ("prefill", 8, 64)])
@pytest.mark.parametrize("side", ["k", "v"])
def test_a_key_or_value_that_is_none_shows(how, bits, hd, side):
    """A NaN in a key every row of its sequence sees makes those rows of the kv head NaN, one
    in a value the elements it stands for; other heads and sequences keep their bits."""
    hq, hkv, gs = 8, 2, 32
    news = [1] * 3 if how == "decode" else [20, 5, 30]
    p = base._problem(71, BF, bits, gs, hq, hkv, hd, 16, [150, 40, 300], news, tree=how == "tree")
    want = base._run(p, how)
    at = p["table"]["rows"][2][130 // 16] * 16 + 130 % 16      # key 130 of the last sequence
    c = p[side + "c"]
    (c if bits == 16 else c.scales).flatten(0, 1)[at, 1, 0] = math.nan
    got = base._run(p, how)
    lost = torch.zeros_like(got, dtype=torch.bool)
    lo = p["cu"][2] if how != "decode" else 2
    if side == "k":
        lost[lo:, hq // 2:] = True
    else:
        lost[lo:, hq // 2:, :1 if bits == 16 else gs] = True
    assert bool(torch.isnan(got[lost]).all())
    assert torch.equal(got[~lost], want[~lost])


# ---------------------------------------------------------------------------- the two rules

@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("bits,hd,gs", [(4, 128, 64), (8, 128, 64), (4, 64, 32), (8, 128, 128)])
def test_append_beside_quantize(t, bits, hd, gs):
    """Values appended to a quantised cache and the same rows through quantize(). Groups
    are the same, bit for bit, unless the larger end lies half way between two codes from
    zero; then one rule may take one neighbour and the other the next, and what the group
    stands for differs by a step and a half at most, with the rounding of scales and
    values.

    Half way: both steps are range / n within 3 * 2^-24 of it (the product's two roundings
    and the reciprocal's; the quotient's one), the end over the step is rounded once more, so
    the two differ only where a half-integer lies within 2^-22 of end * n / range, relatively.

    A step and a half: with the end at m + 1/2 steps, m codes span the range (m + 1/2) / m
    times over and miss a value by half a code, (m + 1/2) / 2m steps; m + 1 codes clip the far
    end by n / 2(m + 1) steps. The larger end is at least n / 2 steps off, m >= (n - 1) / 2:
    0.536 and 1 steps (n = 15). A scale is rounded to t (n codes of it), each value too."""
    hq, hkv, T = 1, 1, 20000
    n = 2 ** bits - 1
    g = base._gen(bits + hd + gs)
    qkv = base._randn(g, T, 3 * hd)
    qkv[:200, 0::gs] = 3.25                       # ends of one magnitude
    qkv[:200, 5::gs] = -3.25
    qkv[:200] = qkv[:200].clamp(-3.25, 3.25)
    qkv = qkv.to(t)
    ids = base._i32(list(range(T)))
    kc, vc = (A.QuantizedKV.zeros(-(-T // 16), 16, hkv, hd, gs, bits, t) for _ in range(2))
    A.rope_kv_append(qkv, ids, ids, kc, vc, hq, hkv, hd, 1e4)
    rows = qkv[:, 2 * hd:].contiguous()
    w, s, b = mxq.quantize(rows, gs, bits)
    mine = [vc.codes.flatten(0, 2)[:T], vc.scales.flatten(0, 2)[:T], vc.biases.flatten(0, 2)[:T]]
    per = gs * bits // 32
    same = (mine[0].view(torch.int32).unflatten(-1, (-1, per)) ==
            w.view(torch.int32).unflatten(-1, (-1, per))).all(-1)
    same &= (mine[1].view(torch.int16) == s.view(torch.int16))
    same &= (mine[2].view(torch.int16) == b.view(torch.int16))
    v = rows.double().unflatten(-1, (-1, gs))
    hi, lo = v.amax(-1), v.amin(-1)
    step = (hi - lo) / n
    ends = torch.maximum(hi.abs(), lo.abs()) / step
    off = (ends - (ends.floor() + 0.5)).abs()
    assert bool((off <= 2.0 ** -22 * ends)[~same].all())
    assert 0 < int((~same).sum()) < same.numel() // 50
    va, vb = (P.values(*x, gs, bits).float().to(t).double().unflatten(-1, (-1, gs))
              for x in (mine, (w, s, b)))
    room = step * (1.54 + 2 * n * 1.08 * P.U[t])
    bound = room[..., None] + P.U[t] * (va.abs() + vb.abs()) * 1.01
    assert bool(((va - vb).abs() <= bound).all())


# ---------------------------------------------------------------------------- variants

ROWS16 = [(14, 2, 128, [2, 1, 2, 0]), (8, 1, 128, [2, 2, 1, 1]), (10, 2, 128, [3, 1, 2, 3]),
          (16, 4, 128, [4, 3, 0, 1]), (4, 4, 128, [16, 9, 1, 5]), (7, 1, 64, [2, 1, 0, 2]),
          (8, 2, 64, [3, 4, 1, 2]), (3, 1, 64, [4, 5, 3, 1])]


@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("bits,gs", base.CACHES)
@pytest.mark.parametrize("hq,hkv,hd,news", [x for x in ROWS16])
@pytest.mark.parametrize("how,page", [("tree", 16), ("prefill", 8), ("tree", 32)])
def test_nine_to_sixteen_rows(t, bits, gs, hq, hkv, hd, news, how, page):
    """A few new tokens over a quantised cache: sixteen rows of a kv head to a chunk."""
    gs = min(gs, hd)
    assert 8 < max(news) * (hq // hkv) <= 16
    lens = [news[0] + 300, news[1], news[2] + 129, news[3] + 31]
    p = base._problem(hq + gs + bits, t, bits, gs, hq, hkv, hd, page, lens, news,
                      tree=how == "tree")
    base._check(p, base._run(p, how))


@pytest.mark.parametrize("bits,gs", [(4, 64), (8, 32)])
def test_nine_to_sixteen_rows_split(bits, gs):
    """The same over lengths that many CTAs share, and masks that are no tree."""
    news, lens = [2, 2, 1], [9000, 2, 3001]
    p = base._problem(81, BF, bits, gs, 28, 4, 128, 16, lens, news, tree=True)
    base._check(p, base._run(p, "tree"))
    p["masks"] = [2, 0, 0, 3, 0]
    got = base._run(p, "tree")
    assert not bool(got[2].any()) and bool(got[4].any())
    base._check(p, got)


@pytest.mark.parametrize("t", [BF, HF])
@pytest.mark.parametrize("page", [8, 16, 32])
@pytest.mark.parametrize("hq,hkv,hd", [(28, 4, 128), (8, 2, 64), (6, 2, 128), (5, 5, 64)])
def test_tree_of_each_page_size(t, page, hq, hkv, hd):
    """16-bit pages as boxes of 8, 16 and 32 rows; sequences that end at every place of a
    page."""
    news = [17, 40, 9, 64]
    lens = [17 + 200, 40 + 23, 9 + 96, 64 + 1]
    p = base._problem(page + hq, t, 16, 0, hq, hkv, hd, page, lens, news, tree=True)
    base._check(p, base._run(p, "tree"))


@pytest.mark.parametrize("bits", [16, 4])
def test_hundreds_of_trees(bits):
    """More sequences than threads that count their tiles."""
    news = [(7 * b) % 23 for b in range(300)]
    lens = [n + (13 * b) % 90 for b, n in enumerate(news)]
    p = base._problem(90, BF, bits, 64, 4, 1, 64, 16, lens, news, tree=True)
    base._check(p, base._run(p, "tree"))


# ---------------------------------------------------------------------------- wide tables

def _peak(call):
    """A call's result and the most memory it held beyond what was held before."""
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = call()
    torch.cuda.synchronize()
    return out, torch.cuda.max_memory_allocated() - before


@pytest.mark.parametrize("bits", [16, 8, 4])
def test_prefill_in_wide_tables(bits):
    """max_kv_len sizes a chunk's work, whatever the block table could hold: the same bits
    and the same memory in a table for 640 keys and in one for 32768."""
    news, lens = [300, 77, 512], [512, 77, 512]
    p = base._problem(14, BF, bits, 64, 28, 4, 128, 16, lens, news)
    cu, kv = base._i32(p["cu"]), base._i32(lens)
    outs = []
    for capacity in (640, 32768):
        bt = base._i32([r + [0] * (capacity // 16 - len(r)) for r in p["table"]["rows"]])
        outs.append(_peak(lambda: A.paged_attention_prefill(
            p["q"], cu, 512, p["kc"], p["vc"], bt, kv, p["scale"], max_kv_len=512)))
    assert torch.equal(outs[0][0], outs[1][0])
    assert outs[0][1] == outs[1][1]
    if bits != 16:
        base._check(p, outs[1][0])
    for bad in (-1, 32769):
        with pytest.raises(ValueError, match="max_kv_len"):
            A.paged_attention_prefill(p["q"], cu, 512, p["kc"], p["vc"], bt, kv, p["scale"],
                                      max_kv_len=bad)


def test_decoder_prefills_in_wide_tables():
    """The decoder gives the prompts' lengths on: its prefill takes no more memory with room
    for 8192 tokens a sequence than with room for 256."""
    c = qwen2.Qwen2Config(**base.CFG)
    model = qwen2.Qwen2ForCausalLM(c, seed=3)
    lengths = [5, 37, 130]
    ids = torch.randint(0, 640, (sum(lengths),), generator=torch.Generator().manual_seed(1),
                        dtype=torch.int32)
    got = []
    for max_len in (256, 256, 8192):       # (the first sets workspaces up)
        cache = A.PagedKVCache(2, 1, 128, num_pages=3 * max_len // 16, bits=8)
        dec = qwen2.GreedyDecoder(model, cache, 3, max_len=max_len)
        got.append(_peak(lambda: dec.prefill(ids, lengths)))
    assert torch.equal(got[1][0], got[2][0])
    assert abs(got[1][1] - got[2][1]) < 1 << 20


# ---------------------------------------------------------------------------- in a model

@pytest.mark.parametrize("bits", [8, 4])
def test_attention_layer_over_a_quantised_cache(bits):
    """The model's attention layer, head norms and all, prefills three prompts and takes a
    decode step over a quantised cache. Its cache rows are the rule's on the rows the 16-bit
    form writes, bit for bit; its output is o_proj of 64-bit attention over those rows.

    The output may be off by what the attention may (carried through the weights' magnitudes),
    by a weight's rounding to T (a half step of its largest term, code * scale or bias), by
    32-bit sums over the inputs, and by its own rounding."""
    cfg = qwen2.Qwen2Config(**base.CFG)
    g = base._gen(17)
    at = qwen2.Qwen2Attention(cfg, device="cuda", dtype=BF, generator=g, norm_jitter=0.1,
                              bias_std=0.5)
    hq, hkv, hd = at.n_heads, at.n_kv_heads, at.head_dim
    cache = A.PagedKVCache(1, hkv, hd, 64, bits=bits)
    plain = A.PagedKVCache(1, hkv, hd, 64)
    k, v = cache.keys[0], cache.values[0]
    kp, vp = plain.keys[0], plain.values[0]
    bt = cache.allocate([200] * 3, generator=torch.Generator().manual_seed(5))
    o = at.o_proj
    W = mxq.dequantize(o.weight, o.scales, o.biases, o.group_size, o.bits).double()
    per = 32 // o.bits
    code = (o.weight.view(torch.int32).long().unsqueeze(-1) >>
            (torch.arange(per, device="cuda") * o.bits)) & (2 ** o.bits - 1)
    code = code.flatten(-2).unflatten(-1, (-1, o.group_size)).double()
    terms = (code * o.scales.double().abs()[..., None] +
             o.biases.double().abs()[..., None]).flatten(-2)
    lens = [5, 37, 130]
    for news in (lens, [1, 1, 1]):
        if news is not lens:
            lens = [n + 1 for n in lens]
        at_pos = [range(L - n, L) for L, n in zip(lens, news)]
        cu = [0] + [sum(news[:i + 1]) for i in range(3)]
        batch = A.PagedBatch(bt, base._i32(lens), base._i32([p for r in at_pos for p in r]),
                             cache.slots(bt, at_pos), max(lens),
                             base._i32(cu) if max(news) > 1 else None, max(news))
        x = base._randn(g, cu[-1], cfg.hidden_size).to(BF)
        y = at(x, batch, k, v)
        qkv = core.quantized_matmul(x, at.qkv_proj.weight, at.qkv_proj.scales, at.qkv_proj.biases,
                                    True, cfg.group_size, cfg.bits, bias=at.qkv_proj.bias)
        q = A.rope_kv_append(qkv, batch.positions, batch.slots, kp, vp, hq, hkv, hd, at.rope_base,
                             at.q_norm, at.k_norm, at.eps)
        held = cache.slots(bt, [range(L) for L in lens]).long()
        kd, vd = A.kv_cache_read(k, v, held.int())
        for got, rows in ((kd, kp), (vd, vp)):
            w, s, b = P.quantized(rows.flatten(0, 1)[held], 64, bits)
            ref = P.values(w, s, b, 64, bits).float().to(BF).cuda()
            assert torch.equal(got, ref)
        starts = [sum(lens[:i]) for i in range(3)]
        parts = [P.attention(q[cu[i]:cu[i + 1]], [0, news[i]],
                             kd[starts[i]:starts[i] + lens[i]].double(),
                             vd[starts[i]:starts[i] + lens[i]].double(),
                             {"page": lens[i], "pages": 1, "rows": [[0]]}, [lens[i]], at.scale,
                             None, BF) for i in range(3)]
        a, tol = (torch.cat(z).flatten(1) for z in zip(*parts))
        ref = a @ W.T
        top = a.abs() + tol
        bound = tol @ W.abs().T + top @ terms.T * (P.U[BF] + (a.shape[1] + 16) * P.F)
        bound = bound + P.U[BF] * (ref.abs() + bound)
        assert bool(((y.double() - ref).abs() <= bound).all())
