"""Argument checks of the paged-cache operators on the CPU: nothing here reaches a device."""
import ctypes

import pytest
import torch

from mlx_server_runtime_b200 import _lib, attention as A

FAKE = 0x1000  # aligned, never dereferenced: validation fails first


def cache(**kw):
    d = dict(k=FAKE, v=FAKE, k_scales=FAKE, k_biases=FAKE, v_scales=FAKE, v_biases=FAKE,
             num_pages=8, page_size=16, n_kv_heads=4, head_dim=128, bits=4, group_size=64,
             dtype=_lib.BF16)
    d.update(kw)
    return _lib.KVCache(**d)


BAD_CACHES = [(dict(dtype=_lib.F32), _lib.ERR_DTYPE), (dict(head_dim=96), _lib.ERR_SHAPE),
              (dict(page_size=64), _lib.ERR_SHAPE), (dict(bits=2), _lib.ERR_BITS),
              (dict(n_kv_heads=0), _lib.ERR_SHAPE), (dict(n_kv_heads=3), _lib.ERR_SHAPE),
              (dict(n_kv_heads=2), _lib.ERR_SHAPE), (dict(num_pages=0), _lib.ERR_SHAPE),
              (dict(num_pages=1 << 28), _lib.ERR_SHAPE), (dict(k=None), _lib.ERR_NULL),
              (dict(v=FAKE + 8), _lib.ERR_ALIGN), (dict(group_size=48), _lib.ERR_GROUP),
              (dict(head_dim=64, group_size=128), _lib.ERR_GROUP),
              (dict(v_biases=None), _lib.ERR_NULL), (dict(k_scales=FAKE + 2), _lib.ERR_ALIGN)]


def append(c, ld=36 * 128, tokens=1, heads=28, base=1e4, eps=1e-6, qkv=FAKE, qn=FAKE):
    return _lib.load().mlxq_norm_rope_kv_append(c, qkv, ld, FAKE, qn, FAKE, eps, FAKE, FAKE,
                                                tokens, heads, base, None)


def rows(c, cu=FAKE, total=5, max_q=4, blocks=4, max_kv=64, mask=FAKE, batch=2, heads=28, q=FAKE,
         ws=None, nbytes=0, scale=0.1, out=FAKE):
    return _lib.load().mlxq_paged_attention_rows(c, q, cu, total, max_q, FAKE, blocks, FAKE,
                                                 max_kv, mask, out, batch, heads, scale, ws,
                                                 nbytes, None)


@pytest.mark.parametrize("kw,code", BAD_CACHES)
def test_cache_is_checked(kw, code):
    c = cache(**kw)
    assert append(c) == code and _lib.last_error()
    assert rows(c) == code
    if "n_kv_heads" not in kw or kw["n_kv_heads"] == 0:
        assert _lib.load().mlxq_kv_cache_read(c, FAKE, 3, FAKE, FAKE, None) == code


def test_append_is_checked():
    c = cache()
    assert append(c, ld=36 * 128 - 8) == _lib.ERR_SHAPE
    assert append(c, ld=36 * 128 + 4) == _lib.ERR_SHAPE
    assert append(c, tokens=-1) == _lib.ERR_SHAPE
    assert append(c, heads=27) == _lib.ERR_SHAPE
    assert append(c, heads=36) == _lib.ERR_SHAPE
    assert append(c, base=1.0) == _lib.ERR_SHAPE
    assert append(c, eps=-1e-6) == _lib.ERR_SHAPE
    assert append(c, eps=float("nan")) == _lib.ERR_SHAPE
    assert append(c, eps=float("inf")) == _lib.ERR_SHAPE
    assert append(c, base=float("inf")) == _lib.ERR_SHAPE
    assert append(c, qkv=None) == _lib.ERR_NULL
    assert append(c, qkv=FAKE + 8) == _lib.ERR_ALIGN
    assert append(c, qn=FAKE + 2) == _lib.ERR_ALIGN
    assert append(c, tokens=0) == _lib.OK
    assert append(None) == _lib.ERR_NULL


def test_read_is_checked():
    L = _lib.load()
    assert L.mlxq_kv_cache_read(cache(), FAKE, -1, FAKE, FAKE, None) == _lib.ERR_SHAPE
    assert L.mlxq_kv_cache_read(cache(), None, 1, FAKE, FAKE, None) == _lib.ERR_NULL
    assert L.mlxq_kv_cache_read(cache(), FAKE, 1, FAKE + 4, FAKE, None) == _lib.ERR_ALIGN
    assert L.mlxq_kv_cache_read(cache(), FAKE, 0, FAKE, FAKE, None) == _lib.OK


def test_rows_are_checked():
    c = cache()
    assert rows(c, max_kv=65) == _lib.ERR_SHAPE          # 4 pages of 16
    assert rows(c, max_q=65) == _lib.ERR_SHAPE           # a tree of 65
    assert rows(c, cu=None, total=3) == _lib.ERR_SHAPE   # rows and sequences differ
    assert rows(c, cu=None, total=2, max_q=4) == _lib.ERR_SHAPE
    assert rows(c, batch=70000) == _lib.ERR_SHAPE
    assert rows(c, blocks=0) == _lib.ERR_SHAPE
    assert rows(c, q=None) == _lib.ERR_NULL
    assert rows(c, q=FAKE + 8) == _lib.ERR_ALIGN
    assert rows(c) == _lib.ERR_WORKSPACE
    need = _lib.load().mlxq_paged_attention_rows_workspace_size(c, 2, 4, 64, 28)
    assert need > 0
    assert rows(c, ws=0x10000, nbytes=need - 1) == _lib.ERR_WORKSPACE
    assert rows(c, ws=0x10010, nbytes=need) == _lib.ERR_ALIGN
    assert rows(c, total=0) == _lib.OK
    for bad in ("nan", "inf", "-inf"):
        assert rows(c, scale=float(bad)) == _lib.ERR_SHAPE
    assert rows(c, out=None) == _lib.ERR_NULL and rows(c, batch=0, out=None) == _lib.ERR_NULL
    # more units of work than 31 bits count
    assert rows(c, total=1 << 24, max_q=1 << 24, mask=None, batch=65535, blocks=1 << 20,
                max_kv=1 << 24) == _lib.ERR_SHAPE


def test_struct_layout():
    assert ctypes.sizeof(_lib.KVCache) == 6 * 8 + 8 + 6 * 4


def test_quantized_kv_is_checked():
    c = A.QuantizedKV.zeros(3, 16, 2, 64, 32, 4, device="cpu")
    assert c.shape == (3, 16, 2, 64) and c.dtype == torch.bfloat16
    assert c.codes.shape == (3, 16, 2, 8) and c.scales.shape == (3, 16, 2, 2)
    ok = dict(codes=c.codes, scales=c.scales, biases=c.biases, group_size=32, bits=4)
    for bad in (dict(bits=2), dict(group_size=16), dict(group_size=64), dict(bits=8),
                dict(scales=c.scales.float()), dict(biases=c.biases.half()),
                dict(scales=c.scales[:2]), dict(codes=c.codes[0]),
                dict(codes=c.codes.view(torch.int32).float()),
                dict(scales=c.scales.transpose(0, 1).contiguous().transpose(0, 1))):
        with pytest.raises(ValueError):
            A.QuantizedKV(**{**ok, **bad})
    with pytest.raises(ValueError):
        A.QuantizedKV.zeros(3, 16, 2, 64, 48, 4, device="cpu")
    with pytest.raises(ValueError):
        A.PagedKVCache(1, 2, 64, 4, bits=2, device="cpu")


def test_functions_refuse():
    q8 = A.QuantizedKV.zeros(4, 16, 2, 64, 32, 8, device="cpu")
    q4 = A.QuantizedKV.zeros(4, 16, 2, 64, 32, 4, device="cpu")
    x16 = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    bt, lens = torch.zeros(3, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    m = torch.zeros(3, dtype=torch.int64)
    cu = torch.zeros(4, dtype=torch.int32)
    slots = torch.zeros(3, dtype=torch.int32)
    qkv = torch.zeros(3, 8 * 64, dtype=torch.bfloat16)
    w = torch.ones(64, dtype=torch.bfloat16)

    def tree(**kw):
        d = dict(q=q, cu_q=cu, max_q_len=4, k_cache=q4, v_cache=q4, block_table=bt, kv_lens=lens,
                 max_kv_len=32, tree_mask=m, scale=0.1)
        return A.paged_attention_tree(**{**d, **kw})

    bad = [dict(v_cache=q8), dict(v_cache=x16), dict(k_cache=x16), dict(q=q.float()),
           dict(q=q[:, :, :32]), dict(q=q[0]), dict(cu_q=cu[:3]), dict(cu_q=cu.long()),
           dict(block_table=bt[0]), dict(block_table=bt.long()), dict(kv_lens=lens[:2]),
           dict(tree_mask=None), dict(tree_mask=m.int()), dict(tree_mask=m[:2]),
           dict(k_cache=x16, v_cache=x16[:2]),
           dict(k_cache=x16.transpose(0, 1), v_cache=x16.transpose(0, 1)),
           dict()]   # (the last: tensors that are not on a CUDA device)
    for kw in bad:
        with pytest.raises(ValueError):
            tree(**kw)
    with pytest.raises(ValueError):
        A.paged_attention_decode(q[:2], q4, q4, bt, lens, 32, 0.1)
    with pytest.raises(ValueError):
        A.paged_attention_prefill(q, cu, 4, q4, x16, bt, lens, 0.1)
    for kw in (dict(v=q8), dict(qkv=qkv.half()), dict(hkv=4), dict(hd=32), dict(hq=5),
               dict(q_norm=w[:32]), dict(k_norm=w.float()), dict(slots=slots[:2]),
               dict(slots=slots.long()), dict(positions=slots[:1]), dict(qkv=qkv.t()), dict()):
        d = {**dict(qkv=qkv, positions=slots, slots=slots, k=q4, v=q4, hq=4, hkv=2, hd=64,
                    q_norm=w, k_norm=w), **kw}
        with pytest.raises(ValueError):
            A.rope_kv_append(d["qkv"], d["positions"], d["slots"], d["k"], d["v"], d["hq"],
                             d["hkv"], d["hd"], 1e4, q_norm=d["q_norm"], k_norm=d["k_norm"])
    for args in ((q4, q8, slots), (q4, q4, slots.long()), (q4, q4, bt), (q4, q4, slots)):
        with pytest.raises(ValueError):
            A.kv_cache_read(*args)


def test_tree_masks():
    m = A.tree_masks([[-1, 0, 0, 1], [], [-1, -1]], device="cpu")
    assert m.dtype == torch.int64 and m.tolist() == [1, 3, 5, 11, 1, 2]
    chain = A.tree_masks([list(range(-1, 63))], device="cpu").tolist()
    assert chain[0] == 1 and chain[62] == 2 ** 63 - 1 and chain[63] == -1
    for bad in ([[0]], [[-1, 1]], [[-2]], [list(range(-1, 64))]):
        with pytest.raises(ValueError):
            A.tree_masks(bad, device="cpu")
