"""What the paged-cache operators promise and no device is needed to check."""
import os
import re

import pytest
import torch

from mlx_server_runtime_b200 import _lib, attention as A

CSRC = os.path.join(os.path.dirname(_lib.__file__), "csrc")


def source(name):
    """A source file without its comments."""
    with open(os.path.join(CSRC, name)) as f:
        s = f.read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", " ", s, flags=re.S)


@pytest.mark.parametrize("name", ["paged_attn.cu", "paged_attn_tc.cu", "paged_cache.cu",
                                  "rows_units.cuh", "kv_dequant.cuh"])
def test_no_read_only_loads(name):
    """With launch overlap these kernels start while the kernel that writes the pools, tables
    and queries they read may still run. A load through the read-only path needs data that
    does not change for as long as the kernel lives, so none is made: neither by hand, nor by
    parameters that allow the compiler to."""
    s = source(name)
    assert not re.search(r"__ldg\b|\bld\.global(\.\w+)*\.nc\b", s)
    assert not re.search(r"\bconst\b[^;,(){}]*\*\s*__restrict__", s)


@pytest.mark.parametrize("name", ["tcgen05.cuh", "kv_dequant.cuh", "rows_units.cuh",
                                  "quant_rule.cuh", "overlap.cuh"])
def test_every_helper_has_a_caller(name):
    all_of_it = "".join(source(f) for f in sorted(os.listdir(CSRC)))
    helpers = set(re.findall(r"__forceinline__[\w:&* ]*?(\w+)\(", source(name)))
    assert helpers
    assert [h for h in sorted(helpers) if len(re.findall(rf"\b{h}\b", all_of_it)) < 2] == []


def test_tensor_memory_loads_are_waited_for():
    """Registers that a tcgen05.ld fills may be used after its wait. Only what one asm statement
    holds, or what passes through a statement behind the wait, is sure to stay in that order."""
    loads = [f for f in re.split(r"(?=__device__ __forceinline__)", source("tcgen05.cuh"))
             if "tcgen05.ld." in f]
    assert loads
    for f in loads:
        statement = f.split("tcgen05.ld.")[-1].split(");")[0]
        tied = re.search(r'wait::ld.*asm volatile\("" : "\+r"', f, flags=re.S)
        assert tied or "tcgen05.wait::ld" in statement, f[:80]


def test_prefill_bounds_its_lengths():
    """max_kv_len is at most what the block table holds (two pages of 16 here)."""
    c = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    i32 = torch.zeros(4, 2, dtype=torch.int32)
    for bad in (-1, 33):
        with pytest.raises(ValueError, match="max_kv_len"):
            A.paged_attention_prefill(q, i32[:, 0], 4, c, c, i32[:3], i32[:3, 0], 0.1,
                                      max_kv_len=bad)


@pytest.mark.parametrize("batch,max_kv,hkv,hd", [(64, 32768, 4, 128), (3, 1 << 20, 8, 128),
                                                 (500, 600, 2, 64), (1, 100, 1, 64)])
def test_expansion_workspace_is_bounded(batch, max_kv, hkv, hd):
    """1 GiB of expanded rows, or one sequence's where they are more; beside them the parts of
    at most two CTAs an SM (two slots of 128 rows each) and 1 KiB a sequence to align."""
    c = _lib.KVCache(*[0x1000] * 6, 8, 16, hkv, hd, 4, 64, _lib.BF16)
    need = _lib.load().mlxq_paged_attention_rows_workspace_size(c, batch, 64, max_kv, 8 * hkv)
    one = -(-max_kv // 64) * 64 * hkv * hd * 4
    parts = 296 * 2 * 128 * (hd * 4 + 8) + 296 * 64
    assert min(one * batch, (1 << 30) - one) <= need <= max(1 << 30, one) + parts + 1024 * batch + 1024


def test_the_warp_that_issues_products_decides_as_one():
    """Its lanes poll barriers each for itself. What it does next follows from a vote, and each
    round begins with all lanes there: a lane left two phases behind would wait for good."""
    s = source("paged_attn_tc.cu")
    role = s[s.index("else if (warp == WARP_MMA)"):]
    loop = role[role.index("while (more || npv < ns)"):role.index("umma_commit_by(leader, smem_u32(&drained))")]
    assert re.match(r"[^;]*\{\s*__syncwarp\(\);", loop)
    voted = "".join(re.findall(r"__all_sync\(0xffffffffu,.*?\)\)\s*\{", loop, flags=re.S))
    assert voted.count("mbar_try_wait(") == loop.count("mbar_try_wait(") > 0
