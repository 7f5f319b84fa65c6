// Launchers of the operators over a paged KV cache held in 16, 8 or 4 bits: the append
// with per-head norms and rotation, the read-back, and attention for several query rows
// per sequence (decode steps, prompt chunks, trees of drafted tokens).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "launch.h"

namespace mlxq {

// Keys and values of one layer. bits 16: rows of T, no scales. bits 8 / 4: packed codes
// [rows, Hkv, hd * bits / 32] with scales and biases [rows, Hkv, hd / gs] of T.
struct KvCache {
    void* k;
    void* v;
    void* ks;
    void* kb;
    void* vs;
    void* vb;
    int pages, page, Hkv, hd, bits, gs, dtype;
};

cudaError_t launch_norm_rope_append(const KvCache& c, const void* qkv, long long ld, void* q_out,
                                    const void* q_norm, const void* k_norm, float eps,
                                    const int32_t* positions, const int32_t* slots, int tokens,
                                    int Hq, double base, bool overlap, cudaStream_t st);
cudaError_t launch_cache_read(const KvCache& c, const int32_t* slots, int n, void* k_out,
                              void* v_out, bool overlap, cudaStream_t st);

// Attention of query rows over the pages. Sequence b owns rows [cu_q[b], cu_q[b + 1]) of q
// and out (cu_q null: row b alone); row i of n sits at position L_b - n + i and sees the
// keys before position L_b - n, and of the n new ones those up to i (mask null) or those
// whose bit is set in mask[row].
struct RowsArgs {
    const void* q;
    void* out;
    const int32_t* cu_q;
    const int32_t* kv_lens;
    const int32_t* table;
    const long long* mask;
    int max_blocks, max_kv, max_q, total, batch, Hq;
    float scale;
    bool tail;  // zero the rows behind the last sequence
};
// Bytes of workspace the launch needs (a function of sizes alone; no zero-fill needed), and
// whether its units of work can be counted in 31 bits.
bool attn_rows_countable(const KvCache& c, const RowsArgs& a);
size_t attn_rows_workspace(const KvCache& c, const RowsArgs& a);
cudaError_t launch_attn_rows(const KvCache& c, const RowsArgs& a, void* workspace, bool overlap,
                             cudaStream_t st);

// The tcgen05 form of the attention (paged_attn_tc.cu): 128 query rows and kRowsTcKeys keys
// to a tile, over 16-bit rows; a quantised cache's are expanded into `expanded` first, which
// takes rows_tc_expand_bytes for each sequence.
constexpr int kRowsTcKeys = 64, kRowsTcThreads = 224;
namespace ra {
struct Params;
}
size_t rows_tc_expand_bytes(const KvCache& c, const RowsArgs& a);
cudaError_t launch_rows_tc(ra::Params& p, void* expanded, bool overlap, cudaStream_t st);
cudaError_t rows_tc_read_error(int* code);

}  // namespace mlxq
