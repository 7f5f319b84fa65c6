// How attention over pages shares its work out: the query rows of every (sequence, kv head)
// in chunks, each chunk's keys in tiles, and the tiles of all (sequence, chunk, kv head)
// items as one sequence of units that the CTAs take in equal contiguous runs. Or, with few
// chunks (a tree's), the tiles of all (sequence, kv head) items, of which C CTAs take the
// same run, each another chunk: they read the same keys at about the same time, so that all
// but one find them in L2. Or, with one chunk (a decode step), the tiles of all sequences, of
// which Hkv CTAs take the same run, each another head: a sector of scales holds several
// heads' (taken head after head, 32 sequences of up to 16384 4-bit keys read 295 MB for the
// 193 they hold). And how the parts of an item that several CTAs computed are joined.
#pragma once

#include "common.cuh"
#include "paged_ops.h"

namespace mlxq {
namespace ra {

// An item whose tiles several CTAs took, recorded by the CTA that took the first of them:
// its partial results are in that CTA's slot `slot`, then in slot 0 of every step-th CTA up
// to `last`, in order of keys.
struct Cut {
    int rows;   // rows of the chunk (0: this CTA began no such item)
    int slot, last, step;
    int row0, rr0, g;  // the sequence's first row of q, the chunk's first row, the kv head
};

struct Params {
    RowsArgs a;
    KvCache c;
    float scale_log2;
    float* part_o;    // [2 P][ROWS][HD] unnormalised outputs
    float2* part_ml;  // [2 P][ROWS] maximum (base 2) and sum
    Cut* cut;         // [P]
    int parts;        // P: CTAs, of which each run of `group` takes the same units
    int group;        // C: 1, the most chunks of a sequence, or its heads: each CTA takes one
};

// One sequence's place in the batch, with everything a bad length or offset could do bounded.
struct Seq {
    int row0, n, L, chunks, tiles;
};
template <int KT>
__device__ __forceinline__ Seq seq_of(const RowsArgs& a, int b, int G, int rows) {
    Seq s;
    int lo = b, hi = b + 1;
    if (a.cu_q) {
        lo = a.cu_q[b];
        hi = a.cu_q[b + 1];
    }
    s.row0 = max(0, min(lo, a.total));
    s.n = max(0, min(min(hi, a.total) - s.row0, a.max_q));
    s.L = max(0, min(a.kv_lens[b], a.max_kv));
    s.chunks = (s.n * G + rows - 1) / rows;
    s.tiles = max(1, (s.L + KT - 1) / KT);  // a sequence without keys still writes its zeros
    return s;
}

// Prefix sums of the batch's units, thread i < SCAN over a run of sequences. Every thread of
// the CTA calls it. (The host refuses a call of 2^31 units or more.)
constexpr int SCAN = 128;
struct Units {
    int total;
    int per;  // sequences per scanning thread
};
template <int KT, bool HEADS>
__device__ __forceinline__ Units scan_units(const RowsArgs& a, int Hkv, int G, int rows, int group,
                                            int* pref /* shared [SCAN + 1] */) {
    __shared__ int wsum[SCAN / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Units u;
    u.per = (a.batch + SCAN - 1) / SCAN;
    int inc = 0;
    if (tid < SCAN) {
        for (int b = tid * u.per; b < min(a.batch, (tid + 1) * u.per); ++b) {
            const Seq s = seq_of<KT>(a, b, G, rows);
            inc += HEADS ? min(s.chunks, 1) * s.tiles
                         : (group > 1 ? min(s.chunks, 1) : s.chunks) * s.tiles * Hkv;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += v;
        }
        if (lane == 31) wsum[warp] = inc;
    }
    __syncthreads();
    if (tid < SCAN) {
        for (int w = 0; w < warp; ++w) inc += wsum[w];
        pref[tid + 1] = inc;
        if (tid == 0) pref[0] = 0;
    }
    __syncthreads();
    u.total = pref[SCAN];
    return u;
}

// A CTA's run of units as segments, each a range of tiles of one item. The first `extra`
// CTAs take share + 1 units, the others share.
// STEPS: items of a sequence follow one another without a division or a load, from more
// words of state: for the specialised warps of the tcgen05 kernel, each with a walk of its
// own in shared memory that its lane 0 moves (see Steps). Otherwise every item is worked out
// anew, from state that the compiler keeps off the main loop's registers (those words would
// be its spills: 32 sequences' decode step 91 -> 105 us).
// HEADS: one chunk to a sequence, and the CTAs of a run take its heads.
template <int KT, bool STEPS, bool HEADS>
struct Walk {
    int u, u_lo, u_hi, start;
    int b, G, Hkv, rows, share, extra, C, ch;
    bool known;  // s is sequence b, whose units end at `end`
    int end, pair, in;
    // the segment
    Seq s;
    int g, rr0, t0, t1;

    __device__ __forceinline__ void begin(const RowsArgs& a, int Hkv_, int rows_, const Units& un,
                                          int parts, int group, const int* pref) {
        Hkv = Hkv_;
        rows = rows_;
        G = a.Hq / Hkv;
        C = group;
        const int P = max(1, min(parts / C, un.total)), i = blockIdx.x / C;  // no share is empty
        ch = blockIdx.x - i * C;
        share = un.total / P;
        extra = un.total - share * P;
        u = u_lo = u_hi = start = b = 0;
        if (STEPS) known = false;
        if (i >= P || un.total == 0) return;
        u = u_lo = i * share + min(i, extra);
        u_hi = u + share + (i < extra ? 1 : 0);
        int lo = 0, hi = SCAN - 1;  // the last run of sequences that begins at or before u
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (pref[mid] <= u) lo = mid;
            else hi = mid - 1;
        }
        start = pref[lo];
        b = lo * un.per;
    }
    // Steps to the segment at u; false at the end of the run.
    __device__ __forceinline__ bool next(const RowsArgs& a) {
        while (u < u_hi) {
            if (!STEPS || !known) {
                s = seq_of<KT>(a, b, G, rows);
                const int n = HEADS ? min(s.chunks, 1) * s.tiles
                                    : (C > 1 ? min(s.chunks, 1) : s.chunks) * s.tiles * Hkv;
                if (u >= start + n) {
                    start += n;
                    ++b;
                    continue;
                }
                if (!HEADS && C > 1 && ch >= s.chunks) {  // no rows of this sequence for this CTA
                    u = min(u_hi, start + n);
                    continue;
                }
                if (STEPS) {
                    known = true;
                    end = start + n;
                }
                const int item = HEADS ? 0 : (u - start) / s.tiles;
                t0 = (u - start) - item * s.tiles;
                pair = C > 1 ? 0 : item / (2 * Hkv);
                in = item - pair * 2 * Hkv;
            } else if (u >= end) {
                start = end;
                ++b;
                known = false;
                continue;
            } else {
                t0 = 0;  // (a segment that ends before its item is the run's last)
                ++in;
                if (C == 1 && in == 2 * Hkv) {
                    in = 0;
                    ++pair;
                }
            }
            t1 = min(s.tiles, t0 + (u_hi - u));
            if (HEADS) {
                g = ch;
                rr0 = 0;
                return true;
            }
            int chunk = ch;
            g = in;
            if (C == 1) {
                // The chunks in pairs from both ends: a causal mask leaves the first ones
                // fewer keys than the last, and a run of items then has its share of both
                const bool lone = 2 * pair + 1 == s.chunks;
                g = lone ? in : in >> 1;
                chunk = !lone && (in & 1) ? s.chunks - 1 - pair : pair;
            }
            rr0 = chunk * rows;
            return true;
        }
        return false;
    }
    __device__ __forceinline__ void advance() { u += t1 - t0; }
    __device__ __forceinline__ bool whole() const { return t0 == 0 && t1 == s.tiles; }
    __device__ __forceinline__ int slot() const { return 2 * blockIdx.x + (u == u_lo ? 0 : 1); }
    // keys the chunk can see (with a causal mask, those up to its last row), of them the
    // ones every row sees, and the position of new token 0
    __device__ __forceinline__ int base() const { return s.L - s.n; }
    __device__ __forceinline__ int kend(const RowsArgs& a) const {
        const int last = min(s.n * G, rr0 + rows) - 1;
        return max(0, a.mask ? s.L : min(s.L, base() + last / G + 1));
    }
    // tiles of the segment that hold such keys
    __device__ __forceinline__ int tile_end(const RowsArgs& a) const {
        return min(t1, (kend(a) + KT - 1) / KT);
    }
    // The CTA (run of CTAs) that owns unit x.
    __device__ __forceinline__ int owner(int x) const {
        const int big = extra * (share + 1);
        return x < big ? x / (share + 1) : extra + (x - big) / share;
    }
    __device__ __forceinline__ Cut cut() const {
        Cut c;
        c.rows = min(s.n * G - rr0, rows);
        c.slot = slot();
        c.last = owner(u - t0 + s.tiles - 1) * C + ch;
        c.step = C;
        c.row0 = s.row0;
        c.rr0 = rr0;
        c.g = g;
        return c;
    }
};

// A warp's way of moving its Walk: every lane calls, lane 0 moves.
template <int KT>
struct Steps {
    Walk<KT, true, false>& w;
    const RowsArgs& a;
    __device__ __forceinline__ void begin(int Hkv, int rows, const Units& un, int parts, int group,
                                          const int* pref) {
        if ((threadIdx.x & 31) == 0) w.begin(a, Hkv, rows, un, parts, group, pref);
        __syncwarp();
    }
    __device__ __forceinline__ bool next() {
        int r = 0;
        __syncwarp();
        if ((threadIdx.x & 31) == 0) r = w.next(a);
        __syncwarp();
        return __shfl_sync(0xffffffffu, r, 0) != 0;
    }
    __device__ __forceinline__ void advance() {
        __syncwarp();
        if ((threadIdx.x & 31) == 0) w.advance();
        __syncwarp();
    }
};

// Rows behind the last sequence are zero.
__device__ __forceinline__ void zero_tail(const RowsArgs& a, int HD, int threads) {
    if (!a.cu_q || !a.tail) return;
    const long long row = static_cast<long long>(a.Hq) * HD / 8;
    const int end = max(0, min(a.cu_q[a.batch], a.total));
    uint4* o = static_cast<uint4*>(a.out);
    for (long long i = end * row + blockIdx.x * threads + threadIdx.x; i < a.total * row;
         i += static_cast<long long>(gridDim.x) * threads)
        o[i] = make_uint4(0u, 0u, 0u, 0u);
}

}  // namespace ra
}  // namespace mlxq
