// Attention of many query rows over a paged KV cache in 16, 8 or 4 bits on tcgen05
// (sm_100a): prompt chunks and trees of drafted tokens.
//
// One tile is 128 query rows (new tokens x the query heads of a kv head) by 128 keys:
//   S = Q K^T   one product of M = 128, N = 128, K = head size: Q and K in shared memory,
//               S in tensor memory (32-bit)
//   softmax     thread = row: S is read back, P = exp2(S * scale - m) goes back into the
//               columns of S as 16-bit pairs. m follows the running maximum only when a
//               score passes it by 2^8, so O is rescaled seldom; P then reaches 256, which
//               costs neither type precision.
//   O += P V    M = 128, N = head size, K = 128: P read from tensor memory, V from shared
//               memory as it lies (key rows, dimensions contiguous)
// Warps 0-3 hold a tensor-memory lane quarter each and do the softmax and the epilogue;
// warps 4-7 bring keys and values into shared memory, dequantised once per tile on the way
// (16-bit rows by cp.async), and a thread of warp 4 issues the products between its loads. The chain S ->
// softmax -> P V of a CTA is serial; two CTAs share an SM (96 KB of shared memory and 256
// columns each), so one's products run under the other's softmax, and a tile's loads have
// most of the chain to land in (K is free once S is done, V once P V is).
// Quantised rows are staged in the order their codes unpack to, eight dims at a time; Q is
// staged in the same order, and the epilogue puts the output's dims back.
// Work is shared out as in rows_units.cuh. Every wait is bounded: on a timeout the CTA
// records an error, its roles stop, what is in flight is waited for, tensor memory is
// freed and the kernel returns.
#include "common.cuh"
#include "kv_dequant.cuh"
#include "overlap.cuh"
#include "paged_ops.h"
#include "rows_units.cuh"
#include "tcgen05.cuh"

namespace mlxq {

__device__ int g_rows_tc_error;  // 0, or the first error code a kernel recorded

namespace rt {
constexpr int ROWS = 128, KT = kRowsTcKeys, THREADS = kRowsTcThreads;
constexpr int WARP_LOAD0 = 4;  // the loads; the first of these warps also issues the products
constexpr uint32_t kCols = 256;   // tensor memory: S (and P) from 0, O from 128
constexpr uint32_t kOCol = 128;
constexpr uint32_t kParkNs = 2000, kParkLimit = 1u << 20;  // ~2 s
constexpr uint32_t kSpinLimit = 1u << 22;
constexpr int kErrTimeout = 3;

template <int HD>
constexpr int tile_bytes() { return KT * HD * 2; }

// Position x of eight staged elements holds dim map(x) of its eight.
template <int BITS>
__host__ __device__ constexpr int staged_dim(int x) {
    return BITS == 16 ? x : pair_dim<BITS>(x / 2, x % 2);
}

// Pairs of 32-bit floats in one register pair: one instruction for two lanes of work.
__device__ __forceinline__ uint64_t pack_f2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float ex2(float x) {  // 2^x, results below 2^-126 as zero
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(r) : "f"(x));
    return r;
}
}  // namespace rt

template <typename T, int HD, int BITS>
__global__ void __launch_bounds__(rt::THREADS, 2)
    attn_rows_tc_kernel(const __grid_constant__ ra::Params p) {
    using namespace rt;
    using namespace ra;
    constexpr int TB = tile_bytes<HD>();
    constexpr int LPR = HD * BITS / 128;     // lanes (16 bytes each) of a cache row
    constexpr int RPI = 32 / LPR;            // rows a warp loads at once
    constexpr int CPU = 16 / BITS;           // staged 16-byte chunks of 16 loaded bytes
    constexpr int RW = HD * BITS / 32;       // words of a cache row
    constexpr uint32_t AB = __is_same(T, __nv_bfloat16) ? 1u : 0u;
    constexpr uint32_t IDESC_S = (1u << 4) | (AB << 7) | (AB << 10) | ((KT / 8) << 17) | ((ROWS / 16) << 24);
    constexpr uint32_t IDESC_O = (1u << 4) | (AB << 7) | (AB << 10) | (1u << 16) | ((HD / 8) << 17) |
                                 ((ROWS / 16) << 24);
    extern __shared__ uint8_t rt_smem_raw[];
    __shared__ long long pref[SCAN + 1];
    __shared__ __align__(8) uint64_t k_full, v_full, s_full, pv_done, p_full, drained;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int s_abort;
    uint8_t* smem = rt_smem_raw + ((1024u - (smem_u32(rt_smem_raw) & 1023u)) & 1023u);
    uint8_t *qs = smem, *ks = smem + ROWS * HD * 2, *vs = ks + TB;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    if (warp == WARP_LOAD0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                         smem_u32(&tmem_slot)),
                     "r"(kCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    if (tid == 0) {
        mbar_init(smem_u32(&k_full), 4);
        mbar_init(smem_u32(&v_full), 4);
        mbar_init(smem_u32(&p_full), 4);
        mbar_init(smem_u32(&s_full), 1);
        mbar_init(smem_u32(&pv_done), 1);
        mbar_init(smem_u32(&drained), 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    pdl_wait();
    const RowsArgs& a = p.a;
    const KvCache& c = p.c;
    const int Hkv = c.Hkv, G = a.Hq / Hkv;
    zero_tail(a, HD, THREADS);
    const Units un = scan_units<KT>(a, Hkv, G, ROWS, pref);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    Walk<KT, ROWS> w;
    w.begin(a, Hkv, un, p.parts, pref);

    auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (s_abort) return false;
        if (mbar_wait_park(smem_u32(bar), parity, kParkLimit, kParkNs)) return true;
        atomicCAS(&g_rows_tc_error, 0, kErrTimeout);
        s_abort = 1;
        return false;
    };
    // tiles of the segment that hold keys its rows can see
    auto tile_end = [&]() { return min(w.t1, (w.kend(a) + KT - 1) / KT); };

    if (warp >= WARP_LOAD0) {
        // ------------------------------ loads and products ---------------------------
        const int lw = warp - WARP_LOAD0;   // this warp's 32 rows of every tile
        const bool issuer = lw == 0 && lane == 0;
        const int c0 = lane % LPR, r0 = lane / LPR;
        const int grp = BITS == 16 ? 0 : c0 * (128 / BITS) / c.gs;
        const int ng = BITS == 16 ? 1 : HD / c.gs;
        // 16-byte chunk ch of row r: eight chunks to a 128-byte row of its half, swizzled
        auto at = [](int r, int ch) -> uint32_t {
            return static_cast<uint32_t>((ch / 8) * (KT * 128) + r * 128 + (((ch % 8) ^ (r & 7)) << 4));
        };
        const bool neg = p.scale_log2 < 0.f;  // the sign of the scale goes into the queries
        const uint64_t qd = sw128_kmajor_desc(smem_u32(qs)), kd = sw128_kmajor_desc(smem_u32(ks));
        const uint64_t vd = sw128_mnmajor_desc(smem_u32(vs), KT * 128);
        uint32_t it = 0;     // tiles so far
        bool ok = true, acc = false;  // acc: the tile before was not its item's first here
        auto spin = [&](uint64_t* bar, uint32_t parity) -> bool {
            // (the issuing thread polls without parking: it wakes fastest)
            if (!s_abort && mbar_wait_bounded(smem_u32(bar), parity, kSpinLimit)) return true;
            atomicCAS(&g_rows_tc_error, 0, kErrTimeout);
            s_abort = 1;
            return false;
        };
        auto issue_s = [&](uint32_t i) {
            if (!spin(&k_full, i & 1)) return;
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < HD / 16; ++j) {  // 16 dims: 32 bytes of a half
                const uint64_t off = static_cast<uint64_t>((j / 4) * (KT * 128 / 16) + (j % 4) * 2);
                umma_f16_ss(tmem, qd + off, kd + off, IDESC_S, j > 0 ? 1u : 0u);
            }
            umma_commit(smem_u32(&s_full));
        };
        auto issue_pv = [&](uint32_t i, bool accumulate) {
            if (!spin(&v_full, i & 1) || !spin(&p_full, i & 1)) return;
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < KT / 16; ++j)  // 16 keys: 8 columns of P, 2 KB of V
                umma_f16_ts(tmem + kOCol, tmem + 8 * j, vd + j * (2048 / 16), IDESC_O,
                            (accumulate || j > 0) ? 1u : 0u);
            umma_commit(smem_u32(&pv_done));
        };
        auto arrive = [&](uint64_t* bar) {  // this warp's rows are in shared memory
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(bar));
        };
        for (; ok && w.next(a); w.advance()) {
            const Seq& s = w.s;
            const int kend = w.kend(a), te = tile_end(), R = s.n * G;
            const int32_t* bt = a.table + static_cast<size_t>(w.b) * a.max_blocks;
            for (int tile = w.t0; tile < te; ++tile, ++it) {
                // lane = key of this warp's rows: its cache row, or -1
                long long mine = -1;
                const int key = tile * KT + lw * 32 + lane;
                if (key < kend) {
                    const int pid = bt[key / c.page];
                    if (pid >= 0 && pid < c.pages)
                        mine = (static_cast<long long>(pid) * c.page + key % c.page) * Hkv + w.g;
                }
                // Quantised rows of the tile, all loads in flight together
                constexpr int NL = BITS == 16 ? 1 : LPR;
                uint4 kr[NL], vr[NL];
                uint16_t ksr[NL], kbr[NL], vsr[NL], vbr[NL];
                uint32_t there = 0;
                if constexpr (BITS != 16) {
#pragma unroll
                    for (int i = 0; i < LPR; ++i) {
                        const long long own = __shfl_sync(0xffffffffu, mine, i * RPI + r0);
                        const long long row = own < 0 ? 0 : own;
                        there |= own < 0 ? 0u : 1u << i;
                        kr[i] = __ldg(reinterpret_cast<const uint4*>(
                            static_cast<const uint32_t*>(c.k) + row * RW + c0 * 4));
                        vr[i] = __ldg(reinterpret_cast<const uint4*>(
                            static_cast<const uint32_t*>(c.v) + row * RW + c0 * 4));
                        const long long g = row * ng + grp;
                        ksr[i] = static_cast<const uint16_t*>(c.ks)[g];
                        kbr[i] = static_cast<const uint16_t*>(c.kb)[g];
                        vsr[i] = static_cast<const uint16_t*>(c.vs)[g];
                        vbr[i] = static_cast<const uint16_t*>(c.vb)[g];
                    }
                }
                // Stages the loaded rows of a tile: 16 bytes of codes become CPU chunks. Lanes
                // of the upper half take theirs in another order, so that the eight lanes of
                // a store phase meet eight different bank groups. A key that is not there is
                // zeros (its stale values must not meet a probability of zero).
                auto stage = [&](uint8_t* dst, const uint4* raw, const uint16_t* sr, const uint16_t* br) {
#pragma unroll
                    for (int i = 0; i < NL; ++i) {
                        const int r = lw * 32 + i * RPI + r0;
                        const bool in = there >> i & 1;
                        const uint32_t s2 = in ? pk_splat(sr[i]) : 0u, b2 = in ? pk_splat(br[i]) : 0u;
                        const bool up = HD == 128 && c0 >= LPR / 2;
                        uint32_t wd[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                        constexpr int flip = CPU / 2;  // chunks exchanged: q ^ flip
#pragma unroll
                        for (int q = 0; q < CPU; ++q) {
                            uint32_t cw[BITS / 4];
#pragma unroll
                            for (int e = 0; e < BITS / 4; ++e) {
                                const uint32_t x = wd[q * (BITS / 4) + e];
                                const uint32_t y = wd[(q ^ flip) * (BITS / 4) + e];
                                cw[e] = up ? y : x;
                            }
                            const int ch = c0 * CPU + (up ? q ^ flip : q);
                            *reinterpret_cast<uint4*>(dst + at(r, ch)) =
                                make_uint4(row_pair<T, BITS>(cw, 0, s2, b2), row_pair<T, BITS>(cw, 1, s2, b2),
                                           row_pair<T, BITS>(cw, 2, s2, b2), row_pair<T, BITS>(cw, 3, s2, b2));
                        }
                    }
                };
                auto copy = [&](uint8_t* dst, const void* pool) {  // 16-bit rows
#pragma unroll
                    for (int i = 0; i < LPR; ++i) {
                        const long long row = __shfl_sync(0xffffffffu, mine, i * RPI + r0);
                        cp_async16(dst + at(lw * 32 + i * RPI + r0, c0),
                                   static_cast<const uint32_t*>(pool) + (row < 0 ? 0 : row) * RW + c0 * 4,
                                   row < 0 ? 0 : 16);
                    }
                    cp_async_commit();
                };
                // K and Q: free once the product before has read them
                if (it > 0 && !wait(&s_full, (it - 1) & 1)) {
                    ok = false;
                    break;
                }
                if (tile == w.t0) {
                    constexpr int QL = HD / 8, QB = 8;  // lanes of a query row; loads at once
#pragma unroll 1
                    for (int i0 = 0; i0 < QL; i0 += QB) {
                        uint4 v[QB];
#pragma unroll
                        for (int i = 0; i < QB; ++i) {
                            const int rr = w.rr0 + lw * 32 + (i0 + i) * (32 / QL) + lane / QL;
                            v[i] = make_uint4(0u, 0u, 0u, 0u);
                            if (rr < R)
                                v[i] = *reinterpret_cast<const uint4*>(
                                    static_cast<const T*>(a.q) +
                                    (static_cast<size_t>(s.row0 + rr / G) * a.Hq + w.g * G + rr % G) * HD +
                                    (lane % QL) * 8);
                        }
#pragma unroll
                        for (int i = 0; i < QB; ++i) {
                            const uint32_t flip = neg ? 0x80008000u : 0u;
                            const uint32_t wd[4] = {v[i].x ^ flip, v[i].y ^ flip, v[i].z ^ flip, v[i].w ^ flip};
                            uint32_t o[4];
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                const int da = staged_dim<BITS>(2 * x), db = staged_dim<BITS>(2 * x + 1);
                                o[x] = prmt(wd[da / 2], wd[db / 2],
                                            (da % 2 ? 0x32u : 0x10u) | (db % 2 ? 0x7600u : 0x5400u));
                            }
                            *reinterpret_cast<uint4*>(
                                qs + at(lw * 32 + (i0 + i) * (32 / QL) + lane / QL, lane % QL)) =
                                make_uint4(o[0], o[1], o[2], o[3]);
                        }
                    }
                }
                // K of this tile goes in while the rows' softmax of the one before runs, then
                // that one's P V and this one's S are issued, then V of this tile goes in
                if constexpr (BITS == 16) {
                    copy(ks, c.k);
                    if (it > 0) {
                        cp_async_wait<1>();
                        arrive(&v_full);
                        if (issuer) issue_pv(it - 1, acc);
                        __syncwarp();
                    }
                    cp_async_wait<0>();
                    arrive(&k_full);
                } else {
                    stage(ks, kr, ksr, kbr);
                    arrive(&k_full);
                    if (issuer && it > 0) issue_pv(it - 1, acc);
                    __syncwarp();
                }
                if (issuer) issue_s(it);
                __syncwarp();
                acc = tile > w.t0;
                if (it > 0 && !wait(&pv_done, (it - 1) & 1)) {
                    ok = false;
                    break;
                }
                if constexpr (BITS == 16) {
                    copy(vs, c.v);
                } else {
                    stage(vs, vr, vsr, vbr);
                    arrive(&v_full);
                }
            }
        }
        if constexpr (BITS == 16) {
            cp_async_wait<0>();
            if (ok && it > 0) arrive(&v_full);
        }
        if (issuer) {
            if (ok && it > 0) issue_pv(it - 1, acc);
            // every product issued has finished before tensor memory is freed
            umma_commit(smem_u32(&drained));
            mbar_wait_bounded(smem_u32(&drained), 0, kSpinLimit);
        }
    } else {
        // ------------------------------ softmax, epilogue -----------------------------
        const int row = tid;  // of the tile; tensor-memory lane
        const uint32_t t_s = tmem + (static_cast<uint32_t>(warp * 32) << 16), t_o = t_s + kOCol;
        const float scale = fabsf(p.scale_log2);
        uint32_t it = 0;
        Cut mine = {};
        bool ok = true;
        for (; ok && w.next(a); w.advance()) {
            const Seq& s = w.s;
            const int kend = w.kend(a), te = tile_end(), base = w.base(), R = s.n * G;
            const int rr = w.rr0 + row;
            const bool active = rr < R, some = w.rr0 + warp * 32 < R;  // this row; any of the warp's
            const int full = min(max(base, 0), kend);  // keys every row sees
            const int32_t* bt = a.table + static_cast<size_t>(w.b) * a.max_blocks;
            unsigned long long vis = 0;  // of the new tokens, those this row sees
            const int tok = active ? rr / G : -1;
            if (a.mask && active) vis = static_cast<unsigned long long>(a.mask[s.row0 + tok]);
            float m = -INFINITY, l = 0.f;
            for (int tile = w.t0; tile < te; ++tile, ++it) {
                const int k0 = tile * KT;
                // which of the tile's keys are there: pages of a warp's lanes, eight keys each
                bool clean = k0 + KT <= full;
                uint32_t pages_ok = 0xffffu;
                {
                    bool good = true;
                    if (lane < KT / 8) {
                        const int key = k0 + 8 * lane;
                        if (key < kend) {
                            const int pid = bt[key / c.page];
                            good = pid >= 0 && pid < c.pages;
                        }
                    }
                    pages_ok = __ballot_sync(0xffffffffu, good) & 0xffffu;
                    clean = clean && pages_ok == 0xffffu;
                }
                if (!wait(&s_full, it & 1)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (some) {
                    // the keys of the tile's q-th 32 that this row sees, a bit each
                    auto seen32 = [&](int q) -> uint32_t {
                        const int kk = k0 + 32 * q, left = kend - kk, j0 = kk - base;
                        uint32_t bits = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;
                        bits &= ((pages_ok >> (4 * q) & 15u) * 0x00204081u & 0x01010101u) * 255u;
                        if (j0 <= -32) return bits;
                        if (a.mask)
                            return bits & (j0 >= 64  ? 0u
                                           : j0 >= 0 ? static_cast<uint32_t>(vis >> j0)
                                                     : static_cast<uint32_t>(vis << -j0) | ((1u << -j0) - 1u));
                        const int n = tok - j0 + 1;
                        return bits & (n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u);
                    };
                    float mx = -INFINITY;
#pragma unroll 1
                    for (int q = 0; q < KT / 32; ++q) {
                        uint32_t v[32];
                        tmem_ld32(t_s + q * 32, v);
                        if (!clean) {
                            const uint32_t bits = seen32(q);
#pragma unroll
                            for (int x = 0; x < 32; ++x)
                                v[x] = bits >> x & 1 ? v[x] : 0xff800000u;
                        }
                        float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int x = 0; x < 32; x += 2)
                            m4[x / 2 & 3] = fmaxf(m4[x / 2 & 3],
                                                  fmaxf(__uint_as_float(v[x]), __uint_as_float(v[x + 1])));
                        mx = fmaxf(mx, fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])));
                    }
                    mx = mx == -INFINITY ? mx : mx * scale;  // (a scale of zero keeps -inf)
                    if (__any_sync(0xffffffffu, mx - m > 8.f)) {
                        const float mn = fmaxf(m, mx);
                        const float f = mn == -INFINITY ? 1.f : exp2f(m - mn);
                        m = mn;
                        l *= f;
                        if (tile > w.t0) {
#pragma unroll 1
                            for (int q = 0; q < HD / 32; ++q) {
                                uint32_t v[32];
                                tmem_ld32(t_o + q * 32, v);
#pragma unroll
                                for (int x = 0; x < 32; ++x) v[x] = __float_as_uint(__uint_as_float(v[x]) * f);
                                tmem_st32(t_o + q * 32, v);
                            }
                        }
                    }
                    const float mr = m == -INFINITY ? 0.f : m;
                    const uint64_t scale2 = pack_f2(scale, scale), mr2 = pack_f2(-mr, -mr);
                    uint64_t l2 = pack_f2(l, 0.f);
#pragma unroll 1
                    for (int q = 0; q < KT / 32; ++q) {
                        uint32_t v[32], o[16];
                        tmem_ld32(t_s + q * 32, v);
#pragma unroll
                        for (int x = 0; x < 32; x += 2) {
                            float e0, e1;
                            unpack_f2(fma_f2(pack_f2(__uint_as_float(v[x]), __uint_as_float(v[x + 1])),
                                             scale2, mr2), e0, e1);
                            v[x] = __float_as_uint(ex2(e0));
                            v[x + 1] = __float_as_uint(ex2(e1));
                        }
                        if (!clean) {
                            const uint32_t bits = seen32(q);
#pragma unroll
                            for (int x = 0; x < 32; ++x) v[x] = bits >> x & 1 ? v[x] : 0u;
                        }
#pragma unroll
                        for (int x = 0; x < 32; x += 2) {
                            const float e0 = __uint_as_float(v[x]), e1 = __uint_as_float(v[x + 1]);
                            l2 = add_f2(l2, pack_f2(e0, e1));
                            o[x / 2] = pk_round<T>(e0, e1);
                        }
                        // (columns 16 q .. 16 q + 15 of S were read in this or an earlier step)
                        tmem_st16(t_s + q * 16, o);
                    }
                    float la, lb;
                    unpack_f2(l2, la, lb);
                    l = la + lb;
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&p_full));
            }
            if (!ok) break;
            const bool whole = w.whole(), any = te > w.t0;
            if (!whole && w.t0 == 0) mine = w.cut();
            if (any && !wait(&pv_done, (it - 1) & 1)) break;
            tc_fence_after();
            if (!some) continue;
            const float inv = m == -INFINITY ? 0.f : 1.0f / l;
            const size_t slot = static_cast<size_t>(w.slot()) * ROWS + row;
            T* dst = nullptr;
            if (active)
                dst = static_cast<T*>(a.out) +
                      (static_cast<size_t>(s.row0 + rr / G) * a.Hq + w.g * G + rr % G) * HD;
#pragma unroll 1
            for (int q = 0; q < HD / 32; ++q) {
                uint32_t v[32];
                if (any) tmem_ld32(t_o + q * 32, v);
                else
#pragma unroll
                    for (int x = 0; x < 32; ++x) v[x] = 0u;
                if (!active) continue;
#pragma unroll
                for (int ch = 0; ch < 4; ++ch) {
                    float d[8];
#pragma unroll
                    for (int x = 0; x < 8; ++x) d[staged_dim<BITS>(x)] = __uint_as_float(v[ch * 8 + x]);
                    if (whole) {
                        *reinterpret_cast<uint4*>(dst + q * 32 + ch * 8) =
                            make_uint4(pk_round<T>(d[0] * inv, d[1] * inv), pk_round<T>(d[2] * inv, d[3] * inv),
                                       pk_round<T>(d[4] * inv, d[5] * inv), pk_round<T>(d[6] * inv, d[7] * inv));
                    } else {
                        float4* o = reinterpret_cast<float4*>(p.part_o + slot * HD + q * 32 + ch * 8);
                        o[0] = make_float4(d[0], d[1], d[2], d[3]);
                        o[1] = make_float4(d[4], d[5], d[6], d[7]);
                    }
                }
            }
            if (!whole && active) p.part_ml[slot] = make_float2(m, l);
        }
        if (row == 0) p.cut[blockIdx.x] = mine;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == WARP_LOAD0) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kCols));
    }
}

namespace {
template <typename T>
const void* tc_fn(int hd, int bits) {
    if (hd == 128)
        return bits == 16  ? reinterpret_cast<const void*>(&attn_rows_tc_kernel<T, 128, 16>)
               : bits == 8 ? reinterpret_cast<const void*>(&attn_rows_tc_kernel<T, 128, 8>)
                           : reinterpret_cast<const void*>(&attn_rows_tc_kernel<T, 128, 4>);
    return bits == 16  ? reinterpret_cast<const void*>(&attn_rows_tc_kernel<T, 64, 16>)
           : bits == 8 ? reinterpret_cast<const void*>(&attn_rows_tc_kernel<T, 64, 8>)
                       : reinterpret_cast<const void*>(&attn_rows_tc_kernel<T, 64, 4>);
}
}  // namespace

const void* rows_tc_fn(int dtype, int hd, int bits) {
    return dtype == kBF16 ? tc_fn<__nv_bfloat16>(hd, bits) : tc_fn<__half>(hd, bits);
}

size_t rows_tc_smem(int hd) {  // Q, K and V tiles, and the slack to align them
    return 3 * static_cast<size_t>(rt::KT) * hd * 2 + 1024;
}

cudaError_t rows_tc_read_error(int* code) {
    int v = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_rows_tc_error, sizeof(int));
    if (e != cudaSuccess) return e;
    if (v) {
        const int zero = 0;
        e = cudaMemcpyToSymbol(g_rows_tc_error, &zero, sizeof(int));
    }
    *code = v;
    return e;
}

}  // namespace mlxq
