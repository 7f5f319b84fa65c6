// Attention of many query rows over keys and values in 16 bits on tcgen05 (sm_100a): prompt
// chunks and trees of drafted tokens. A quantised cache's rows are expanded to 16 bits once
// by kv_expand_kernel (every chunk of rows would otherwise dequantise them again, and 128
// rows by 64 keys leave no issue slots for it: staged in the kernel itself, two prompts'
// chunks of 2048 tokens over 8200 4-bit keys took 599 to 945 us in four arrangements).
//
// One tile is 128 query rows (new tokens x the query heads of a kv head) by 64 keys:
//   S = Q K^T   M = 128, N = 64, K = head size: Q and K in shared memory, S in tensor
//               memory (32-bit)
//   softmax     thread = row: S is read back, P = exp2(S * scale - m) goes back into the
//               columns of S as 16-bit pairs. m follows the running maximum only when a
//               score passes it by 2^8, so O is rescaled seldom; P then reaches 256, which
//               costs neither type precision. (Rounded to T as a 16-bit product's operand: half
//               a step each, 2.0e-3 to 2.3e-3 of a bf16 result where unrounded ones leave 1.7e-3.)
//   O += P V    M = 128, N = head size, K = 64: P read from tensor memory, V from shared
//               memory as it lies (key rows, dimensions contiguous)
// S, K and V have two buffers each, so S of the next tile is there when the softmax of this
// one ends, and P V runs under the next softmax. Warps 0-3 hold a tensor-memory lane quarter
// each and do the softmax and the epilogue; warp 4 brings keys in by TMA and warp 6 values, a
// box to a page and 64 dims (one warp for both takes 2100 cycles a tile of 16-key pages,
// longer than the softmax); warp 5 issues the products. A chunk is whole tokens, 128 / G of
// them, so that its queries are one box too (64 dims, G heads, the tokens): loaded by a
// warp's lanes they took 5000 cycles of every item. Two CTAs share an SM: 105 KB of dynamic
// shared memory (heads of 128) and 256 of the 512 columns each. For heads of 64 it is registers,
// 128 a thread, that leave no room for a third, which would wait for columns.
// Work is shared out as in rows_units.cuh. Every wait is bounded: on a timeout the CTA
// records an error, its roles stop, what is in flight is waited for, tensor memory is
// freed and the kernel returns.
#include <cudaTypedefs.h>

#include <mutex>

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
constexpr int WARP_K = 4, WARP_MMA = 5, WARP_V = 6;
constexpr uint32_t kCols = 256;   // tensor memory: S (and P) from 0 and 64, O from 128
constexpr uint32_t kOCol = 128;
constexpr uint32_t kParkNs = 2000, kParkLimit = 1u << 20;  // ~2 s
constexpr uint32_t kSpinLimit = 1u << 22;
constexpr int kErrTimeout = 3;

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

__device__ __forceinline__ void st_shared16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ uint4 ld_shared16(uint32_t at) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
    return v;
}

// 3-D TMA load of one box (64 dims, one head, some rows); no cluster multicast.
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar,
                                            int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%3, %4, %5}], [%2];\n" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
}  // namespace rt

// One warp's 32 rows of O on their way out, whole (scaled, rounded to T, to their rows of the
// output) or as a part (32-bit). They go by way of 2 KB of shared memory, 64 bytes of each at
// a time, so that a store covers whole sectors: 16 bytes from each of 32 rows took 5000 to
// 10000 cycles an item. Sixteen-byte chunks are swizzled: no bank conflicts. (Not inlined:
// its registers would be the softmax's spills.)
struct Leave {
    uint32_t t_o;    // O's first column, or kNoCols: zeros
    uint32_t stage;
    int rows, x0, G, Hq;  // rows that are there, the first one's place in the chunk
};
constexpr uint32_t kNoCols = ~0u;

template <typename T, int HD, bool WHOLE>
__device__ __noinline__ void rows_leave(const Leave lv, float scale, void* base) {
    using namespace rt;
    constexpr int COLS = WHOLE ? 32 : 16;  // of O in 64 bytes
    const int lane = threadIdx.x & 31, ch = lane & 3;
    uint32_t off[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // a lane stores 16 bytes of rows lane / 4 + 8 i
        const int r = 8 * i + (lane >> 2), x = lv.x0 + r, dn = x * (65536 / lv.G + 1) >> 16;
        off[i] = WHOLE ? (dn * lv.Hq + x - dn * lv.G) * HD + ch * 8 : r * HD + ch * 4;
    }
#pragma unroll 1
    for (int q = 0; q < HD / COLS; ++q) {
        uint32_t v[COLS], o[16];
        if (lv.t_o == kNoCols) {
#pragma unroll
            for (int x = 0; x < COLS; ++x) v[x] = 0u;
        } else if constexpr (WHOLE) {
            tmem_ld32(lv.t_o + q * COLS, v);
        } else {
            tmem_ld16(lv.t_o + q * COLS, v);
        }
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            if constexpr (WHOLE)
                o[x] = pk_round<T>(__uint_as_float(v[2 * x]) * scale, __uint_as_float(v[2 * x + 1]) * scale);
            else
                o[x] = v[x];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            st_shared16(lv.stage + lane * 64 + ((i ^ (lane >> 1 & 3)) << 4), o[4 * i], o[4 * i + 1],
                        o[4 * i + 2], o[4 * i + 3]);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 8 * i + (lane >> 2);
            if (r < lv.rows) {
                const uint4 d = ld_shared16(lv.stage + r * 64 + ((ch ^ (r >> 1 & 3)) << 4));
                if constexpr (WHOLE) *reinterpret_cast<uint4*>(static_cast<T*>(base) + off[i] + q * COLS) = d;
                else *reinterpret_cast<uint4*>(static_cast<float*>(base) + off[i] + q * COLS) = d;
            }
        }
        __syncwarp();
    }
}

// Where the 16-bit rows are: the cache's pages (box = page size), or the expanded rows of
// sequence b from row b * rows_per_seq on, whole tiles of them, zeros behind the last key.
struct RowSource {
    int box, rows_per_seq, rows;  // rows_per_seq 0: pages; rows: of the whole source
};

template <typename T, int HD>
__global__ void __launch_bounds__(rt::THREADS, 2)
    attn_rows_tc_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                        const __grid_constant__ CUtensorMap tv,
                        const __grid_constant__ ra::Params p, const RowSource src) {
    using namespace rt;
    using namespace ra;
    constexpr int HB = KT * HD * 2;  // bytes of a tile of keys or values
    constexpr int HALVES = HD / 64;  // 128-byte wide halves of a row
    constexpr uint32_t AB = __is_same(T, __nv_bfloat16) ? 1u : 0u;
    constexpr uint32_t IDESC_S = (1u << 4) | (AB << 7) | (AB << 10) | ((KT / 8) << 17) | ((ROWS / 16) << 24);
    constexpr uint32_t IDESC_O = (1u << 4) | (AB << 7) | (AB << 10) | (1u << 16) | ((HD / 8) << 17) |
                                 ((ROWS / 16) << 24);
    extern __shared__ uint8_t rt_smem_raw[];
    __shared__ int pref[SCAN + 1];
    __shared__ __align__(8) uint64_t k_full[2], v_full[2], s_full[2], pv_done[2], p_full[2], q_full,
        q_free, v_land, drained;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile int s_abort;
    uint8_t* smem = rt_smem_raw + ((1024u - (smem_u32(rt_smem_raw) & 1023u)) & 1023u);
    uint8_t *qs = smem, *ks = smem + ROWS * HD * 2, *vs = ks + 2 * HB;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    if (warp == WARP_MMA) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(
                         smem_u32(&tmem_slot)),
                     "r"(kCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(k_full + i), 1);
            mbar_init(smem_u32(v_full + i), 1);
            mbar_init(smem_u32(p_full + i), 4);
            mbar_init(smem_u32(s_full + i), 1);
            mbar_init(smem_u32(pv_done + i), 1);
        }
        mbar_init(smem_u32(&q_full), 1);
        mbar_init(smem_u32(&q_free), 1);
        mbar_init(smem_u32(&v_land), 1);
        mbar_init(smem_u32(&drained), 1);
        s_abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == WARP_K && lane == 0) {
        tma_prefetch_map(&tq);
        tma_prefetch_map(&tk);
    }
    if (warp == WARP_V && lane == 0) tma_prefetch_map(&tv);
    pdl_wait();
    const RowsArgs& a = p.a;
    const KvCache& c = p.c;
    const int Hkv = c.Hkv, G = a.Hq / Hkv, chunk = ROWS / G * G;
    zero_tail(a, HD, THREADS);
    const Units un = scan_units<KT, false>(a, Hkv, G, chunk, p.group, pref);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    const int page_shift = 31 - __clz(c.page);
    __shared__ Walk<KT, true, false> walks[THREADS / 32];
    const Walk<KT, true, false>& w = walks[warp];
    Steps<KT> steps = {walks[warp], a};
    steps.begin(Hkv, chunk, un, p.parts, p.group, pref);

    // Tile j of the CTA's run uses buffer j & 1 of K, V, S and P, and that buffer's barriers'
    // phase j >> 1; item i the queries' barriers' phase i. No role is ever two phases behind
    // another: each buffer's next use waits for its last.
    auto wait_at = [&](uint64_t* bar, uint32_t parity) -> bool {
        if (mbar_try_wait(smem_u32(bar), parity & 1)) return true;
        for (uint32_t i = 0; i < kParkLimit && !s_abort; ++i)
            if (mbar_try_wait_hint(smem_u32(bar), parity & 1, kParkNs)) return true;
        atomicCAS(&g_rows_tc_error, 0, kErrTimeout);
        s_abort = 1;
        return false;
    };
    auto wait = [&](uint64_t* bars, uint32_t j) -> bool { return wait_at(bars + (j & 1), j >> 1); };
    // The tiles of the run one after another, whatever item they belong to.
    int tile = 0, te = 0, kend = 0;
    auto step = [&]() -> bool {  // to the next tile; false behind the last
        if (++tile < te) return true;
        while (te >= 0) {
            if (te > 0) steps.advance();
            if (!steps.next()) {
                te = -1;
                break;
            }
            kend = w.kend(a);
            te = w.tile_end(a);
            tile = w.t0;
            if (tile < te) return true;
            te = max(te, 1);  // (an item without keys: step over it)
        }
        return false;
    };

    if (warp == WARP_K || warp == WARP_V) {
        // ------------------------------ keys, values ---------------------------------
        // lane = (box of the tile, 64-dim half); a box that is not there is read from behind
        // the source's last row, which gives zeros
        const bool is_v = warp == WARP_V;
        const CUtensorMap* map = is_v ? &tv : &tk;
        uint64_t *full = is_v ? v_full : k_full, *freed = is_v ? pv_done : s_full;
        uint8_t* tiles = is_v ? vs : ks;
        const int nbox = KT / src.box, half = lane % HALVES, box = lane / HALVES;
        const bool loads = box < nbox;
        const uint32_t off = static_cast<uint32_t>(half * (KT * 128) + box * src.box * 128);
        auto page_of = [&]() -> int {  // (loaded a tile before it is used)
            const int key = tile * KT + box * src.box;
            if (!loads || key >= kend) return -1;
            if (src.rows_per_seq) return w.b * src.rows_per_seq + key;
            return a.table[static_cast<size_t>(w.b) * a.max_blocks + (key >> page_shift)];
        };
        uint32_t j = 0, lands = 0, items = 0;
        bool more = step();
        int page = more ? page_of() : -1;
        for (; more; ++j) {
            const int g = w.g, left = kend - tile * KT;  // keys of the tile
            if (!is_v && tile == w.t0) {  // the item's queries, once the last S of the one before is done
                if (items > 0 && !wait_at(&q_free, items - 1)) break;
                ++items;
                if (lane == 0) mbar_arrive_expect_tx(smem_u32(&q_full), chunk * HD * 2);
                __syncwarp();
                if (lane < HALVES)
                    tma_load_3d(smem_u32(qs) + lane * (ROWS * 128), &tq, smem_u32(&q_full), lane * 64, g * G,
                                w.s.row0 + w.rr0 / G);
            }
            const int row = page < 0 ? src.rows
                            : src.rows_per_seq ? page
                            : page < c.pages   ? page << page_shift
                                               : src.rows;
            more = step();
            page = more ? page_of() : -1;
            if (j > 1 && !wait(freed, j - 2)) {
                more = true;
                break;
            }
            uint8_t* dst = tiles + (j & 1) * HB;
            const uint32_t bar = smem_u32(full + (j & 1));
            // A page's rows behind the last key hold anything, and a probability of zero does
            // not make a number of what is none: those rows of V are zeroed once they landed.
            const bool ragged = is_v && left < KT && (left & (src.box - 1)) && !src.rows_per_seq;
            const uint32_t to = ragged ? smem_u32(&v_land) : bar;
            if (lane == 0) mbar_arrive_expect_tx(to, HB);
            __syncwarp();
            if (loads) tma_load_3d(smem_u32(dst) + off, map, to, half * 64, g, row);
            if (ragged) {
                if (!wait_at(&v_land, lands++)) {
                    more = true;
                    break;
                }
                const int end = min(KT, (left + src.box - 1) & ~(src.box - 1));
                for (int i = left * 8 + lane; i < end * 8; i += 32)
#pragma unroll
                    for (int h = 0; h < HALVES; ++h)
                        *reinterpret_cast<uint4*>(dst + h * (KT * 128) + i * 16) = make_uint4(0u, 0u, 0u, 0u);
                fence_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            }
        }
        if (more) {  // stopped early: the copies under way land before the CTA ends
            for (uint32_t i = j > 1 ? j - 2 : 0; i < j; ++i)
                mbar_wait_bounded(smem_u32(full + (i & 1)), (i >> 1) & 1, kSpinLimit);
            if (lands) mbar_wait_bounded(smem_u32(&v_land), (lands - 1) & 1, kSpinLimit);
            if (items) mbar_wait_bounded(smem_u32(&q_full), (items - 1) & 1, kSpinLimit);
        }
    } else if (warp == WARP_MMA) {
        // ------------------------------ products -------------------------------------
        // The whole warp walks along, so that descriptors stay in uniform registers (by one
        // thread in a branch of its own, issuing took 2600 cycles a tile, twice what the
        // softmax takes); one thread of it issues.
        const uint32_t leader = elect_leader();
        auto spin = [&](uint64_t* bar, uint32_t parity) -> bool {
            // (polls without parking: it wakes fastest)
            if (mbar_wait_bounded(smem_u32(bar), parity & 1, 64)) return true;
            for (uint32_t i = 0; i < kSpinLimit / 64 && !s_abort; ++i)
                if (mbar_wait_bounded(smem_u32(bar), parity & 1, 64)) return true;
            atomicCAS(&g_rows_tc_error, 0, kErrTimeout);
            s_abort = 1;
            return false;
        };
        const uint64_t qd = sw128_kmajor_desc(smem_u32(qs)), kd = sw128_kmajor_desc(smem_u32(ks));
        const uint64_t vd = sw128_mnmajor_desc(smem_u32(vs), KT * 128);
        uint32_t ns = 0, npv = 0, nq = 0;  // S and P V issued, items of queries met
        uint32_t begins = 0;               // tiles that begin an item, by their last five bits
        bool more = step();                // a tile whose S is to come
        while (more || npv < ns) {
            // S runs up to two tiles ahead of P V. An item's first waits for its queries, and
            // they for the last S of the item before: P V goes first then.
            // (One poll's answer is each lane's own: they vote on it, and lanes that left a wait
            // early are waited for, or some could fall behind by the two phases a barrier holds.)
            __syncwarp();
            const bool begin = tile == w.t0;
            const uint32_t sb = ns & 1, vb = npv & 1;
            if (more && ns - npv < 2 &&
                (!begin || npv == ns ||
                 __all_sync(0xffffffffu, mbar_try_wait(smem_u32(&q_full), nq & 1) &&
                                             mbar_try_wait(smem_u32(k_full + sb), ns >> 1 & 1)))) {
                if ((begin && !spin(&q_full, nq++)) || !spin(k_full + sb, ns >> 1)) break;
                tc_fence_after();
                const uint32_t bit = 1u << (ns & 31);
                begins = begin ? begins | bit : begins & ~bit;
                const uint64_t kb = kd + sb * (HB / 16);
                const uint32_t d = tmem + sb * KT;
#pragma unroll
                for (int i = 0; i < HD / 16; ++i)  // 16 dims: 32 bytes of a half of them
                    umma_f16_ss_by(leader, d, qd + (i / 4) * (ROWS * 128 / 16) + (i % 4) * 2,
                                   kb + (i / 4) * (KT * 128 / 16) + (i % 4) * 2, IDESC_S, i > 0 ? 1u : 0u);
                umma_commit_by(leader, smem_u32(s_full + sb));
                if (tile + 1 == te) umma_commit_by(leader, smem_u32(&q_free));
                ++ns;
                more = step();
                continue;
            }
            if (!spin(v_full + vb, npv >> 1) || !spin(p_full + vb, npv >> 1)) break;
            tc_fence_after();
            const uint64_t vt = vd + vb * (HB / 16);
            const uint32_t pa = tmem + vb * KT;
            const bool fresh = begins >> (npv & 31) & 1;
#pragma unroll
            for (int i = 0; i < KT / 16; ++i)  // 16 keys: 8 columns of P, 2 KB of V
                umma_f16_ts_by(leader, tmem + kOCol, pa + 8 * i, vt + i * (2048 / 16), IDESC_O,
                               (!fresh || i > 0) ? 1u : 0u);
            umma_commit_by(leader, smem_u32(pv_done + vb));
            ++npv;
        }
        // every product issued has finished before tensor memory is freed
        umma_commit_by(leader, smem_u32(&drained));
        mbar_wait_bounded(smem_u32(&drained), 0, kSpinLimit);
    } else {
        // ------------------------------ softmax, epilogue -----------------------------
        const int row = tid;  // of the tile; tensor-memory lane
        const uint32_t t_w = tmem + (static_cast<uint32_t>(warp * 32) << 16), t_o = t_w + kOCol;
        const float scale = fmaxf(fabsf(p.scale_log2), 0x1p-100f);  // (zero times -inf is no number)
        uint32_t it = 0;  // tiles so far
        Cut mine = {};
        bool ok = true;
        for (; ok && steps.next(); steps.advance()) {
            const Seq s = w.s;
            const int kend = w.kend(a), te = w.tile_end(a), base = w.base(), R = s.n * G;
            const int rr = w.rr0 + row;
            // this row; any of the warp's
            const bool active = rr < R && row < chunk, some = w.rr0 + warp * 32 < R;
            const int full = min(max(base, 0), kend);  // keys every row sees
            const int32_t* bt = a.table + static_cast<size_t>(w.b) * a.max_blocks;
            unsigned long long vis = 0;  // of the new tokens, those this row sees
            const int tok = active ? rr / G : -1;
            if (a.mask && active) vis = static_cast<unsigned long long>(a.mask[s.row0 + tok]);
            float m = -INFINITY, l = 0.f;
            // which eights of a tile's keys are on pages of the pool: looked up a tile ahead
            auto page_at = [&](int k0) -> int {
                const int key = k0 + 8 * (lane & 7);
                return key < kend ? bt[key >> page_shift] : 0;
            };
            int pid = page_at(w.t0 * KT);
            for (int tile = w.t0; tile < te; ++tile, ++it) {
                const int k0 = tile * KT;
                const uint32_t t_s = t_w + (it & 1) * KT;
                const uint32_t pages_ok = __ballot_sync(0xffffffffu, pid >= 0 && pid < c.pages) & 0xffu;
                pid = page_at(k0 + KT);
                const bool clean = k0 + KT <= full && pages_ok == 0xffu;
                if (!wait(s_full, it)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                if (some) {
                    uint32_t v[2][32];
                    tmem_ld64(t_s, v[0], v[1]);
                    if (p.scale_log2 < 0.f) {  // the sign of the scale goes into the scores
#pragma unroll
                        for (int x = 0; x < 64; ++x) v[x / 32][x % 32] ^= 0x80000000u;
                    }
                    if (!clean) {
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            // the keys of these 32 that this row sees, a bit each
                            const int kk = k0 + 32 * q, left = kend - kk, j0 = kk - base;
                            uint32_t bits = left >= 32 ? ~0u : left <= 0 ? 0u : (1u << left) - 1u;
                            bits &= ((pages_ok >> (4 * q) & 15u) * 0x00204081u & 0x01010101u) * 255u;
                            if (j0 > -32) {
                                if (a.mask) {
                                    bits &= j0 >= 64  ? 0u
                                            : j0 >= 0 ? static_cast<uint32_t>(vis >> j0)
                                                      : static_cast<uint32_t>(vis << -j0) | ((1u << -j0) - 1u);
                                } else {
                                    const int n = tok - j0 + 1;
                                    bits &= n >= 32 ? ~0u : n <= 0 ? 0u : (1u << n) - 1u;
                                }
                            }
#pragma unroll
                            for (int x = 0; x < 32; ++x) v[q][x] = bits >> x & 1 ? v[q][x] : 0xff800000u;
                        }
                    }
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int x = 0; x < 64; x += 2)
                        m4[x / 2 & 3] = fmaxf(m4[x / 2 & 3], fmaxf(__uint_as_float(v[x / 32][x % 32]),
                                                                   __uint_as_float(v[x / 32][x % 32 + 1])));
                    const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * scale;
                    // (rows that are not there hold anything: they have no say in when the others
                    // rescale, or results would change from call to call by a rounding)
                    if (__any_sync(0xffffffffu, active && mx - m > 8.f)) {
                        const float mn = fmaxf(m, mx);
                        const float f = mn == -INFINITY ? 1.f : exp2f(m - mn);
                        m = mn;
                        l *= f;
                        if (tile > w.t0) {  // O so far: every P V issued has to be in it
                            if (!wait(pv_done, it - 1)) {
                                ok = false;
                                break;
                            }
                            tc_fence_after();
#pragma unroll 1
                            for (int q = 0; q < HD / 16; ++q) {
                                uint32_t o[16];
                                tmem_ld16(t_o + q * 16, o);
#pragma unroll
                                for (int x = 0; x < 16; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
                                tmem_st16(t_o + q * 16, o);
                            }
                        }
                    }
                    // a row that has seen nothing yet: its scores are -inf, 2^-inf = 0
                    const float mr = m == -INFINITY ? 0.f : m;
                    const uint64_t scale2 = pack_f2(scale, scale), mr2 = pack_f2(-mr, -mr);
                    uint64_t l2 = pack_f2(l, 0.f);
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        uint32_t o[16];
#pragma unroll
                        for (int x = 0; x < 32; x += 2) {
                            float e0, e1;
                            unpack_f2(fma_f2(pack_f2(__uint_as_float(v[q][x]), __uint_as_float(v[q][x + 1])),
                                             scale2, mr2), e0, e1);
                            e0 = ex2(e0);
                            e1 = ex2(e1);
                            l2 = add_f2(l2, pack_f2(e0, e1));
                            o[x / 2] = pk_round<T>(e0, e1);
                        }
                        tmem_st16(t_s + q * 16, o);
                    }
                    float la, lb;
                    unpack_f2(l2, la, lb);
                    l = la + lb;
                    tmem_wait_st();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(p_full + (it & 1)));
            }
            if (!ok) break;
            const bool whole = w.whole(), any = te > w.t0;
            if (!whole && w.t0 == 0) mine = w.cut();
            if (any && !wait(pv_done, it - 1)) break;
            tc_fence_after();
            if (!some) continue;
            Leave lv;
            lv.t_o = any ? t_o : kNoCols;
            lv.stage = smem_u32(smem + ROWS * HD * 2 + 4 * HB + warp * 2048);
            lv.rows = min(min(R - w.rr0, chunk) - warp * 32, 32);
            lv.x0 = warp * 32;
            lv.G = G;
            lv.Hq = a.Hq;
            if (whole) {
                rows_leave<T, HD, true>(lv, m == -INFINITY ? 0.f : 1.0f / l,
                                        static_cast<T*>(a.out) +
                                            (static_cast<size_t>(s.row0 + w.rr0 / G) * a.Hq + w.g * G) * HD);
            } else {
                const size_t slot = static_cast<size_t>(w.slot()) * ROWS + warp * 32;
                rows_leave<T, HD, false>(lv, 1.f, p.part_o + slot * HD);
                if (lane < lv.rows) p.part_ml[slot + lane] = make_float2(m, l);
            }
        }
        if (row == 0) p.cut[blockIdx.x] = mine;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == WARP_MMA) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(kCols));
    }
}

// The values of every sequence's keys, from the first to the end of its last tile (zeros
// behind the last key and for pages outside the pool): block (tile of 64 keys, sequence,
// keys or values), thread = (eight values of a row, row), so that a warp reads and writes
// one span; eight rows in flight. (Ordinary loads: see ldw in paged_attn.cu.)
template <typename T, int BITS>
__global__ void __launch_bounds__(256)
    kv_expand_kernel(const KvCache c, const RowsArgs a, int rows_per_seq, T* __restrict__ k_out,
                     T* __restrict__ v_out) {
    constexpr int AHEAD = 8;
    pdl_launch_dependents();
    pdl_wait();
    const bool is_v = blockIdx.z != 0;
    const int b = blockIdx.y, k0 = blockIdx.x * rt::KT;
    const int L = max(0, min(a.kv_lens[b], a.max_kv));
    if (k0 >= L) return;
    const uint32_t cpr = c.Hkv * c.hd / 8;                       // chunks of eight values in a row
    const int page_shift = 31 - __clz(c.page), gs_shift = 28 - __clz(c.gs);  // (of chunks)
    const uint32_t gpr = cpr >> gs_shift;                        // groups in a row
    const int32_t* bt = a.table + static_cast<size_t>(b) * a.max_blocks;
    for (uint32_t col = threadIdx.x; col < cpr; col += blockDim.x) {
        const uint32_t* codes = static_cast<const uint32_t*>(is_v ? c.v : c.k) + col * (BITS / 4);
        const uint16_t* sp = static_cast<const uint16_t*>(is_v ? c.vs : c.ks) + (col >> gs_shift);
        const uint16_t* bp = static_cast<const uint16_t*>(is_v ? c.vb : c.kb) + (col >> gs_shift);
        uint4* out = reinterpret_cast<uint4*>(is_v ? v_out : k_out) +
                     (static_cast<size_t>(b) * rows_per_seq + k0) * cpr + col;
        for (uint32_t r0 = threadIdx.y; r0 < rt::KT; r0 += AHEAD * blockDim.y) {
            uint32_t raw[AHEAD][BITS / 4], there = 0;
            uint16_t s[AHEAD], z[AHEAD];
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int r = r0 + j * blockDim.y, key = k0 + r;
                int pid = -1;
                if (r < rt::KT && key < L) pid = bt[key >> page_shift];
                const bool in = pid >= 0 && pid < c.pages;
                there |= in ? 1u << j : 0u;
                // (a row that is not there is read from the pool's first, and not used)
                const uint32_t row = in ? (static_cast<uint32_t>(pid) << page_shift) + (key & (c.page - 1)) : 0u;
                const uint32_t* at = codes + static_cast<size_t>(row) * (cpr * (BITS / 4));
                if constexpr (BITS == 8) {
                    const uint2 v = *reinterpret_cast<const uint2*>(at);
                    raw[j][0] = v.x;
                    raw[j][1] = v.y;
                } else {
                    raw[j][0] = *at;
                }
                s[j] = sp[static_cast<size_t>(row) * gpr];
                z[j] = bp[static_cast<size_t>(row) * gpr];
            }
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const uint32_t r = r0 + j * blockDim.y;
                if (r >= rt::KT) break;
                uint4 o = make_uint4(0u, 0u, 0u, 0u);
                if (there >> j & 1u) o = in_order<T, BITS>(raw[j], pk_splat(s[j]), pk_splat(z[j]));
                out[static_cast<size_t>(r) * cpr] = o;
            }
        }
    }
}

namespace {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
    });
    return fn;
}

// [rows, heads, hd] of 16-bit elements, boxes of 64 dims of `box_heads` heads and `box` rows.
cudaError_t row_map(CUtensorMap* m, const void* base, int dtype, int hd, int heads, long long rows,
                    int box_heads, int box) {
    const PFN_cuTensorMapEncodeTiled_v12000 enc = encode_fn();
    if (!enc) return cudaErrorNotSupported;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(hd), static_cast<cuuint64_t>(heads),
                                static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(hd) * 2,
                                   static_cast<cuuint64_t>(heads) * hd * 2};
    const cuuint32_t boxes[3] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box)};
    const cuuint32_t ones[3] = {1, 1, 1};
    const CUresult r = enc(m, dtype == kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           3, const_cast<void*>(base), dims, strides, boxes, ones,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

size_t tc_smem(int hd) {  // Q, two tiles each of K and V, the epilogue's 8 KB, slack to align
    return (rt::ROWS + 4 * static_cast<size_t>(rt::KT)) * hd * 2 + 8192 + 1024;
}

// (a tile at least, so that a tensor map of a call without keys has rows)
int rows_per_seq(const RowsArgs& a) { return ((a.max_kv > 0 ? a.max_kv : 1) + rt::KT - 1) / rt::KT * rt::KT; }

}  // namespace

size_t rows_tc_expand_bytes(const KvCache& c, const RowsArgs& a) {
    return static_cast<size_t>(rows_per_seq(a)) * c.Hkv * c.hd * 4;
}

cudaError_t launch_rows_tc(ra::Params& p, void* expanded, bool overlap, cudaStream_t st) {
    const KvCache& c = p.c;
    const bool bf = c.dtype == kBF16, big = c.hd == 128;
    RowSource src = {c.page, 0, c.pages * c.page};
    const void *k = c.k, *v = c.v;
    if (c.bits != 16) {
        int rps = rows_per_seq(p.a);
        const size_t each = static_cast<size_t>(p.a.batch) * rps * c.Hkv * c.hd * 2;
        void *ko = expanded, *vo = static_cast<char*>(expanded) + each;
        const int cpr = c.Hkv * c.hd / 8, x = cpr < 256 ? cpr : 256;
        KvCache cc = c;
        RowsArgs aa = p.a;
        void* args[] = {&cc, &aa, &rps, &ko, &vo};
        const void* f = bf ? (c.bits == 8 ? reinterpret_cast<const void*>(&kv_expand_kernel<__nv_bfloat16, 8>)
                                          : reinterpret_cast<const void*>(&kv_expand_kernel<__nv_bfloat16, 4>))
                           : (c.bits == 8 ? reinterpret_cast<const void*>(&kv_expand_kernel<__half, 8>)
                                          : reinterpret_cast<const void*>(&kv_expand_kernel<__half, 4>));
        static PerDevice cfg[4];
        const cudaError_t e = launch_ex(f, cfg[(bf ? 0 : 2) + (c.bits == 8 ? 0 : 1)],
                                        dim3(rps / rt::KT, p.a.batch, 2), dim3(x, 256 / x), 0, st,
                                        overlap, args);
        if (e != cudaSuccess) return e;
        overlap = true;  // (the attention waits for the whole of it)
        k = ko;
        v = vo;
        src = {rt::KT, rps, p.a.batch * rps};
    }
    const int G = p.a.Hq / c.Hkv;
    CUtensorMap tq, tk, tv;
    cudaError_t e = row_map(&tq, p.a.q, c.dtype, c.hd, p.a.Hq, p.a.total, G, rt::ROWS / G);
    if (e == cudaSuccess) e = row_map(&tk, k, c.dtype, c.hd, c.Hkv, src.rows, 1, src.box);
    if (e == cudaSuccess) e = row_map(&tv, v, c.dtype, c.hd, c.Hkv, src.rows, 1, src.box);
    if (e != cudaSuccess) return e;
    void* args[] = {&tq, &tk, &tv, &p, &src};
    const void* f = bf ? (big ? reinterpret_cast<const void*>(&attn_rows_tc_kernel<__nv_bfloat16, 128>)
                              : reinterpret_cast<const void*>(&attn_rows_tc_kernel<__nv_bfloat16, 64>))
                       : (big ? reinterpret_cast<const void*>(&attn_rows_tc_kernel<__half, 128>)
                              : reinterpret_cast<const void*>(&attn_rows_tc_kernel<__half, 64>));
    static PerDevice cfg[4];
    return launch_ex(f, cfg[(bf ? 0 : 2) + (big ? 0 : 1)], dim3(p.parts), dim3(kRowsTcThreads),
                     tc_smem(c.hd), st, overlap, args);
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
