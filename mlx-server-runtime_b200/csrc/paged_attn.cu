// Attention of query rows over a paged KV cache in 16, 8 or 4 bits (sm_100a): decode steps,
// prompt chunks and trees of drafted tokens.
//
// Reference (huydt84/mlx-server-runtime, python/mlx_worker/native_mlx/): append_and_attend
// (attention.py:215-298) over pages, with a causal or, for drafted trees, an ancestor mask.
//
//   s = scale * q . k over the visible keys, p = exp(s - m), out = sum p v / sum p
//
// Rows: sequence b has R = n * G query rows per kv head (its n new tokens times the G query
// heads that share the head). This file's kernel takes up to eight of them (a decode step's
// heads) or sixteen (of a quantised cache); more are tcgen05's M rows (paged_attn_tc.cu).
// The rows' keys are taken in tiles of 128, a warp 32 of them, and the tiles of all sequences
// form one sequence of units that the CTAs share out evenly, whatever the lengths
// (rows_units.cuh). A part of an item goes to a workspace slot of its CTA, and
// attn_combine_kernel joins the parts in order of keys.
//
// Keys are the M rows of the m16n8k16 products and query rows the N columns, so eight rows
// fill a tile without padding:
//   S^T = K Q^T    A = 16 keys x 16 dims, straight from global memory: a lane's dims are
//                  contiguous in its key's row, and q is permuted to match once
//   O^T = V^T P^T  A = 16 dims x 16 keys, pairs of keys joined by byte permutes; P^T is S^T
//                  rounded to T (a 16-bit product's operand: half a step each, 2.0e-3 to
//                  2.3e-3 of a bf16 result where unrounded ones leave 1.7e-3, the result's own
//                  rounding) and transposed in registers (movmatrix)
// so packed codes go from their load through registers into the product; shared memory
// holds only the four warps' results at the end of an item. Rows are loaded into registers a
// tile ahead, page ids two.
//
// What bounds it is how rows arrive: 32 sequences of up to 16384 4-bit keys (4 kv heads of 128,
// 192 MB, 16384 down to 4500 keys) take 80 us, 2.4 TB/s, of which 15 do not depend on the
// lengths; with the loads left out they take 47, with the unpacking left out 74, and with
// keys that fit L2 the rate is the same. Sixteen-key pages of one head are 64-byte pieces, and
// a head's scales a quarter of their sectors. 8-bit codes of the same heads move 3.5 TB/s,
// 16-bit rows 4.7. Shorter runs (94 to 115 us) were slower, as were four heads' warps in one
// CTA, which share those sectors but join four times the parts (75 us here, but 32 for 23 with
// 64 sequences of 1000 keys and 89 for 82 over 16 bits).
#include "common.cuh"
#include "kv_dequant.cuh"
#include "overlap.cuh"
#include "paged_ops.h"
#include "rows_units.cuh"
#include "sm100.cuh"

namespace mlxq {

namespace ra {
constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int KT = 32 * WARPS;  // keys per tile

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
    return r;
}

// Everything here may have been written by a kernel of the same stream that still ran when
// this one was launched (launch overlap): ordinary loads, which the wait for that kernel
// orders, and not the read-only path, whose data must not change while a kernel runs.
template <int N>
__device__ __forceinline__ void ldw(const void* at, uint32_t (&r)[N]) {
    if constexpr (N == 1) {
        r[0] = *static_cast<const uint32_t*>(at);
    } else if constexpr (N == 2) {
        const uint2 v = *static_cast<const uint2*>(at);
        r[0] = v.x;
        r[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 v = static_cast<const uint4*>(at)[i];
            r[4 * i] = v.x;
            r[4 * i + 1] = v.y;
            r[4 * i + 2] = v.z;
            r[4 * i + 3] = v.w;
        }
    }
}

// CTAs of an SM: what the registers of a variant allow (and the launch bounds ask for).
// Three rather than four for heads of 128, which spills nothing: 32 sequences of up to 16384
// 4-bit keys 80 us (four: 78), 64 of 1000 22.7 (23.7), 16 of 4097 20.7 (21.2), and over 8 bits
// 32 of up to 16384 105 (130).
constexpr int resident(int hd, int bits, int nt) {
    return nt == 2 ? 2 : bits == 16 ? (hd == 64 ? 3 : 2) : hd == 64 ? 4 : 3;
}
}  // namespace ra

// NG: quantisation groups of a head's row (1 for 16-bit rows).
template <typename T, int HD, int BITS, int NG, int NT>
__global__ void __launch_bounds__(ra::THREADS, ra::resident(HD, BITS, NT))
    attn_rows_kernel(const __grid_constant__ ra::Params p) {
    using namespace ra;
    constexpr int ROWS = 8 * NT;
    constexpr int RB = HD * BITS / 8;  // bytes of a row
    constexpr int MT = HD / 16;
    constexpr int KW = HD / 4 * BITS / 32, VW = HD / 8 * BITS / 32;  // a lane's words of a row
    __shared__ int pref[SCAN + 1];
    __shared__ float wo[WARPS][ROWS][HD + 4];
    __shared__ float wm[WARPS][ROWS], wl[WARPS][ROWS];
    pdl_launch_dependents();
    pdl_wait();
    const RowsArgs& a = p.a;
    const KvCache& c = p.c;
    const int Hkv = c.Hkv, G = a.Hq / Hkv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r8 = lane >> 2, c4 = lane & 3;
    const int page_shift = 31 - __clz(c.page);
    const T* q = static_cast<const T*>(a.q);
    T* out = static_cast<T*>(a.out);

    zero_tail(a, HD, THREADS);
    const Units un = scan_units<KT, true>(a, Hkv, G, ROWS, p.group, pref);
    Walk<KT, false, true> w;
    w.begin(a, Hkv, ROWS, un, p.parts, p.group, pref);
    Cut mine = {};

    const float scale = fmaxf(fabsf(p.scale_log2), 0x1p-100f);  // (zero times -inf is no number)
    const int kg = NG == 1 ? 0 : c4 * NG / 4;  // this lane's group of a key row
    const int vg = NG == 1 ? 0 : r8 * NG / 8;  // and of a value row
    const uint32_t row_bytes = static_cast<uint32_t>(Hkv) * RB;  // of a token: its heads' rows

    for (; w.next(a); w.advance()) {
        const Seq& s = w.s;
        const int g = w.g, row_lo = w.rr0, t0 = w.t0, R = s.n * G;
        const int base = w.base(), kend = w.kend(a), full = min(max(base, 0), kend);
        const int32_t* bt = a.table + static_cast<size_t>(w.b) * a.max_blocks;
        const int te = w.tile_end(a);

        // A warp takes 32 keys of each tile, lane = key of them for the page ids. Eight keys
        // share a page: eight e of the 32 begins at the row lane 8 e holds. Page ids are
        // loaded two steps before their use, rows one. A row that is not there is read from
        // the pool's first rows (and not used).
        auto page_id = [&](int tile) -> int {
            const int key = tile * KT + warp * 32 + lane;
            return tile < te && key < kend ? bt[key >> page_shift] : -1;
        };
        auto row_id = [&](int tile, int pid) -> uint32_t {
            const uint32_t in = static_cast<uint32_t>(tile * KT + warp * 32 + lane) & (c.page - 1);
            return (pid >= 0 && pid < c.pages ? static_cast<uint32_t>(pid) << page_shift : 0u) + in;
        };
        // Words of key rows r8 and r8 + 8 of each sixteen (a quarter of each), of value rows
        // 2 c4, 2 c4 + 1 and eight on (an eighth of each); of 32 keys x NG groups in order,
        // NG to a lane: scales and biases.
        uint32_t kw[2][2][KW], vw[2][4][VW];
        uint16_t ks[NG], kb[NG], vs[NG], vb[NG];
        const char* k_at = static_cast<const char*>(c.k) + static_cast<size_t>(r8) * row_bytes + g * RB + c4 * (RB / 4);
        const char* v_at = static_cast<const char*>(c.v) + static_cast<size_t>(2 * c4) * row_bytes + g * RB + r8 * (RB / 8);
        auto load_k = [&](uint32_t rows) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    ldw(k_at + static_cast<size_t>(__shfl_sync(0xffffffffu, rows, 16 * mt + 8 * h)) * row_bytes,
                        kw[mt][h]);
            if constexpr (BITS != 16) {
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const int id = 32 * i + lane;
                    const size_t at = static_cast<size_t>(__shfl_sync(0xffffffffu, rows, id / NG)) * (Hkv * NG) +
                                      (g * NG + id % NG);
                    ks[i] = static_cast<const uint16_t*>(c.ks)[at];
                    kb[i] = static_cast<const uint16_t*>(c.kb)[at];
                }
            }
        };
        auto load_v = [&](uint32_t rows) {
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // (the pair's rows follow one another: one page)
                    const char* at = v_at +
                        static_cast<size_t>(__shfl_sync(0xffffffffu, rows, 16 * mt + 8 * h)) * row_bytes;
                    ldw(at, vw[mt][2 * h]);
                    ldw(at + row_bytes, vw[mt][2 * h + 1]);
                }
            if constexpr (BITS != 16) {
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const int id = 32 * i + lane;
                    const size_t at = static_cast<size_t>(__shfl_sync(0xffffffffu, rows, id / NG)) * (Hkv * NG) +
                                      (g * NG + id % NG);
                    vs[i] = static_cast<const uint16_t*>(c.vs)[at];
                    vb[i] = static_cast<const uint16_t*>(c.vb)[at];
                }
            }
        };
        int pid = page_id(t0);

        // Queries: lane (row r8 of the n-tile, quarter c4) holds its quarter's dims in the
        // order the key words unpack to.
        const uint32_t sign = p.scale_log2 < 0.f ? 0x80008000u : 0u;  // (the scale's goes into them)
        uint32_t bq[NT][MT][2];
        int qpos[NT][2];                // column 2 c4 + e: its index among the new tokens
        unsigned long long vis[NT][2];  // and its ancestors
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int rr = row_lo + 8 * nt + r8;
            uint32_t qw[HD / 8];
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) qw[i] = 0u;
            if (rr < R)
                ldw(q + (static_cast<size_t>(s.row0 + rr / G) * a.Hq + g * G + rr % G) * HD +
                        c4 * (HD / 4),
                    qw);
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                const int da = pair_dim<BITS>(i, 0), db = pair_dim<BITS>(i, 1);
                bq[nt][i / 2][i % 2] =
                    prmt(qw[da / 2], qw[db / 2], (da % 2 ? 0x32u : 0x10u) | (db % 2 ? 0x7600u : 0x5400u)) ^
                    sign;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int rc = row_lo + 8 * nt + 2 * c4 + e;
                qpos[nt][e] = rc < R ? rc / G : -1;
                vis[nt][e] = ~0ull;
                if (a.mask) vis[nt][e] = rc < R ? static_cast<unsigned long long>(a.mask[s.row0 + rc / G]) : 0ull;
            }
        }

        const uint32_t rows = row_id(t0, pid);
        bool mine_there = pid >= 0 && pid < c.pages;
        load_k(rows);
        load_v(rows);
        pid = page_id(t0 + 1);

        float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }

        for (int tile = t0; tile < te; ++tile) {
            const int k0 = tile * KT + warp * 32;
            // the keys of the 32 that are there, a bit each
            const uint32_t there = __ballot_sync(0xffffffffu, mine_there);
            const bool clean = there == ~0u;
            float sc[NT][2][4];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                uint32_t s2[2] = {0u, 0u}, b2[2] = {0u, 0u};
                if constexpr (BITS != 16) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // (the set that holds the id: a constant for each number of groups)
                        const int set = NG == 1 ? 0 : NG == 2 ? mt : 2 * mt + h;
                        const int id = (16 * mt + 8 * h + r8) * NG + kg;
                        const uint32_t sb = __shfl_sync(
                            0xffffffffu, ks[set] | static_cast<uint32_t>(kb[set]) << 16, id & 31);
                        s2[h] = pk_splat(sb);
                        b2[h] = prmt(sb, 0u, 0x3232u);
                    }
                }
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    const uint32_t a0 = row_pair<T, BITS>(kw[mt][0], 2 * j, s2[0], b2[0]);
                    const uint32_t a1 = row_pair<T, BITS>(kw[mt][1], 2 * j, s2[1], b2[1]);
                    const uint32_t a2 = row_pair<T, BITS>(kw[mt][0], 2 * j + 1, s2[0], b2[0]);
                    const uint32_t a3 = row_pair<T, BITS>(kw[mt][1], 2 * j + 1, s2[1], b2[1]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (j == 0) mma16816z<T>(sc[nt][mt], a0, a1, a2, a3, bq[nt][j][0], bq[nt][j][1]);
                        else mma16816<T>(sc[nt][mt], a0, a1, a2, a3, bq[nt][j][0], bq[nt][j][1]);
                    }
                }
            }
            // the next tile's keys come in from here on
            const uint32_t next = row_id(tile + 1, pid);
            mine_there = pid >= 0 && pid < c.pages;
            if (tile + 1 < te) load_k(next);
            pid = page_id(tile + 2);

            if (!clean || k0 + 32 > full) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int x = 16 * mt + 8 * (e >> 1) + r8, j = k0 + x - base;
                            const bool see = (there >> x & 1u) &&
                                             (j < 0 || (a.mask ? j < 64 && (vis[nt][e & 1] >> (j & 63) & 1)
                                                               : j <= qpos[nt][e & 1]));
                            sc[nt][mt][e] = see ? sc[nt][mt][e] : -INFINITY;
                        }
            }
            float top[NT][2];
            bool grow = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    top[nt][e] = fmaxf(fmaxf(sc[nt][0][e], sc[nt][0][e + 2]),
                                       fmaxf(sc[nt][1][e], sc[nt][1][e + 2])) * scale;
                    grow |= top[nt][e] > m[nt][e] + 8.f;
                }
            // The reference of the exponentials follows the running maximum only when a
            // score passes it by 2^8: the probabilities then reach 256, the sums lose nothing.
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = top[nt][e];
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                        mx = fmaxf(mx, m[nt][e]);
                        const float f = mx == -INFINITY ? 1.f : ex2(m[nt][e] - mx);
                        m[nt][e] = mx;
                        l[nt][e] *= f;
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            o[nt][i][e] *= f;
                            o[nt][i][e + 2] *= f;
                        }
                    }
            }
            uint32_t pb[NT][2][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float mr[2] = {m[nt][0] == -INFINITY ? 0.f : m[nt][0],
                                     m[nt][1] == -INFINITY ? 0.f : m[nt][1]};
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    float pr[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        pr[e] = ex2(fmaf(sc[nt][mt][e], scale, -mr[e & 1]));
                        l[nt][e & 1] += pr[e];
                    }
                    pb[nt][mt][0] = transpose8x8(pk_round<T>(pr[0], pr[1]));
                    pb[nt][mt][1] = transpose8x8(pk_round<T>(pr[2], pr[3]));
                }
            }
#pragma unroll
            for (int mt = 0; mt < 2; ++mt) {
                uint32_t s2[2] = {0u, 0u}, b2[2] = {0u, 0u};  // of value rows 2 c4, 2 c4 + 1; eight on
                // values of keys that are not there multiply zeros: make them zeros
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int x = 16 * mt + 8 * h + 2 * c4;
                    uint32_t keep = 0xffffffffu;
                    if (!clean)
                        keep = (there >> x & 1u ? 0xffffu : 0u) | (there >> x & 2u ? 0xffff0000u : 0u);
                    if constexpr (BITS == 16) {
                        if (!clean) {
#pragma unroll
                            for (int i = 0; i < VW; ++i) {
                                if (!(keep & 0xffffu)) vw[mt][2 * h][i] = 0u;
                                if (!(keep >> 16)) vw[mt][2 * h + 1][i] = 0u;
                            }
                        }
                    } else {
                        const int set = NG == 1 ? 0 : NG == 2 ? mt : 2 * mt + h;
                        const uint32_t sb = vs[set] | static_cast<uint32_t>(vb[set]) << 16;
                        const uint32_t e0 = __shfl_sync(0xffffffffu, sb, (x * NG + vg) & 31);
                        const uint32_t e1 = __shfl_sync(0xffffffffu, sb, ((x + 1) * NG + vg) & 31);
                        s2[h] = prmt(e0, e1, 0x5410u) & keep;
                        b2[h] = prmt(e0, e1, 0x7632u) & keep;
                    }
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    const uint32_t a0 = cross_pair<T, BITS>(vw[mt][0], vw[mt][1], i, s2[0], b2[0]);
                    const uint32_t a1 = cross_pair<T, BITS>(vw[mt][0], vw[mt][1], MT + i, s2[0], b2[0]);
                    const uint32_t a2 = cross_pair<T, BITS>(vw[mt][2], vw[mt][3], i, s2[1], b2[1]);
                    const uint32_t a3 = cross_pair<T, BITS>(vw[mt][2], vw[mt][3], MT + i, s2[1], b2[1]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
                        mma16816<T>(o[nt][i], a0, a1, a2, a3, pb[nt][mt][0], pb[nt][mt][1]);
                }
            }
            if (tile + 1 < te) load_v(next);
        }

        // Join the warps: (max, sum, O) of every row through shared memory.
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float sum = l[nt][e];
                sum += __shfl_xor_sync(0xffffffffu, sum, 4);
                sum += __shfl_xor_sync(0xffffffffu, sum, 8);
                sum += __shfl_xor_sync(0xffffffffu, sum, 16);
                const int col = 8 * nt + 2 * c4 + e;
                if (r8 == 0) {
                    wm[warp][col] = m[nt][e];
                    wl[warp][col] = sum;
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    wo[warp][col][r8 * (HD / 8) + i] = o[nt][i][e];
                    wo[warp][col][r8 * (HD / 8) + MT + i] = o[nt][i][e + 2];
                }
            }
        __syncthreads();
        const bool whole = w.whole();
        if (!whole && t0 == 0) mine = w.cut();
        const size_t slot = static_cast<size_t>(w.slot()) * ROWS;
        for (int i = tid; i < ROWS * HD / 2; i += THREADS) {
            const int row = i / (HD / 2), d = 2 * (i % (HD / 2)), rr = row_lo + row;
            if (rr >= R) continue;
            float M = -INFINITY, den = 0.f, x = 0.f, y = 0.f;
#pragma unroll
            for (int i = 0; i < WARPS; ++i) M = fmaxf(M, wm[i][row]);
#pragma unroll
            for (int i = 0; i < WARPS; ++i) {
                const float f = wm[i][row] == -INFINITY ? 0.f : ex2(wm[i][row] - M);
                den = fmaf(f, wl[i][row], den);
                x = fmaf(f, wo[i][row][d], x);
                y = fmaf(f, wo[i][row][d + 1], y);
            }
            if (whole) {
                const float inv = M == -INFINITY ? 0.f : 1.0f / den;
                T* dst = out + (static_cast<size_t>(s.row0 + rr / G) * a.Hq + g * G + rr % G) * HD + d;
                *reinterpret_cast<uint32_t*>(dst) = pk_round<T>(x * inv, y * inv);
            } else {
                *reinterpret_cast<float2*>(p.part_o + (slot + row) * HD + d) = make_float2(x, y);
                if (d == 0) p.part_ml[slot + row] = make_float2(M, den);
            }
        }
        __syncthreads();  // the shared results are read before the next item writes its own
    }
    if (tid == 0) p.cut[blockIdx.x] = mine;
}

// Joins the parts of the items that several CTAs took: block (CTA that began one, a few of
// its rows), lane = HD / 32 dimensions. Eight rows in 128 are many: a warp to a row. A
// decode step's eight are few, and a long sequence alone on the GPU has a part on every
// fourth CTA: two rows to a block, four warps to a row, each a run of the parts. Parts are
// taken in order of keys, eight loads ahead.
template <typename T, int HD, int ROWS>
__global__ void __launch_bounds__(256) attn_combine_kernel(const __grid_constant__ ra::Params p) {
    using namespace ra;
    constexpr int DPL = HD / 32, AHEAD = 8, S = ROWS == 128 ? 1 : 4, RPB = 8 / S;
    __shared__ float so[S > 1 ? 8 : 1][HD];
    __shared__ float2 sml[8];
    pdl_launch_dependents();
    pdl_wait();
    const Cut c = p.cut[blockIdx.x];
    const RowsArgs& a = p.a;
    const int G = a.Hq / p.c.Hkv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (static_cast<int>(blockIdx.y) * RPB >= c.rows) return;
    const int r = blockIdx.y * RPB + warp / S;
    const bool live = r < c.rows;
    const int first = blockIdx.x;
    // the warp's run of parts
    const int n = (c.last - first) / c.step + 1, per = (n + S - 1) / S;
    const int lo = warp % S * per, hi = live ? min(n, lo + per) : 0;
    float M = -INFINITY, den = 0.f, acc[DPL];
#pragma unroll
    for (int e = 0; e < DPL; ++e) acc[e] = 0.f;
    for (int i0 = lo; i0 < hi; i0 += AHEAD) {
        float2 ml[AHEAD];
        float v[AHEAD][DPL];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            ml[i] = make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int e = 0; e < DPL; ++e) v[i][e] = 0.f;
            if (i0 + i >= hi) continue;
            const int k = first + (i0 + i) * c.step;
            const size_t at = static_cast<size_t>(k == first ? c.slot : 2 * k) * ROWS + r;
            ml[i] = __ldcg(&p.part_ml[at]);
            if constexpr (DPL == 4) {
                const float4 t = __ldcg(reinterpret_cast<const float4*>(p.part_o + at * HD) + lane);
                v[i][0] = t.x; v[i][1] = t.y; v[i][2] = t.z; v[i][3] = t.w;
            } else {
                const float2 t = __ldcg(reinterpret_cast<const float2*>(p.part_o + at * HD) + lane);
                v[i][0] = t.x; v[i][1] = t.y;
            }
        }
        // one maximum for the eight and what went before
        float Mn = M;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) Mn = fmaxf(Mn, ml[i].x);
        const float co = M == -INFINITY ? 0.f : ex2(M - Mn);
        den *= co;
#pragma unroll
        for (int e = 0; e < DPL; ++e) acc[e] *= co;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const float cn = ml[i].x == -INFINITY ? 0.f : ex2(ml[i].x - Mn);
            den = fmaf(cn, ml[i].y, den);
#pragma unroll
            for (int e = 0; e < DPL; ++e) acc[e] = fmaf(cn, v[i][e], acc[e]);
        }
        M = Mn;
    }
    if constexpr (S > 1) {  // the row's warps, in order
        if (lane == 0) sml[warp] = make_float2(M, den);
#pragma unroll
        for (int e = 0; e < DPL; ++e) so[warp][lane * DPL + e] = acc[e];
        __syncthreads();
        if (warp % S != 0) return;
        float Mn = -INFINITY;
#pragma unroll
        for (int i = 0; i < S; ++i) Mn = fmaxf(Mn, sml[warp + i].x);
        den = 0.f;
#pragma unroll
        for (int e = 0; e < DPL; ++e) acc[e] = 0.f;
#pragma unroll
        for (int i = 0; i < S; ++i) {
            const float2 ml = sml[warp + i];
            const float cn = ml.x == -INFINITY ? 0.f : ex2(ml.x - Mn);
            den = fmaf(cn, ml.y, den);
#pragma unroll
            for (int e = 0; e < DPL; ++e) acc[e] = fmaf(cn, so[warp + i][lane * DPL + e], acc[e]);
        }
        M = Mn;
    }
    if (!live) return;
    const float inv = M == -INFINITY ? 0.f : 1.0f / den;
    const int rr = c.rr0 + r;
    T* dst = static_cast<T*>(a.out) +
             (static_cast<size_t>(c.row0 + rr / G) * a.Hq + c.g * G + rr % G) * HD + lane * DPL;
    if constexpr (DPL == 4)
        *reinterpret_cast<uint2*>(dst) = make_uint2(pk_round<T>(acc[0] * inv, acc[1] * inv),
                                                    pk_round<T>(acc[2] * inv, acc[3] * inv));
    else
        *reinterpret_cast<uint32_t*>(dst) = pk_round<T>(acc[0] * inv, acc[1] * inv);
}

namespace {

// How a call is run: eight rows to a chunk where a decode step's heads fit them; sixteen
// of a quantised cache; and from then on up to 128, whole tokens of them, as the M rows of
// tcgen05 products. The kernel of few rows takes one chunk a sequence. Nine to sixteen rows
// over 4 bits, 28/4 heads of 128, with sixteen rows to a chunk and as M rows, whose keys are
// expanded first: one sequence of 512 keys 11.7 and 14.6 us, of 16384 19.5 and 38; eight of 1024
// 14.6 and 24.5, of 4096 22 and 36, of 16384 40 and 94; 32 of 4096 41 and 90. Over 8 bits the
// same within a fifth. Over 16 bits, where nothing is expanded, eight of 4096 take 33 and 26.
struct Plan {
    bool tc;
    int rows, kt, parts, group;
    int chunk;  // rows of a chunk: `rows`, or the whole tokens of them
};
Plan plan_of(const KvCache& c, const RowsArgs& a) {
    const int G = a.Hq / c.Hkv;
    const long long r = static_cast<long long>(a.max_q) * G;
    Plan p;
    p.tc = r > (c.bits == 16 ? 8 : 16);
    p.rows = p.tc ? 128 : r > 8 ? 16 : 8;
    p.chunk = p.tc ? 128 / G * G : p.rows;
    p.kt = p.tc ? kRowsTcKeys : ra::KT;
    // CTAs the units are shared out to, in groups that take the same ones: what the GPU holds
    // at once, at most a group per unit
    const long long most = 148LL * (p.tc ? 2 : ra::resident(c.hd, c.bits, p.rows / 8));
    const long long tiles = a.max_kv > 0 ? (a.max_kv + p.kt - 1) / p.kt : 1;
    const long long chunks = (r + p.chunk - 1) / p.chunk;
    p.group = !p.tc ? c.Hkv : chunks >= 2 && chunks <= 8 ? static_cast<int>(chunks) : 1;
    long long units = tiles * (p.tc ? c.Hkv * (p.group > 1 ? 1 : chunks) : 1);  // of a sequence
    long long groups = most / p.group > 1 ? most / p.group : 1;
    // runs of fewer than four tiles cost more to join than they save: two CTAs an SM then
    // (a sequence of 32768 4-bit keys 18 us, with three 19; 16 of 4097 8-bit ones 17.6 and 19)
    const long long few = 296 / p.group;
    if (!p.tc && units * a.batch < 4 * groups && few < groups) groups = few > 1 ? few : 1;
    if (units < groups && units * a.batch < groups) groups = units * a.batch > 1 ? units * a.batch : 1;
    p.parts = static_cast<int>(groups * p.group);
    return p;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

template <typename T, int HD, int BITS, int NG>
const void* rows_fn(int rows) {
    if constexpr (BITS != 16) {
        if (rows == 16) return reinterpret_cast<const void*>(&attn_rows_kernel<T, HD, BITS, NG, 2>);
    }
    return reinterpret_cast<const void*>(&attn_rows_kernel<T, HD, BITS, NG, 1>);
}
template <typename T, int HD, int BITS>
const void* rows_fn(int groups, int rows) {
    if constexpr (HD == 128) {
        if (groups == 4) return rows_fn<T, HD, BITS, 4>(rows);
    }
    return groups == 2 ? rows_fn<T, HD, BITS, 2>(rows) : rows_fn<T, HD, BITS, 1>(rows);
}
template <typename T, int HD>
const void* rows_fn(int bits, int groups, int rows) {
    return bits == 16 ? rows_fn<T, HD, 16, 1>(rows) : bits == 8 ? rows_fn<T, HD, 8>(groups, rows)
                                                                : rows_fn<T, HD, 4>(groups, rows);
}
template <typename T, int HD>
const void* combine_fn(int rows) {
    return rows == 8    ? reinterpret_cast<const void*>(&attn_combine_kernel<T, HD, 8>)
           : rows == 16 ? reinterpret_cast<const void*>(&attn_combine_kernel<T, HD, 16>)
                        : reinterpret_cast<const void*>(&attn_combine_kernel<T, HD, 128>);
}

}  // namespace

bool attn_rows_countable(const KvCache& c, const RowsArgs& a) {
    const Plan pl = plan_of(c, a);
    const long long r = static_cast<long long>(a.max_q) * (a.Hq / c.Hkv);
    const double units = static_cast<double>((r + pl.chunk - 1) / pl.chunk) * c.Hkv * a.batch *
                         (a.max_kv / pl.kt + 1);
    return units < 2147483647.0;
}

namespace {

// Sequences whose expanded rows are held at once: as many as 1 GiB takes, one at least.
int group_of(const KvCache& c, const RowsArgs& a, const Plan& pl) {
    if (!pl.tc || c.bits == 16) return a.batch;
    const size_t each = rows_tc_expand_bytes(c, a);
    const size_t n = each ? (size_t{1} << 30) / each : a.batch;
    return static_cast<int>(n < 1 ? 1 : n < static_cast<size_t>(a.batch) ? n : a.batch);
}

}  // namespace

size_t attn_rows_workspace(const KvCache& c, const RowsArgs& a) {
    const Plan pl = plan_of(c, a);
    const size_t rows = 2 * static_cast<size_t>(pl.parts) * pl.rows;
    size_t n = round256(rows * c.hd * sizeof(float)) + round256(rows * sizeof(float2)) +
               round256(pl.parts * sizeof(ra::Cut));
    if (pl.tc && c.bits != 16) n += group_of(c, a, pl) * (rows_tc_expand_bytes(c, a) + 1024);
    return n;
}

cudaError_t launch_attn_rows(const KvCache& c, const RowsArgs& all, void* workspace, bool overlap,
                             cudaStream_t st) {
    const Plan pl = plan_of(c, all);
    const size_t rows = 2 * static_cast<size_t>(pl.parts) * pl.rows;
    ra::Params p;
    p.a = all;
    p.c = c;
    p.scale_log2 = all.scale * 1.4426950408889634f;
    p.parts = pl.parts;
    p.group = pl.group;
    char* ws = static_cast<char*>(workspace);
    p.part_o = reinterpret_cast<float*>(ws);
    ws += round256(rows * c.hd * sizeof(float));
    p.part_ml = reinterpret_cast<float2*>(ws);
    ws += round256(rows * sizeof(float2));
    p.cut = reinterpret_cast<ra::Cut*>(ws);
    ws += round256(pl.parts * sizeof(ra::Cut));
    const bool bf = c.dtype == kBF16, big = c.hd == 128;
    const int type = (bf ? 0 : 1) * 2 + (big ? 0 : 1);
    const int size = pl.rows == 8 ? 0 : pl.rows == 16 ? 1 : 2;
    // sequences [b, b + n) at a time; the whole batch but for large expansions
    const int group = group_of(c, all, pl);
    for (int b = 0; b < all.batch; b += group) {
        const int n = all.batch - b < group ? all.batch - b : group;
        if (group < all.batch) {
            p.a.cu_q = all.cu_q + b;  // (tcgen05 calls have offsets: a row each is no such call)
            p.a.kv_lens = all.kv_lens + b;
            p.a.table = all.table + static_cast<size_t>(b) * all.max_blocks;
            p.a.batch = n;
            p.a.tail = all.tail && b + n == all.batch;
        }
        void* args[] = {&p};
        cudaError_t e;
        if (pl.tc) {
            e = launch_rows_tc(p, ws, overlap, st);
        } else {
            const int ng = c.hd / c.gs;  // 1, 2 or 4
            const void* f = bf ? (big ? rows_fn<__nv_bfloat16, 128>(c.bits, ng, pl.rows)
                                      : rows_fn<__nv_bfloat16, 64>(c.bits, ng, pl.rows))
                               : (big ? rows_fn<__half, 128>(c.bits, ng, pl.rows)
                                      : rows_fn<__half, 64>(c.bits, ng, pl.rows));
            static PerDevice cfg[72];
            e = launch_ex(f,
                          cfg[((type * 3 + (c.bits == 16 ? 0 : c.bits == 8 ? 1 : 2)) * 3 + ng / 2) * 2 + size],
                          dim3(pl.parts), dim3(ra::THREADS), 0, st, overlap, args);
        }
        if (e != cudaSuccess) return e;
        overlap = true;  // (from here on every launch waits for the one before)
        if (pl.parts == pl.group) continue;  // (one run of units: nothing is cut)
        const void* fc = bf ? (big ? combine_fn<__nv_bfloat16, 128>(pl.rows)
                                   : combine_fn<__nv_bfloat16, 64>(pl.rows))
                            : (big ? combine_fn<__half, 128>(pl.rows) : combine_fn<__half, 64>(pl.rows));
        static PerDevice cfgc[12];
        e = launch_ex(fc, cfgc[type * 3 + size], dim3(pl.parts - 1, pl.rows == 128 ? 16 : pl.rows / 2), dim3(256), 0,
                      st, true, args);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace mlxq
