// Attention of query rows over a paged KV cache in 16, 8 or 4 bits (sm_100a): decode steps,
// prompt chunks and trees of drafted tokens.
//
// Reference (huydt84/mlx-server-runtime, python/mlx_worker/native_mlx/): append_and_attend
// (attention.py:215-298) over pages, with a causal or, for drafted trees, an ancestor mask.
//
//   s = scale * q . k over the visible keys, p = exp(s - m), out = sum p v / sum p
//
// Rows: sequence b has R = n * G query rows per kv head (its n new tokens times the G query
// heads that share the head). They are taken in chunks of ROWS; the chunk's keys in tiles
// of 64. The tiles of all (sequence, kv head, chunk) items form one sequence of units that
// the CTAs share out evenly, whatever the lengths: a CTA's share is a contiguous run that
// may end one item and begin another. A part of an item goes to a workspace slot of its
// CTA, and attn_combine_kernel joins the parts in order of keys.
//
// Keys are the M rows of the m16n8k16 products and query rows the N columns, so eight rows
// (a decode step's heads) fill a tile without padding:
//   S^T = K Q^T    A = 16 keys x 16 dims, straight from global memory: a lane's dims are
//                  contiguous in its key's row, and q is permuted to match once
//   O^T = V^T P^T  A = 16 dims x 16 keys, pairs of keys joined by byte permutes; P^T is S^T
//                  rounded to T and transposed in registers (movmatrix)
// so packed codes go from their load through registers into the product; shared memory
// holds only the four warps' results at the end of an item.
#include "common.cuh"
#include "kv_dequant.cuh"
#include "overlap.cuh"
#include "paged_ops.h"
#include "rows_units.cuh"
#include "sm100.cuh"

namespace mlxq {

namespace ra {
constexpr int WARPS = 4, THREADS = 32 * WARPS;
constexpr int KT = 16 * WARPS;  // keys per tile

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(r) : "r"(v));
    return r;
}

template <int N>
__device__ __forceinline__ void ldw(const void* at, uint32_t (&r)[N]) {
    if constexpr (N == 1) {
        r[0] = __ldg(static_cast<const uint32_t*>(at));
    } else if constexpr (N == 2) {
        const uint2 v = __ldg(static_cast<const uint2*>(at));
        r[0] = v.x;
        r[1] = v.y;
    } else {
#pragma unroll
        for (int i = 0; i < N / 4; ++i) {
            const uint4 v = __ldg(static_cast<const uint4*>(at) + i);
            r[4 * i] = v.x;
            r[4 * i + 1] = v.y;
            r[4 * i + 2] = v.z;
            r[4 * i + 3] = v.w;
        }
    }
}

// CTAs of an SM: what the registers of a variant allow (and the launch bounds ask for).
constexpr int resident(int hd, int bits, int nt) {
    return nt == 2 ? 2 : hd == 64 ? 4 : bits == 4 ? 4 : bits == 8 ? 3 : 2;
}

// A lane's part of 16 keys on its way: words of key rows r8 and r8 + 8 (a quarter of each),
// of value rows 2 c4, 2 c4 + 1 and eight on (an eighth of each); and of (key lane % 16,
// group lane / 16, and with four groups lane / 16 + 2) scale | bias << 16.
template <int HD, int BITS>
struct Raw {
    uint32_t k[2][HD / 4 * BITS / 32], v[4][HD / 8 * BITS / 32];
    uint32_t ks[2], vs[2];
};
}  // namespace ra

template <typename T, int HD, int BITS, int NT>
__global__ void __launch_bounds__(ra::THREADS, ra::resident(HD, BITS, NT))
    attn_rows_kernel(const __grid_constant__ ra::Params p) {
    using namespace ra;
    constexpr int ROWS = 8 * NT;
    constexpr int RB = HD * BITS / 8;  // bytes of a row
    constexpr int MT = HD / 16;
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
    const Units un = scan_units<KT>(a, Hkv, G, ROWS, p.group, pref);
    Walk<KT, ROWS> w;
    w.begin(a, Hkv, un, p.parts, p.group, pref);
    Cut mine = {};

    const int ng = BITS == 16 ? 1 : HD / c.gs;
    const int kg = BITS == 16 ? 0 : c4 * (HD / 4) / c.gs;  // this lane's group of a key row
    const int vg = BITS == 16 ? 0 : r8 * (HD / 8) / c.gs;  // and of a value row
    const uint32_t row_bytes = static_cast<uint32_t>(Hkv) * RB;  // of a token: its heads' rows

    for (; w.next(a); w.advance()) {
        const Seq& s = w.s;
        const int g = w.g, row_lo = w.rr0, t0 = w.t0, R = s.n * G;
        const int base = w.base(), kend = w.kend(a), full = min(max(base, 0), kend);
        const int32_t* bt = a.table + static_cast<size_t>(w.b) * a.max_blocks;

        // Queries: lane (row r8 of the n-tile, quarter c4) holds its quarter's dims in the
        // order the key words unpack to.
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
                    prmt(qw[da / 2], qw[db / 2], (da % 2 ? 0x32u : 0x10u) | (db % 2 ? 0x7600u : 0x5400u));
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int rc = row_lo + 8 * nt + 2 * c4 + e;
                qpos[nt][e] = rc < R ? rc / G : -1;
                vis[nt][e] = ~0ull;
                if (a.mask) vis[nt][e] = rc < R ? static_cast<unsigned long long>(a.mask[s.row0 + rc / G]) : 0ull;
            }
        }

        float o[NT][MT][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }

        // Sixteen keys per warp and step. Eight keys share a page: the two page ids of a
        // step are loaded a step before its rows, the rows a step before their use (16-bit
        // rows, which would not fit registers twice, K after S and V after P V).
        const int te = w.tile_end(a);
        auto pages = [&](int tile, int (&pid)[2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int key = tile * KT + warp * 16 + 8 * h;
                pid[h] = key < kend ? __ldg(bt + (key >> page_shift)) : -1;
            }
        };
        // rows of the pool the two eights begin at; which of them are there, a bit each
        auto rows = [&](int tile, const int (&pid)[2], uint32_t (&row)[2]) -> uint32_t {
            uint32_t ok = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const bool good = pid[h] >= 0 && pid[h] < c.pages;
                const uint32_t in = static_cast<uint32_t>(tile * KT + warp * 16 + 8 * h) & (c.page - 1);
                ok |= good ? 1u << h : 0u;
                row[h] = good ? (static_cast<uint32_t>(pid[h]) << page_shift) + in : 0u;  // (page 0: in bounds)
            }
            return ok;
        };
        auto load_k = [&](Raw<HD, BITS>& x, const uint32_t (&row)[2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
                ldw(static_cast<const char*>(c.k) + static_cast<size_t>(row[h] + r8) * row_bytes + g * RB +
                        c4 * (RB / 4),
                    x.k[h]);
        };
        auto load_v = [&](Raw<HD, BITS>& x, const uint32_t (&row)[2]) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const char* at = static_cast<const char*>(c.v) +
                                 static_cast<size_t>(row[h] + 2 * c4) * row_bytes + g * RB + r8 * (RB / 8);
                ldw(at, x.v[2 * h]);
                ldw(at + row_bytes, x.v[2 * h + 1]);
            }
            if constexpr (BITS != 16) {
                const size_t token = row[lane >> 3 & 1] + (lane & 7);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (i == 1 && ng < 4) break;
                    const size_t at = (token * Hkv + g) * ng + min(lane >> 4, ng - 1) + 2 * i;
                    x.ks[i] = __ldg(static_cast<const uint16_t*>(c.ks) + at) |
                              static_cast<uint32_t>(__ldg(static_cast<const uint16_t*>(c.kb) + at)) << 16;
                    x.vs[i] = __ldg(static_cast<const uint16_t*>(c.vs) + at) |
                              static_cast<uint32_t>(__ldg(static_cast<const uint16_t*>(c.vb) + at)) << 16;
                }
            }
        };
        // scale | bias of (key, this lane's group) from the lane that loaded it
        auto sb_of = [&](const uint32_t (&x)[2], int key, int group) -> uint32_t {
            const int from = key + 16 * (group & 1);
            uint32_t r = __shfl_sync(0xffffffffu, x[0], from);
            if (ng == 4) {
                const uint32_t hi = __shfl_sync(0xffffffffu, x[1], from);
                r = group & 2 ? hi : r;
            }
            return r;
        };

        auto tile_of = [&](int tile, Raw<HD, BITS>& x, uint32_t ok, auto after_s, auto after_pv) {
            const int k0 = tile * KT + warp * 16;
            const bool clean = k0 + 16 <= kend && ok == 3u;
            float sc[NT][4];
            {
                uint32_t s2[2] = {0u, 0u}, b2[2] = {0u, 0u};
                if constexpr (BITS != 16) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t sb = sb_of(x.ks, r8 + 8 * h, kg);
                        s2[h] = pk_splat(sb);
                        b2[h] = prmt(sb, 0u, 0x3232u);
                    }
                }
#pragma unroll
                for (int j = 0; j < MT; ++j) {
                    const uint32_t a0 = row_pair<T, BITS>(x.k[0], 2 * j, s2[0], b2[0]);
                    const uint32_t a1 = row_pair<T, BITS>(x.k[1], 2 * j, s2[1], b2[1]);
                    const uint32_t a2 = row_pair<T, BITS>(x.k[0], 2 * j + 1, s2[0], b2[0]);
                    const uint32_t a3 = row_pair<T, BITS>(x.k[1], 2 * j + 1, s2[1], b2[1]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        if (j == 0) mma16816z<T>(sc[nt], a0, a1, a2, a3, bq[nt][j][0], bq[nt][j][1]);
                        else mma16816<T>(sc[nt], a0, a1, a2, a3, bq[nt][j][0], bq[nt][j][1]);
                    }
                }
            }
            after_s();
            const bool plain = clean && k0 + 16 <= full;
            float grow = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float y = sc[nt][e] * p.scale_log2;
                    if (!plain) {
                        const int key = k0 + r8 + 8 * (e >> 1), j = key - base;
                        const bool see = key < kend && (ok >> (e >> 1) & 1u) &&
                                         (j < 0 || (a.mask ? j < 64 && (vis[nt][e & 1] >> (j & 63) & 1)
                                                           : j <= qpos[nt][e & 1]));
                        y = see ? y : -INFINITY;
                    }
                    sc[nt][e] = y;
                    grow = fmaxf(grow, y - m[nt][e & 1]);
                }
            // The reference of the exponentials follows the running maximum only when a
            // score passes it by 2^8: the probabilities then reach 256, the sums lose nothing.
            if (__any_sync(0xffffffffu, grow > 8.f)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mx = fmaxf(sc[nt][e], sc[nt][e + 2]);
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
            uint32_t pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float pr[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float mr = m[nt][e & 1];
                    pr[e] = ex2(sc[nt][e] - (mr == -INFINITY ? 0.f : mr));
                    l[nt][e & 1] += pr[e];
                }
                pb[nt][0] = transpose8x8(pk_round<T>(pr[0], pr[1]));
                pb[nt][1] = transpose8x8(pk_round<T>(pr[2], pr[3]));
            }
            uint32_t s2[2] = {0u, 0u}, b2[2] = {0u, 0u};  // of value rows 2 c4, 2 c4 + 1; eight on
            // values of keys that are not there multiply zeros: make them zeros
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t keep = 0xffffffffu;
                if (!clean) {
                    const int k = k0 + 8 * h + 2 * c4;
                    const bool there = ok >> h & 1u;
                    keep = (there && k < kend ? 0xffffu : 0u) | (there && k + 1 < kend ? 0xffff0000u : 0u);
                }
                if constexpr (BITS == 16) {
                    if (!clean) {
#pragma unroll
                        for (int i = 0; i < HD / 16; ++i) {
                            if (!(keep & 0xffffu)) x.v[2 * h][i] = 0u;
                            if (!(keep >> 16)) x.v[2 * h + 1][i] = 0u;
                        }
                    }
                } else {
                    const uint32_t e0 = sb_of(x.vs, 8 * h + 2 * c4, vg), e1 = sb_of(x.vs, 8 * h + 2 * c4 + 1, vg);
                    s2[h] = prmt(e0, e1, 0x5410u) & keep;
                    b2[h] = prmt(e0, e1, 0x7632u) & keep;
                }
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const uint32_t a0 = cross_pair<T, BITS>(x.v[0], x.v[1], i, s2[0], b2[0]);
                const uint32_t a1 = cross_pair<T, BITS>(x.v[0], x.v[1], MT + i, s2[0], b2[0]);
                const uint32_t a2 = cross_pair<T, BITS>(x.v[2], x.v[3], i, s2[1], b2[1]);
                const uint32_t a3 = cross_pair<T, BITS>(x.v[2], x.v[3], MT + i, s2[1], b2[1]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) mma16816<T>(o[nt][i], a0, a1, a2, a3, pb[nt][0], pb[nt][1]);
            }
            after_pv();
        };
        auto nothing = [] {};

        if (t0 < te) {
            int pid[2];
            uint32_t row[2];
            pages(t0, pid);
            uint32_t ok = rows(t0, pid, row);
            Raw<HD, BITS> x;
            load_k(x, row);
            load_v(x, row);
            pages(t0 + 1, pid);
            if constexpr (BITS == 16) {
                for (int tile = t0; tile < te; ++tile) {
                    uint32_t ok1 = 0;
                    tile_of(
                        tile, x, ok,
                        [&] {
                            ok1 = rows(tile + 1, pid, row);
                            if (tile + 1 < te) load_k(x, row);
                            pages(tile + 2, pid);
                        },
                        [&] {
                            if (tile + 1 < te) load_v(x, row);
                        });
                    ok = ok1;
                }
            } else {
                Raw<HD, BITS> y;
                for (int tile = t0; tile < te; tile += 2) {
                    const uint32_t ok1 = rows(tile + 1, pid, row);
                    if (tile + 1 < te) {
                        load_k(y, row);
                        load_v(y, row);
                    }
                    pages(tile + 2, pid);
                    tile_of(tile, x, ok, nothing, nothing);
                    if (tile + 1 >= te) break;
                    ok = rows(tile + 2, pid, row);
                    if (tile + 2 < te) {
                        load_k(x, row);
                        load_v(x, row);
                    }
                    pages(tile + 3, pid);
                    tile_of(tile + 1, y, ok1, nothing, nothing);
                }
            }
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

// Joins the parts of the items that several CTAs took: block (CTA that began one, eight
// rows), warp = row, lane = HD / 32 dimensions. Parts are taken in order of keys, eight
// loads ahead.
template <typename T, int HD, int ROWS>
__global__ void __launch_bounds__(256) attn_combine_kernel(const __grid_constant__ ra::Params p) {
    using namespace ra;
    constexpr int DPL = HD / 32, AHEAD = 8;
    pdl_launch_dependents();
    pdl_wait();
    const Cut c = p.cut[blockIdx.x];
    const RowsArgs& a = p.a;
    const int G = a.Hq / p.c.Hkv, lane = threadIdx.x & 31;
    const int r = blockIdx.y * 8 + (threadIdx.x >> 5);
    if (r >= c.rows) return;
    const int first = blockIdx.x;
    float M = -INFINITY, den = 0.f, acc[DPL];
#pragma unroll
    for (int e = 0; e < DPL; ++e) acc[e] = 0.f;
    for (int k0 = first; k0 <= c.last; k0 += AHEAD * c.step) {
        float2 ml[AHEAD];
        float v[AHEAD][DPL];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int k = min(k0 + i * c.step, c.last);
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
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            if (k0 + i * c.step > c.last) break;
            const float Mn = fmaxf(M, ml[i].x);
            const float co = M == -INFINITY ? 0.f : exp2f(M - Mn);
            const float cn = ml[i].x == -INFINITY ? 0.f : exp2f(ml[i].x - Mn);
            den = fmaf(cn, ml[i].y, den * co);
#pragma unroll
            for (int e = 0; e < DPL; ++e) acc[e] = fmaf(cn, v[i][e], acc[e] * co);
            M = Mn;
        }
    }
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

// How a call is run: eight rows to a chunk where a decode step's heads fit them, sixteen
// up to there, and from then on 128 of them as the M rows of tcgen05 products.
struct Plan {
    bool tc;
    int rows, kt, parts, group;
};
Plan plan_of(const KvCache& c, const RowsArgs& a) {
    const long long r = static_cast<long long>(a.max_q) * (a.Hq / c.Hkv);
    Plan p;
    p.tc = r > 16;
    p.rows = p.tc ? 128 : r > 8 ? 16 : 8;
    p.kt = p.tc ? kRowsTcKeys : ra::KT;
    // CTAs the units are shared out to: what the GPU holds at once, at most one per unit
    const long long most = 148LL * (p.tc ? 2 : ra::resident(c.hd, c.bits, p.rows / 8));
    const long long tiles = (a.max_kv + p.kt - 1) / p.kt;
    long long units = (r + p.rows - 1) / p.rows * (tiles > 0 ? tiles : 1) * c.Hkv;
    units = units < most ? units * a.batch : most;
    p.parts = static_cast<int>(units < 1 ? 1 : units < most ? units : most);
    // up to eight chunks go side by side
    const int chunks = static_cast<int>((r + p.rows - 1) / p.rows);
    p.group = p.tc && chunks >= 2 && chunks <= 8 ? chunks : 1;
    if (p.group > 1) p.parts = (p.parts + p.group - 1) / p.group * p.group > most
                                   ? static_cast<int>(most / p.group * p.group)
                                   : (p.parts + p.group - 1) / p.group * p.group;
    return p;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

template <typename T, int HD, int BITS>
const void* rows_fn(int rows) {
    return rows == 8 ? reinterpret_cast<const void*>(&attn_rows_kernel<T, HD, BITS, 1>)
                     : reinterpret_cast<const void*>(&attn_rows_kernel<T, HD, BITS, 2>);
}
template <typename T, int HD>
const void* rows_fn(int bits, int rows) {
    return bits == 16 ? rows_fn<T, HD, 16>(rows) : bits == 8 ? rows_fn<T, HD, 8>(rows)
                                                             : rows_fn<T, HD, 4>(rows);
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
    const double units = static_cast<double>((r + pl.rows - 1) / pl.rows) * c.Hkv * a.batch *
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
            const void* f = bf ? (big ? rows_fn<__nv_bfloat16, 128>(c.bits, pl.rows)
                                      : rows_fn<__nv_bfloat16, 64>(c.bits, pl.rows))
                               : (big ? rows_fn<__half, 128>(c.bits, pl.rows)
                                      : rows_fn<__half, 64>(c.bits, pl.rows));
            static PerDevice cfg[24];
            e = launch_ex(f, cfg[(type * 3 + (c.bits == 16 ? 0 : c.bits == 8 ? 1 : 2)) * 2 + size],
                          dim3(pl.parts), dim3(ra::THREADS), 0, st, overlap, args);
        }
        if (e != cudaSuccess) return e;
        overlap = true;  // (from here on every launch waits for the one before)
        if (pl.parts == 1) continue;
        const void* fc = bf ? (big ? combine_fn<__nv_bfloat16, 128>(pl.rows)
                                   : combine_fn<__nv_bfloat16, 64>(pl.rows))
                            : (big ? combine_fn<__half, 128>(pl.rows) : combine_fn<__half, 64>(pl.rows));
        static PerDevice cfgc[12];
        e = launch_ex(fc, cfgc[type * 3 + size], dim3(pl.parts - 1, pl.rows / 8), dim3(256), 0,
                      st, true, args);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace mlxq
