// What writes and reads back a paged KV cache (sm_100a): RMSNorm of each query and key
// head, rotation, and the append of keys and values to their cache rows, 16-bit or
// quantised as they are written; and the read-back of cache rows.
//
// Reference (huydt84/mlx-server-runtime, python/mlx_worker/native_mlx/): the head norms
// of Qwen3-style attention (models/qwen3.py), mx.fast.rope, the append of
// cache.py:485-520; the quantised form follows quantize()'s rule per row.
#include <cmath>

#include "common.cuh"
#include "kv_dequant.cuh"
#include "overlap.cuh"
#include "paged_ops.h"
#include "quant_rule.cuh"

namespace mlxq {

namespace {

struct AppendArgs {
    const void* qkv;
    long long ld;
    void* q_out;
    const void* q_norm;
    const void* k_norm;
    float eps;
    const int32_t* positions;
    const int32_t* slots;
    int Hq, rounds;      // rounds: head groups of a warp's share
    KvCache c;
    double turns[64];    // rotation of pair i per position, in full turns
};

__device__ __forceinline__ uint2 ld8(const void* p) { return *reinterpret_cast<const uint2*>(p); }

// Minimum and maximum that are no number where one of the two is none (fminf and fmaxf
// return the other).
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

}  // namespace

// One warp takes `rounds` groups of 32 / LPH heads of a token; the LPH = HD / 8 lanes of a
// head hold four elements of its lower half and the four they rotate with, so that neither
// the rotation nor the loads cross lanes:
//   y = x * rsqrt(mean x^2 + eps) * w          (32-bit; no rounding before the last)
//   (y_i, y_{i+hd/2}) -> (y_i cos - y_{i+hd/2} sin, y_i sin + y_{i+hd/2} cos), rounded to T
// The angle is position * turns[i] reduced to one turn in 64 bits (at position 10^5 a
// 32-bit product is off by several 2^-8 rad, more than the rounding of the result), then
// 32-bit sine and cosine of the rest, one pair to a thread and through shared memory to the
// CTA's warps: worked out by every warp for itself, they were a third of the instructions,
// which is what bounds a prompt's append. In a quantised cache the row rounded to T is
// quantised by quantize()'s rule (see quant_group): a group's least and largest value by
// shuffles over its lanes, four codes per lane and half. A NaN in a group makes both of them
// one, an infinity the range, and so the group's scale: it then stands for NaN, as its row does
// in 16 bits, and not for a number that nothing computed.
template <typename T, int HD, int BITS>
__global__ void __launch_bounds__(128) norm_rope_append_kernel(const __grid_constant__ AppendArgs a) {
    constexpr int LPH = HD / 8, HPW = 32 / LPH, HALF = HD / 2;
    pdl_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int li = lane % LPH, e0 = 4 * li;
    const KvCache& c = a.c;
    __shared__ float4 cos4[HALF / 4], sin4[HALF / 4];
    const T* qn = static_cast<const T*>(a.q_norm);
    const T* kn = static_cast<const T*>(a.k_norm);
    pdl_wait();
    const int t = blockIdx.x;
    const int slot = a.slots[t];
    const bool keep = slot >= 0 && slot < c.pages * static_cast<long long>(c.page);
    const int heads = a.Hq + 2 * c.Hkv;
    // groups of heads in turn, so that the warps share the heads that are quantised
    const int stride = gridDim.y * (blockDim.x >> 5) * HPW;
    const int first = (blockIdx.y * (blockDim.x >> 5) + warp) * HPW + lane / LPH;
    const T* src = static_cast<const T*>(a.qkv) + t * a.ld;
    uint2 next[2] = {make_uint2(0u, 0u), make_uint2(0u, 0u)};
    auto fetch = [&](int h) {  // a head's elements, a round before they are used
        if (h < heads) {
            next[0] = ld8(src + static_cast<size_t>(h) * HD + e0);
            next[1] = ld8(src + static_cast<size_t>(h) * HD + HALF + e0);
        }
    };
    fetch(first);
    const double pos = static_cast<double>(a.positions[t]);
    for (int i = threadIdx.x; i < HALF; i += blockDim.x) {
        const double x = pos * a.turns[i];
        float sine, cosine;
        sincospif(2.0f * static_cast<float>(x - rint(x)), &sine, &cosine);
        reinterpret_cast<float*>(cos4)[i] = cosine;
        reinterpret_cast<float*>(sin4)[i] = sine;
    }
    __syncthreads();
    const float cs[4] = {cos4[li].x, cos4[li].y, cos4[li].z, cos4[li].w};
    const float sn[4] = {sin4[li].x, sin4[li].y, sin4[li].z, sin4[li].w};
    for (int r = 0; r < a.rounds; ++r) {
        const int h = first + r * stride;
        const bool live = h < heads;
        uint2 lo = next[0], hi = next[1];
        if (r + 1 < a.rounds) fetch(h + stride);
        float x[4] = {Elem<T>::lo(lo.x), Elem<T>::hi(lo.x), Elem<T>::lo(lo.y), Elem<T>::hi(lo.y)};
        float y[4] = {Elem<T>::lo(hi.x), Elem<T>::hi(hi.x), Elem<T>::lo(hi.y), Elem<T>::hi(hi.y)};
        const bool is_q = h < a.Hq, is_v = h >= a.Hq + c.Hkv;
        const T* w = is_q ? qn : is_v ? nullptr : kn;
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) ss = fmaf(x[j], x[j], fmaf(y[j], y[j], ss));
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        if (w) {
            const float rs = rsqrtf(ss / static_cast<float>(HD) + a.eps);
            const uint2 wl = ld8(w + e0), wh = ld8(w + HALF + e0);
            x[0] *= rs * Elem<T>::lo(wl.x); x[1] *= rs * Elem<T>::hi(wl.x);
            x[2] *= rs * Elem<T>::lo(wl.y); x[3] *= rs * Elem<T>::hi(wl.y);
            y[0] *= rs * Elem<T>::lo(wh.x); y[1] *= rs * Elem<T>::hi(wh.x);
            y[2] *= rs * Elem<T>::lo(wh.y); y[3] *= rs * Elem<T>::hi(wh.y);
        }
        if (!is_v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float u = x[j], v = y[j];
                x[j] = u * cs[j] - v * sn[j];
                y[j] = u * sn[j] + v * cs[j];
            }
            lo = make_uint2(pk_round<T>(x[0], x[1]), pk_round<T>(x[2], x[3]));
            hi = make_uint2(pk_round<T>(y[0], y[1]), pk_round<T>(y[2], y[3]));
        }
        if (is_q) {
            T* dst = static_cast<T*>(a.q_out) + (static_cast<size_t>(t) * a.Hq + h) * HD;
            *reinterpret_cast<uint2*>(dst + e0) = lo;
            *reinterpret_cast<uint2*>(dst + HALF + e0) = hi;
        }
        const int g = is_v ? h - a.Hq - c.Hkv : h - a.Hq;  // kv head
        const bool put = live && !is_q && keep;
        const size_t row = put ? static_cast<size_t>(slot) * c.Hkv + g : 0;
        if constexpr (BITS == 16) {
            if (put) {
                T* dst = static_cast<T*>(is_v ? c.v : c.k) + row * HD;
                *reinterpret_cast<uint2*>(dst + e0) = lo;
                *reinterpret_cast<uint2*>(dst + HALF + e0) = hi;
            }
        } else if (__any_sync(0xffffffffu, put)) {
            // (a warp of query heads is done: quantising them all the same took 117 us where
            // the 16-bit append of 8190 tokens takes 34.) Every lane takes part in the
            // shuffles; lanes of a query head store nothing.
            const float p[4] = {Elem<T>::lo(lo.x), Elem<T>::hi(lo.x), Elem<T>::lo(lo.y),
                                Elem<T>::hi(lo.y)};
            const float q[4] = {Elem<T>::lo(hi.x), Elem<T>::hi(hi.x), Elem<T>::lo(hi.y),
                                Elem<T>::hi(hi.y)};
            float mn[2] = {INFINITY, INFINITY}, mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mn[0] = min_nan(mn[0], p[j]); mx[0] = max_nan(mx[0], p[j]);
                mn[1] = min_nan(mn[1], q[j]); mx[1] = max_nan(mx[1], q[j]);
            }
            const bool whole = c.gs == HD;  // one group: both halves
            if (whole) {
                mn[0] = mn[1] = min_nan(mn[0], mn[1]);
                mx[0] = mx[1] = max_nan(mx[0], mx[1]);
            }
            const int seg = min(LPH, c.gs / 4);  // lanes of a group
            // even lanes go on with the lower half's group, odd lanes with the upper half's
            const int side = li & 1;
            float lo_s = min_nan(mn[side], __shfl_xor_sync(0xffffffffu, mn[side ^ 1], 1));
            float hi_s = max_nan(mx[side], __shfl_xor_sync(0xffffffffu, mx[side ^ 1], 1));
            for (int o = seg >> 1; o > 1; o >>= 1) {
                lo_s = min_nan(lo_s, __shfl_xor_sync(0xffffffffu, lo_s, o));
                hi_s = max_nan(hi_s, __shfl_xor_sync(0xffffffffu, hi_s, o));
            }
            constexpr float n_bins = static_cast<float>((1 << BITS) - 1);
            float sc[2], bi[2], rc[2];
            quant_group(lo_s, hi_s, __fmul_rn(__fsub_rn(hi_s, lo_s), 1.0f / n_bins), sc[0], bi[0]);
            rc[0] = __frcp_rn(sc[0]);
            sc[1] = __shfl_xor_sync(0xffffffffu, sc[0], 1);
            bi[1] = __shfl_xor_sync(0xffffffffu, bi[0], 1);
            rc[1] = __shfl_xor_sync(0xffffffffu, rc[0], 1);
            uint32_t code[2] = {0u, 0u};
#pragma unroll
            for (int s = 0; s < 2; ++s) {  // this half's: the lane's own, or its neighbour's
                const float scale = side == s ? sc[0] : sc[1], bias = side == s ? bi[0] : bi[1];
                const float r = side == s ? rc[0] : rc[1];
                const bool fast = fabsf(r) >= 0x1p-126f && fabsf(r) <= 0x1p126f;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    code[s] |= quant_code(__fsub_rn(s ? q[j] : p[j], bias), scale, r, n_bins, fast)
                               << (BITS * j);
            }
            uint32_t* words = static_cast<uint32_t*>(is_v ? c.v : c.k) + row * (HD * BITS / 32);
            if constexpr (BITS == 8) {
                if (put) {
                    words[li] = code[0];
                    words[HALF / 4 + li] = code[1];
                }
            } else {
                // a word holds two lanes' codes: even lanes join the lower half's, odd lanes
                // the upper half's
                const bool odd = li & 1;
                const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? code[0] : code[1], 1);
                const uint32_t word = odd ? (got | code[1] << 16) : (code[0] | got << 16);
                if (put) words[(odd ? HALF / 8 : 0) + li / 2] = word;
            }
            // the first two lanes of a group hold its halves' scales and biases
            if (put && (li & (seg - 1)) < 2 && !(whole && side)) {
                const size_t at = row * (HD / c.gs) + (side ? HALF + e0 - 4 : e0) / c.gs;
                static_cast<T*>(is_v ? c.vs : c.ks)[at] = Elem<T>::from_f(sc[0]);
                static_cast<T*>(is_v ? c.vb : c.kb)[at] = Elem<T>::from_f(bi[0]);
            }
        }
    }
}

namespace {

template <typename T>
const void* append_fn(int hd, int bits) {
    if (hd == 128)
        return bits == 16  ? reinterpret_cast<const void*>(&norm_rope_append_kernel<T, 128, 16>)
               : bits == 8 ? reinterpret_cast<const void*>(&norm_rope_append_kernel<T, 128, 8>)
                           : reinterpret_cast<const void*>(&norm_rope_append_kernel<T, 128, 4>);
    return bits == 16  ? reinterpret_cast<const void*>(&norm_rope_append_kernel<T, 64, 16>)
           : bits == 8 ? reinterpret_cast<const void*>(&norm_rope_append_kernel<T, 64, 8>)
                       : reinterpret_cast<const void*>(&norm_rope_append_kernel<T, 64, 4>);
}

int variant(const KvCache& c) {  // index of a kernel's instance by type, head size and bits
    return (c.dtype == kBF16 ? 0 : 6) + (c.hd == 128 ? 0 : 3) + (c.bits == 16 ? 0 : c.bits == 8 ? 1 : 2);
}

}  // namespace

cudaError_t launch_norm_rope_append(const KvCache& c, const void* qkv, long long ld, void* q_out,
                                    const void* q_norm, const void* k_norm, float eps,
                                    const int32_t* positions, const int32_t* slots, int tokens,
                                    int Hq, double base, bool overlap, cudaStream_t st) {
    AppendArgs a;
    a.qkv = qkv;
    a.ld = ld;
    a.q_out = q_out;
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.eps = eps;
    a.positions = positions;
    a.slots = slots;
    a.Hq = Hq;
    a.c = c;
    // turns of pair i: base^(-2i/hd) / 2 pi, each from the one before (64 products keep
    // 2^-46 of the value; at position 2^24 the angle is then off by less than 2^-21 rad)
    const double step = std::pow(base, -2.0 / c.hd);
    double turn = 0.15915494309189533577;
    for (int i = 0; i < 64; ++i) {
        a.turns[i] = i < c.hd / 2 ? turn : 0.0;
        turn *= step;
    }
    // A warp takes one group of heads while that leaves warps idle, more (sharing the
    // sines) once the tokens alone fill the GPU.
    const int groups = (Hq + 2 * c.Hkv + 256 / c.hd - 1) / (256 / c.hd);
    const int want = 148 * 16;
    int rounds = 1;
    while (rounds < 8 && static_cast<long long>(tokens) * groups / (2 * rounds) >= want) rounds *= 2;
    const int warps = (groups + rounds - 1) / rounds;
    a.rounds = (groups + warps - 1) / warps;  // (evened out)
    const int wpc = warps < 4 ? warps : 4;
    void* args[] = {&a};
    static PerDevice cfg[12];
    const void* f = c.dtype == kBF16 ? append_fn<__nv_bfloat16>(c.hd, c.bits)
                                     : append_fn<__half>(c.hd, c.bits);
    return launch_ex(f, cfg[variant(c)], dim3(tokens, (warps + wpc - 1) / wpc), dim3(32 * wpc), 0,
                     st, overlap, args);
}

// ------------------------------------------------------------------------------------
// Rows of the cache as values: thread = eight elements of one head of row slots[i], from
// the keys (blockIdx.y 0) or the values (1). Slots outside the pool give zeros.
template <typename T, int BITS>
__global__ void __launch_bounds__(256)
    cache_read_kernel(const KvCache c, const int32_t* slots, long long n8,
                      T* k_out, T* v_out) {
    pdl_launch_dependents();
    pdl_wait();
    const bool is_v = blockIdx.y != 0;
    const int cpr = c.Hkv * c.hd / 8;  // chunks of eight in a row
    const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= n8) return;
    const int ch = static_cast<int>(i % cpr);
    const int slot = slots[i / cpr];
    uint4 o = make_uint4(0u, 0u, 0u, 0u);
    if (slot >= 0 && slot < c.pages * static_cast<long long>(c.page)) {
        o = cache_chunk<T, BITS>(c, is_v, static_cast<size_t>(slot) * cpr + ch);
    }
    reinterpret_cast<uint4*>(is_v ? v_out : k_out)[i] = o;
}

cudaError_t launch_cache_read(const KvCache& c, const int32_t* slots, int n, void* k_out,
                              void* v_out, bool overlap, cudaStream_t st) {
    long long n8 = static_cast<long long>(n) * c.Hkv * c.hd / 8;
    KvCache cc = c;
    void* args[] = {&cc, &slots, &n8, &k_out, &v_out};
    const void* f;
    if (c.dtype == kBF16)
        f = c.bits == 16  ? reinterpret_cast<const void*>(&cache_read_kernel<__nv_bfloat16, 16>)
            : c.bits == 8 ? reinterpret_cast<const void*>(&cache_read_kernel<__nv_bfloat16, 8>)
                          : reinterpret_cast<const void*>(&cache_read_kernel<__nv_bfloat16, 4>);
    else
        f = c.bits == 16  ? reinterpret_cast<const void*>(&cache_read_kernel<__half, 16>)
            : c.bits == 8 ? reinterpret_cast<const void*>(&cache_read_kernel<__half, 8>)
                          : reinterpret_cast<const void*>(&cache_read_kernel<__half, 4>);
    static PerDevice cfg[12];
    return launch_ex(f, cfg[variant(c)], dim3(static_cast<unsigned>((n8 + 255) / 256), 2),
                     dim3(256), 0, st, overlap, args);
}

}  // namespace mlxq
