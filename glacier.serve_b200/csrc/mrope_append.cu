// Rotary positions with several axes, fused with the q/k/v prologue and the KV append.
//
// gkv_rope_append's steps (bias, per-head RMSNorm of q and k, rotation, Store) for tokens whose
// position has several axes, as image and video patches have: pair i of a head turns by
//   angle_i = position[axis(i)] * inv_freq[i],   (a, b) -> (a cos - b sin, b cos + a sin) * mscale.
// The angle is formed in 64 bits: exact for positions below 2^29 (29 + 24 bits of factors), above off by
// at most 2^-53 of itself, 2^-22 rad.  It is reduced by pi/2 there and only then rounded: at position
// 10^6 a product in 32 bits is off by up to 2^-5 rad.  Everything else is 32 bits, rounded once to each
// destination's type.
//
// Roofline: HBM for prompts, launch latency for single tokens.  A block takes up to 16 tokens (one
// where there are few), puts their cos and sin into shared memory once for all heads, and hands
// each group of head_dim / 16 lanes one head row: a lane holds 8 pairs, read as two vectors of 8
// elements (pairs (i, i + R/2)) or one of 16 (pairs (2i, 2i + 1)), so partners meet in a lane and
// the norm's sum crosses lanes only log2(head_dim / 16) times.
//
// Measured (28 q and 4 kv heads of 128, 16 bits): 64 tokens 3.9 us; 8192 tokens with biases 35.7 us =
// 4.7 TB/s, 72 % of the measured copy rate; 2049 tokens of 32 q and 8 kv heads with norms, 32 bits into an
// 8-bit arena, 21 us = 4.1 TB/s (513 blocks, one wave of 592).  What is left is latency: 47 % of the issue
// slots are used and the warps wait for their rows.  3 or 5 blocks an SM, rows prefetched into registers and
// rows staged in shared memory were all slower.
#include "gkv_device.cuh"
#include "kernels.h"
#include "rope_math.cuh"
#include "../../include/glacier_kv.h"

namespace gkv {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;    // tokens per block
constexpr int kPlaces = 148 * 4;  // blocks that the card holds at a time
// Blocks come in as few waves as kMaxTokens tokens each allow, and then take no more tokens than fill those: a
// block's cos and sin and the loads of its bias cost once a block.  (4 a block for 8192 tokens: 39.2 instead of 35.7 us.)
__host__ __device__ constexpr int block_waves(int n_tok) { return (n_tok - 1) / (kPlaces * kMaxTokens) + 1; }
__host__ __device__ constexpr int block_tokens(int n_tok) { return (n_tok - 1) / (kPlaces * block_waves(n_tok)) + 1; }

__device__ __forceinline__ float2 unpack(uint32_t w, __nv_bfloat16) {
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// 8 consecutive elements as floats, from a 16-byte boundary.  Plain loads, not the read-only path:
// q may be rewritten in place by the lane that read it.
__device__ __forceinline__ void load8(const float* p, float (&x)[8]) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    const uint4 w = *reinterpret_cast<const uint4*>(p);
    const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 f = unpack(q[e], T{});
        x[2 * e] = f.x;
        x[2 * e + 1] = f.y;
    }
}

// 8 consecutive elements, rounded to nearest even (fp8: times `inv`, the reciprocal of the head's
// scale, saturated).
__device__ __forceinline__ void store8(float* p, const float (&x)[8], float) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8], float) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ void store8(__half* p, const float (&x)[8], float) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack_f16x2(x[0], x[1]), pack_f16x2(x[2], x[3]), pack_f16x2(x[4], x[5]), pack_f16x2(x[6], x[7]));
}
__device__ __forceinline__ void store8(__nv_fp8_e4m3* p, const float (&x)[8], float inv) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)
        w[e] = __nv_cvt_float2_to_fp8x2(make_float2(x[2 * e] * inv, x[2 * e + 1] * inv), __NV_SATFINITE, __NV_E4M3);
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
}
__device__ __forceinline__ void store8_as(void* base, int dtype, int64_t at, const float (&x)[8]) {
    if (dtype == GKV_DTYPE_F32) store8(static_cast<float*>(base) + at, x, 1.f);
    else if (dtype == GKV_DTYPE_BF16) store8(static_cast<__nv_bfloat16*>(base) + at, x, 1.f);
    else store8(static_cast<__half*>(base) + at, x, 1.f);
}

// 8 floats of a bias or norm weight, from a 16-byte boundary.
__device__ __forceinline__ void weights8(const float* w, float (&x)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(w)), b = __ldg(reinterpret_cast<const float4*>(w) + 1);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// T: the type of q, k and v; KV: the arena's; NORM: q or k has a norm weight.  Bound by issued
// instructions as much as by memory: what does not depend on the token is computed once per head row.
template <typename T, typename KV, bool NORM>
__global__ void __launch_bounds__(kThreads, 4) mrope_append_kernel(const ArenaGeom g, const __grid_constant__ MropeParams a, int tokens) {
    pdl_launch_dependents();  // the decode that follows waits for this grid before reading q or the arena
    // (cos, sin) * mscale of each token's pairs: pair 8 l + 2 e + f at ((e * half / 8) + l) * 2 + f, so that the
    // lanes of a row read neighbouring 16 bytes.  (In the pairs' own order the lanes are 64 bytes apart and
    // four of them meet in a bank.)
    __shared__ __align__(16) float2 turn[kMaxTokens * kMropeMaxPairs];
    __shared__ int64_t k_row[kMaxTokens], v_row[kMaxTokens];            // each token's row of head 0 in the arenas, -1: not stored
    int n_tok = a.n_tok;
    if (a.dyn_tok) {  // the rows that are there decide, not those reserved
        n_tok = min(__ldg(a.dyn_tok), n_tok);
        tokens = block_tokens(n_tok);
    }
    if (static_cast<int64_t>(blockIdx.x) * tokens >= n_tok) return;
    const int t0 = blockIdx.x * tokens;
    const int nt = min(tokens, n_tok - t0);
    const int half = a.rope_dim / 2;
    // The tables are in the parameters, but are read as memory: 32 different addresses of the constant
    // bank are 32 reads one after the other.
    const float* inv_freq = a.inv_freq;
    const uint8_t* axis = a.axis;
    asm volatile("" : "+l"(inv_freq), "+l"(axis));
    for (int i = threadIdx.x; i < nt * half; i += kThreads) {
        const int t = i / half, j = i - t * half;
        const int pos = __ldg(a.positions + axis[j] * a.pos_stride + t0 + t);
        float s, c;
        rope_sincos_f64(static_cast<double>(pos) * static_cast<double>(inv_freq[j]), s, c);
        turn[t * half + ((j >> 1 & 3) * (half >> 3) + (j >> 3)) * 2 + (j & 1)] = make_float2(c * a.mscale, s * a.mscale);
    }
    if (threadIdx.x < nt) {
        const int64_t s = __ldg(a.slots + t0 + threadIdx.x);
        k_row[threadIdx.x] = v_row[threadIdx.x] = -1;
        if (s >= static_cast<int64_t>(g.total_blocks) * g.block_size) {
            atomicOr(a.err, kErrBadSlot);
        } else if (s >= 0) {
            const int64_t blk = s / g.block_size, off = s - blk * g.block_size;
            k_row[threadIdx.x] = blk * g.k_block_stride + a.layer * g.k_layer_stride + off * g.head_dim;
            v_row[threadIdx.x] = blk * g.v_block_stride + a.layer * g.v_layer_stride + off * g.v_head_dim;
        }
    }
    __syncthreads();

    const int d = g.head_dim, hk = g.heads_kv, lane = threadIdx.x & 31;
    const int tpr = d / 16;  // lanes of a head row: 2, 4, 8 or 16
    const int tpr_log2 = 31 - __clz(tpr);
    const int units = (a.n_heads + hk) * tpr;
    const bool neox = a.style == GKV_ROPE_NEOX;
    // A lane takes one place of one head, of one token after the other.  Whole warps run every pass: the
    // norm's sums cross lanes.
    for (int i = threadIdx.x; i - lane < units; i += kThreads) {
        const bool live = i < units;
        const int r = live ? i >> tpr_log2 : 0, u = live ? (i - (r << tpr_log2)) * 8 : 0;  // pairs u .. u + 7 of d / 2
        const bool is_q = r < a.n_heads;
        const int h = is_q ? r : r - a.n_heads;
        // NEOX: 8 first elements of pairs, then their 8 partners; the unrotated elements [R, d) pair
        // up as halves too.  Interleaved: 16 adjacent elements.  R is a multiple of 16, so a vector
        // lies on one side of it.
        const int ia = neox ? (u < half ? u : u + half) : 2 * u;
        const int ib = neox ? (u < half ? u + half : u + d / 2) : 2 * u + 8;
        const int64_t ts = is_q ? a.q_ts : a.k_ts;
        const T* src = (is_q ? static_cast<const T*>(a.q) + h * a.q_hs : static_cast<const T*>(a.k) + h * a.k_hs) + t0 * ts;
        const float* bias = is_q ? a.q_bias : a.k_bias;
        if (bias) bias += h * d;
        const float* norm = NORM ? (is_q ? a.q_norm : a.k_norm) : nullptr;
        void* out = is_q ? a.q_out : a.k_out;
        const int out_stride = (is_q ? a.n_heads : hk) * d;
        int64_t at = static_cast<int64_t>(t0) * out_stride + h * d;
        KV* k_dst = static_cast<KV*>(g.k) + h * g.k_head_stride;
        const float k_inv = !is_q && g.k_inv ? __ldg(g.k_inv + a.layer * hk + h) : 1.f;
        const float4* w4 = reinterpret_cast<const float4*>(turn) + (u >> 3);
#pragma unroll 1
        for (int t = 0; t < nt; ++t, src += ts, at += out_stride, w4 += half / 2) {
            float x[8], y[8];
            load8(src + ia, x);
            load8(src + ib, y);
            if (bias) {
                float w[8];
                weights8(bias + ia, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] += w[e];
                weights8(bias + ib, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) y[e] += w[e];
            }
            if constexpr (NORM) {
                float p = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) p = fmaf(x[e], x[e], fmaf(y[e], y[e], p));
                for (int o = tpr >> 1; o >= 1; o >>= 1) p += __shfl_xor_sync(~0u, p, o);
                if (norm) {
                    const float inv = 1.f / sqrtf(p / static_cast<float>(d) + a.eps);
                    float w[8];
                    weights8(norm + ia, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] *= inv * w[e];
                    weights8(norm + ib, w);
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] *= inv * w[e];
                }
            }
            if (!live) continue;
            if (u < half) {  // all 8 pairs, or none
                float c[8], s[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float4 w = w4[e * (half >> 3)];
                    c[2 * e] = w.x, s[2 * e] = w.y, c[2 * e + 1] = w.z, s[2 * e + 1] = w.w;
                }
                if (neox) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float p = x[e];
                        x[e] = p * c[e] - y[e] * s[e];
                        y[e] = y[e] * c[e] + p * s[e];
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e += 2) {
                        const int e0 = e / 2, e1 = 4 + e / 2;
                        const float p = x[e], q = y[e];
                        x[e] = p * c[e0] - x[e + 1] * s[e0];
                        x[e + 1] = x[e + 1] * c[e0] + p * s[e0];
                        y[e] = q * c[e1] - y[e + 1] * s[e1];
                        y[e + 1] = y[e + 1] * c[e1] + q * s[e1];
                    }
                }
            }
            if (out) {
                store8_as(out, a.out_dtype, at + ia, x);
                store8_as(out, a.out_dtype, at + ib, y);
            }
            if (!is_q && k_row[t] >= 0) {
                store8(k_dst + k_row[t] + ia, x, k_inv);
                store8(k_dst + k_row[t] + ib, y, k_inv);
            }
        }
    }
    // v: 8 elements per lane
    const int dv = g.v_head_dim, vpr = dv / 8, v_units = hk * vpr;
    for (int i = threadIdx.x; i < nt * v_units; i += kThreads) {
        const int t = i / v_units, r = i - t * v_units;
        const int h = r / vpr, e = (r - h * vpr) * 8;
        const int64_t tok = t0 + t;
        float x[8];
        load8(static_cast<const T*>(a.v) + tok * a.v_ts + h * a.v_hs + e, x);
        if (a.v_bias) {
            float w[8];
            weights8(a.v_bias + h * dv + e, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) x[k] += w[k];
        }
        if (a.v_out) store8_as(a.v_out, a.out_dtype, (tok * hk + h) * dv + e, x);
        if (v_row[t] >= 0)
            store8(static_cast<KV*>(g.v) + v_row[t] + h * g.v_head_stride + e, x, g.v_inv ? __ldg(g.v_inv + a.layer * hk + h) : 1.f);
    }
}

template <typename T, typename KV>
cudaError_t launch_typed(const ArenaGeom& g, const MropeParams& p, cudaStream_t st) {
    const int tokens = block_tokens(p.n_tok);
    unsigned blocks = static_cast<unsigned>((p.n_tok - 1) / tokens) + 1;
    if (p.dyn_tok) {  // enough for any smaller count
        const int64_t places = static_cast<int64_t>(kPlaces) * block_waves(p.n_tok);
        blocks = static_cast<unsigned>(p.n_tok < places ? p.n_tok : places);
    }
    if (p.q_norm || p.k_norm) mrope_append_kernel<T, KV, true><<<blocks, kThreads, 0, st>>>(g, p, tokens);
    else mrope_append_kernel<T, KV, false><<<blocks, kThreads, 0, st>>>(g, p, tokens);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_arena(const ArenaGeom& g, const MropeParams& p, cudaStream_t st) {
    if (g.dtype == GKV_DTYPE_BF16) return launch_typed<T, __nv_bfloat16>(g, p, st);
    if (g.dtype == GKV_DTYPE_F16) return launch_typed<T, __half>(g, p, st);
    if (g.dtype == GKV_DTYPE_FP8_E4M3) return launch_typed<T, __nv_fp8_e4m3>(g, p, st);
    return launch_typed<T, float>(g, p, st);
}

}  // namespace

cudaError_t launch_mrope_append(const ArenaGeom& g, const MropeParams& p, cudaStream_t st) {
    if (p.n_tok <= 0) return cudaSuccess;
    if (p.in_dtype == GKV_DTYPE_BF16) return launch_arena<__nv_bfloat16>(g, p, st);
    if (p.in_dtype == GKV_DTYPE_F16) return launch_arena<__half>(g, p, st);
    return launch_arena<float>(g, p, st);
}

}  // namespace gkv
