// Causal attention of packed prompts in 32-bit arithmetic: every type, head dims up to 256.
//
//   out_t = sum_{s <= t} p_ts v_s / l_t,  p_ts = exp(scale q_t . k_s - m_t),
//   l_t = sum_s p_ts [+ exp(sink - m_t)],  lse_t = m_t + ln l_t
// with the running maximum m and sum l of an online softmax over tiles of 64 keys.  A block of 256
// threads takes M = 128 queries of one (prompt, head) (64 where head dims above 128 leave no room):
// thread (i, j) of a 16 x 16 grid holds scores of rows R i .. R i + R - 1, R = M / 16, and keys j, j + 16,
// j + 32, j + 48, and output columns 4 j + 64 c.  The bound is the 32-bit FMA rate: per 4 dims (or 4 keys)
// R + 4 (R + D / 16) vector reads of shared memory feed 16 R (R D / 4) products, in pairs (one
// instruction, which leaves issue slots to the reads).  Scores keep two sums each, of even and odd dims.
// 32-bit keys and values are copied asynchronously: values while the scores are formed, the next keys
// while they are used.
//
// Measured (32 q and 8 kv heads of 128, 32 bits): 4 prompts of 4096 tokens 45 TFLOP/s, 60 % of the FMA rate of
// 74.5; 6 ragged prompts of 1 to 1500 tokens 0.71 ms = 36.4 TFLOP/s; bf16 with head dims of 96, 256 and 192/128, which
// the tensor-core kernel does not take, 30 to 37 TFLOP/s.  A key tile takes 13.5 us where its FMAs take
// 8.3: shared memory gives 128 bytes a cycle to the registers, which the values (4 FMA a float) just live on
// and the scores (8 / 3 FMA a float) do not, and one block of 8 warps an SM (184 KB) hides little of the softmax.
#include "gkv_device.cuh"
#include "kernels.h"
#include "prompt_tiles.cuh"
#include "../../include/glacier_kv.h"

namespace gkv {

namespace {

constexpr int kN = 64, kThreads = 256;
// Batches up to which every block sorts the prompts for itself, to take the tiles with the most keys first; the others
// go prompt by prompt.  Here every tile of every head does that, so the limit is lower than kListed.  Sorted against
// prompt by prompt, 28 heads and 4 heads, us: prompts of 1 to 2000 tokens (median 100) 64: 1723 / 1697 and 409 / 523,
// 128: 1917 / 1846 and 290 / 326, 512: 15657 / 12203 and 2252 / 1818; prompts of 16 tokens 64: 237 / 224 and 39 / 37,
// 512: 3302 / 1683 and 481 / 246.
constexpr int kSorted = 64;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xffff0000u));
}
__device__ __forceinline__ float4 load4(const __half* p) {
    const uint2 w = *reinterpret_cast<const uint2*>(p);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
}
__device__ __forceinline__ void store4(__half* p, float4 v) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack_f16x2(v.x, v.y), pack_f16x2(v.z, v.w));
}

__device__ __forceinline__ void copy_async(float* to, const float* from, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// Rows [0, ROWS) x D of shared memory from `rows` rows x dim of the tensor, the rest zero.  32-bit rows
// arrive behind copies_done(), the others at once.
template <int ROWS, int D, typename T>
__device__ __forceinline__ void fill(float* to, const T* from, int64_t ts, int rows, int dim) {
    for (int i = threadIdx.x; i < ROWS * (D / 4); i += kThreads) {
        const int r = i / (D / 4), e = (i - r * (D / 4)) * 4;
        const bool there = r < rows && e < dim;
        float* dst = to + r * (D + 4) + e;
        if constexpr (sizeof(T) == 4) copy_async(dst, there ? from + r * ts + e : from, there);
        else *reinterpret_cast<float4*>(dst) = there ? load4(from + r * ts + e) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
}

// D: head dims padded to a multiple of 64 (the padding is zero in shared memory).
template <typename T, int D, int R>
__global__ void __launch_bounds__(kThreads) prompt_simt_kernel(const PromptArgs a) {
    constexpr int M = 16 * R;
    constexpr int LD = D + 4;  // row stride in floats: 16-byte aligned, rows 4 banks apart
    constexpr int LP = kN + 4;
    constexpr int C = D / 64;  // output column groups of 4 per thread
    extern __shared__ __align__(16) float sm[];
    float* sQ = sm;
    float* sK = sQ + M * LD;
    float* sV = sK + kN * LD;
    float* sP = sV + kN * LD;  // [M][LP]
    const int x = blockIdx.x / a.n_heads, head = blockIdx.x - x * a.n_heads;
    if (blockIdx.x == 0) check_prompts(a, threadIdx.x, kThreads);
    PromptTile pt;
    if (a.batch <= kSorted) {
        PromptList& list = *reinterpret_cast<PromptList*>(sP + M * LP);
        count_prompt_tiles<M>(a, list, threadIdx.x, kThreads);
        __syncthreads();
        sort_prompts(a, list, threadIdx.x, kThreads);
        __syncthreads();
        if (x >= sum_prompt_levels(a, list)) return;  // every warp for itself, with the same result
        listed_prompt_tile(a, list, x, pt);
    } else if (!find_prompt_tile<M>(a, static_cast<int>(gridDim.x / a.n_heads) - 1 - x, pt)) {
        return;
    }
    const int hkv = head / (a.n_heads / a.heads_kv);
    const int q0 = pt.tile * M, nq = min(M, pt.len - q0);
    const T* Q = static_cast<const T*>(a.q) + (pt.row0 + q0) * a.q_ts + head * a.q_hs;
    const T* K = static_cast<const T*>(a.k) + pt.row0 * a.k_ts + hkv * a.k_hs;
    const T* V = static_cast<const T*>(a.v) + pt.row0 * a.v_ts + hkv * a.v_hs;
    const int ti = threadIdx.x >> 4, tj = threadIdx.x & 15;
    const float sl = a.scale * kLog2e;
    float m[R], l[R];
    float2 o[R][C][2];
    const float sink = a.sinks ? __ldg(a.sinks + head) * kLog2e : -INFINITY;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) o[r][c][0] = o[r][c][1] = make_float2(0.f, 0.f);
    }
    const int n_keys = q0 + nq;
    fill<M, D>(sQ, Q, a.q_ts, nq, a.d);
    fill<kN, D>(sK, K, a.k_ts, min(kN, n_keys), a.d);
#pragma unroll 1
    for (int k0 = 0; k0 < n_keys; k0 += kN) {
        const int nk = min(kN, n_keys - k0);
        copies_done();
        __syncthreads();  // the keys are there, and the last tile's values and weights have been used
        fill<kN, D>(sV, V + k0 * a.v_ts, a.v_ts, nk, a.dv);
        // keys of the tile that a row of this warp sees (a multiple of 2 R): the products with the others are left out
        const int seen = min(kN, q0 + ((ti & ~1) + 2) * R - k0);
        float2 s2[R][4];
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int c = 0; c < 4; ++c) s2[r][c] = make_float2(0.f, 0.f);
        if (seen > 0)
#pragma unroll 2
        for (int e = 0; e < D; e += 4) {
            float4 kv[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) kv[c] = *reinterpret_cast<const float4*>(sK + (tj + 16 * c) * LD + e);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float4 qv = *reinterpret_cast<const float4*>(sQ + (ti * R + r) * LD + e);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    s2[r][c] = __ffma2_rn(make_float2(qv.x, qv.y), make_float2(kv[c].x, kv[c].y), s2[r][c]);
                    s2[r][c] = __ffma2_rn(make_float2(qv.z, qv.w), make_float2(kv[c].z, kv[c].w), s2[r][c]);
                }
            }
        }
        const bool masked = k0 + kN > q0;  // the tile reaches past some row's own position, or past the prompt
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int row = q0 + ti * R + r;
            float s[4];
            float mx = m[r];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[c] = k0 + tj + 16 * c <= row && tj + 16 * c < nk ? (s2[r][c].x + s2[r][c].y) * sl : -INFINITY;
                mx = fmaxf(mx, s[c]);
            }
#pragma unroll
            for (int off = 8; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, off));
            const float base = mx == -INFINITY ? 0.f : mx;
            const float alpha = fast_exp2(m[r] - base);
            m[r] = mx;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float p = fast_exp2(s[c] - base);
                sP[(ti * R + r) * LP + tj + 16 * c] = p;
                sum += p;
            }
            l[r] = l[r] * alpha + sum;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                o[r][c][0] = __fmul2_rn(o[r][c][0], make_float2(alpha, alpha));
                o[r][c][1] = __fmul2_rn(o[r][c][1], make_float2(alpha, alpha));
            }
        }
        copies_done();
        __syncthreads();  // the values are there, and the keys have been used (weights are a warp's own)
        if (k0 + kN < n_keys) fill<kN, D>(sK, K + (k0 + kN) * a.k_ts, a.k_ts, min(kN, n_keys - k0 - kN), a.d);
        // Masked weights are 0, but a masked value must not reach the row even where it is not finite
        // (0 * inf is not 0): such a tile is looked over, and only with such a value in it goes key by key.
        bool finite = true;
        if (masked) {
            float acc = 0.f;
            for (int i = threadIdx.x; i < kN * (D / 4); i += kThreads) {
                const float4 v = *reinterpret_cast<const float4*>(sV + i / (D / 4) * LD + i % (D / 4) * 4);
                acc = fmaf(v.x, 0.f, fmaf(v.y, 0.f, fmaf(v.z, 0.f, fmaf(v.w, 0.f, acc))));
            }
            finite = !__syncthreads_or(acc != 0.f);  // NaN differs from everything
        }
        if (finite) {
#pragma unroll 1
            for (int n = 0; n < seen; n += 4) {
                float4 p[R];
#pragma unroll
                for (int r = 0; r < R; ++r) p[r] = *reinterpret_cast<const float4*>(sP + (ti * R + r) * LP + n);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float4 vv[C];
#pragma unroll
                    for (int c = 0; c < C; ++c) vv[c] = *reinterpret_cast<const float4*>(sV + (n + i) * LD + tj * 4 + 64 * c);
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const float pi = i == 0 ? p[r].x : i == 1 ? p[r].y : i == 2 ? p[r].z : p[r].w;
#pragma unroll
                        for (int c = 0; c < C; ++c) {
                            o[r][c][0] = __ffma2_rn(make_float2(pi, pi), make_float2(vv[c].x, vv[c].y), o[r][c][0]);
                            o[r][c][1] = __ffma2_rn(make_float2(pi, pi), make_float2(vv[c].z, vv[c].w), o[r][c][1]);
                        }
                    }
                }
            }
        } else {
#pragma unroll 1
            for (int n = 0; n < nk; ++n) {
                float4 vv[C];
#pragma unroll
                for (int c = 0; c < C; ++c) vv[c] = *reinterpret_cast<const float4*>(sV + n * LD + tj * 4 + 64 * c);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    if (k0 + n > q0 + ti * R + r) continue;
                    const float p = sP[(ti * R + r) * LP + n];
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        o[r][c][0] = __ffma2_rn(make_float2(p, p), make_float2(vv[c].x, vv[c].y), o[r][c][0]);
                        o[r][c][1] = __ffma2_rn(make_float2(p, p), make_float2(vv[c].z, vv[c].w), o[r][c][1]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float sum = l[r];
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) sum += __shfl_xor_sync(~0u, sum, off);
        // the sink joins the denominator against the larger of the two maxima
        const float top = fmaxf(m[r], sink);
        const float base = top == -INFINITY ? 0.f : top;
        const float alpha = fast_exp2(m[r] - base);
        const float total = sum * alpha + (sink == base ? 1.f : fast_exp2(sink - base));  // also where both are infinite
        const float inv = alpha / total;
        const int row = ti * R + r;
        if (row >= nq) continue;
        const int64_t at = (pt.row0 + q0 + row) * a.n_heads + head;
        T* out = static_cast<T*>(a.out) + at * a.dv;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e = tj * 4 + 64 * c;
            if (e < a.dv) store4(out + e, make_float4(o[r][c][0].x * inv, o[r][c][0].y * inv, o[r][c][1].x * inv, o[r][c][1].y * inv));
        }
        if (a.lse && tj == 0) a.lse[at] = (top + log2f(total)) * 0.6931471805599453f;
    }
}

template <typename T, int D, int R>
cudaError_t launch_d(const PromptArgs& a, cudaStream_t st) {
    constexpr size_t smem = ((16 * R + 2 * kN) * (D + 4) + 16 * R * (kN + 4)) * sizeof(float) + sizeof(PromptList);
    static_assert(smem <= 232448, "shared memory of a block");
    cudaError_t e = cudaFuncSetAttribute(prompt_simt_kernel<T, D, R>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    const int64_t grid = prompt_tile_bound(a, 16 * R) * a.n_heads;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    prompt_simt_kernel<T, D, R><<<static_cast<unsigned>(grid), kThreads, smem, st>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_t(const PromptArgs& a, cudaStream_t st) {
    const int d = a.d > a.dv ? a.d : a.dv;
    if (d <= 64) return launch_d<T, 64, 8>(a, st);
    if (d <= 128) return launch_d<T, 128, 8>(a, st);
    if (d <= 192) return launch_d<T, 192, 4>(a, st);
    return launch_d<T, 256, 4>(a, st);
}

}  // namespace

cudaError_t launch_prompt_simt(const PromptArgs& a, cudaStream_t st) {
    if (a.batch <= 0 || a.total <= 0) return cudaSuccess;
    if (a.dtype == GKV_DTYPE_BF16) return launch_t<__nv_bfloat16>(a, st);
    if (a.dtype == GKV_DTYPE_F16) return launch_t<__half>(a, st);
    return launch_t<float>(a, st);
}

}  // namespace gkv
