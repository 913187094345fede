// Causal attention of packed prompts in 32-bit arithmetic: every type, head dims up to 256.
//
//   out_t = sum_{s <= t} p_ts v_s / l_t,  p_ts = exp(scale q_t . k_s - m_t),
//   l_t = sum_s p_ts [+ exp(sink - m_t)],  lse_t = m_t + ln l_t
// with the running maximum m and sum l of an online softmax over tiles of 64 keys.  A block of 256
// threads takes 64 queries of one (prompt, head); thread (i, j) of a 16 x 16 grid holds scores of rows
// 4 i .. 4 i + 3 and keys j, j + 16, j + 32, j + 48, and output columns j * 4 + 64 c.  The bound is the
// 32-bit FMA rate: each pair of operands read from shared memory feeds 16 products.
#include "gkv_device.cuh"
#include "kernels.h"
#include "prompt_tiles.cuh"
#include "../../include/glacier_kv.h"

namespace gkv {

namespace {

constexpr int kM = 64, kN = 64, kThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float4 load4(const float* p) { return *reinterpret_cast<const float4*>(p); }
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

// D: head dims padded to a multiple of 64 (the padding is zero in shared memory).
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) prompt_simt_kernel(const PromptArgs a) {
    constexpr int LD = D + 4;  // row stride in floats: 16-byte aligned, rows 4 banks apart
    constexpr int C = D / 64;  // output column groups of 4 per thread
    extern __shared__ __align__(16) float sm[];
    float* sQ = sm;
    float* sK = sQ + kM * LD;
    float* sV = sK + kN * LD;
    float* sP = sV + kN * LD;  // [kM][kN + 4]
    constexpr int LP = kN + 4;
    const int x = blockIdx.x / a.n_heads, head = blockIdx.x - x * a.n_heads;
    if (blockIdx.x == 0) check_prompts(a, threadIdx.x, kThreads);
    PromptTile pt;
    if (!find_prompt_tile<kM>(a, static_cast<int>(gridDim.x / a.n_heads) - 1 - x, pt)) return;
    const int hkv = head / (a.n_heads / a.heads_kv);
    const int q0 = pt.tile * kM, nq = min(kM, pt.len - q0);
    const T* Q = static_cast<const T*>(a.q) + (pt.row0 + q0) * a.q_ts + head * a.q_hs;
    const T* K = static_cast<const T*>(a.k) + pt.row0 * a.k_ts + hkv * a.k_hs;
    const T* V = static_cast<const T*>(a.v) + pt.row0 * a.v_ts + hkv * a.v_hs;
    auto fill = [&](float* to, const T* from, int64_t ts, int rows, int dim) {
        for (int i = threadIdx.x; i < 64 * (D / 4); i += kThreads) {
            const int r = i / (D / 4), e = (i - r * (D / 4)) * 4;
            *reinterpret_cast<float4*>(to + r * LD + e) = r < rows && e < dim ? load4(from + r * ts + e) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    fill(sQ, Q, a.q_ts, nq, a.d);
    const int ti = threadIdx.x >> 4, tj = threadIdx.x & 15;
    const float sl = a.scale * kLog2e;
    float m[4], l[4], o[4][C][4];
    const float sink = a.sinks ? __ldg(a.sinks + head) * kLog2e : -INFINITY;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        m[r] = -INFINITY;
        l[r] = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[r][c][e] = 0.f;
    }
    const int n_keys = q0 + nq;
    for (int k0 = 0; k0 < n_keys; k0 += kN) {
        const int nk = min(kN, n_keys - k0);
        __syncthreads();  // the last tile's reads are done
        fill(sK, K + k0 * a.k_ts, a.k_ts, nk, a.d);
        fill(sV, V + k0 * a.v_ts, a.v_ts, nk, a.dv);
        __syncthreads();
        float s[4][4] = {};
#pragma unroll 4
        for (int e = 0; e < D; e += 4) {
            float4 kv[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) kv[c] = *reinterpret_cast<const float4*>(sK + (tj + 16 * c) * LD + e);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float4 qv = *reinterpret_cast<const float4*>(sQ + (ti * 4 + r) * LD + e);
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    s[r][c] = fmaf(qv.x, kv[c].x, fmaf(qv.y, kv[c].y, fmaf(qv.z, kv[c].z, fmaf(qv.w, kv[c].w, s[r][c]))));
            }
        }
        const bool masked = k0 + kN > q0;  // the tile reaches past some row's own position, or past the prompt
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = q0 + ti * 4 + r;
            float mx = m[r];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[r][c] = k0 + tj + 16 * c <= row && tj + 16 * c < nk ? s[r][c] * sl : -INFINITY;
                mx = fmaxf(mx, s[r][c]);
            }
#pragma unroll
            for (int off = 8; off >= 1; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, off));
            const float base = mx == -INFINITY ? 0.f : mx;
            const float alpha = fast_exp2(m[r] - base);
            m[r] = mx;
            float sum = 0.f;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float p = fast_exp2(s[r][c] - base);
                sP[(ti * 4 + r) * LP + tj + 16 * c] = p;
                sum += p;
            }
            l[r] = l[r] * alpha + sum;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[r][c][e] *= alpha;
        }
        __syncwarp();  // a row's p are written and read by the same 16 lanes
        if (!masked) {
#pragma unroll 4
            for (int n = 0; n < kN; ++n) {
                float4 vv[C];
#pragma unroll
                for (int c = 0; c < C; ++c) vv[c] = *reinterpret_cast<const float4*>(sV + n * LD + tj * 4 + 64 * c);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float p = sP[(ti * 4 + r) * LP + n];
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        o[r][c][0] = fmaf(p, vv[c].x, o[r][c][0]);
                        o[r][c][1] = fmaf(p, vv[c].y, o[r][c][1]);
                        o[r][c][2] = fmaf(p, vv[c].z, o[r][c][2]);
                        o[r][c][3] = fmaf(p, vv[c].w, o[r][c][3]);
                    }
                }
            }
        } else {
            // a masked value must not reach the row even where it is not finite: 0 * inf is not 0
            for (int n = 0; n < nk; ++n) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (k0 + n > q0 + ti * 4 + r) continue;
                    const float p = sP[(ti * 4 + r) * LP + n];
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        const float4 v = *reinterpret_cast<const float4*>(sV + n * LD + tj * 4 + 64 * c);
                        o[r][c][0] = fmaf(p, v.x, o[r][c][0]);
                        o[r][c][1] = fmaf(p, v.y, o[r][c][1]);
                        o[r][c][2] = fmaf(p, v.z, o[r][c][2]);
                        o[r][c][3] = fmaf(p, v.w, o[r][c][3]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float sum = l[r];
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) sum += __shfl_xor_sync(~0u, sum, off);
        // the sink joins the denominator against the larger of the two maxima
        const float top = fmaxf(m[r], sink);
        const float base = top == -INFINITY ? 0.f : top;
        const float alpha = fast_exp2(m[r] - base);
        const float total = sum * alpha + fast_exp2(sink - base);
        const float inv = alpha / total;
        const int row = ti * 4 + r;
        if (row >= nq) continue;
        const int64_t at = (pt.row0 + q0 + row) * a.n_heads + head;
        T* out = static_cast<T*>(a.out) + at * a.dv;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int e = tj * 4 + 64 * c;
            if (e < a.dv) store4(out + e, make_float4(o[r][c][0] * inv, o[r][c][1] * inv, o[r][c][2] * inv, o[r][c][3] * inv));
        }
        if (a.lse && tj == 0) a.lse[at] = (top + log2f(total)) * 0.6931471805599453f;
    }
}

template <typename T, int D>
cudaError_t launch_d(const PromptArgs& a, cudaStream_t st) {
    constexpr size_t smem = (3 * 64 * (D + 4) + 64 * 68) * sizeof(float);
    cudaError_t e = cudaFuncSetAttribute(prompt_simt_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    const int64_t grid = prompt_tile_bound(a, kM) * a.n_heads;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    prompt_simt_kernel<T, D><<<static_cast<unsigned>(grid), kThreads, smem, st>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_t(const PromptArgs& a, cudaStream_t st) {
    const int d = a.d > a.dv ? a.d : a.dv;
    if (d <= 64) return launch_d<T, 64>(a, st);
    if (d <= 128) return launch_d<T, 128>(a, st);
    if (d <= 192) return launch_d<T, 192>(a, st);
    return launch_d<T, 256>(a, st);
}

}  // namespace

cudaError_t launch_prompt_simt(const PromptArgs& a, cudaStream_t st) {
    if (a.batch <= 0 || a.total <= 0) return cudaSuccess;
    if (a.dtype == GKV_DTYPE_BF16) return launch_t<__nv_bfloat16>(a, st);
    if (a.dtype == GKV_DTYPE_F16) return launch_t<__half>(a, st);
    return launch_t<float>(a, st);
}

}  // namespace gkv
