// Rules on the logits of T rows before the pick, gfx950: repetition, frequency
// and presence penalties from each row's tokens so far, biases, a mask of the
// allowed ids, and optionally the greedy pick.
//
//   s(n)    id n is among the row's tokens; c(n): how often among the generated ones
//   l' = (s ? (l > 0 ? l / r : l r) : l) - (f c + p [c > 0]) + bias(n)
//   out = allowed(n) ? l' : -inf;  pick: the largest l' of the allowed ids
//
// A workgroup takes a slice of one row's vocabulary.  It counts the row's tokens
// that fall into the slice in LDS (integer adds and maxima: the order does not
// matter), then passes over the slice once.  The history is read again by every
// slice, 8 bytes a token from the L2, against 8 bytes per id from HBM.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "rv12_device.h"
#include "rv12_internal.h"

namespace rv12 {

// counts of a slice: bit 31 set once the id is among the row's tokens, below it
// the generated ones
constexpr uint32_t kSeen = 0x80000000u;

// VEC: the rows of x and y at 16-byte addresses, V a multiple of 4 (a slice is one)
template <bool VEC>
__global__ __launch_bounds__(kAdjustThreads) void k_adjust(AdjustParams p) {
    constexpr int W = VEC ? 4 : 1;  // ids of a thread at once
    constexpr int U = VEC ? 4 : 8;  // loads of a thread in flight
    extern __shared__ uint32_t cnt[];  // [slice], then the bias entries' places [slice]
    const int r = blockIdx.y, t = threadIdx.x, lane = t & 63;
    const int64_t n0 = (int64_t)blockIdx.x * p.slice;
    const int ns = (int)min((int64_t)p.slice, p.V - n0);
    int* bias_at = reinterpret_cast<int*>(cnt + p.slice);
    const int L = p.tokens ? (int)min(max(p.length[r], 0), p.max_tokens) : 0;
    const int made = p.prompt ? max(p.prompt[r], 0) : 0;
    const bool counts = L > 0, biased = p.n_bias > 0;
    if (counts || biased) {
        for (int i = t; i < ns; i += kAdjustThreads) {
            cnt[i] = 0;
            if (biased) bias_at[i] = 0;
        }
        __syncthreads();
        const int64_t* tok = p.tokens + (int64_t)r * p.tokens_stride;
#pragma unroll 8
        for (int i = t; i < L; i += kAdjustThreads) {
            const int64_t n = tok[i] - n0;
            if (n >= 0 && n < ns) {
                atomicOr(&cnt[n], kSeen);
                if (i >= made) atomicAdd(&cnt[n], 1u);
            }
        }
        const int64_t* id = p.bias_ids + (int64_t)r * p.bias_stride;
        for (int i = t; i < p.n_bias; i += kAdjustThreads) {
            const int64_t n = id[i] - n0;
            if (n >= 0 && n < ns) atomicMax(&bias_at[n], i + 1);  // the last entry of an id counts
        }
        __syncthreads();
    }
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (p.penalties) {
        rep = p.penalties[3 * r];
        freq = p.penalties[3 * r + 1];
        pres = p.penalties[3 * r + 2];
    }
    const float* x = p.x + (int64_t)r * p.x_stride + n0;
    float* y = p.y + (int64_t)r * p.y_stride + n0;
    // (a slice starts at a multiple of 32 ids)
    const uint32_t* mask = p.mask ? p.mask + (int64_t)r * p.mask_stride + (n0 >> 5) : nullptr;
    const float* bias = p.bias + (int64_t)r * p.bias_stride;
    float bv = -INFINITY;
    int bi = 0x7FFFFFFF;
    for (int i0 = t * W; i0 < ns; i0 += U * kAdjustThreads * W) {
        float v[U][W];
        uint32_t ok[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kAdjustThreads * W;
            ok[u] = 0;
            if (i >= ns) break;
            if constexpr (VEC) {
                const f32x4 q = *reinterpret_cast<const f32x4*>(x + i);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[u][e] = q[e];
            } else {
                v[u][0] = x[i];
            }
            ok[u] = mask ? mask[i >> 5] >> (i & 31) : 0xFu;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kAdjustThreads * W;
            if (i >= ns) break;
#pragma unroll
            for (int e = 0; e < W; ++e) {
                float f = v[u][e];
                if (counts) {
                    const uint32_t c = cnt[i + e];
                    if (c) {
                        f = f > 0.0f ? f / rep : f * rep;
                        const uint32_t k = c & ~kSeen;
                        if (k) f -= freq * (float)k + pres;
                    }
                }
                if (biased && bias_at[i + e]) f += bias[bias_at[i + e] - 1];
                const bool may = ok[u] >> e & 1u;
                f = may ? f : -INFINITY;
                v[u][e] = f;
                if (may && pick_beats(f, (int)n0 + i + e, bv, bi)) {
                    bv = f;
                    bi = (int)n0 + i + e;
                }
            }
            if constexpr (VEC) *reinterpret_cast<f32x4*>(y + i) = f32x4{v[u][0], v[u][1], v[u][2], v[u][3]};
            else y[i] = v[u][0];
        }
    }
    if (!p.pv) return;
    __shared__ float sv[kAdjustThreads / 64];
    __shared__ int si[kAdjustThreads / 64];
#pragma unroll
    for (int j = 1; j < 64; j <<= 1) {
        const float ov = __shfl_xor(bv, j);
        const int oi = __shfl_xor(bi, j);
        if (pick_beats(ov, oi, bv, bi)) {
            bv = ov;
            bi = oi;
        }
    }
    if (lane == 0) {
        sv[t >> 6] = bv;
        si[t >> 6] = bi;
    }
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < kAdjustThreads / 64; ++w)
            if (pick_beats(sv[w], si[w], bv, bi)) {
                bv = sv[w];
                bi = si[w];
            }
        p.pv[(int64_t)r * gridDim.x + blockIdx.x] = bv;
        p.pi[(int64_t)r * gridDim.x + blockIdx.x] = bi;
    }
}

// the pick over a row's slices; -1 where no id is allowed
__global__ __launch_bounds__(64) void k_adjust_pick(const float* pv, const int32_t* pi, int n, int64_t* ids) {
    const int r = blockIdx.x, lane = threadIdx.x;
    float bv = -INFINITY;
    int bi = 0x7FFFFFFF;
    for (int i = lane; i < n; i += 64) {
        const float v = pv[(int64_t)r * n + i];
        const int k = pi[(int64_t)r * n + i];
        if (pick_beats(v, k, bv, bi)) {
            bv = v;
            bi = k;
        }
    }
#pragma unroll
    for (int j = 1; j < 64; j <<= 1) {
        const float ov = __shfl_xor(bv, j);
        const int oi = __shfl_xor(bi, j);
        if (pick_beats(ov, oi, bv, bi)) {
            bv = ov;
            bi = oi;
        }
    }
    if (lane == 0) ids[r] = bi == 0x7FFFFFFF ? -1 : bi;
}

void launch_adjust(const AdjustParams& pa, int T, int64_t* ids, hipStream_t st) {
    AdjustParams p = pa;
    const int ns = (int)((p.V + p.slice - 1) / p.slice);
    const bool vec = p.V % 4 == 0 && (((uintptr_t)p.x | (uintptr_t)p.y) & 15u) == 0 &&
                     (T == 1 || (p.x_stride % 4 == 0 && p.y_stride % 4 == 0));
    const dim3 grid((unsigned)ns, (unsigned)T);
    const size_t lds = (size_t)p.slice * (p.n_bias ? 8 : 4);
    if (vec) hipLaunchKernelGGL((k_adjust<true>), grid, dim3(kAdjustThreads), lds, st, p);
    else hipLaunchKernelGGL((k_adjust<false>), grid, dim3(kAdjustThreads), lds, st, p);
    if (ids) hipLaunchKernelGGL(k_adjust_pick, dim3((unsigned)T), dim3(64), 0, st, p.pv, p.pi, ns, ids);
}

}  // namespace rv12
