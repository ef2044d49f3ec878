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
//
// 64 rows of 151936 logits: 14.5 us without rules (the bytes' rate), 24 with
// histories up to 6000 tokens, 32 biases, masks and the pick's first pass (the
// barriers between clearing, counting and the pass, which eight workgroups a CU
// overlap in part); the pick's second pass 4 us, a launch.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "rv12_device.h"
#include "rv12_internal.h"

namespace rv12 {

// the word of an id: bit 31 set once it is among the row's tokens, bits 20 .. 30 the
// place of its last bias entry plus one, below them how often it was generated
constexpr uint32_t kSeen = 0x80000000u, kCount = (1u << kAdjustCountBits) - 1u;
constexpr int kNoId = 0x7FFFFFFF;

// four floats at a 4-byte address (one 16-byte access all the same): rows of an odd
// vocabulary start anywhere
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

__global__ __launch_bounds__(kAdjustThreads) void k_adjust(AdjustParams p) {
    constexpr int U = 4;               // 16-byte loads of a thread in flight
    constexpr int TB = 8;              // tokens of a thread in flight
    constexpr int kStep = 4 * kAdjustThreads;
    extern __shared__ u32x4 lds[];     // the slice's words
    uint32_t* word = reinterpret_cast<uint32_t*>(lds);
    const int r = blockIdx.y, t = threadIdx.x, lane = t & 63;
    const int64_t n0 = (int64_t)blockIdx.x * p.slice;
    const int ns = (int)min((int64_t)p.slice, p.V - n0);
    const int L = p.tokens ? (int)min(max(p.length[r], 0), p.max_tokens) : 0;
    const int made = p.prompt ? max(p.prompt[r], 0) : 0;
    const bool any = L > 0 || p.n_bias > 0;
    const float* x = p.x + (int64_t)r * p.x_stride + n0;
    float* y = p.y + (int64_t)r * p.y_stride + n0;
    // (a slice starts at a multiple of 32 ids)
    const uint32_t* mask = p.mask ? p.mask + (int64_t)r * p.mask_stride + (n0 >> 5) : nullptr;
    const float* bias = p.bias + (int64_t)r * p.bias_stride;
    f32x4 v[U];
    uint32_t ok[U];
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kStep;
            if (i >= ns) break;
            if (i + 4 <= ns) {
                v[u] = *reinterpret_cast<const f32x4u*>(x + i);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[u][e] = i + e < ns ? x[i + e] : 0.0f;
            }
            // past the row's end no id is allowed
            ok[u] = (mask ? mask[i >> 5] >> (i & 31) : 0xFu) & (i + 4 <= ns ? 0xFu : (1u << (ns - i)) - 1u);
        }
    };
    load(4 * t);  // the slice's first logits are on their way while its tokens are counted
    if (any) {
        const int64_t* tok = p.tokens + (int64_t)r * p.tokens_stride;
        const int64_t* id = p.bias_ids + (int64_t)r * p.bias_stride;
        int64_t n[TB];
#pragma unroll
        for (int u = 0; u < TB; ++u) n[u] = L ? tok[min(t + u * kAdjustThreads, L - 1)] : 0;
        int64_t nb = t < p.n_bias ? id[t] : -1;
        for (int i = t; i < p.slice / 4; i += kAdjustThreads) lds[i] = u32x4{0, 0, 0, 0};
        __syncthreads();
        if (p.n_bias) {  // the biases first, while a word holds nothing else: the last entry of an id stays
            for (int i = t; i < p.n_bias; i += kAdjustThreads) {
                const int64_t k = nb - n0;
                if (k >= 0 && k < ns) atomicMax(&word[k], (uint32_t)(i + 1) << kAdjustCountBits);
                if (i + kAdjustThreads < p.n_bias) nb = id[i + kAdjustThreads];
            }
            __syncthreads();
        }
        for (int i0 = t; i0 < L; i0 += TB * kAdjustThreads) {
#pragma unroll
            for (int u = 0; u < TB; ++u) {
                const int i = i0 + u * kAdjustThreads;
                const int64_t k = n[u] - n0;
                if (i < L && k >= 0 && k < ns) {
                    atomicOr(&word[k], kSeen);
                    if (i >= made) atomicAdd(&word[k], 1u);
                }
            }
            if (i0 + TB * kAdjustThreads < L) {
#pragma unroll
                for (int u = 0; u < TB; ++u) n[u] = tok[min(i0 + (TB + u) * kAdjustThreads, L - 1)];
            }
        }
        __syncthreads();
    }
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (p.penalties) {
        rep = p.penalties[3 * r];
        freq = p.penalties[3 * r + 1];
        pres = p.penalties[3 * r + 2];
    }
    float bv = -INFINITY;
    int bi = kNoId;
    for (int i0 = 4 * t; i0 < ns; i0 += U * kStep) {
        if (i0 != 4 * t) load(i0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * kStep;
            if (i >= ns) break;
            u32x4 c = {0, 0, 0, 0};
            if (any) c = lds[i >> 2];
            if (c[0] | c[1] | c[2] | c[3]) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float f = v[u][e];
                    if (c[e] & kSeen) {
                        f = f > 0.0f ? f / rep : f * rep;
                        const uint32_t k = c[e] & kCount;
                        if (k) f -= freq * (float)k + pres;
                    }
                    const uint32_t b = (c[e] & ~kSeen) >> kAdjustCountBits;
                    if (b) f += bias[b - 1];
                    v[u][e] = f;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const bool may = ok[u] >> e & 1u;
                const float f = may ? v[u][e] : -INFINITY;
                v[u][e] = f;
                // (the thread's ids ascend: the first, a larger one, the first NaN)
                if (may && (bi == kNoId || (!(f <= bv) && bv == bv))) {
                    bv = f;
                    bi = (int)n0 + i + e;
                }
            }
            if (i + 4 <= ns) {
                *reinterpret_cast<f32x4u*>(y + i) = v[u];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e < ns) y[i + e] = v[u][e];
            }
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
    int bi = kNoId;
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
    if (lane == 0) ids[r] = bi == kNoId ? -1 : bi;
}

void launch_adjust(const AdjustParams& pa, int T, int64_t* ids, hipStream_t st) {
    AdjustParams p = pa;
    const int ns = (int)((p.V + p.slice - 1) / p.slice);
    hipLaunchKernelGGL(k_adjust, dim3((unsigned)ns, (unsigned)T), dim3(kAdjustThreads),
                       (size_t)p.slice * 4, st, p);
    if (ids) hipLaunchKernelGGL(k_adjust_pick, dim3((unsigned)T), dim3(64), 0, st, p.pv, p.pi, ns, ids);
}

}  // namespace rv12
