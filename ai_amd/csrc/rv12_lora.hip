// Low-rank adapters of many requests beside a shared projection, gfx950:
//   out[t] = y[t] + scale_a B_a (A_a x'[t]),  a = idx[t]
// with A [count][R][K] and B [count][N][R] in bf16 and x' as the shared linear
// has it (the RMSNorm or silu(g) u prologue).  Two passes: h = A x' in K splits,
// then out.  Both work on tiles of 16 consecutive rows and one adapter of the
// tile: slot s of a tile takes its s-th distinct adapter (in row order) and the
// rows that use it, so rows of one request share the adapter's weights and rows
// of 16 requests run side by side.
//
// Products run on the bf16 matrix cores with x' and h split into three bf16 parts
// (24 bits), sums in float32.  v_mfma_f32_16x16x32_bf16: A operand row l % 16, k
// slot 8 (l / 16) + 0..7 of lane l (the adapter's weights, 16 bytes a lane
// straight from memory), B operand column l % 16 (the token), result rows
// 4 (l / 16) + 0..3.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "rv12_device.h"
#include "rv12_internal.h"

namespace rv12 {

// the s-th distinct adapter of the tile's rows t0 .. t0 + 15; id -1: rows without
// an adapter.  False: the tile has fewer.  `mine`: the lane's row t0 + lane % 16
// uses it.
__device__ __forceinline__ bool tile_slot(const LoraParams& p, int t0, int s, int* id, bool* mine) {
    const int c = threadIdx.x & 15;
    int a = -2;  // past the last row
    if (t0 + c < p.T) {
        a = p.idx[t0 + c];
        if (a < 0 || a >= p.count) a = -1;
    }
    bool lead = a != -2;
    for (int j = 0; j < 15; ++j) lead = lead && !(j < c && __builtin_amdgcn_readlane(a, j) == a);
    uint64_t m = __ballot(lead) & 0xFFFFull;
    for (int j = 0; j < s && m; ++j) m &= m - 1;
    if (!m) return false;
    *id = __builtin_amdgcn_readlane(a, __builtin_ctzll(m));
    *mine = a == *id;
    return true;
}

// 1. h[split][t][j] = sum over the split's columns of A[j] x'[t] (before the
// RMSNorm's factor), ssq[split][t] = their sum of squares (scaled).  Four waves
// share the split's steps of 32 columns and join in LDS.
template <int RB>  // blocks of 16 ranks
__global__ __launch_bounds__(256) void k_lora_down(LoraParams p) {
    __shared__ f32x4 acc_lds[4][RB][64];
    __shared__ float ssq_lds[4][16];
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q4 = lane >> 4, c16 = lane & 15;
    const int sp = blockIdx.x, t0 = blockIdx.y * 16;
    for (int slot = blockIdx.z;; slot += gridDim.z) {
        int id;
        bool mine;
        if (!tile_slot(p, t0, slot, &id, &mine)) return;
        if (id < 0) continue;
        const int rank = p.ranks ? min(max(p.ranks[id], 0), p.R) : p.R;
        const int nb = (rank + 15) / 16;
        const int steps = p.K / 32;
        const int s0 = (int)((int64_t)sp * steps / p.S), s1 = (int)((int64_t)(sp + 1) * steps / p.S);
        const float* x = p.x + (int64_t)(t0 + c16) * (p.mode == 2 ? 2 * (int64_t)p.K : p.K) + 8 * q4;
        const uint16_t* A = p.A + (int64_t)id * p.R * p.K + 8 * q4;
        f32x4 acc[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b] = f32x4{0, 0, 0, 0};
        float ss = 0.0f;
        for (int s = s0 + wv; s < s1; s += 4) {
            float v[8];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                f32x4 g = {0, 0, 0, 0};
                if (mine) g = *reinterpret_cast<const f32x4*>(x + 32 * s + 4 * c);
                if (p.mode == 2) {
                    f32x4 u = {0, 0, 0, 0};
                    if (mine) u = *reinterpret_cast<const f32x4*>(x + p.K + 32 * s + 4 * c);
#pragma unroll
                    for (int e = 0; e < 4; ++e) g[e] = silu_mul(g[e], u[e]);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * c + e] = g[e];
            }
            if (p.lnw) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(p.lnw + 32 * s + 8 * q4);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float sv = v[e] * kSsqScale;
                    ss = fmaf(sv, sv, ss);
                    v[e] *= (e & 1) ? hi_f(w[e >> 1]) : lo_f(w[e >> 1]);
                }
            }
            u32x4 h, m, l;
            split3(v, h, m, l);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                if (b >= nb) break;
                const int j = min(16 * b + c16, p.R - 1);
                const u32x4 a = *reinterpret_cast<const u32x4*>(A + (int64_t)j * p.K + 32 * s);
                acc[b] = mfma(a, h, acc[b]);
                acc[b] = mfma(a, m, acc[b]);
                acc[b] = mfma(a, l, acc[b]);
            }
        }
        ss += __shfl_xor(ss, 16);
        ss += __shfl_xor(ss, 32);
#pragma unroll
        for (int b = 0; b < RB; ++b) acc_lds[wv][b][lane] = acc[b];
        if (q4 == 0) ssq_lds[wv][c16] = ss;
        __syncthreads();
        float* h = p.h + ((int64_t)sp * p.T + t0 + c16) * (16 * RB);
        for (int b = wv; b < nb; b += 4) {
            f32x4 v = acc_lds[0][b][lane];
            for (int w = 1; w < 4; ++w) v += acc_lds[w][b][lane];
            if (mine) *reinterpret_cast<f32x4*>(h + 16 * b + 4 * q4) = v;
        }
        if (wv == 0 && q4 == 0 && mine && p.lnw)
            p.ssq[(int64_t)sp * p.T + t0 + c16] = (ssq_lds[0][c16] + ssq_lds[1][c16]) + (ssq_lds[2][c16] + ssq_lds[3][c16]);
        __syncthreads();
    }
}

// 2. out[t][n] = y[t][n] + sum_j B[n][j] (factor h[t][j]), factor = scale times
// the RMSNorm's.  A wave has the tile's h in registers and takes blocks of 16
// output rows.
template <int RB, bool VEC>  // VEC: y and out rows at 16-byte addresses, N % 4 == 0
__global__ __launch_bounds__(256) void k_lora_up(LoraParams p) {
    constexpr int RS = (RB + 1) / 2;  // steps of 32 ranks
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q4 = lane >> 4, c16 = lane & 15;
    const int t0 = blockIdx.y * 16, t = t0 + c16;
    const int nb0 = blockIdx.x * p.nbw * 4 + wv;  // first block of 16 rows, every fourth from there
    const int nblk = (p.N + 15) / 16;
    if (nb0 >= nblk) return;
    for (int slot = blockIdx.z;; slot += gridDim.z) {
        int id;
        bool mine;
        if (!tile_slot(p, t0, slot, &id, &mine)) return;
        if (id < 0 && p.y == p.out) continue;
        const int rank = id < 0 ? 0 : (p.ranks ? min(max(p.ranks[id], 0), p.R) : p.R);
        u32x4 hp[RS][3];
        if (rank > 0) {
            float f = mine ? p.scale[id] : 0.0f;
            if (p.lnw) {
                float ss = 0.0f;
                for (int s = 0; s < p.S; ++s) ss += mine ? p.ssq[(int64_t)s * p.T + t] : 0.0f;
                f *= rms_scale(ss, p.K, p.eps);
            }
#pragma unroll
            for (int s = 0; s < RS; ++s) {
                float v[8];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    f32x4 a = {0, 0, 0, 0};
                    const int j = 32 * s + 8 * q4 + 4 * c;
                    if (mine && j < rank)
                        for (int k = 0; k < p.S; ++k)
                            a += *reinterpret_cast<const f32x4*>(p.h + ((int64_t)k * p.T + t) * (16 * RB) + j);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[4 * c + e] = j + e < rank ? a[e] * f : 0.0f;
                }
                split3(v, hp[s][0], hp[s][1], hp[s][2]);
            }
        }
        const uint16_t* B = p.B + (int64_t)max(id, 0) * p.N * p.R + 8 * q4;
        for (int i = 0; i < p.nbw; ++i) {
            const int nb = nb0 + 4 * i;
            if (nb >= nblk) break;
            f32x4 acc = {0, 0, 0, 0};
            const int n = min(16 * nb + c16, p.N - 1);
#pragma unroll
            for (int s = 0; s < RS; ++s) {
                if (32 * s >= rank) break;
                u32x4 b = {0, 0, 0, 0};
                if (32 * s + 8 * q4 < p.R) b = *reinterpret_cast<const u32x4*>(B + (int64_t)n * p.R + 32 * s);
#pragma unroll
                for (int c = 0; c < 3; ++c) acc = mfma(b, hp[s][c], acc);
            }
            if (!mine) continue;
            const int no = 16 * nb + 4 * q4;
            const float* y = p.y + (int64_t)t * p.y_stride + no;
            float* o = p.out + (int64_t)t * p.out_stride + no;
            if constexpr (VEC) {
                if (no < p.N) *reinterpret_cast<f32x4*>(o) = *reinterpret_cast<const f32x4*>(y) + acc;
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (no + e < p.N) o[e] = y[e] + acc[e];
            }
        }
    }
}

template <int RB>
static void launch_lora_t(const LoraParams& p, bool vec, hipStream_t st) {
    const unsigned tiles = (unsigned)((p.T + 15) / 16), nblk = (unsigned)((p.N + 15) / 16);
    hipLaunchKernelGGL((k_lora_down<RB>), dim3((unsigned)p.S, tiles, (unsigned)p.slots), dim3(256), 0, st, p);
    const dim3 g((nblk + 4 * p.nbw - 1) / (4 * p.nbw), tiles, (unsigned)p.slots);
    if (vec) hipLaunchKernelGGL((k_lora_up<RB, true>), g, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((k_lora_up<RB, false>), g, dim3(256), 0, st, p);
}

void launch_lora(const LoraParams& p, bool vec, hipStream_t st) {
    switch (lora_rank_blocks(p.R)) {
        case 1: launch_lora_t<1>(p, vec, st); break;
        case 2: launch_lora_t<2>(p, vec, st); break;
        case 4: launch_lora_t<4>(p, vec, st); break;
        default: launch_lora_t<8>(p, vec, st); break;
    }
}

}  // namespace rv12
