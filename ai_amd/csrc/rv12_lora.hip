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
//
// A prompt is bound by its bytes (rank 64, 2051 rows of 4096 beside 24576 outputs, y
// and out: 448 MB in 15 + 93 us, 4.2 TB/s; behind the gate, 2 x 12288 beside 4096, x:
// the 138 MB of the 1368 rows with an adapter in 45 us, 3.1 TB/s, then 28); a few rows
// by two launches of dependent round trips (4 + 5 us for one row, 7 + 7 for 16 of 13
// adapters).
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
    uint64_t left = __ballot(a != -2) & 0xFFFFull;
    for (; left; --s) {
        const int first = __builtin_amdgcn_readlane(a, __builtin_ctzll(left));
        if (s == 0) {
            *id = first;
            *mine = a == first;
            return true;
        }
        left &= ~__ballot(a == first);
    }
    return false;
}

// 1. h[split][t][j] = sum over the split's columns of A[j] x'[t] (before the
// RMSNorm's factor), ssq[split][t] = their sum of squares (scaled).  Four waves
// share the split's steps of 32 columns and join in LDS.  The splits spread the
// adapter's weights over the CUs (a CU reads them from HBM at some 20 GB/s: 16
// rows of 13 adapters, rank 32, 4096 columns, take 6.7 us in 8 splits of 4 waves,
// 17.5 in one of 16).
template <int RB, bool MODE2>  // blocks of 16 ranks; x' = silu(g) u
__global__ __launch_bounds__(256) void k_lora_down(LoraParams p) {
    constexpr int NW = 4;
    __shared__ f32x4 acc_lds[NW][RB][64];
    __shared__ float ssq_lds[NW][16];
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
        const float* x = p.x + (int64_t)(t0 + c16) * (MODE2 ? 2 : 1) * p.K + 8 * q4;
        const uint16_t* A = p.A + (int64_t)id * p.R * p.K + 8 * q4;
        f32x4 acc[RB];
#pragma unroll
        for (int b = 0; b < RB; ++b) acc[b] = f32x4{0, 0, 0, 0};
        float ss = 0.0f;
        // the loads of a step, one step ahead of its products
        f32x4 xg[2], xu[2];
        u32x4 w, av[RB];
        auto load = [&](int s) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                xg[c] = xu[c] = f32x4{0, 0, 0, 0};
                if (mine) xg[c] = *reinterpret_cast<const f32x4*>(x + 32 * s + 4 * c);
                if (mine && MODE2) xu[c] = *reinterpret_cast<const f32x4*>(x + p.K + 32 * s + 4 * c);
            }
            if (!MODE2 && p.lnw) w = *reinterpret_cast<const u32x4*>(p.lnw + 32 * s + 8 * q4);
#pragma unroll
            for (int b = 0; b < RB; ++b)
                if (b < nb) av[b] = *reinterpret_cast<const u32x4*>(A + (int64_t)min(16 * b + c16, p.R - 1) * p.K + 32 * s);
        };
        if (s0 + wv < s1) load(s0 + wv);
        for (int s = s0 + wv; s < s1; s += NW) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = xg[e >> 2][e & 3];
                if constexpr (MODE2) v[e] = silu_mul(v[e], xu[e >> 2][e & 3]);
            }
            if (!MODE2 && p.lnw) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float sv = v[e] * kSsqScale;
                    ss = fmaf(sv, sv, ss);
                    v[e] *= (e & 1) ? hi_f(w[e >> 1]) : lo_f(w[e >> 1]);
                }
            }
            u32x4 a[RB];
#pragma unroll
            for (int b = 0; b < RB; ++b) a[b] = av[b];
            if (s + NW < s1) load(s + NW);
            u32x4 h, m, l;
            split3(v, h, m, l);
#pragma unroll
            for (int b = 0; b < RB; ++b) {
                if (b >= nb) break;
                acc[b] = mfma(a[b], h, acc[b]);
                acc[b] = mfma(a[b], m, acc[b]);
                acc[b] = mfma(a[b], l, acc[b]);
            }
        }
        ss += __shfl_xor(ss, 16);
        ss += __shfl_xor(ss, 32);
        if (q4 == 0) ssq_lds[wv][c16] = ss;
#pragma unroll
        for (int b = 0; b < RB; ++b) acc_lds[wv][b][lane] = acc[b];
        __syncthreads();
        float* h = p.h + ((int64_t)sp * p.T + t0 + c16) * (16 * RB);
        for (int b = wv; b < nb; b += NW) {
            f32x4 v = acc_lds[0][b][lane];
#pragma unroll
            for (int w = 1; w < NW; ++w) v += acc_lds[w][b][lane];
            if (mine) *reinterpret_cast<f32x4*>(h + 16 * b + 4 * q4) = v;
        }
        if (wv == 0 && q4 == 0 && mine && !MODE2 && p.lnw) {
            float v = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) v += ssq_lds[w][c16];
            p.ssq[(int64_t)sp * p.T + t0 + c16] = v;
        }
        __syncthreads();
    }
}

// 2. out[t][n] = y[t][n] + sum_j B[n][j] (factor h[t][j]), factor = scale times
// the RMSNorm's.  The workgroup adds the splits' h (every thread one part of it, all
// loads at once) and leaves it in LDS as the products' operand; then a wave takes
// p.nbw consecutive blocks of 16 output rows, UB at a time, the weights and y of
// the next UB loaded ahead of the products and stores of these.  The products leave
// 4 rows of a token per lane; they go through LDS to whole token rows, so that y is
// read and out written in runs of 64 UB bytes.
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));  // at any float's address

template <int RB>
__global__ __launch_bounds__(256, RB == 8 ? 2 : 3) void k_lora_up(LoraParams p) {
    constexpr int RS = (RB + 1) / 2;  // steps of 32 ranks
    constexpr int UB = RB == 8 ? 2 : 4;
    constexpr int LR = 4 * UB, RI = 64 / LR;  // lanes of one token row, rows at once (UB times)
    constexpr int kRow = 16 * UB + 4;         // LDS floats of a token row
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q4 = lane >> 4, c16 = lane & 15;
    const int tr = lane / LR, cr = 4 * (lane % LR);  // the lane's first token row and its 4 outputs
    const int t0 = blockIdx.y * 16;
    const int nb0 = (blockIdx.x * 4 + wv) * p.nbw, nb1 = min(nb0 + p.nbw, (p.N + 15) / 16);
    constexpr int HE = 64 * RB;             // float4 parts of the tile's h
    constexpr int GR = HE < 256 ? 256 / HE : 1;  // thread groups that share the splits
    constexpr int PE = HE > 256 ? HE / 256 : 1;  // parts of a thread
    __shared__ f32x4 part[GR][HE];
    __shared__ u32x4 hl[RS][3][64];
    __shared__ float factor[16];
    __shared__ __align__(16) float sums[4][16 * kRow];
    for (int slot = blockIdx.z;; slot += gridDim.z) {
        int id;
        bool mine;
        if (!tile_slot(p, t0, slot, &id, &mine)) return;
        if (id < 0 && p.y == p.out) continue;
        const uint32_t rows = (uint32_t)__ballot(mine);  // bit of every token row
        const int rank = id < 0 ? 0 : (p.ranks ? min(max(p.ranks[id], 0), p.R) : p.R);
        const uint16_t* B = p.B + (int64_t)max(id, 0) * p.N * p.R + 8 * q4;
        u32x4 bv[UB][RS];
        f32x4 yv[UB];
        auto load = [&](int nb) {
            const int n1 = min(16 * nb1, p.N);
#pragma unroll
            for (int u = 0; u < UB; ++u) {
                const int n = min(16 * (nb + u) + c16, p.N - 1);
#pragma unroll
                for (int s = 0; s < RS; ++s) {
                    bv[u][s] = u32x4{0, 0, 0, 0};
                    if (nb + u < nb1 && 32 * s < rank && 32 * s + 8 * q4 < p.R)
                        bv[u][s] = *reinterpret_cast<const u32x4*>(B + (int64_t)n * p.R + 32 * s);
                }
            }
#pragma unroll
            for (int u = 0; u < UB; ++u) {
                const int t = u * RI + tr, no = 16 * nb + cr;
                const float* y = p.y + (int64_t)(t0 + t) * p.y_stride + no;
                if (rows >> t & 1u) {
                    if (no + 4 <= n1) {
                        yv[u] = *reinterpret_cast<const f32x4u*>(y);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) yv[u][e] = no + e < n1 ? y[e] : 0.0f;
                    }
                }
            }
        };
        load(nb0);
        if (rank > 0) {  // (the same for the whole workgroup)
            const int tid = threadIdx.x;
            {
                // the factor of row tid / 16: its 16 lanes take a split each
                const int r = min(t0 + (tid >> 4), p.T - 1), k = tid & 15;
                float ss = p.lnw && k < p.S ? p.ssq[(int64_t)k * p.T + r] : 0.0f;
                ss += dpp<kDppXor1>(ss);
                ss += dpp<kDppXor2>(ss);
                ss += dpp<kDppHalfMirror>(ss);
                ss += dpp<kDppMirror>(ss);
                if (k == 0) factor[tid >> 4] = p.scale[id] * (p.lnw ? rms_scale(ss, p.K, p.eps) : 1.0f);
            }
#pragma unroll
            for (int i = 0; i < PE; ++i) {
                const int e = tid % HE + 256 * i, r = e / (4 * RB), grp = tid / HE;
                // (rows past the last are clamped and what is another adapter's, or
                // past the rank, dropped below: no condition on the loads)
                const float* h = p.h + (int64_t)min(t0 + r, p.T - 1) * (16 * RB) + 4 * (e % (4 * RB));
                f32x4 a = {0, 0, 0, 0};
#pragma unroll 4
                for (int k = grp; k < p.S; k += GR) a += *reinterpret_cast<const f32x4*>(h + (int64_t)k * p.T * (16 * RB));
                part[grp][e] = a;
            }
            __syncthreads();
            for (int s = wv; s < RS; s += 4) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = 0.0f;
                if (32 * s + 8 * q4 < 16 * RB) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        f32x4 a = part[0][c16 * 4 * RB + 8 * s + 2 * q4 + c];
#pragma unroll
                        for (int i = 1; i < GR; ++i) a += part[i][c16 * 4 * RB + 8 * s + 2 * q4 + c];
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            v[4 * c + e] = mine && 32 * s + 8 * q4 + 4 * c + e < rank ? a[e] * factor[c16] : 0.0f;
                    }
                }
                u32x4 hi, mid, lo;
                split3(v, hi, mid, lo);
                hl[s][0][lane] = hi;
                hl[s][1][lane] = mid;
                hl[s][2][lane] = lo;
            }
            __syncthreads();
        }
        for (int nb = nb0; nb < nb1; nb += UB) {
            const int n1 = min(16 * nb1, p.N);
            float* tile = sums[wv];
            // (h's parts are read again for every UB blocks: 12 RS registers less, which
            // would spill at rank 64)
            asm volatile("" ::: "memory");
            u32x4 hp[RS][3];
#pragma unroll
            for (int s = 0; s < RS; ++s)
#pragma unroll
                for (int c = 0; c < 3; ++c) hp[s][c] = hl[s][c][lane];
#pragma unroll
            for (int u = 0; u < UB; ++u) {
                f32x4 acc = {0, 0, 0, 0};
#pragma unroll
                for (int s = 0; s < RS; ++s) {
                    if (32 * s >= rank) break;
#pragma unroll
                    for (int c = 0; c < 3; ++c) acc = mfma(bv[u][s], hp[s][c], acc);
                }
                *reinterpret_cast<f32x4*>(tile + c16 * kRow + 16 * u + 4 * q4) = acc;
            }
            f32x4 yo[UB];
#pragma unroll
            for (int u = 0; u < UB; ++u) yo[u] = yv[u];
            if (nb + UB < nb1) load(nb + UB);
            // (a wave's LDS accesses keep their order: its own rows are there)
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int u = 0; u < UB; ++u) {
                const int t = u * RI + tr, no = 16 * nb + cr;
                const f32x4 o = yo[u] + *reinterpret_cast<const f32x4*>(tile + t * kRow + cr);
                float* out = p.out + (int64_t)(t0 + t) * p.out_stride + no;
                if (rows >> t & 1u) {
                    if (no + 4 <= n1) {
                        *reinterpret_cast<f32x4u*>(out) = o;
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (no + e < n1) out[e] = o[e];
                    }
                }
            }
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
        }
    }
}

template <int RB>
static void launch_lora_t(const LoraParams& p, hipStream_t st) {
    const unsigned tiles = (unsigned)((p.T + 15) / 16), nblk = (unsigned)((p.N + 15) / 16);
    const dim3 d((unsigned)p.S, tiles, (unsigned)p.slots);
    if (p.mode == 2) hipLaunchKernelGGL((k_lora_down<RB, true>), d, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((k_lora_down<RB, false>), d, dim3(256), 0, st, p);
    const dim3 g((nblk + 4 * p.nbw - 1) / (4 * p.nbw), tiles, (unsigned)p.slots);
    hipLaunchKernelGGL((k_lora_up<RB>), g, dim3(256), 0, st, p);
}

void launch_lora(const LoraParams& p, hipStream_t st) {
    switch (lora_rank_blocks(p.R)) {
        case 1: launch_lora_t<1>(p, st); break;
        case 2: launch_lora_t<2>(p, st); break;
        case 4: launch_lora_t<4>(p, st); break;
        default: launch_lora_t<8>(p, st); break;
    }
}

}  // namespace rv12
