// Paged key-value cache, gfx950: the cache of many sequences in pages, the
// append of a pass's keys and values to it, and the attention that reads it.
//
// A pass has T token rows; row r is the token at position pos[r] of sequence
// seq[r] (seq NULL: sequence r).  Position j of sequence s lives in page
// table[s][j / page] at slot j % page; the caches are [n_pages][n_kv][page][HD],
// so the 16 positions of an aligned block of one kv head are contiguous (pages
// hold a power of two of positions, at least 16).  A row whose sequence or
// position is outside the table (padding) gives zeros and writes nothing; a
// page id outside [0, n_pages) is no page: an append to it writes nothing, its
// positions take no part in the attention.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "rv12_device.h"
#include "rv12_internal.h"

namespace rv12 {

// ---------------------------------------------------------------------------
// Append: q and k get their head RMSNorm and the rotate-half RoPE at the row's
// position, q goes to q_out as float32, k and v into the row's page slot,
// rounded once to the cache type.
//
// Bound by bytes (4 (H + 2 KV) HD read, 4 H HD + 2 KV HD EB written per row); at
// a few rows by its latency.  HD / 8 lanes hold a head, 4 consecutive dims of
// either rotation half each, so every access is 16 bytes (8 where bf16 is
// stored) and the norm's sum stays within 16 lanes.  A workgroup of 256 threads
// takes a share of one row's heads: the row's HD / 2 angles are computed once
// per workgroup, while the heads' loads are in flight.
//
// The angle pos inv[i] passes 2^24 turns' worth of float32 steps in a long
// context (its float32 product is off by 0.004 rad at position 120000), so it
// is formed and reduced to [-pi, pi] in 64 bits; sine and cosine of the reduced
// angle are float32.
template <int HD, bool BF16>
__global__ __launch_bounds__(256) void k_paged_append(PagedParams p) {
    constexpr int half = HD / 2, LPH = HD / 8;  // lanes per head
    __shared__ float2 cs[half];                 // (cos, sin) of the row's angles
    const int r = blockIdx.x, t = threadIdx.x;
    const int H = p.n_heads, KV = p.n_kv, NH = H + 2 * KV;
    const int slots = 256 / LPH;  // heads at once
    const int hl = t % LPH;       // the lane's dims: 4 hl .. + 3 of both halves
    const int64_t sq = p.seq ? (int64_t)p.seq[r] : r;
    const int64_t pos = p.pos[r];
    const bool live = sq >= 0 && sq < p.n_seq && pos >= 0 && pos < p.cap;
    const float* row = p.qkv + (int64_t)r * NH * HD;
    int h = blockIdx.y * slots + t / LPH;
    f32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
    if (h < NH) {
        a = *reinterpret_cast<const f32x4*>(row + (int64_t)h * HD + 4 * hl);
        b = *reinterpret_cast<const f32x4*>(row + (int64_t)h * HD + half + 4 * hl);
    }
    if (!live) {
        for (; h < H; h += slots * gridDim.y) {
            float* dst = p.qo + ((int64_t)r * H + h) * HD;
            *reinterpret_cast<f32x4*>(dst + 4 * hl) = f32x4{0, 0, 0, 0};
            *reinterpret_cast<f32x4*>(dst + half + 4 * hl) = f32x4{0, 0, 0, 0};
        }
        return;
    }
    const int64_t pid = p.table[sq * p.table_stride + (pos >> p.page_log)];
    if (t < half) {
        constexpr double two_pi_hi = 6.283185307179586232, two_pi_lo = 2.449293598294706414e-16;
        const double ang = (double)pos * (double)p.inv[t];
        const double n = rint(ang * 0.15915494309189535);
        const float red = (float)fma(-n, two_pi_lo, fma(-n, two_pi_hi, ang));
        float sn, c;
        sincosf(red, &sn, &c);
        cs[t] = float2{c, sn};
    }
    const bool paged = pid >= 0 && pid < p.n_pages;
    const int64_t slot = ((paged ? pid : 0) * KV << p.page_log) + (pos & ((1 << p.page_log) - 1));
    __syncthreads();
    for (; h < NH; h += slots * gridDim.y) {
        f32x4 o0 = a, o1 = b;
        if (h < H + KV) {
            const float* nw = h < H ? p.qn : p.kn;
            const f32x4 wa = *reinterpret_cast<const f32x4*>(nw + 4 * hl);
            const f32x4 wb = *reinterpret_cast<const f32x4*>(nw + half + 4 * hl);
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) s = fmaf(a[e], a[e], fmaf(b[e], b[e], s));
            s += dpp<kDppXor1>(s);
            s += dpp<kDppXor2>(s);
            s += dpp<kDppHalfMirror>(s);
            if constexpr (LPH == 16) s += dpp<kDppMirror>(s);
            const float rs = 1.0f / sqrtf(s / (float)HD + p.eps);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 c = cs[4 * hl + e];
                const float x = wa[e] * (a[e] * rs), y = wb[e] * (b[e] * rs);
                o0[e] = x * c.x - y * c.y;
                o1[e] = y * c.x + x * c.y;
            }
        }
        const int hn = h + slots * gridDim.y;
        if (hn < NH) {
            a = *reinterpret_cast<const f32x4*>(row + (int64_t)hn * HD + 4 * hl);
            b = *reinterpret_cast<const f32x4*>(row + (int64_t)hn * HD + half + 4 * hl);
        }
        if (h < H) {
            float* dst = p.qo + ((int64_t)r * H + h) * HD;
            *reinterpret_cast<f32x4*>(dst + 4 * hl) = o0;
            *reinterpret_cast<f32x4*>(dst + half + 4 * hl) = o1;
        } else if (paged) {
            const int g = h < H + KV ? h - H : h - H - KV;
            void* c = h < H + KV ? p.kc : p.vc;
            const int64_t off = (slot + ((int64_t)g << p.page_log)) * HD + 4 * hl;
            if constexpr (BF16) {
                uint16_t* dst = static_cast<uint16_t*>(c) + off;
                *reinterpret_cast<uint2*>(dst) =
                    uint2{bf16_bits(o0[0]) | bf16_bits(o0[1]) << 16, bf16_bits(o0[2]) | bf16_bits(o0[3]) << 16};
                *reinterpret_cast<uint2*>(dst + half) =
                    uint2{bf16_bits(o1[0]) | bf16_bits(o1[1]) << 16, bf16_bits(o1[2]) | bf16_bits(o1[3]) << 16};
            } else {
                float* dst = static_cast<float*>(c) + off;
                *reinterpret_cast<f32x4*>(dst) = o0;
                *reinterpret_cast<f32x4*>(dst + half) = o1;
            }
        }
    }
}

void launch_paged_append(const PagedParams& p, hipStream_t st) {
    // every head of a row at once while the rows are few
    const int slots = 256 / (p.head_dim / 8), nh = p.n_heads + 2 * p.n_kv;
    const dim3 grid((unsigned)p.T, (unsigned)((nh + slots - 1) / slots));
    if (p.head_dim == 128) {
        if (p.kv_bf16) hipLaunchKernelGGL((k_paged_append<128, true>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((k_paged_append<128, false>), grid, dim3(256), 0, st, p);
    } else {
        if (p.kv_bf16) hipLaunchKernelGGL((k_paged_append<64, true>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((k_paged_append<64, false>), grid, dim3(256), 0, st, p);
    }
}

// ---------------------------------------------------------------------------
// Attention of the T rows over their sequences' pages: row r attends over
// positions 0 .. pos[r] of its sequence, softmax(q . K scale) V per head.
//
// A workgroup takes 16 columns (query rows x the G query heads of one kv head)
// over a chunk of positions.  Rows of one sequence that follow each other within
// an aligned tile of RT = 2^floor(log2(16 / G)) rows share the columns (a chunk
// of a prompt, speculated tokens); the first of them leads, and a new token
// alone has G columns.  The lengths are on the device, so every workgroup works
// out the same plan from pos and seq: the chunk length C that gives about
// `target` workgroups in all (long rows get many chunks, short ones one), and
// from prefix sums over the rows which row and chunk it has.  The host bounds
// the grid by target / n_kv + T per kv head.
//
// Per block of 16 positions a wave has the scores transposed, S^T = K . Q^T
// (rows = positions, columns = the 16 query columns): lane l holds positions
// 4(l/16) + 0..3 of column l % 16, which is at once the operand layout of
// O^T = V^T . P^T, so the probabilities never leave their lane.  Operand maps,
// the same for both operands of a product: scores, k slot 8 (l/16) + b of
// MFMA a is dim 32 a + 8 (l/16) + b; values, tile row m of output tile d is dim
// DT m + d (DT = HD / 16), so a lane loads DT consecutive dims of a position.
// bf16 caches: exact products on the bf16 matrix cores with q and the
// probabilities split into three bf16 parts (24 bits), 32 positions per value
// product; float32 caches: the float32 matrix cores.  Sums, maxima and the
// running rescale are float32.  (An infinite cache value gives NaN, as a part of
// 0 meets it.)
//
// The four waves of a workgroup take blocks in turn, each with its own running
// maximum and sum, and join in LDS.  A row in one chunk is written at once; the
// chunks of the others leave (sums, m, l) and k_paged_combine joins them in
// chunk order.

// the rows r = base + lane of a plan step: leader rows have the number of rows
// they lead (nr) and the positions to cover (n, 0 for a padding row)
struct PlanRows {
    bool leader;
    int nr, n;
};

__device__ __forceinline__ PlanRows plan_rows(const PagedParams& p, int base) {
    const int lane = threadIdx.x & 63, r = base + lane;
    int key = -1 - r, n = 0;  // rows without a sequence share nothing
    if (r < p.T) {
        const int64_t sq = p.seq ? (int64_t)p.seq[r] : r;
        const int64_t pos = p.pos[r];
        if (sq >= 0 && sq < p.n_seq) {
            key = (int)sq;
            if (pos >= 0 && pos < p.cap) n = (int)pos + 1;
        }
    }
    PlanRows o;
    const int before = __shfl_up(key, 1), in_tile = r & (p.rt - 1);
    o.leader = r < p.T && (in_tile == 0 || before != key);
    o.nr = 1;
    o.n = n;
    bool same = true;
    for (int j = 1; j < p.rt; ++j) {
        const int k2 = __shfl_down(key, j), n2 = __shfl_down(n, j);
        same = same && in_tile + j < p.rt && lane + j < 64 && k2 == key;
        if (same) {
            ++o.nr;
            o.n = max(o.n, n2);
        }
    }
    return o;
}

// chunk length of the plan: all positions over the target, in steps of 128
__device__ __forceinline__ int plan_chunk(const PagedParams& p) {
    int64_t total = 0;
    for (int base = 0; base < p.T; base += 64) {
        const PlanRows o = plan_rows(p, base);
        total += o.leader ? o.n : 0;
    }
#pragma unroll
    for (int j = 1; j < 64; j <<= 1) total += __shfl_xor(total, j);
    const int64_t c = (total * p.n_kv + p.target - 1) / p.target;
    return (int)(max(c, (int64_t)p.min_chunk) + 127) & ~127;
}

struct PlanItem {
    int row, nr, n;     // leader row, rows, positions
    int chunk, chunks;  // of this row
    int slot;           // first partial of the row (rows of several chunks only)
};

// item `want` among the chunks of all rows; `several` true: row `want` among the
// rows of several chunks.  False if there is none.
__device__ __forceinline__ bool plan_find(const PagedParams& p, int C, int want, bool several, PlanItem* it) {
    const int lane = threadIdx.x & 63;
    int items0 = 0, slots0 = 0;
    for (int base = 0; base < p.T; base += 64) {
        const PlanRows o = plan_rows(p, base);
        const int ch = o.leader ? max(1, (o.n + C - 1) / C) : 0;
        const int sl = ch > 1 ? ch : 0;
        const int mine = several ? (ch > 1 ? 1 : 0) : ch;
        int items = mine, slots = sl;
#pragma unroll
        for (int j = 1; j < 64; j <<= 1) {
            const int a = __shfl_up(items, j), b = __shfl_up(slots, j);
            if (lane >= j) {
                items += a;
                slots += b;
            }
        }
        const int e = items0 + items - mine;
        const uint64_t hit = __ballot(want >= e && want < e + mine);
        if (hit) {
            const int s = __builtin_ctzll(hit);
            it->row = base + s;
            it->nr = __builtin_amdgcn_readlane(o.nr, s);
            it->n = __builtin_amdgcn_readlane(o.n, s);
            it->chunk = want - __builtin_amdgcn_readlane(e, s);
            it->chunks = __builtin_amdgcn_readlane(ch, s);
            it->slot = slots0 + __builtin_amdgcn_readlane(slots - sl, s);
            return true;
        }
        items0 += __builtin_amdgcn_readlane(items, 63);
        slots0 += __builtin_amdgcn_readlane(slots, 63);
    }
    return false;
}

__device__ __forceinline__ float max4rows(float v) {
    return rows_and_halves(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float sum4rows(float v) {
    return rows_and_halves(v, [](float x, float y) { return x + y; });
}

// partial p of kv head g: [columns][HD + 2]
__device__ __forceinline__ float* paged_part(const PagedParams& p, int HD, int slot, int g) {
    return p.part + ((int64_t)slot * p.n_kv + g) * (p.rt * p.g) * (HD + 2);
}

template <int HD, bool BF16>
__global__ __launch_bounds__(256, 2) void k_paged_attend(PagedParams p) {
    constexpr int EB = BF16 ? 2 : 4;   // cache bytes per value
    constexpr int NB = BF16 ? 2 : 1;   // blocks of 16 positions per step
    constexpr int PB = 16 * NB;
    constexpr int NA = HD / 32;        // 8-dim score chunks per lane
    constexpr int DT = HD / 16;        // output dim tiles = value dims per lane
    constexpr int KW = 8 * EB / 4;     // words of one 8-dim key chunk
    constexpr int VW = DT * EB / 4;    // words of one lane's value dims
    constexpr int NW = 4;              // waves
    constexpr int ROWB = HD * EB;      // bytes of one position
    __shared__ float lds[NW * (DT * 256 + 128)];
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q4 = lane >> 4, c16 = lane & 15;
    const int g = blockIdx.x % p.n_kv, item = blockIdx.x / p.n_kv;
    const int G = p.g, H = p.n_heads;

    const int C = plan_chunk(p);
    PlanItem it;
    if (!plan_find(p, C, item, false, &it)) return;

    // this lane's column: head cg of row r0 + rt
    const int rt = c16 / G, cg = c16 - rt * G;
    const bool col = rt < it.nr;
    const int row = it.row + (col ? rt : 0);
    const int64_t prow = p.pos[row];
    const int lim = col && it.n > 0 && prow >= 0 && prow < p.cap ? (int)prow : -1;  // last position it sees
    const int lo = it.chunk * C, hi = min(it.n, lo + C);
    const int64_t sq = p.seq ? (int64_t)p.seq[it.row] : it.row;
    // the smallest of the columns' limits: up to it every column sees every position
    int first = col ? lim : 0x7FFFFFFF;
#pragma unroll
    for (int j = 1; j < 16; j <<= 1) first = min(first, __shfl_xor(first, j));
    first = __builtin_amdgcn_readfirstlane(first);

    // q of the column, times scale log2(e): the scores are exponents of 2
    float qv[NA][8];
    {
        const float* src = p.q + ((int64_t)row * H + g * G + cg) * HD + 8 * q4;
        const float f = p.scale * 1.44269504088896341f;
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                f32x4 v = {0, 0, 0, 0};
                if (col) v = *reinterpret_cast<const f32x4*>(src + 32 * a + 4 * c);
#pragma unroll
                for (int e = 0; e < 4; ++e) qv[a][4 * c + e] = v[e] * f;
            }
    }
    u32x4 qp[BF16 ? NA : 1][3];
    if constexpr (BF16) {
#pragma unroll
        for (int a = 0; a < NA; ++a) split3(qv[a], qp[a][0], qp[a][1], qp[a][2]);
    }

    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;

    const int steps = (max(hi - lo, 0) + PB - 1) / PB;
    const int32_t* trow = p.table + (hi > lo ? sq * p.table_stride : 0);
    // page ids of this wave's next 64 blocks, one per lane (-1: none)
    constexpr int SPR = 64 / NB;  // steps per refill
    int ids = -1;
    auto refill = [&](int s0) {
        const int ps = lo + (s0 + (lane / NB) * NW) * PB + (lane % NB) * 16;
        ids = ps < hi ? trow[ps >> p.page_log] : -1;
        if (ids >= p.n_pages) ids = -1;
    };
    uint32_t kw[NB][NA][KW], vw[NB][4][VW];
    // descriptor of block b of step s (k: kc or vc): its positions below hi
    auto block = [&](const void* cache, int s, int b, int id) {
        const int ps = lo + s * PB + 16 * b;
        const int rows = id < 0 ? 0 : min(16, hi - ps);
        const int64_t off =
            ((((int64_t)max(id, 0) * p.n_kv + g) << p.page_log) + (ps & ((1 << p.page_log) - 1))) * ROWB;
        return make_rsrc(static_cast<const char*>(cache) + off, (uint32_t)max(rows, 0) * ROWB);
    };
    auto load_k = [&](int s, const int (&id)[NB]) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const __amdgpu_buffer_rsrc_t r = block(p.kc, s, b, id[b]);
#pragma unroll
            for (int a = 0; a < NA; ++a)
#pragma unroll
                for (int c = 0; c < KW / 4; ++c) {
                    const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, c16 * ROWB + (32 * a + 8 * q4) * EB + c * 16, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) kw[b][a][4 * c + e] = v[e];
                }
        }
    };
    auto load_v = [&](int s, const int (&id)[NB]) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const __amdgpu_buffer_rsrc_t r = block(p.vc, s, b, id[b]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int off = (4 * q4 + j) * ROWB + DT * c16 * EB;
                if constexpr (VW == 2) {
                    const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, off, 0, 0);
                    vw[b][j][0] = v[0];
                    vw[b][j][1] = v[1];
                } else {
#pragma unroll
                    for (int c = 0; c < VW / 4; ++c) {
                        const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, off + c * 16, 0, 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e) vw[b][j][4 * c + e] = v[e];
                    }
                }
            }
        }
    };
    auto word_f = [](const uint32_t* w, int i) -> float { return __uint_as_float(w[i]); };
    auto ids_of = [&](int k, int (&id)[NB]) {  // step number k of this wave
#pragma unroll
        for (int b = 0; b < NB; ++b) id[b] = __builtin_amdgcn_readlane(ids, (k % SPR) * NB + b);
    };
    // o[d] += V^T P^T over the step's positions
    auto values = [&](const uint32_t (&w)[NB][4][VW], const float (&pr)[NB][4], f32x4 (&acc)[DT]) {
        if constexpr (BF16) {
            float p8[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) p8[j] = pr[j >> 2][j & 3];
            u32x4 ph, pm, pl;
            split3(p8, ph, pm, pl);
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                // the same dim of the 4 + 4 positions: two 16-bit picks per word
                u32x4 va;
                const uint32_t sel = (d & 1) ? 0x07060302u : 0x05040100u;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    va[j] = __builtin_amdgcn_perm(w[j >> 1][2 * (j & 1) + 1][d >> 1], w[j >> 1][2 * (j & 1)][d >> 1], sel);
                acc[d] = mfma(va, ph, acc[d]);
                acc[d] = mfma(va, pm, acc[d]);
                acc[d] = mfma(va, pl, acc[d]);
            }
        } else {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(word_f(w[0][j], d), pr[0][j], acc[d], 0, 0, 0);
        }
    };

    int id[NB];
    if (wv < steps) {
        refill(wv);
        ids_of(0, id);
        load_k(wv, id);
        load_v(wv, id);
    }
    for (int s = wv, k = 0; s < steps; s += NW, ++k) {
        const int p0 = lo + s * PB;
        // scores of positions p0 + 16 b + 4 q4 + r for the lane's column
        f32x4 sc[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            f32x4 acc = {0, 0, 0, 0};
#pragma unroll
            for (int a = 0; a < NA; ++a) {
                if constexpr (BF16) {
                    const u32x4 ka = {kw[b][a][0], kw[b][a][1], kw[b][a][2], kw[b][a][3]};
#pragma unroll
                    for (int c = 0; c < 3; ++c) acc = mfma(ka, qp[a][c], acc);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(word_f(kw[b][a], e), qv[a][e], acc, 0, 0, 0);
                }
            }
            sc[b] = acc;
        }
        int cur[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) cur[b] = id[b];
        const bool more = s + NW < steps;
        if (more) {
            if ((k + 1) % SPR == 0) refill(s + NW);
            ids_of(k + 1, id);
            load_k(s + NW, id);
        }
        float pr[NB][4];
        float mb = -INFINITY;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int ps = p0 + 16 * b + 4 * q4 + r;
                pr[b][r] = ps <= lim && cur[b] >= 0 && ps < hi ? sc[b][r] : -INFINITY;
                mb = fmaxf(mb, pr[b][r]);
            }
        mb = max4rows(mb);
        // (before the first score above -inf the exponent offset is 0: masked
        // scores add nothing, NaN stays)
        const float mn = fmaxf(m, mb);
        const float mr = mn == -INFINITY ? 0.0f : mn;
        if (__any(mn > m)) {
            const float alpha = __builtin_amdgcn_exp2f(m - mr);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d) o[d] *= alpha;
            m = mn;
        }
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                pr[b][r] = __builtin_amdgcn_exp2f(pr[b][r] - mr);
                l += pr[b][r];
            }
        if (it.nr == 1 || p0 + PB - 1 <= first) {
            values(vw, pr, o);
        } else {
            // the columns' limits differ within these positions: per row, the values
            // past its limit as zeros, so that one row's NaN or infinity does not meet
            // another row's probability of 0
            for (int rr = 0; rr < it.nr; ++rr) {
                const int lm = __builtin_amdgcn_readlane(lim, rr * G);
                uint32_t w[NB][4][VW];
                f32x4 t[DT];
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < VW; ++i) w[b][j][i] = p0 + 16 * b + 4 * q4 + j <= lm ? vw[b][j][i] : 0u;
#pragma unroll
                for (int d = 0; d < DT; ++d) t[d] = o[d];
                values(w, pr, t);
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[d][r] = rt == rr ? t[d][r] : o[d][r];
            }
        }
        if (more) load_v(s + NW, id);
    }
    l = sum4rows(l);

    // join of the waves: wave w adds the sums of tiles d = w, w + 4, ..
    constexpr int kPart = DT * 256 + 128;
    float* mine = lds + wv * kPart;
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<f32x4*>(mine + d * 256 + lane * 4) = o[d];
    mine[DT * 256 + lane] = m;
    mine[DT * 256 + 64 + lane] = l;
    __syncthreads();
    float wm[NW], wl[NW], mj = -INFINITY, lj = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        wm[w] = lds[w * kPart + DT * 256 + lane];
        wl[w] = lds[w * kPart + DT * 256 + 64 + lane];
        mj = fmaxf(mj, wm[w]);
    }
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        // a wave without a finite score: its sums are zero, or NaN and stay so
        wm[w] = wm[w] == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(wm[w] - mj);
        lj = fmaf(wl[w], wm[w], lj);
    }
    if (!col) return;
    const bool whole = it.chunks == 1;
    const float inv_l = lj == 0.0f ? 0.0f : 1.0f / lj;  // nothing to attend: zeros
    float* part = paged_part(p, HD, it.slot + it.chunk, g) + c16 * (HD + 2);
    float* dst = whole ? p.out + ((int64_t)row * H + g * G + cg) * HD : part;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
        if ((d & (NW - 1)) != wv) continue;
        f32x4 v = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < NW; ++w) v += *reinterpret_cast<const f32x4*>(lds + w * kPart + d * 256 + lane * 4) * wm[w];
#pragma unroll
        for (int r = 0; r < 4; ++r) dst[DT * (4 * q4 + r) + d] = whole ? (lj == 0.0f ? 0.0f : v[r] * inv_l) : v[r];
    }
    if (!whole && wv == 0 && q4 == 0) {
        part[HD] = mj;
        part[HD + 1] = lj;
    }
}

// joins the chunks of the rows that have several: out = sum e^(m_c - M) acc_c /
// sum e^(m_c - M) l_c.  Workgroup (row among them, kv head, column); the chunks go
// round the thread groups of HD threads, whose sums are added in a fixed order.
constexpr int kCombineThreads = 512;
template <int HD>
__global__ __launch_bounds__(kCombineThreads) void k_paged_combine(PagedParams p) {
    constexpr int NG = kCombineThreads / HD;
    __shared__ float acc[NG][HD], ssum[NG];
    const int t = threadIdx.x, d = t % HD, grp = t / HD;
    const int g = blockIdx.y, c = blockIdx.z, G = p.g;
    const int C = plan_chunk(p);
    PlanItem it;
    if (!plan_find(p, C, blockIdx.x, true, &it)) return;
    if (c >= it.nr * G) return;
    const float* src = paged_part(p, HD, it.slot, g) + c * (HD + 2);
    const int64_t stride = (int64_t)p.n_kv * p.rt * G * (HD + 2);
    float mx = -INFINITY;
    for (int i = 0; i < it.chunks; ++i) mx = fmaxf(mx, src[i * stride + HD]);
    float a = 0.0f, l = 0.0f;
    for (int i = grp; i < it.chunks; i += NG) {
        const float m = src[i * stride + HD];
        const float w = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
        a = fmaf(src[i * stride + d], w, a);
        l = fmaf(src[i * stride + HD + 1], w, l);
    }
    acc[grp][d] = a;
    if (d == 0) ssum[grp] = l;
    __syncthreads();
    if (grp) return;
#pragma unroll
    for (int i = 1; i < NG; ++i) {
        a += acc[i][d];
        l += ssum[i];
    }
    const int rt = c / G;
    p.out[((int64_t)(it.row + rt) * p.n_heads + g * G + c - rt * G) * HD + d] = l == 0.0f ? 0.0f : a / l;
}

template <int HD, bool BF16>
static void launch_paged_t(const PagedParams& p, hipStream_t st) {
    hipLaunchKernelGGL((k_paged_attend<HD, BF16>), dim3((unsigned)(paged_items(p) * p.n_kv)), dim3(256), 0, st, p);
    const int rows = paged_split_rows(p);
    if (rows)
        hipLaunchKernelGGL((k_paged_combine<HD>), dim3((unsigned)rows, (unsigned)p.n_kv, (unsigned)(p.rt * p.g)),
                           dim3(kCombineThreads), 0, st, p);
}

void launch_paged_attend(const PagedParams& p, hipStream_t st) {
    if (p.head_dim == 128) {
        if (p.kv_bf16) launch_paged_t<128, true>(p, st);
        else launch_paged_t<128, false>(p, st);
    } else {
        if (p.kv_bf16) launch_paged_t<64, true>(p, st);
        else launch_paged_t<64, false>(p, st);
    }
}

}  // namespace rv12
