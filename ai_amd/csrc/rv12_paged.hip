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

#include <type_traits>

#include "rv12_device.h"
#include "rv12_internal.h"

namespace rv12 {

// ---------------------------------------------------------------------------
// Append: q and k get their head RMSNorm and the rotate-half RoPE at the row's
// position, q goes to q_out as float32, k and v into the row's page slot,
// rounded once to the cache type.
//
// Bound by bytes (4 (H + 2 KV) HD read, 4 H HD + 2 KV HD EB written per row: 4099
// rows of 32 heads over 8 take 37 us into bf16 pages, 5.0 TB/s, and 42 into float32
// ones, 4.8: the rate of a copy); at a few rows by its latency (2.2 us for one, 3.3
// for 64).  HD / 8 lanes hold a head, 4 consecutive dims of either rotation half
// each, so every access is 16 bytes (8 where bf16 is stored) and the norm's sum
// stays within 16 lanes.  A workgroup of 256 threads takes a share of one row's
// heads: the row's HD / 2 angles are computed once per workgroup, while the heads'
// loads are in flight.
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
    const int slots = 256 / LPH;  // heads of a workgroup
    const int hl = t % LPH;       // the lane's dims: 4 hl .. + 3 of both halves
    const int64_t sq = p.seq ? (int64_t)p.seq[r] : r;
    const int64_t pos = p.pos[r];
    const bool live = sq >= 0 && sq < p.n_seq && pos >= 0 && pos < p.cap;
    const float* row = p.qkv + (int64_t)r * NH * HD;
    const int h = blockIdx.y * slots + t / LPH;
    f32x4 a = {0, 0, 0, 0}, b = {0, 0, 0, 0};
    if (h < NH) {
        a = *reinterpret_cast<const f32x4*>(row + (int64_t)h * HD + 4 * hl);
        b = *reinterpret_cast<const f32x4*>(row + (int64_t)h * HD + half + 4 * hl);
    }
    if (!live) {
        if (h < H) {
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
    if (h >= NH) return;
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
            a[e] = x * c.x - y * c.y;
            b[e] = y * c.x + x * c.y;
        }
    }
    if (h < H) {
        float* dst = p.qo + ((int64_t)r * H + h) * HD;
        *reinterpret_cast<f32x4*>(dst + 4 * hl) = a;
        *reinterpret_cast<f32x4*>(dst + half + 4 * hl) = b;
    } else if (paged) {
        const int g = h < H + KV ? h - H : h - H - KV;
        void* c = h < H + KV ? p.kc : p.vc;
        const int64_t off = (slot + ((int64_t)g << p.page_log)) * HD + 4 * hl;
        if constexpr (BF16) {
            uint16_t* dst = static_cast<uint16_t*>(c) + off;
            *reinterpret_cast<uint2*>(dst) =
                uint2{bf16_bits(a[0]) | bf16_bits(a[1]) << 16, bf16_bits(a[2]) | bf16_bits(a[3]) << 16};
            *reinterpret_cast<uint2*>(dst + half) =
                uint2{bf16_bits(b[0]) | bf16_bits(b[1]) << 16, bf16_bits(b[2]) | bf16_bits(b[3]) << 16};
        } else {
            float* dst = static_cast<float*>(c) + off;
            *reinterpret_cast<f32x4*>(dst) = a;
            *reinterpret_cast<f32x4*>(dst + half) = b;
        }
    }
}

void launch_paged_append(const PagedParams& p, hipStream_t st) {
    // a thread group for every head of a row
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
// running rescale are float32.  (An infinite value of a bf16 cache gives NaN where a
// part of 0 meets it; a float32 one gives what its product does.)
//
// The four waves of a workgroup take blocks in turn, each with its own running
// maximum and sum, and join in LDS.  A row in one chunk is written at once; the
// chunks of the others leave (sums, m, l) and k_paged_combine joins them in
// chunk order.
//
// Bound by the cache's bytes once they are many: 64 rows of 500 to 8200 positions,
// 32 heads over 8, bf16, 730 MB in 130 us (5.6 TB/s) and the join in 6; 32771
// positions of one row 25 + 4 us.  One row of 16 positions takes 6.2 us, all of it
// dependent round trips (rows, table, keys, values, the join in LDS); 8 float32 rows
// of 60 to 700 positions, 16 heads over 8, take that, 3.8 for their 18 MB, and 4 in
// the join's own launch: 10.3 + 4.  A prompt of 2048 rows, 32 heads over 8, takes 187 us
// in bf16 and 361 in float32, the plan's 7 and the join's 5 among them: 34 GFLOP, in
// bf16 in three parts each, that keep the matrix cores busy 22 % of the time; the
// waves wait a third of theirs.

// the rows r = base + lane of a plan step: leader rows have the number of rows
// they lead (nr) and the positions to cover (n, 0 for a padding row); key: the row's
// sequence, another negative number for every row without one
struct PlanRows {
    bool leader;
    int nr, n, key;
};

template <int CTRL, int ROWS = 0xF>
__device__ __forceinline__ int dpp_int(int v) {  // 0 where no lane is named
    return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
constexpr int kDppDown1 = 0x101, kDppDown2 = 0x102, kDppDown4 = 0x104, kDppDown8 = 0x108;  // lane i gets i + n of its 16
constexpr int kDppUp1 = 0x111, kDppUp2 = 0x112, kDppUp4 = 0x114, kDppUp8 = 0x118;          // i - n
// inclusive sum over the wave's lanes
__device__ __forceinline__ int wave_scan(int v) {
    v += dpp_int<kDppUp1>(v);
    v += dpp_int<kDppUp2>(v);
    v += dpp_int<kDppUp4>(v);
    v += dpp_int<kDppUp8>(v);
    v += dpp_int<0x142, 0xA>(v);  // lane 15 of rows 0 and 2 to the row after
    v += dpp_int<0x143, 0xC>(v);  // lane 31 to rows 2 and 3
    return v;
}

__device__ __forceinline__ PlanRows plan_rows(const PagedParams& p, int base) {
    const int lane = threadIdx.x & 63, r = base + lane;
    int key = -1 - r, n = 0;  // rows without a sequence share nothing
    if (r < p.T) {
        const int64_t pos = p.pos[r];
        const int64_t sq = p.seq ? (int64_t)p.seq[r] : r;
        if (sq >= 0 && sq < p.n_seq) {
            key = (int)sq;
            if (pos >= 0 && pos < p.cap) n = (int)pos + 1;
        }
    }
    // tiles are aligned to rt <= 16 rows, so a tile stays within 16 lanes
    const int before = dpp_int<kDppUp1>(key);  // (every lane active: no part of a condition)
    const bool joins = r < p.T && (r & (p.rt - 1)) != 0 && before == key;
    const uint64_t m = __ballot(joins);
    PlanRows o;
    o.leader = r < p.T && !joins;
    o.nr = 1;
    o.n = n;
    o.key = key;
    if (m) {
        o.nr = 1 + __builtin_ctzll(~((m >> lane) >> 1));
        int k;
        k = dpp_int<kDppDown1>(o.n);
        if (o.nr > 1) o.n = max(o.n, k);
        k = dpp_int<kDppDown2>(o.n);
        if (o.nr > 2) o.n = max(o.n, k);
        k = dpp_int<kDppDown4>(o.n);
        if (o.nr > 4) o.n = max(o.n, k);
        k = dpp_int<kDppDown8>(o.n);
        if (o.nr > 8) o.n = max(o.n, k);
    }
    return o;
}

// chunk length of the plan over `total` blocks of 32 positions
__device__ __forceinline__ int plan_chunk(const PagedParams& p, int total) {
    // up to 512 positions a chunk's own cost (its round trips, its partials) counts,
    // and two workgroups per CU are best; above it smaller chunks even out the
    // workgroups' ends (both passes, us with the target's workgroups and with half of
    // them: 8 rows of one sequence at 4104 positions, 64 query heads over 8, 25.3,
    // 21.7; 64 rows of 500 to 8200 positions, 32 heads over 8, 141, 156)
    const int64_t all = (int64_t)total * p.n_kv;
    constexpr int64_t kKnee = 512;
    const int64_t half_c = (all + p.target / 2 - 1) / (p.target / 2) * 32;
    const int64_t c = half_c <= kKnee ? half_c : max((all + p.target - 1) / p.target * 32, kKnee);
    return (int)((max(c, (int64_t)1) + p.grain - 1) & ~(int64_t)(p.grain - 1));
}
__device__ __forceinline__ int plan_blocks(const PlanRows& o) { return o.leader ? (o.n + 31) >> 5 : 0; }
__device__ __forceinline__ int plan_chunks(const PlanRows& o, int C) { return o.leader ? max(1, (o.n + C - 1) / C) : 0; }

// item `want` among the chunks of all rows, or (SEVERAL) row `want` among the rows
// of several chunks.  False if there is none.  Up to 64 rows every workgroup works
// it out from one load of the rows; of more the list of k_paged_plan has it.
template <bool SEVERAL>
__device__ __forceinline__ bool plan_find(const PagedParams& p, int want, PlanItem* it) {
    if (p.plan) {
        if (want >= p.plan[0].row && !SEVERAL) return false;
        if (want >= p.plan[0].nr && SEVERAL) return false;
        *it = p.plan[1 + want + (SEVERAL ? p.plan_items : 0)];
        return true;
    }
    const PlanRows o = plan_rows(p, 0);
    const int C = plan_chunk(p, __builtin_amdgcn_readlane(wave_scan(plan_blocks(o)), 63));
    const int ch = plan_chunks(o, C), sl = ch > 1 ? ch : 0;
    const int mine = SEVERAL ? (ch > 1 ? 1 : 0) : ch;
    // both sums at once: at most 2 target slots and target + 64 items
    const int both = wave_scan(sl << 16 | mine);
    const int e = (both & 0xFFFF) - mine;
    const uint64_t hit = __ballot(want >= e && want < e + mine);
    if (!hit) return false;
    const int s = __builtin_ctzll(hit);
    it->row = s;
    it->nr = __builtin_amdgcn_readlane(o.nr, s);
    it->n = __builtin_amdgcn_readlane(o.n, s);
    it->C = C;
    it->chunk = want - __builtin_amdgcn_readlane(e, s);
    it->chunks = __builtin_amdgcn_readlane(ch, s);
    it->slot = __builtin_amdgcn_readlane((both >> 16) - sl, s);
    const int key = __builtin_amdgcn_readlane(o.key, s), e1 = s + it->nr;
    it->once = !((s > 0 && __builtin_amdgcn_readlane(o.key, max(s - 1, 0)) == key) ||
                 (e1 < p.T && __builtin_amdgcn_readlane(o.key, min(e1, 63)) == key));
    return true;
}

// the plan of more than 64 rows, one workgroup: entry 0 the counts (row: items, nr:
// rows of several chunks), then every item, then the rows of several chunks.  The
// waves take the steps of 64 rows in turn, in three passes over them: the sum of
// the positions, the numbers of items and slots, the entries.  (Worked out in every
// workgroup, as for up to 64 rows, a prompt of 2048 rows took 850 us in all, not 187.)
constexpr int kPlanThreads = 1024;
__global__ __launch_bounds__(kPlanThreads) void k_paged_plan(PagedParams p) {
    constexpr int NW = kPlanThreads / 64;
    __shared__ int sums[3][NW];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int steps = (p.T + 63) / 64;
    const int s0 = (int)((int64_t)wv * steps / NW), s1 = (int)((int64_t)(wv + 1) * steps / NW);
    int v = 0;
    for (int s = s0; s < s1; ++s) v += plan_blocks(plan_rows(p, 64 * s));
    v = wave_scan(v);
    if (lane == 63) sums[0][wv] = v;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < NW; ++w) total += sums[0][w];
    const int C = plan_chunk(p, total);
    __syncthreads();
    int items = 0, slots = 0, rows = 0;
    for (int s = s0; s < s1; ++s) {
        const int ch = plan_chunks(plan_rows(p, 64 * s), C);
        items += ch;
        slots += ch > 1 ? ch : 0;
        rows += ch > 1 ? 1 : 0;
    }
    items = wave_scan(items);
    slots = wave_scan(slots);
    rows = wave_scan(rows);
    if (lane == 63) {
        sums[0][wv] = items;
        sums[1][wv] = slots;
        sums[2][wv] = rows;
    }
    __syncthreads();
    items = slots = rows = 0;
    for (int w = 0; w < wv; ++w) {
        items += sums[0][w];
        slots += sums[1][w];
        rows += sums[2][w];
    }
    if (threadIdx.x == kPlanThreads - 1) {
        p.plan[0].row = items + sums[0][NW - 1];
        p.plan[0].nr = rows + sums[2][NW - 1];
    }
    for (int s = s0; s < s1; ++s) {
        const PlanRows o = plan_rows(p, 64 * s);
        const int ch = plan_chunks(o, C), sl = ch > 1 ? ch : 0, se = ch > 1 ? 1 : 0;
        const int ie = wave_scan(ch), le = wave_scan(sl), re = wave_scan(se);
        PlanItem it;
        it.row = 64 * s + lane;
        it.nr = o.nr;
        it.n = o.n;
        it.C = C;
        it.chunks = ch;
        it.slot = slots + le - sl;
        it.chunk = 0;
        it.once = 1;
        if (p.seq && o.leader && o.key >= 0) {
            const int r0 = it.row, r1 = it.row + it.nr;
            it.once = !((r0 > 0 && p.seq[r0 - 1] == o.key) || (r1 < p.T && p.seq[r1] == o.key));
        }
        if (se) p.plan[1 + p.plan_items + rows + re - 1] = it;
        for (int i = 0; i < ch; ++i) {
            it.chunk = i;
            p.plan[1 + items + ie - ch + i] = it;
        }
        items += __builtin_amdgcn_readlane(ie, 63);
        slots += __builtin_amdgcn_readlane(le, 63);
        rows += __builtin_amdgcn_readlane(re, 63);
    }
}

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
// split3 with a pair of values per conversion
__device__ __forceinline__ uint32_t bf16_pair(f32x2 v) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ void split3_pairs(const float (&v)[8], u32x4& hi, u32x4& mid, u32x4& lo) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        f32x2 a = {v[2 * j], v[2 * j + 1]};
        hi[j] = bf16_pair(a);
        a = f32x2{a.x - lo_f(hi[j]), a.y - hi_f(hi[j])};
        mid[j] = bf16_pair(a);
        a = f32x2{a.x - lo_f(mid[j]), a.y - hi_f(mid[j])};
        lo[j] = bf16_pair(a);
    }
}

__device__ __forceinline__ float max4rows(float v) {
    return rows_and_halves(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float sum4rows(float v) {
    return rows_and_halves(v, [](float x, float y) { return x + y; });
}

// the partial of a slot and kv head: [columns][HD + 4], the sums, m and l
__device__ __forceinline__ float* paged_part(const PagedParams& p, int HD, int slot, int g) {
    return p.part + ((int64_t)slot * p.n_kv + g) * (p.rt * p.g) * (HD + 4);
}

template <int HD, bool BF16>
struct AttendLds {
    float part[4 * (HD / 16 * 256 + 128)];
    u32x4 qp[BF16 ? HD / 32 : 1][3][BF16 ? 64 : 1];
    f32x4 qf[BF16 ? 1 : HD / 32][2][BF16 ? 1 : 64];
};

template <int HD, bool BF16, bool ONCE>
__device__ __forceinline__ void attend_item(const PagedParams& p, const PlanItem& it, AttendLds<HD, BF16>& sh) {
    constexpr int EB = BF16 ? 2 : 4;   // cache bytes per value
    constexpr int NB = BF16 ? 2 : 1;   // blocks of 16 positions per step
    constexpr int PB = 16 * NB;
    constexpr int NA = HD / 32;        // 8-dim score chunks per lane
    constexpr int DT = HD / 16;        // output dim tiles = value dims per lane
    constexpr int KW = 8 * EB / 4;     // words of one 8-dim key chunk
    constexpr int VW = DT * EB / 4;    // words of one lane's value dims
    constexpr int NW = 4;              // waves
    constexpr int ROWB = HD * EB;      // bytes of one position
    constexpr int kPolicy = ONCE ? kNonTemporal : 0;
    float* lds = sh.part;
    auto& qp = sh.qp;
    auto& qf = sh.qf;
    const int lane = threadIdx.x & 63;
    const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int q4 = lane >> 4, c16 = lane & 15;
    const int g = blockIdx.x % p.n_kv;
    const int G = p.g, H = p.n_heads;

    // this lane's column: head cg of row r0 + rt
    const int rt = c16 / G, cg = c16 - rt * G;
    const bool col = rt < it.nr;
    const int row = it.row + (col ? rt : 0);
    const int64_t prow = p.pos[row];
    const int lim = col && it.n > 0 && prow >= 0 && prow < p.cap ? (int)prow : -1;  // last position it sees
    const int lo = it.chunk * it.C, hi = min(it.n, lo + it.C);
    const int64_t sq = p.seq ? (int64_t)p.seq[it.row] : it.row;
    // the smallest of the columns' limits: up to it every column sees every position
    int first = it.n - 1;
    if (it.nr > 1) {
        first = col ? lim : 0x7FFFFFFF;
#pragma unroll
        for (int j = 1; j < 16; j <<= 1) first = min(first, __shfl_xor(first, j));
    }
    first = __builtin_amdgcn_readfirstlane(first);

    // q of the column: wave w loads the 8-dim chunks w, w + 4, .., before anything
    // waits
    constexpr int QC = (NA + NW - 1) / NW;
    f32x4 qin[QC][2];
#pragma unroll
    for (int i = 0; i < QC; ++i) {
        const float* src = p.q + ((int64_t)row * H + g * G + cg) * HD + 8 * q4 + 32 * (wv + NW * i);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            qin[i][c] = f32x4{0, 0, 0, 0};
            if (col && wv + NW * i < NA) qin[i][c] = *reinterpret_cast<const f32x4*>(src + 4 * c);
        }
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
    const int koff = c16 * ROWB + 8 * q4 * EB, voff = 4 * q4 * ROWB + DT * c16 * EB;
    // descriptor of block b of step s (k: kc or vc): its positions below hi
    auto block = [&](const void* cache, int s, int b, int id) {
        const int ps = lo + s * PB + 16 * b;
        const int rows = id < 0 ? 0 : min(16, hi - ps);
        const int64_t off =
            ((((int64_t)max(id, 0) * p.n_kv + g) << p.page_log) + (ps & ((1 << p.page_log) - 1))) * ROWB;
        // (a clamp is a vector instruction: back to a scalar register)
        return make_rsrc(static_cast<const char*>(cache) + off,
                         (uint32_t)__builtin_amdgcn_readfirstlane(max(rows, 0) * ROWB));
    };
    auto load_k = [&](int s, const int (&id)[NB]) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            const __amdgpu_buffer_rsrc_t r = block(p.kc, s, b, id[b]);
#pragma unroll
            for (int a = 0; a < NA; ++a)
#pragma unroll
                for (int c = 0; c < KW / 4; ++c) {
                    const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, koff, 32 * a * EB + c * 16, kPolicy);
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
                if constexpr (VW == 2) {
                    const auto v = __builtin_amdgcn_raw_buffer_load_b64(r, voff, j * ROWB, kPolicy);
                    vw[b][j][0] = v[0];
                    vw[b][j][1] = v[1];
                } else {
#pragma unroll
                    for (int c = 0; c < VW / 4; ++c) {
                        const auto v = __builtin_amdgcn_raw_buffer_load_b128(r, voff, j * ROWB + c * 16, kPolicy);
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
    // o[d] += V^T P^T over the step's positions; MASKED: the positions past lm as
    // zeros, and only the columns of row rr
    auto values = [&](const float (&pr)[NB][4], auto masked, int p0, int lm, int rr) {
        constexpr bool MASKED = decltype(masked)::value;
        if constexpr (BF16) {
            float p8[8];
            uint32_t keep[4];
#pragma unroll
            for (int j = 0; j < 8; ++j) p8[j] = pr[j >> 2][j & 3];
            u32x4 ph, pm, pl;
            split3_pairs(p8, ph, pm, pl);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int ps = p0 + 16 * (j >> 1) + 4 * q4 + 2 * (j & 1);
                keep[j] = (ps <= lm ? 0xFFFFu : 0u) | (ps + 1 <= lm ? 0xFFFF0000u : 0u);
            }
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                // the same dim of the 4 + 4 positions: two 16-bit picks per word
                u32x4 va;
                const uint32_t sel = (d & 1) ? 0x07060302u : 0x05040100u;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    va[j] = __builtin_amdgcn_perm(vw[j >> 1][2 * (j & 1) + 1][d >> 1], vw[j >> 1][2 * (j & 1)][d >> 1], sel);
                    if constexpr (MASKED) va[j] &= keep[j];
                }
                f32x4 t = mfma(va, ph, o[d]);
                t = mfma(va, pm, t);
                t = mfma(va, pl, t);
                if constexpr (MASKED) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[d][r] = rt == rr ? t[r] : o[d][r];
                } else {
                    o[d] = t;
                }
            }
        } else {
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                f32x4 t = o[d];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float v = !MASKED || p0 + 4 * q4 + j <= lm ? word_f(vw[0][j], d) : 0.0f;
                    t = __builtin_amdgcn_mfma_f32_16x16x4f32(v, pr[0][j], t, 0, 0, 0);
                }
                if constexpr (MASKED) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) o[d][r] = rt == rr ? t[r] : o[d][r];
                } else {
                    o[d] = t;
                }
            }
        }
    };

    int id[NB];
    if (wv < steps) {
        refill(wv);
        ids_of(0, id);
        load_k(wv, id);
        // keys before values, as in the loop: its first wait is then for the keys alone
        __builtin_amdgcn_sched_barrier(0);
        load_v(wv, id);
    }
    // q times scale log2(e) (the scores are exponents of 2) stays in LDS (bf16
    // caches: its three parts), the same for the four waves: 48 (float32: 32)
    // registers less, a third workgroup on every CU
#pragma unroll
    for (int i = 0; i < QC; ++i) {
        const int a = wv + NW * i;
        if (a >= NA) continue;
        const float f = p.scale * 1.44269504088896341f;
        qin[i][0] *= f;
        qin[i][1] *= f;
        if constexpr (BF16) {
            float v8[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v8[e] = qin[i][e >> 2][e & 3];
            u32x4 h, m, l;
            split3_pairs(v8, h, m, l);
            qp[a][0][lane] = h;
            qp[a][1][lane] = m;
            qp[a][2][lane] = l;
        } else {
            qf[a][0][lane] = qin[i][0];
            qf[a][1][lane] = qin[i][1];
        }
    }
    __syncthreads();
    auto step = [&](int s, int k, auto apart) {
        const int p0 = lo + s * PB;
        asm volatile("" ::: "memory");  // q is read again, not kept in registers
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
                    for (int c = 0; c < 3; ++c) acc = mfma(ka, qp[a][c][lane], acc);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        acc = __builtin_amdgcn_mfma_f32_16x16x4f32(word_f(kw[b][a], e), qf[a][e >> 2][lane][e & 3], acc, 0, 0, 0);
                }
            }
            sc[b] = acc;
        }
        int cur[NB];
#pragma unroll
        for (int b = 0; b < NB; ++b) cur[b] = id[b];
        // the next step's keys; past the last step the ids are -1, and the loads
        // read zeros without an access (no branch, so that each wait below is for
        // the loads that it needs alone)
        if ((k + 1) % SPR == 0) refill(s + NW);
        ids_of(k + 1, id);
        load_k(s + NW, id);
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
        if constexpr (decltype(apart)::value) {
            for (int rr = 0; rr < it.nr; ++rr)
                values(pr, std::true_type{}, p0, __builtin_amdgcn_readlane(lim, rr * G), rr);
        } else {
            values(pr, std::false_type{}, 0, 0, 0);
        }
        load_v(s + NW, id);
    };
    int s = wv, k = 0;
    // the steps that every column sees whole (with one row: all), then those within
    // which the columns' limits differ: per row, the values past its limit as zeros,
    // so that one row's NaN or infinity does not meet another row's probability of 0
    const int whole_steps = it.nr == 1 ? steps : min(steps, max(first + 1 - lo, 0) / PB);
    for (; s < whole_steps; s += NW, ++k) step(s, k, std::false_type{});
    for (; s < steps; s += NW, ++k) step(s, k, std::true_type{});
    l = sum4rows(l);

    // join of the waves: wave w adds the sums of its quarter of the tiles
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
    float* part = paged_part(p, HD, it.slot + it.chunk, g) + c16 * (HD + 4);
    float* dst = whole ? p.out + ((int64_t)row * H + g * G + cg) * HD : part;
    constexpr int TW = DT / NW;  // tiles per wave: consecutive dims
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        float v[TW];
#pragma unroll
        for (int i = 0; i < TW; ++i) {
            v[i] = 0.0f;
#pragma unroll
            for (int w = 0; w < NW; ++w) v[i] = fmaf(lds[w * kPart + (TW * wv + i) * 256 + lane * 4 + r], wm[w], v[i]);
            if (whole) v[i] = lj == 0.0f ? 0.0f : v[i] * inv_l;
        }
        float* to = dst + DT * (4 * q4 + r) + TW * wv;
        if constexpr (TW == 2) *reinterpret_cast<float2*>(to) = float2{v[0], v[1]};
        else to[0] = v[0];
    }
    if (!whole && wv == 0 && q4 == 0) *reinterpret_cast<float2*>(part + HD) = float2{mj, lj};
}

// Loads past the caches: where the item's rows have their sequence to themselves
// (the rows before and after them are of others), every key and value of bf16 caches
// is read once and the loads stream: a pass over a model's layers comes back to a
// layer's keys when the other layers' have gone by.  Both passes, 32 heads over 8, us
// streaming and through the caches: 8 rows at 1000 positions 15.1, 16.2; 24 at 4100
// 78, 85; 64 at 8200 344, 385.  (Keys still in the 256 MB cache from a call just
// before are the exception: 8 rows at 4100 36.8, 31.6.)  Items that share a sequence
// find its keys in the L2 (64 heads over 8, 8 rows at 4104 positions: 21.7, 22.6 past
// it), and a float32 key row takes two loads of one line (64 rows of 500 to 8200
// positions: 278, 299 past it).  The policy is a part of the instructions, so bf16 has
// the body twice, chosen before anything of it is issued: chosen inside it, the waits
// of both merged (142 -> 146 us for the 64 rows in bf16).
template <int HD, bool BF16>
__global__ __launch_bounds__(256, 3) void k_paged_attend(PagedParams p) {
    __shared__ AttendLds<HD, BF16> sh;
    PlanItem it;
    if (!plan_find<false>(p, blockIdx.x / p.n_kv, &it)) return;
    // (said to be uniform, so that the loads' descriptors stay in scalar registers)
    it.row = __builtin_amdgcn_readfirstlane(it.row);
    it.nr = __builtin_amdgcn_readfirstlane(it.nr);
    it.n = __builtin_amdgcn_readfirstlane(it.n);
    it.C = __builtin_amdgcn_readfirstlane(it.C);
    it.chunk = __builtin_amdgcn_readfirstlane(it.chunk);
    it.chunks = __builtin_amdgcn_readfirstlane(it.chunks);
    it.slot = __builtin_amdgcn_readfirstlane(it.slot);
    if (BF16 && __builtin_amdgcn_readfirstlane(it.once)) attend_item<HD, BF16, BF16>(p, it, sh);
    else attend_item<HD, BF16, false>(p, it, sh);
}

// joins the chunks of the rows that have several: out = sum 2^(m_c - M) acc_c /
// sum 2^(m_c - M) l_c.  Workgroup (row among them, kv head, query head of it); HD /
// 4 threads hold a head's dims, the chunks go round the groups of threads, each
// with a running maximum (one pass over the partials), and the groups join in
// LDS in order.
constexpr int kCombineThreads = 256;
template <int HD>
__global__ __launch_bounds__(kCombineThreads) void k_paged_combine(PagedParams p) {
    constexpr int TD = HD / 4, NG = kCombineThreads / TD;
    __shared__ f32x4 acc[NG][TD];
    __shared__ float2 ml[NG];
    const int t = threadIdx.x, d = t % TD, grp = t / TD;
    const int g = blockIdx.y, G = p.g;
    PlanItem it;
    if (!plan_find<true>(p, blockIdx.x, &it)) return;
    const int64_t stride = (int64_t)p.n_kv * p.rt * G * (HD + 4);
    for (int rr = 0; rr < it.nr; ++rr) {
        const float* src = paged_part(p, HD, it.slot, g) + (rr * G + (int)blockIdx.z) * (HD + 4);
        f32x4 a = {0, 0, 0, 0};
        float l = 0.0f, m = -INFINITY;
#pragma unroll 4
        for (int i = grp; i < it.chunks; i += NG) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(src + i * stride + 4 * d);
            const float2 s = *reinterpret_cast<const float2*>(src + i * stride + HD);
            // chunks and groups without a finite score: their sums are zero, or NaN and stay so
            const float mn = fmaxf(m, s.x);
            const float f0 = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            const float f1 = s.x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(s.x - mn);
            a = a * f0 + v * f1;
            l = l * f0 + s.y * f1;
            m = mn;
        }
        acc[grp][d] = a;
        if (d == 0) ml[grp] = float2{m, l};
        __syncthreads();
        if (grp == 0) {
            float mx = m;
#pragma unroll
            for (int i = 1; i < NG; ++i) mx = fmaxf(mx, ml[i].x);
            const float f = m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
            a *= f;
            l *= f;
#pragma unroll
            for (int i = 1; i < NG; ++i) {
                const float fi = ml[i].x == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ml[i].x - mx);
                a += acc[i][d] * fi;
                l = fmaf(ml[i].y, fi, l);
            }
            float* o = p.out + ((int64_t)(it.row + rr) * p.n_heads + g * G + (int)blockIdx.z) * HD + 4 * d;
            *reinterpret_cast<f32x4*>(o) = l == 0.0f ? f32x4{0, 0, 0, 0} : a / l;
        }
        __syncthreads();
    }
}

template <int HD, bool BF16>
static void launch_paged_t(const PagedParams& p, hipStream_t st) {
    const dim3 grid((unsigned)(paged_items(p) * p.n_kv));
    hipLaunchKernelGGL((k_paged_attend<HD, BF16>), grid, dim3(256), 0, st, p);
    const int rows = paged_split_rows(p);
    if (rows)
        hipLaunchKernelGGL((k_paged_combine<HD>), dim3((unsigned)rows, (unsigned)p.n_kv, (unsigned)p.g),
                           dim3(kCombineThreads), 0, st, p);
}

void launch_paged_attend(const PagedParams& p, hipStream_t st) {
    if (p.plan) hipLaunchKernelGGL(k_paged_plan, dim3(1), dim3(kPlanThreads), 0, st, p);
    if (p.head_dim == 128) {
        if (p.kv_bf16) launch_paged_t<128, true>(p, st);
        else launch_paged_t<128, false>(p, st);
    } else {
        if (p.kv_bf16) launch_paged_t<64, true>(p, st);
        else launch_paged_t<64, false>(p, st);
    }
}

}  // namespace rv12
