// The paged key-value cache of an attention decoder: append (rows into pages), attend (one new token per sequence over
// its pages) and evict (the cache cut to a budget by the attention its tokens have drawn). include/taco.h has the
// formulas. The pool holds pages of page_size tokens per kv head; a sequence names its pages in a table row, slot s of
// it lives in row s % page_size of page table[b][s / page_size].
//
// Nothing on the device trusts a length or a page id: lengths are clamped to the table's capacity, a slot whose page id
// is outside the pool is treated as masked (attend) or not written (append, evict), and either sets a bit of the pool's
// status word. Offsets into the pool and the side tables are 64-bit.
#include "kernels.h"

#include <atomic>
#include <type_traits>

namespace taco {
namespace {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// a lambda that is not inlined would keep the registers it refers to in memory
#define INLINE __attribute__((always_inline))

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }   // (flushes results below 2^-126)

// log of sum 2^ref, the same bits wherever it is computed.
__device__ __forceinline__ float log_sum(float ref, float sum) { return __builtin_fmaf(ref, LN2, logf(sum)); }

__device__ __forceinline__ int clamp_len(int n, int cap, int32_t* status, bool report) {
    if (n >= 0 && n <= cap) return n;
    if (report) atomicOr(status, KV_BAD_LENGTH);
    return n < 0 ? 0 : cap;
}

// Element offset of slot s (page id already checked) in a pool with strides st = {page, head, token}.
__device__ __forceinline__ int64_t slot_off(const int64_t* st, int page, int h, int in_page) {
    return (int64_t)page * st[0] + (int64_t)h * st[1] + (int64_t)in_page * st[2];
}

__global__ void kv_take_status_kernel(int32_t* status, int32_t* bits) { *bits = atomicExch(status, 0); }

// ---------------------------------------------------------------------------------------
// append

// 16-byte pieces per lane. (8 x 4097 tokens of 8 heads, bf16, take 50 us with 2, 49 with 4, 62 with 1 and through the caches;
// 32 x 150 of one head, fp32, 6.6, 8.0 and 7.1.)
constexpr int AP_ITEMS = 2;

// Planes 0 / 1 of the grid copy K / V, 16-byte pieces (t, h, column) with the column fastest, AP_ITEMS per lane, all read
// before the first is written; plane 2 writes the side tables, (h, t) with t fastest. Nothing but the copy bounds it: rows
// come in once and go out once, past the caches.
__global__ __launch_bounds__(256) void kv_append_kernel(const KvPool p, const KvTable tb, const KvAppend a) {
    const int b = blockIdx.y, plane = blockIdx.z;
    const int cap = tb.max_pages << p.page_shift;
    const bool first_thread = blockIdx.x == 0 && threadIdx.x == 0 && plane == 0;
    const int start = clamp_len(a.starts[b], cap, p.status, first_thread);
    int count = a.counts ? clamp_len(a.counts[b], a.T, p.status, first_thread) : a.T;
    if (count > cap - start) {
        count = cap - start;
        if (first_thread) atomicOr(p.status, KV_BAD_LENGTH);
    }
    if (first_thread) a.lengths_out[b] = start + count;
    if (plane == 2) {
        const uint32_t n = (uint32_t)p.heads * (uint32_t)a.T;
        for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) {
            const int t = (int)(i % a.T), h = (int)(i / a.T);
            if (t >= count) continue;
            const int64_t o = ((int64_t)b * p.heads + h) * a.side_ld + start + t;
            if (a.mass) a.mass[o] = 0.f;
            if (a.positions) a.positions[o] = (a.first ? a.first[b] : start) + t;
        }
        return;
    }
    const int vec_shift = 31 - __builtin_clz((p.dim * p.esize) >> 4);      // pieces per row: a power of two
    const uint32_t n = ((uint32_t)count * (uint32_t)p.heads) << vec_shift;
    const uint32_t i0 = blockIdx.x * (256 * AP_ITEMS) + threadIdx.x;
    if (i0 >= n) return;
    const int64_t* xs = plane ? a.v_st : a.k_st;
    const int64_t* ps = plane ? p.v_st : p.k_st;
    const char* src = (const char*)(plane ? a.v : a.k) + (int64_t)b * xs[0] * p.esize;
    char* dst = (char*)(plane ? p.v : p.k);
    const int32_t* row = tb.table + (int64_t)b * tb.ld;
    u32x4 x[AP_ITEMS];
    int64_t to[AP_ITEMS];
#pragma unroll
    for (int j = 0; j < AP_ITEMS; ++j) {
        const uint32_t i = min(i0 + 256 * j, n - 1), th = i >> vec_shift;      // (behind the end: the last piece, not written)
        const int c = (int)(i & ((1u << vec_shift) - 1)), t = (int)(th / (uint32_t)p.heads), h = (int)(th - (uint32_t)t * p.heads), s = start + t;
        const int page = row[s >> p.page_shift];
        to[j] = -1;
        if ((unsigned)page >= (unsigned)p.num_pages) atomicOr(p.status, KV_BAD_PAGE);
        else if (i0 + 256 * j < n) to[j] = slot_off(ps, page, h, s & (p.page_size - 1)) * p.esize + 16 * c;
        x[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + ((int64_t)t * xs[1] + (int64_t)h * xs[2]) * p.esize + 16 * c));
    }
#pragma unroll
    for (int j = 0; j < AP_ITEMS; ++j)
        if (to[j] >= 0) __builtin_nontemporal_store(x[j], reinterpret_cast<u32x4*>(dst + to[j]));
}

// ---------------------------------------------------------------------------------------
// attend
//
// One pass over the pages with the running maximum and sum of the softmax, on the matrix cores, the token axis cut into
// equal shares. What bounds it is reading K and V once.
//
// Shares. The tokens of a (sequence, kv head) are tiles of TW; all tiles of the call, sequence by sequence and head by head,
// are one line, and wave w of W takes the w-th W-th of it. The line is laid out on the device from the lengths, so the
// split follows the lengths that are there when the kernel (or a captured graph) runs, a ragged batch is as balanced as
// an even one, and one long sequence fills the chip. A wave walks its share tile by tile, from one head into the next, with
// the next tile's K always in flight, and meets no barrier; four waves to a CU keep enough loads in flight (64 KB; eight at
// D = 64). Heads that end up in several waves leave {maximum, sum, unnormalised output} of each in the workspace and
// kv_join_kernel joins them.
//
// Products. Query heads of one kv head are the columns of a 16-wide tile, or of two where a group has more than 16 (one over
// 32 takes several passes over K and V). A group under 16 leaves columns idle: the matrix cores have the room, the reads
// of K and V are what counts.
//   S^T = K Q^T: a lane of the A operand is a token (lane & 15) with 16 bytes of its row at 16 (lane >> 4) + 64 j; the
//     order of the summed dimension is free as long as Q has the same, so both are plain 16-byte loads.
//   O^T += V^T P^T: the C layout of S^T leaves lane (g = lane >> 4, head = lane & 15) with rows 4 g + i of every 16, which
//     is the B operand as it stands when the summed tokens are taken in that order. Row r of 16-token block s of a
//     tile is token 8 (r / 4) + 4 s + r % 4, so a lane's eight tokens are consecutive: they share a page (pages hold 8 or
//     more), their scores leave in one piece. A lane loads VEC consecutive dims of each of its tokens, 16 lanes
//     a whole row; for 16-bit types the 8 x VEC block it holds is transposed in registers (one v_perm per dword). No
//     LDS, no barrier in the loop.
// fp32 runs on v_mfma_f32_16x16x4_f32, 16-bit types on the 16x16x32 ones.

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef f16_t f16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int AT_WAVES = 4;

// Workgroups to a CU, which share its 160 KB of LDS. A tile of D = 64 is half as much to have in flight: two (32 x 16384
// tokens of 8 heads: 188 us with one, 169 with two, 174 with three). Above, a second one costs more in parts to join than it
// brings (64 heads over 4 of 128, 64 x 4096: 65 us with one, 73 with two).
constexpr int attend_per_cu(int dim) { return dim == 64 ? 2 : 1; }

// Query heads of a group that one pass over K and V serves: 32 where there are more than 16 (32 heads over one of 128, 32 x
// 8192 tokens, bf16: 32 us in one pass, 39 in two), but at fp32 and D = 256, where two tiles' sums do not fit the registers
// (124 us against 119). 16-bit types at 256 just about do: ten registers go to scratch, and one pass still wins everywhere (32 x
// 8192 tokens, bf16, weights collected: 84 us against 117 with 32 heads, 71 against 112 with 17; 128 x 512 47 against 50).
__host__ __device__ constexpr int attend_columns(int dtype, int dim, int group) { return group > 16 && !(dtype == KV_F32 && dim == 256) ? 32 : 16; }
static int attend_columns(const KvPool& p, int group) { return attend_columns(p.dtype, p.dim, group); }
static int attend_passes(const KvPool& p, int group) { return (group + attend_columns(p, group) - 1) / attend_columns(p, group); }

template <int DT, int D>
struct AttendShape {
    static constexpr int ES = DT == KV_F32 ? 4 : 2;
    static constexpr int TW = DT == KV_F32 ? 16 : 32;          // tokens of a tile
    static constexpr int VEC = DT != KV_F32 && D >= 128 ? 8 : 4;   // dims per lane and V row
    static constexpr int NX = D / (16 * VEC);
    static constexpr int NACC = D / 16;
    static constexpr int KL = D * ES / 64;                     // 16-byte loads per lane and K row
    static constexpr int GATHER = 39 * 1024 / attend_per_cu(D);        // bytes of scores a wave gathers in LDS
};

int attend_tile(int dtype) { return dtype == KV_F32 ? AttendShape<KV_F32, 64>::TW : AttendShape<KV_BF16, 64>::TW; }

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int x) { return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }

// Inclusive sums over the lanes of a wave: within rows of 16 by shifts of 1, 2, 4, 8, then row ends into the rows behind.
__device__ __forceinline__ int wave_scan(int x) {
    x = dpp_add<0x111, 0xf>(x);
    x = dpp_add<0x112, 0xf>(x);
    x = dpp_add<0x114, 0xf>(x);
    x = dpp_add<0x118, 0xf>(x);
    x = dpp_add<0x142, 0xa>(x);
    return dpp_add<0x143, 0xc>(x);
}

__device__ __forceinline__ int wave_sum(int x) { return __builtin_amdgcn_readlane(wave_scan(x), 63); }

template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_max(int x) { return max(x, __builtin_amdgcn_update_dpp(-0x7fffffff - 1, x, CTRL, ROWS, 0xf, false)); }

__device__ __forceinline__ int wave_max(int x) {
    x = dpp_max<0x118, 0xf>(dpp_max<0x114, 0xf>(dpp_max<0x112, 0xf>(dpp_max<0x111, 0xf>(x))));
    return __builtin_amdgcn_readlane(dpp_max<0x143, 0xc>(dpp_max<0x142, 0xa>(x)), 63);
}

// f over the four lanes of a column (lane, lane ^ 16, lane ^ 32, lane ^ 48), for each of them.
template <class F>
__device__ __forceinline__ float column_all(float x, F f) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = f(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return f(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// The line of tiles: sequence b has tiles(len_b) of them for each of H head groups.
struct Line {
    int base, rem;                       // share w: base tiles, and one more for w < rem
    __device__ __forceinline__ Line(int U, int W) : base(U / W), rem(U % W) {}
    __device__ __forceinline__ int begin(int w) const { return w * base + min(w, rem); }
    __device__ __forceinline__ int share_of(int u) const {
        const int big = rem * (base + 1);
        return u < big ? u / (base + 1) : rem + (u - big) / base;
    }
};

__device__ __forceinline__ int tiles_of(const KvTable& tb, const int32_t* lengths, int b, int cap, int tw) {
    const int n = lengths[b];
    return n <= 0 ? 0 : (min(n, cap) + tw - 1) / tw;
}

template <int DT>
struct Mma;
template <>
struct Mma<KV_BF16> {
    static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mma<KV_F16> {
    static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
};
template <>
struct Mma<KV_F32> {
    static __device__ __forceinline__ f32x4 run(u32x4 a, u32x4 b, f32x4 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
        return c;
    }
};

// A weight as a sum of 16-bit numbers, each what the ones before leave: three of bf16 hold all its 24 bits, two of fp16 hold it to
// 2^-22. A matrix instruction each; the kernel waits for memory either way (64 x 4096 tokens of 8 heads of 128, bf16: 178.7 us with
// two, 16 bits, and 179.1 with three; one sequence of 8190 15.4 and 15.5; the short kernel at 16 x 8 heads over 128 slots 6.07 and
// 6.17).
template <typename V8, int N>
__device__ __forceinline__ void split8(const float* p, u32x4 (&parts)[N]) {
    float rest[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) rest[i] = p[i];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        V8 h;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            h[i] = (decltype(h[0] + h[0]))rest[i];
            rest[i] -= (float)h[i];
        }
        parts[n] = __builtin_bit_cast(u32x4, h);
    }
}

// What a wave holds of one head group and tile, and the steps of a tile. NG 16-wide tiles of heads: a lane has heads
// col + 16 g of the group's stretch, g < NG.
template <int DT, int D, int NG>
struct AttendWave {
    using S = AttendShape<DT, D>;
    static constexpr int TW = S::TW, VEC = S::VEC, NX = S::NX, NACC = S::NACC, KL = S::KL, ES = S::ES;
    static constexpr int NS = TW / 16, NV = TW / 4;  // 16-token blocks; tokens a lane holds, NV (lane >> 4) and on
    static constexpr int COLS = 16 * NG;
    static constexpr int WEIGHT_PARTS = DT == KV_BF16 ? 3 : 2;       // (16-bit types)
    // fp16 weights are kept 2^14 too large (the sums with them): at most 16384, and 2^-28 is still a normal number, so that
    // many small weights beside a large one are not lost
    static constexpr float OFF = DT == KV_F16 ? 14.f : 0.f;
    typedef typename std::conditional<VEC * ES == 16, u32x4, u32x2>::type vload_t;

    const KvPool& p;
    const KvTable& tb;
    const KvAttend& a;
    int lane, col, grp, ktok;                        // ktok: token of this lane's K row, block 0
    int ngrp, hq;
    u32x4 kf[NS][KL], qf[NG][KL];
    vload_t vf[NV][NX];
    float sc[NG][NV];                                // scores of the lane's tokens, in units of ln 2
    float m[NG], l[NG], ref[NG];                     // maximum (column-wide), sum (this lane's), exponent the sums refer to
    f32x4 acc[NG][NACC];                             // component i of x VEC + e: dim 16 VEC x + (4 grp + i) VEC + e

    __device__ __forceinline__ AttendWave(const KvPool& p_, const KvTable& tb_, const KvAttend& a_) : p(p_), tb(tb_), a(a_) {
        lane = threadIdx.x & 63;
        col = lane & 15;
        grp = lane >> 4;
        ktok = NS == 2 ? 8 * (col >> 2) + (col & 3) : col;
        ngrp = (a.group + COLS - 1) / COLS;
        hq = p.heads * a.group;
        reset();
    }
    __device__ __forceinline__ void reset() {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            m[g] = -INFINITY;
            l[g] = 0.f;
#pragma unroll
            for (int n = 0; n < NACC; ++n) acc[g][n] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ int head0(int hg) const { return hg / ngrp * a.group + hg % ngrp * COLS; }
    __device__ __forceinline__ int heads(int hg) const { return min(COLS, a.group - hg % ngrp * COLS); }

    // Page of slot t of sequence b; of its last one where t lies behind it, so that every row below is in the pool (and of page
    // 0 where the id is bad): what is masked is read and thrown away. A lane's NV tokens share a page.
    __device__ __forceinline__ int page_of(int b, int len, int t) const { return tb.table[(int64_t)b * tb.ld + (min(t, len - 1) >> p.page_shift)]; }
    __device__ __forceinline__ bool bad_id(int page) const { return (unsigned)page >= (unsigned)p.num_pages; }
    __device__ __forceinline__ int k_page(int b, int len, int t) const { return page_of(b, len, t + ktok); }
    __device__ __forceinline__ int v_page(int b, int len, int t) const { return page_of(b, len, t + NV * grp); }

    __device__ __forceinline__ void load_q(int b, int hg) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int head = head0(hg) + min(col + 16 * g, heads(hg) - 1);      // (idle columns: the last head again)
            const char* q = (const char*)a.q + ((int64_t)b * a.q_st[0] + (int64_t)head * a.q_st[1]) * ES + grp * 16;
#pragma unroll
            for (int j = 0; j < KL; ++j) qf[g][j] = *reinterpret_cast<const u32x4*>(q + j * 64);
        }
    }
    // K and V rows of the tile at t. (Past the caches: read once.)
    __device__ __forceinline__ void load_k(int hg, int t, int page) {
        const char* r = (const char*)p.k + ((int64_t)(hg / ngrp) * p.k_st[1] + (int64_t)(bad_id(page) ? 0 : page) * p.k_st[0] +
                                            (int64_t)((t + ktok) & (p.page_size - 1)) * p.k_st[2]) * ES + grp * 16;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < KL; ++j)
                kf[s][j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(r + 4 * s * p.k_st[2] * ES + j * 64));
    }
    __device__ __forceinline__ void load_v(int hg, int t, int page) {
        const char* r = (const char*)p.v + ((int64_t)(hg / ngrp) * p.v_st[1] + (int64_t)(bad_id(page) ? 0 : page) * p.v_st[0] +
                                            (int64_t)((t + NV * grp) & (p.page_size - 1)) * p.v_st[2]) * ES + col * VEC * ES;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int x = 0; x < NX; ++x)
                vf[i][x] = __builtin_nontemporal_load(reinterpret_cast<const vload_t*>(r + i * p.v_st[2] * ES + x * 16 * VEC * ES));
    }
    __device__ __forceinline__ void scores() {
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < KL; ++j) c = Mma<DT>::run(kf[s][j], qf[g][j], c);
#pragma unroll
                for (int i = 0; i < 4; ++i) sc[g][4 * s + i] = c[i] * a.scale2;
            }
    }
    // Slots behind the length or of a bad page: score -inf, and no row that 0 could be multiplied with to give NaN.
    __device__ __forceinline__ void mask(int len, int t, int page) {
        const int tok = t + NV * grp;
        const bool bad = bad_id(page);
        if (t + TW <= len && !__any(bad)) return;
        if (bad && tok < len) atomicOr(p.status, KV_BAD_PAGE);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (bad || tok + i >= len) {
#pragma unroll
                for (int g = 0; g < NG; ++g) sc[g][i] = -INFINITY;
#pragma unroll
                for (int x = 0; x < NX; ++x) vf[i][x] = vload_t{};
            }
    }
    // The lane's scores of head tile g as they go into a [head][TW] table.
    __device__ __forceinline__ void put_scores(int g, f32x4* to) const {
#pragma unroll
        for (int s = 0; s < NS; ++s) to[s] = f32x4{sc[g][4 * s], sc[g][4 * s + 1], sc[g][4 * s + 2], sc[g][4 * s + 3]};
    }
    __device__ __forceinline__ void accumulate() {
        float pr[NG][NV];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            float mx = sc[g][0];
#pragma unroll
            for (int i = 1; i < NV; ++i) mx = fmaxf(mx, sc[g][i]);
            if (__any(mx > m[g])) {
                const float mn = fmaxf(m[g], column_all(mx, [](float x, float y) { return fmaxf(x, y); }));
                const float alpha = m[g] == -INFINITY ? 0.f : ex2(m[g] - mn);
                m[g] = mn;
                l[g] *= alpha;
#pragma unroll
                for (int n = 0; n < NACC; ++n) acc[g][n] *= alpha;
            }
            ref[g] = m[g] == -INFINITY ? 0.f : m[g] - OFF;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < NV; ++i) { pr[g][i] = ex2(sc[g][i] - ref[g]); sum += pr[g][i]; }
            l[g] += sum;
        }
        if constexpr (DT == KV_F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < NX; ++x)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int g = 0; g < NG; ++g)
                            acc[g][4 * x + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vf[i][x][e]), pr[g][i], acc[g][4 * x + e], 0, 0, 0);
        } else {
            u32x4 w[NG][WEIGHT_PARTS];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if constexpr (DT == KV_BF16) split8<bf16x8>(pr[g], w[g]);
                else split8<f16x8>(pr[g], w[g]);
            }
#pragma unroll
            for (int x = 0; x < NX; ++x)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    u32x4 v;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        v[i] = __builtin_amdgcn_perm(vf[2 * i + 1][x][e >> 1], vf[2 * i][x][e >> 1], e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
                    for (int n = 0; n < WEIGHT_PARTS; ++n)
#pragma unroll
                        for (int g = 0; g < NG; ++g) acc[g][x * VEC + e] = Mma<DT>::run(v, w[g][n], acc[g][x * VEC + e]);
                }
        }
    }
    __device__ __forceinline__ float sum_of(int g) const { return column_all(l[g], [](float x, float y) { return x + y; }); }
    __device__ __forceinline__ float exponent_of(int g) const { return m[g] == -INFINITY ? -INFINITY : m[g] - OFF; }
};

template <int DT>
__device__ __forceinline__ void store_out(void* out, int64_t at, float x) {
    if constexpr (DT == KV_F32) ((float*)out)[at] = x;
    else if constexpr (DT == KV_BF16) ((bf16_t*)out)[at] = (bf16_t)x;
    else ((f16_t*)out)[at] = (f16_t)x;
}

// A tile of the line.
struct Cursor {
    int b, hg, tile;                     // sequence, head group, tile of its tokens
    int nb, len;                         // tiles and tokens of the sequence
};

// What it reaches, with the weights collected: 32 sequences of up to 32768 tokens (655 k in all), 32 heads over 8 of 128, bf16,
// pages of 32: 405 us for 2.65 GB of K and V, 6.5 TB/s (and 84 MB of scores written); without the weights 32 x 16384 tokens
// 6.4 / 6.85 / 6.7 TB/s at pages of 16 / 32 / 128, 5.8 where a page keeps its heads side by side. A plain read of as many
// bytes in order reaches 7.0 to 7.4. A call of nothing much takes 8 us here, five loads one after the other.
template <int DT, int D, bool MASS, int NG>
__global__ __launch_bounds__(64 * AT_WAVES) void kv_attend_kernel(const KvPool p, const KvTable tb, const KvAttend a) {
    using S = AttendShape<DT, D>;
    using Wave = AttendWave<DT, D, NG>;
    constexpr int TW = S::TW, VEC = S::VEC, NX = S::NX, ES = S::ES, COLS = Wave::COLS;
    __shared__ f32x4 gathered[MASS ? AT_WAVES : 1][MASS ? S::GATHER / 16 : 1];
    Wave x(p, tb, a);
    const int lane = x.lane, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int cap = tb.max_pages << p.page_shift, w = blockIdx.x * AT_WAVES + wave;
    const int H = p.heads * x.ngrp, hq = x.hq;

    // the line, from the tiles of the first 64 sequences (a lane each; their lengths stay at hand) and, 64 by 64, the rest
    auto tiles = [](int len) { return (len + TW - 1) / TW; };
    const int raw64 = lane < tb.B ? a.lengths[lane] : 0, len64 = max(0, min(raw64, cap));
    auto len_of = [&](int b) INLINE { return b < 64 ? __builtin_amdgcn_readlane(len64, b) : __builtin_amdgcn_readfirstlane(max(0, min(a.lengths[b], cap))); };
    const int first64 = tiles(len64), scan64 = wave_scan(first64);
    int total = __builtin_amdgcn_readlane(scan64, 63);
    if (tb.B > 64) {
        int more = 0;
        for (int i = lane + 64; i < tb.B; i += 64) more += tiles_of(tb, a.lengths, i, cap, TW);
        total += wave_sum(more);
    }
    const Line line(total * H, gridDim.x * AT_WAVES);
    const int u0 = line.begin(w), u1 = line.begin(w + 1);

    // the check of the lengths, and sequences without tokens
    if (w == 0 && len64 != raw64) atomicOr(p.status, KV_BAD_LENGTH);
    for (int b = w; b < tb.B; b += gridDim.x * AT_WAVES) {
        if (b >= 64) (void)clamp_len(a.lengths[b], cap, p.status, lane == 0);
        if (len_of(b)) continue;
        for (int i = lane; i < hq * D * ES / 4; i += 64) ((uint32_t*)a.out)[(int64_t)b * (hq * D * ES / 4) + i] = 0;
        for (int i = lane; i < hq; i += 64) a.lse[(int64_t)b * hq + i] = -INFINITY;
    }
    if (u0 == u1) return;

    int b0 = 0, before = 0;                          // the sequence of tile u0, and the tiles before it
    for (int n = first64, inc = scan64;;) {
        const unsigned long long hit = __ballot(before + inc * H > u0);
        if (hit) {
            const int at = __ffsll(hit) - 1;
            b0 += at;
            before += __builtin_amdgcn_readlane(inc - n, at) * H;
            break;
        }
        before += __builtin_amdgcn_readlane(inc, 63) * H;
        b0 += 64;
        n = b0 + lane < tb.B ? tiles_of(tb, a.lengths, b0 + lane, cap, TW) : 0;
        inc = wave_scan(n);
    }
    auto at_sequence = [&](Cursor& c) INLINE {
        c.len = len_of(c.b);
        c.nb = tiles(c.len);
    };
    // (called for tiles of the share only, so there is a next one)
    auto advance = [&](Cursor c) INLINE {
        if (++c.tile == c.nb) {
            c.tile = 0;
            if (++c.hg == H) {
                c.hg = 0;
                do {
                    ++c.b;
                    at_sequence(c);
                } while (c.nb == 0);
            }
        }
        return c;
    };
    Cursor cur;
    cur.b = __builtin_amdgcn_readfirstlane(b0);
    at_sequence(cur);
    cur.hg = (u0 - before) / cur.nb;
    cur.tile = (u0 - before) % cur.nb;
    auto k_page = [&](const Cursor& c) INLINE { return x.k_page(c.b, c.len, c.tile * TW); };
    auto v_page = [&](const Cursor& c) INLINE { return x.v_page(c.b, c.len, c.tile * TW); };

    // Scores for the weights of `mass`: [tile][score_rows][TW]. A wave gathers those of tiles gather0, gather0 + 1, ... and
    // writes them out when there is room for no more, and at the end: a trickle of writes among the reads costs far more of
    // the memory's time than their bytes.
    const int tile_vecs = a.score_rows * TW / 4, room = S::GATHER / 16 / tile_vecs;
    int gather0 = u0;
    auto flush = [&](int upto) INLINE {
        f32x4* to = (f32x4*)a.scores + (int64_t)gather0 * tile_vecs;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        for (int j = lane; j < (upto - gather0) * tile_vecs; j += 64) to[j] = gathered[wave][j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        gather0 = upto;
    };

    int vpage = v_page(cur);
    x.load_q(cur.b, cur.hg);
    x.load_k(cur.hg, cur.tile * TW, k_page(cur));
    Cursor next = u0 + 1 < u1 ? advance(cur) : cur;
    int kpage1 = k_page(next), vpage1 = v_page(next);
    int seg0 = u0;                                   // where this wave began with the head

    for (int u = u0;;) {
        // pages of the tile after the next, then V of this one: in flight during the first product
        const bool last = u + 1 == u1;
        const Cursor next2 = u + 2 < u1 ? advance(next) : next;
        const int kpage2 = k_page(next2), vpage2 = v_page(next2);
        x.load_v(cur.hg, cur.tile * TW, vpage);
        x.scores();
        const bool end = last || next.tile == 0;     // of the head, as far as it is this wave's
        const int nh = x.heads(cur.hg);
        if (!last) {
            if (end) x.load_q(next.b, next.hg);
            x.load_k(next.hg, next.tile * TW, kpage1);
        }
        x.mask(cur.len, cur.tile * TW, vpage);
        if constexpr (MASS) {
            if (u - gather0 == room) flush(u);
#pragma unroll
            for (int g = 0; g < NG; ++g)
                if (x.col + 16 * g < nh)
                    x.put_scores(g, gathered[wave] + (u - gather0) * tile_vecs + ((x.col + 16 * g) * TW + Wave::NV * x.grp) / 4);
        }
        x.accumulate();
        if (end) {
            const bool whole = seg0 + cur.nb == u + 1;
            const int d0 = 4 * x.grp * VEC, slot = 2 * w + (seg0 != u0);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float L = x.sum_of(g);
                const int c = x.col + 16 * g;
                if (c >= nh) continue;
                if (whole) {
                    // no weight at all (every page bad, or every score -inf): as a row without tokens
                    const float inv = L == 0.f ? 0.f : 1.f / L;
                    const int64_t head = (int64_t)cur.b * hq + x.head0(cur.hg) + c;
                    if (x.grp == 0) a.lse[head] = L == 0.f ? -INFINITY : log_sum(x.ref[g], L);
#pragma unroll
                    for (int n = 0; n < NX; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < VEC; ++e)
                                store_out<DT>(a.out, head * D + n * 16 * VEC + d0 + i * VEC + e, x.acc[g][n * VEC + e][i] * inv);
                } else {
                    if (x.grp == 0) a.part_ml[slot * COLS + c] = float2{x.exponent_of(g), L};
                    float* po = a.part_out + ((int64_t)slot * a.score_rows + c) * D + d0;
#pragma unroll
                    for (int n = 0; n < NX; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int e = 0; e < VEC; ++e) po[n * 16 * VEC + i * VEC + e] = x.acc[g][n * VEC + e][i];
                }
            }
            if (last) break;
            seg0 = u + 1;
            x.reset();
        }
        ++u;
        cur = next;
        next = next2;
        vpage = vpage1;
        kpage1 = kpage2;
        vpage1 = vpage2;
    }
    if constexpr (MASS) flush(u1);
}

// {reference exponent, sum} of two disjoint sets of weights as one.
__device__ __forceinline__ float2 stat_join(float2 x, float2 y) {
    const float M = fmaxf(x.x, y.x), ref = M == -INFINITY ? 0.f : M;
    return float2{M, x.y * ex2(x.x - ref) + y.y * ex2(y.x - ref)};
}

// Short memories (an utterance's encoder outputs): a workgroup has a head group to itself, tile after tile dealt to its eight
// waves, and everything that takes the long way a workspace and a second launch stays in its LDS: the waves' parts and the
// scores of the whole memory, from which the weights are added to `mass`. Bound by its loads one after the other. Long way
// against this one, with the weights, lengths from an eighth of the slots to all of them: 16 x 8 heads over 128 slots of 128,
// bf16, four query heads each: 10.7 us, 6.5; 64 x 8: 15.8, 11.3; 64 x 8 over 512 slots of 64: 18.9, 13.7.
constexpr int SHORT_WAVES = 8;

// Tokens of memory that the short way takes: as many as have 64 KB of K, two rounds of the waves' tiles at D = 64, one at 128.
// (Twice as many: 32 x 1 heads over 512 slots of 128, bf16: 10.6 us the long way, 11.2 the short; over 256 of fp32 10.7 and 12.5.)
// And how many heads, to a CU: at D = 128 a CU holds one workgroup at a time (1024 heads, 4 a CU, over 256 slots, bf16: 25.7 us
// the long way, 27.3 the short; 512: 16.5 and 15.0), at 64 three (4096 over 64 slots, no weights: 23.1 and 26.9; 2048: 14.9 and
// 15.3, with weights 20.2 and 16.7). At D = 256 eight waves' registers do not fit a CU's (32 x 1 over 128 to 256 slots lost).
constexpr int short_slots(int dtype, int dim) { return 65536 / (dim * (dtype == KV_F32 ? 4 : 2)); }
constexpr int short_per_cu(int dim) { return dim == 64 ? 8 : dim == 128 ? 2 : 0; }

template <int DT, int D, bool MASS>
__global__ __launch_bounds__(64 * SHORT_WAVES) void kv_attend_short_kernel(const KvPool p, const KvTable tb, const KvAttend a) {
    using Wave = AttendWave<DT, D, 1>;
    constexpr int NW = SHORT_WAVES, HALF = NW / 2, TW = Wave::TW, VEC = Wave::VEC, NACC = Wave::NACC, STEP = NW * TW;
    __shared__ f32x4 parts[HALF][NACC][64];          // a wave's accumulators, by lane
    __shared__ float2 ml[NW][16];
    __shared__ f32x4 score[MASS ? short_slots(DT, D) * 16 / 4 : 1];      // [tile][head][TW]
    __shared__ float lse2[16];
    Wave x(p, tb, a);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = blockIdx.x / p.heads, h = blockIdx.x % p.heads, nh = a.group;
    const int len = clamp_len(a.lengths[b], tb.max_pages << p.page_shift, p.status, h == 0 && tid == 0);
    const int64_t head0 = (int64_t)b * x.hq + h * a.group;
    int t = wave * TW, kpage, vpage;
    if (t < len) {
        kpage = x.k_page(b, len, t);
        vpage = x.v_page(b, len, t);
        x.load_q(b, h);
        x.load_k(h, t, kpage);
        kpage = x.k_page(b, len, t + STEP);
        for (;; t += STEP) {
            const int kpage2 = x.k_page(b, len, t + 2 * STEP), vpage2 = x.v_page(b, len, t + STEP);
            const bool last = t + STEP >= len;
            x.load_v(h, t, vpage);
            x.scores();
            if (!last) x.load_k(h, t + STEP, kpage);
            x.mask(len, t, vpage);
            if (MASS && x.col < nh) x.put_scores(0, score + ((t / TW * 16 + x.col) * TW + Wave::NV * x.grp) / 4);
            x.accumulate();
            if (last) break;
            kpage = kpage2;
            vpage = vpage2;
        }
    }
    // the waves' parts: the upper four into the lower four, those into the output
    const float2 own = {x.exponent_of(0), x.sum_of(0)};
    if (wave >= HALF) {
        if (x.grp == 0) ml[wave][x.col] = own;
#pragma unroll
        for (int n = 0; n < NACC; ++n) parts[wave - HALF][n][x.lane] = x.acc[0][n];
    }
    __syncthreads();
    if (wave < HALF) {
        const float2 other = ml[wave + HALF][x.col], both = stat_join(own, other);
        const float ref = both.x == -INFINITY ? 0.f : both.x, f = ex2(own.x - ref), g = ex2(other.x - ref);
#pragma unroll
        for (int n = 0; n < NACC; ++n) x.acc[0][n] = x.acc[0][n] * f + parts[wave][n][x.lane] * g;
        if (x.grp == 0) ml[wave][x.col] = both;
#pragma unroll
        for (int n = 0; n < NACC; ++n) parts[wave][n][x.lane] = x.acc[0][n];
    }
    __syncthreads();
    // {exponent, sum} of head c; a memory without tokens, or without a score above -inf, has sum 0
    auto total = [&](int c) INLINE {
        float2 y = ml[0][c];
#pragma unroll
        for (int i = 1; i < HALF; ++i) y = stat_join(y, ml[i][c]);
        return y;
    };
    for (int i = tid; i < NACC * 64; i += 64 * NW) {
        const int n = i >> 6, l = i & 63, c = l & 15;
        if (c >= nh) continue;
        const float2 y = total(c);
        const float ref = y.x == -INFINITY ? 0.f : y.x, inv = y.y == 0.f ? 0.f : 1.f / y.y;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < HALF; ++w) o += parts[w][n][l] * ex2(ml[w][c].x - ref);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            store_out<DT>(a.out, (head0 + c) * D + n / VEC * 16 * VEC + (4 * (l >> 4) + e) * VEC + n % VEC, o[e] * inv);
    }
    if (tid < nh) {
        const float2 y = total(tid);
        const float ref = y.x == -INFINITY ? 0.f : y.x;
        a.lse[head0 + tid] = y.y == 0.f ? -INFINITY : log_sum(ref, y.y);
        lse2[tid] = y.y == 0.f ? 0.f : ref + __log2f(y.y);         // (no weight at all: every score is -inf)
    }
    if constexpr (MASS) {
        __syncthreads();
        float* mass = a.mass + ((int64_t)b * p.heads + h) * a.side_ld;
        for (int s = tid; s < len; s += 64 * NW) {
            const float* sc = (const float*)score + (s / TW * 16) * TW + s % TW;
            float w = 0.f;
            for (int c = 0; c < nh; ++c) w += ex2(sc[c * TW] - lse2[c]);
            mass[s] += w;
        }
    }
}

// Parts of one (sequence, head group): waves w0 .. w1, and where part w of them lies in the workspace.
struct Parts {
    int first, w0, w1;                   // first tile
    __device__ __forceinline__ int slot(const Line& line, int w) const { return 2 * w + (line.begin(w) < first); }
};

// The first `joins` workgroups join the parts of a (sequence, query head): one each, or, WAVES, one per wave. The rest
// do mass_tokens tokens (a multiple of 1024) of mass[b][h] += sum over the query heads of h of exp(score - lse) each, from
// the scores that kv_attend_kernel left. The lse of a head in parts is computed by whoever needs it (a few values), so
// that both fit one launch. Short work that waits for one dependent load after the other, so every step loads all it needs
// at once: a part's {exponent, sum} per lane, eight or sixteen rows of the parts' outputs per lane, four tokens of a head's
// scores per lane, the first of them beside the statistics. (5 us where there is little to do; 31 us for the 126 MB of scores and masses of 32 sequences up to 32768.)
template <int D, bool WAVES>
__global__ __launch_bounds__(256) void kv_join_kernel(const KvPool p, const KvTable tb, const KvAttend a, int W, int tw, int joins,
                                                      int mass_tokens) {
    constexpr int COLS = D / 4;                      // a lane joins four dims of every ROWS-th part
    constexpr int ROWS = (WAVES ? 64 : 256) / COLS;
    constexpr int AHEAD = WAVES ? 8 : 16;            // parts a lane loads at once
    __shared__ f32x4 sums[WAVES ? 1 : ROWS][WAVES ? 1 : COLS];
    __shared__ float lse2[32];
    __shared__ float2 wave_stat[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cap = tb.max_pages << p.page_shift;
    const int cols = attend_columns(p.dtype, D, a.group), ngrp = (a.group + cols - 1) / cols, H = p.heads * ngrp, hq = p.heads * a.group;
    const bool join = (int)blockIdx.x < joins;
    int b, kvh, h0 = 0, t0 = 0;                      // h0: query head within the group
    if (join) {
        const int i = WAVES ? blockIdx.x * 4 + wave : blockIdx.x;
        b = i / hq;
        if (b >= tb.B) return;                       // (no barrier where a wave has its own head)
        kvh = i % hq / a.group;
        h0 = i % hq % a.group;
    } else {
        const int chunks = (cap + mass_tokens - 1) / mass_tokens, i = blockIdx.x - joins;
        b = i / (chunks * p.heads);
        kvh = i / chunks % p.heads;
        t0 = i % chunks * mass_tokens;
    }
    b = __builtin_amdgcn_readfirstlane(b);
    const int len64 = lane < tb.B ? max(0, min(a.lengths[lane], cap)) : 0;
    const int len = b < 64 ? __builtin_amdgcn_readlane(len64, b) : max(0, min(a.lengths[b], cap));
    if (t0 >= len) return;
    const int nb = (len + tw - 1) / tw;
    if (join && nb == 1) return;                     // a single tile is never in parts
    int total = (len64 + tw - 1) / tw, before = lane < b ? total : 0;
    for (int i = lane + 64; i < tb.B; i += 64) {
        const int n = tiles_of(tb, a.lengths, i, cap, tw);
        total += n;
        before += i < b ? n : 0;
    }
    total = wave_sum(total);
    before = wave_sum(before);
    const Line line(total * H, W);
    auto parts_of = [&](int g) {
        Parts q;
        q.first = before * H + (kvh * ngrp + g) * nb;
        q.w0 = line.share_of(q.first);
        q.w1 = line.share_of(q.first + nb - 1);
        return q;
    };
    // {exponent, sum} of head c over parts from, from + step, ...: the caller's lanes together, then the wave's
    auto stats = [&](const Parts& q, int c, int from, int step) {
        float2 x = {-INFINITY, 0.f};
        for (int w = q.w0 + from; w <= q.w1; w += step) x = stat_join(x, a.part_ml[q.slot(line, w) * cols + c]);
        for (int o = 32; o; o >>= 1) x = stat_join(x, float2{__shfl_xor(x.x, o), __shfl_xor(x.y, o)});
        return x;
    };
    if (join) {
        const Parts q = parts_of(h0 / cols);
        if (q.w0 == q.w1) return;
        const int c = h0 % cols, n = q.w1 - q.w0 + 1;
        const int id = WAVES ? lane : tid, d4 = id % COLS, k = id / COLS;
        f32x4 v[AHEAD];
        float f[AHEAD];
        auto load = [&](int i) INLINE {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) {
                const int slot = q.slot(line, q.w0 + min(i + j * ROWS, n - 1));      // (beyond the last part: not added)
                v[j] = *reinterpret_cast<const f32x4*>(a.part_out + ((int64_t)slot * a.score_rows + c) * D + 4 * d4);
                f[j] = a.part_ml[slot * cols + c].x;
            }
        };
        load(k);                                     // beside the statistics
        float2 x = stats(q, c, WAVES ? lane : tid, WAVES ? 64 : 256);
        if (!WAVES) {
            if (lane == 0) wave_stat[wave] = x;
            __syncthreads();
            x = stat_join(stat_join(wave_stat[0], wave_stat[1]), stat_join(wave_stat[2], wave_stat[3]));
        }
        const float ref = x.x == -INFINITY ? 0.f : x.x, L = x.y;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int i = k;;) {
#pragma unroll
            for (int j = 0; j < AHEAD; ++j)
                if (i + j * ROWS < n) o += v[j] * ex2(f[j] - ref);
            i += AHEAD * ROWS;
            if (i >= n) break;
            load(i);
        }
        if constexpr (WAVES) {
#pragma unroll
            for (int step = COLS; step < 64; step *= 2)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], step);
        } else {
            sums[k][d4] = o;
            __syncthreads();
        }
        if (k) return;
        if constexpr (!WAVES) {
#pragma unroll
            for (int i = 1; i < ROWS; ++i) o += sums[i][d4];
        }
        o *= L == 0.f ? 0.f : 1.f / L;
        const int64_t head = (int64_t)b * hq + kvh * a.group + h0;
        if (id == 0) a.lse[head] = L == 0.f ? -INFINITY : log_sum(ref, L);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int64_t at = head * D + 4 * d4 + e;
            if (p.dtype == KV_F32) ((float*)a.out)[at] = o[e];
            else if (p.dtype == KV_BF16) ((bf16_t*)a.out)[at] = (bf16_t)o[e];
            else ((f16_t*)a.out)[at] = (f16_t)o[e];
        }
        return;
    }
    float* mass = a.mass + ((int64_t)b * p.heads + kvh) * a.side_ld;
    const bool whole4 = ((uintptr_t)mass & 15) == 0;
    for (int g = 0; g < ngrp; ++g) {
        const Parts q = parts_of(g);
        const int nh = min(cols, a.group - cols * g);
        for (int c = wave; c < nh; c += 4) {
            float x;
            if (q.w0 == q.w1) x = a.lse[(int64_t)b * hq + kvh * a.group + cols * g + c] * LOG2E;
            else {
                const float2 st = stats(q, c, lane, 64);
                x = st.y == 0.f ? -INFINITY : (st.x == -INFINITY ? 0.f : st.x) + __log2f(st.y);
            }
            // no weight at all: every score is -inf, and so is every difference to a finite number
            if (lane == 0) lse2[c] = x == -INFINITY ? 0.f : x;
        }
        __syncthreads();
        for (int t = t0 + 4 * tid; t < min(len, t0 + mass_tokens); t += 1024) {
            const float* s = a.scores + (int64_t)(q.first + t / tw) * a.score_rows * tw + t % tw;
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int c = 0; c < nh; ++c) {           // (tiles are multiples of 4 tokens: four scores lie together)
                const f32x4 x = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(s + c * tw));
#pragma unroll
                for (int e = 0; e < 4; ++e) sum[e] += ex2(x[e] - lse2[c]);
            }
            if (whole4 && t + 4 <= len) *reinterpret_cast<f32x4*>(mass + t) += sum;
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (t + e < len) mass[t + e] += sum[e];
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------
// evict

constexpr int EV_THREADS = 1024, EV_WAVES = EV_THREADS / 64;
constexpr int EV_LIST = 4096;            // keys that are looked at again from LDS
constexpr int EV_ROWS = 16;              // rows of 64 slots a wave holds in registers, at most
constexpr int EV_CHUNK = 8192;           // slots per workgroup where several share a head

// Order-preserving bits of a mass: NaN above everything, -0 as +0; protected slots above that. Never 0.
__device__ __forceinline__ uint32_t mass_key(float x) {
    if (x != x) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct SelectShared {
    uint32_t hist[2048];
    uint32_t list[EV_LIST];
    int wave_a[EV_WAVES], wave_b[EV_WAVES];
    uint32_t digit;
    int left, same, listed, newest;                  // same: keys with the digit
};

// One (sequence, kv head) as the select kernels see it.
struct Head {
    int len, n;
    const float* mass; const int32_t* pos;
    float* mass_out; int32_t* pos_out;
    int32_t* gaps; int32_t* late; int32_t* counts;
    int border;                                      // positions above it are protected
    __device__ __forceinline__ Head(const KvPool& p, const KvTable& tb, const KvEvict& a, int h, int b, bool report) {
        len = clamp_len(a.lengths[b], tb.max_pages << p.page_shift, p.status, report);
        n = min(len, a.budget);
        const int64_t row = (int64_t)b * p.heads + h;
        mass = a.mass + row * a.side_ld;
        pos = a.positions + row * a.side_ld;
        mass_out = a.mass_out + row * a.side_ld;
        pos_out = a.positions_out + row * a.side_ld;
        gaps = a.lists + row * 2 * a.list_ld;
        late = gaps + a.list_ld;
        counts = a.counts + 2 * row;
        border = 0x7fffffff;
    }
    __device__ __forceinline__ void protect(int newest, int recent) {
        if (recent > 0) border = (int)max((int64_t)newest - recent, (int64_t)(-0x7fffffff - 1));
    }
};

// f(i) for rows i < per of a wave, in groups of 4 (rows behind per up to a group's end too). i is a compile-time constant, as
// an index into registers has to be.
template <int R, int I = 0, class F>
__device__ __forceinline__ void for_rows(int per, F f) {
    if constexpr (I < R) {
        if (I < per) {
            f(std::integral_constant<int, I>{});
            f(std::integral_constant<int, I + 1>{});
            f(std::integral_constant<int, I + 2>{});
            f(std::integral_constant<int, I + 3>{});
            __builtin_amdgcn_sched_barrier(0);       // keeps one group's masks from living through all of them
            for_rows<R, I + 4>(per, f);
        }
    }
}

// A lane's slots of a head: rows of 64 slots, first + 64 i. Masses and positions come in once; keys are made of them.
template <int R>
struct Slots {
    float mass[R];
    int pos[R];
    uint32_t key[R];                                 // 0 for no slot
    int first, stop;                                 // slots from stop on are none
    // (rows behind per, and slots behind stop, read the last slot; the wave has slots, or nothing is read)
    __device__ __forceinline__ void load(const Head& h, int first_, int stop_, int per) {
        first = first_;
        stop = stop_;
        if (first - (int)(threadIdx.x & 63) >= stop) return;
        for_rows<R>(per, [&](auto i) INLINE {
            const int t = min(first + 64 * i, stop - 1);
            mass[i] = h.mass[t];
            pos[i] = h.pos[t];
        });
    }
    __device__ __forceinline__ int slot(int i) const { return first + 64 * i; }
    __device__ __forceinline__ int newest(int per) const {
        int x = -0x7fffffff - 1;
        for_rows<R>(per, [&](auto i) INLINE {
            if (i < per && slot(i) < stop) x = max(x, pos[i]);
        });
        return x;
    }
    // Made once, each of the passes below would be bound by making them again.
    __device__ __forceinline__ void make_keys(const Head& h, int per) {
        for_rows<R>(per, [&](auto i) INLINE {
            const uint32_t k = pos[i] > h.border ? 0xffffffffu : mass_key(mass[i]);
            key[i] = i < per && slot(i) < stop ? k : 0u;
        });
    }
};

// n and the set bits of a wave's mask below this lane's.
__device__ __forceinline__ int lanes_below(unsigned long long mask, int n) {
    return (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, (uint32_t)n));
}

// Counts a key's digit if `in`. Equal digits side by side (fresh tokens, protected ones) would queue for one counter: where
// a wave has only one digit it adds once.
__device__ __forceinline__ void count_digit(SelectShared& sh, bool in, uint32_t digit) {
    const unsigned long long who = __ballot(in);
    if (!who) return;
    const uint32_t one = (uint32_t)__builtin_amdgcn_readlane((int)digit, __ffsll(who) - 1);
    if (__ballot(in && digit == one) == who) {
        if ((threadIdx.x & 63) == 0) atomicAdd(&sh.hist[one], (uint32_t)__popcll(who));
    } else if (in) atomicAdd(&sh.hist[digit], 1u);
}

__device__ __forceinline__ void clear_hist(SelectShared& sh) {
    for (int i = threadIdx.x; i < 2048; i += EV_THREADS) sh.hist[i] = 0;
}

// Sum of x over the workgroup, for every thread. Two barriers; wave_a is free again behind the second.
__device__ __forceinline__ int block_sum(SelectShared& sh, int x) {
    x = wave_sum(x);
    if ((threadIdx.x & 63) == 0) sh.wave_a[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < EV_WAVES; ++w) x += sh.wave_a[w];
    __syncthreads();
    return x;
}

// The greatest digit d of a histogram of 2048 bins with at least `want` keys at it or above (sh.digit), how many of the
// want are left for d itself (sh.left), how many keys have it (sh.same). A thread brings the counts of bins
// 2047 - 2 tid and 2046 - 2 tid. Ends with a barrier.
__device__ __forceinline__ void pick_digit(SelectShared& sh, int want, int c0, int c1) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, top = 2047 - 2 * tid;
    int inc = wave_scan(c0 + c1);
    if (lane == 63) sh.wave_a[wave] = inc;
    __syncthreads();
    for (int w = 0; w < EV_WAVES; ++w) inc += w < wave ? sh.wave_a[w] : 0;
    const int over = inc - c0 - c1;                  // keys above this thread's bins
    if (over < want && want <= inc) {
        const bool upper = over + c0 >= want;
        sh.digit = (uint32_t)(upper ? top : top - 1);
        sh.left = want - over - (upper ? 0 : c0);
        sh.same = upper ? c0 : c1;
    }
    __syncthreads();
}

__device__ __forceinline__ void pick_digit(SelectShared& sh, int want) {
    pick_digit(sh, want, (int)sh.hist[2047 - 2 * threadIdx.x], (int)sh.hist[2046 - 2 * threadIdx.x]);
}

// Digits two and three of the threshold. each(f) calls f(key) for all keys, 0 for none, in whole waves. sh.hist is clear.
template <class E>
__device__ __forceinline__ void pick_rest(SelectShared& sh, E each, uint32_t* thr, int* need) {
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
        const int shift = pass ? 0 : 10, bits = pass ? 10 : 11;
        const uint32_t t = *thr;
        each([&](uint32_t k) INLINE { count_digit(sh, k != 0u && k >> (shift + bits) == t >> (shift + bits), k >> shift & ((1u << bits) - 1)); });
        __syncthreads();
        pick_digit(sh, *need);
        *thr |= sh.digit << shift;
        *need = sh.left;
        if (!pass) {
            clear_hist(sh);
            __syncthreads();
        }
    }
}

// Greatest of x over the workgroup, in sh.newest (set to the least before). Ends with a barrier.
__device__ __forceinline__ int block_max(SelectShared& sh, int x) {
    x = wave_max(x);
    if ((threadIdx.x & 63) == 0) atomicMax(&sh.newest, x);
    __syncthreads();
    return sh.newest;
}

// The outcome for a workgroup's slots: waves one after the other, `per` rows of 64 each. gt, eq: keys above the threshold
// and at it in the slots before the workgroup's. All above it are kept and the first `need` at it. A gap below n is the
// (slot - kept before it)-th, a kept slot from n on has rank `kept before it`: both lists come out ascending without a
// sort.
template <int R>
__device__ __forceinline__ void emit(SelectShared& sh, const Head& a, const Slots<R>& x, int per, uint32_t thr, int need, int gt, int eq) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int g = 0, e0 = 0;
    for_rows<R>(per, [&](auto i) INLINE {
        const uint32_t k = x.key[i];
        g += __popcll(__ballot(k > thr));
        e0 += __popcll(__ballot(k == thr));
    });
    if (lane == 0) { sh.wave_a[wave] = g; sh.wave_b[wave] = e0; }
    __syncthreads();
    for (int w = 0; w < EV_WAVES; ++w) {
        gt += w < wave ? sh.wave_a[w] : 0;
        eq += w < wave ? sh.wave_b[w] : 0;
    }
    const bool copy = a.mass_out != a.mass, copy_pos = a.pos_out != a.pos;
    for_rows<R>(per, [&](auto i) INLINE {
        const int s = x.slot(i);
        const uint32_t k = x.key[i];
        const unsigned long long bg = __ballot(k > thr), be = __ballot(k == thr);
        const int e = lanes_below(be, eq), before = lanes_below(bg, gt) + min(e, need);
        const bool keep = k > thr || (k == thr && e < need);
        gt += __popcll(bg);
        eq += __popcll(be);
        if (k == 0u) return;
        if (s == a.n) a.counts[0] = before;
        if (s < a.n) {
            if (!keep) a.gaps[s - before] = s;
            else {
                if (copy) a.mass_out[s] = x.mass[i];
                if (copy_pos) a.pos_out[s] = x.pos[i];
            }
        } else if (keep) a.late[before] = s;         // the move empties it
        else { a.mass_out[s] = 0.f; a.pos_out[s] = -1; }
    });
}

// Slots from .. to - 1 of a head that keeps what it has, and emptiness behind its length.
__device__ __forceinline__ void keep_all(const Head& a, int64_t from, int64_t to) {
    for (int64_t s = from + threadIdx.x; s < to; s += EV_THREADS) {
        if (s >= a.len) { a.mass_out[s] = 0.f; a.pos_out[s] = -1; }
        else if (a.len == a.n) {
            if (a.mass_out != a.mass) a.mass_out[s] = a.mass[s];
            if (a.pos_out != a.pos) a.pos_out[s] = a.pos[s];
        }
    }
    if (from == 0 && threadIdx.x == 0) {
        if (a.len == a.n) a.counts[0] = a.n;
        a.counts[1] = a.n;
    }
}

// Keys that share the threshold's first digit, from x into list (n of them so far), one wave's after another's.
template <int R>
__device__ __forceinline__ void list_keys(const Head& a, const Slots<R>& x, int per, uint32_t digit, uint32_t* list, int* n) {
    const int lane = threadIdx.x & 63;
    for_rows<R>(per, [&](auto i) INLINE {
        const uint32_t k = x.key[i];
        const bool in = k != 0u && k >> 21 == digit;
        const unsigned long long who = __ballot(in);
        if (who) {
            int at = 0;
            if (lane == 0) at = atomicAdd(n, __popcll(who));
            at = __builtin_amdgcn_readfirstlane(at);
            if (in) list[lanes_below(who, at)] = k;
        }
    });
}

// A head of one workgroup.
template <int R>
__device__ __forceinline__ void select_head(SelectShared& sh, Head& a, int recent) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (a.len + EV_THREADS - 1) / EV_THREADS;
    Slots<R> x;
    x.load(a, wave * per * 64 + lane, min(a.len, (wave + 1) * per * 64), per);
    if (tid == 0) { sh.newest = -0x7fffffff - 1; sh.listed = 0; }
    clear_hist(sh);
    __syncthreads();
    if (recent > 0) a.protect(block_max(sh, x.newest(per)), recent);
    x.make_keys(a, per);
    for_rows<R>(per, [&](auto i) INLINE { count_digit(sh, x.key[i] != 0u, x.key[i] >> 21); });
    __syncthreads();
    pick_digit(sh, a.n);
    uint32_t thr = sh.digit << 21;
    int need = sh.left;
    const bool few = sh.same <= EV_LIST;
    clear_hist(sh);
    if (few) list_keys<R>(a, x, per, thr >> 21, sh.list, &sh.listed);      // only these are looked at from here on
    __syncthreads();
    if (few)
        pick_rest(sh, [&](auto f) INLINE { for (int i = tid; i - lane < sh.listed; i += EV_THREADS) f(i < sh.listed ? sh.list[i] : 0u); }, &thr, &need);
    else pick_rest(sh, [&](auto f) INLINE { for_rows<R>(per, [&](auto i) INLINE { f(x.key[i]); }); }, &thr, &need);
    emit<R>(sh, a, x, per, thr, need, 0, 0);
}

// Row late[low + i] -> row gaps[i] of a head, K and V and the side tables, 16-byte pieces first, first + step, ...
__device__ __forceinline__ void move_rows(const KvPool& p, const KvTable& tb, const KvEvict& a, int h, int b, int low, int n, int first, int step) {
    const int64_t row = (int64_t)b * p.heads + h;
    const int32_t* gaps = a.lists + row * 2 * a.list_ld;
    const int32_t* late = gaps + a.list_ld + low;
    const int32_t* table = tb.table + (int64_t)b * tb.ld;
    const int vecs = (p.dim * p.esize) >> 4, vec_shift = 31 - __builtin_clz(vecs), mask = p.page_size - 1;
    for (int64_t i = first; i < (int64_t)(n - low) * vecs; i += step) {
        const int c = (int)i & (vecs - 1), r = (int)(i >> vec_shift);
        const int to = gaps[r], from = late[r];
        if (c == 0) {
            const int64_t o = row * a.side_ld;
            a.mass_out[o + to] = a.mass[o + from];
            a.positions_out[o + to] = a.positions[o + from];
            a.mass_out[o + from] = 0.f;
            a.positions_out[o + from] = -1;
        }
        const int pt = table[to >> p.page_shift], pf = table[from >> p.page_shift];
        if ((unsigned)pt >= (unsigned)p.num_pages || (unsigned)pf >= (unsigned)p.num_pages) {
            if (c == 0) atomicOr(p.status, KV_BAD_PAGE);
            continue;
        }
        const int64_t kt = slot_off(p.k_st, pt, h, to & mask) * p.esize, kf = slot_off(p.k_st, pf, h, from & mask) * p.esize;
        const int64_t vt = slot_off(p.v_st, pt, h, to & mask) * p.esize, vf = slot_off(p.v_st, pf, h, from & mask) * p.esize;
        const u32x4 k = reinterpret_cast<const u32x4*>((const char*)p.k + kf)[c];
        const u32x4 v = reinterpret_cast<const u32x4*>((const char*)p.v + vf)[c];
        reinterpret_cast<u32x4*>((char*)p.k + kt)[c] = k;
        reinterpret_cast<u32x4*>((char*)p.v + vt)[c] = v;
    }
}

// Greatest of a waves' value in wave_x, one of each, over the workgroup.
__device__ __forceinline__ int waves_max(const int* wave_x, int none) {
    const int lane = threadIdx.x & 63;
    return wave_max(lane < EV_WAVES ? wave_x[lane] : none);
}

// A head one token over its budget, as every step of a decoder that holds one leaves it: the token that goes is the least key's,
// of equal ones the last, found in two barriers without a select, and at most one row moves, that of slot n, which is loaded
// meanwhile. (32 x 8 heads of 2049 tokens: 11.3 us by the select, 6.3 here.)
template <int R>
__device__ __forceinline__ void drop_one(SelectShared& sh, const KvPool& p, const KvTable& tb, Head& a, int recent, int h, int b) {
    constexpr int NONE = -0x7fffffff - 1;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n;
    const int per = (a.len + EV_THREADS - 1) / EV_THREADS, vecs = (p.dim * p.esize) >> 4, mask = p.page_size - 1;
    const int32_t* table = tb.table + (int64_t)b * tb.ld;
    Slots<R> x;
    x.load(a, wave * per * 64 + lane, min(a.len, (wave + 1) * per * 64), per);
    const bool is_k = tid < vecs, mover = tid < 2 * vecs;      // a piece of row n each
    const int pf = table[n >> p.page_shift], c = is_k ? tid : tid - vecs;
    const bool bad_from = (unsigned)pf >= (unsigned)p.num_pages;
    char* pool = (char*)(is_k ? p.k : p.v);
    auto at = [&](int page, int s) INLINE {
        const int64_t k = slot_off(p.k_st, page, h, s & mask), v = slot_off(p.v_st, page, h, s & mask);
        return reinterpret_cast<u32x4*>(pool + (is_k ? k : v) * p.esize) + c;
    };
    u32x4 piece = {};
    if (mover && !bad_from) piece = *at(pf, n);
    if (recent > 0) {
        const int newest = wave_max(x.newest(per));
        if (lane == 0) sh.wave_a[wave] = newest;
        __syncthreads();
        a.protect(waves_max(sh.wave_a, NONE), recent);
    }
    x.make_keys(a, per);
    int least = NONE, slot = -1;                     // the key's bits in descending order, as a number with a sign
    for_rows<R>(per, [&](auto i) INLINE {
        const uint32_t k = x.key[i];
        const int v = (int)(~k ^ 0x80000000u);
        if (k != 0u && v >= least) { least = v; slot = x.slot(i); }
    });
    int m = wave_max(least);
    slot = wave_max(least == m ? slot : -1);
    if (lane == 0) { sh.hist[wave] = (uint32_t)m; sh.wave_b[wave] = slot; }
    __syncthreads();
    least = lane < EV_WAVES ? (int)sh.hist[lane] : NONE;
    m = wave_max(least);
    const int gone = wave_max(lane < EV_WAVES && least == m ? sh.wave_b[lane] : -1);
    const bool copy = a.mass_out != a.mass, copy_pos = a.pos_out != a.pos;
    for_rows<R>(per, [&](auto i) INLINE {
        const int s = x.slot(i);
        if (i >= per || s >= x.stop) return;
        if (s == n) {
            if (gone != n) { a.mass_out[gone] = x.mass[i]; a.pos_out[gone] = x.pos[i]; }
            a.mass_out[n] = 0.f;
            a.pos_out[n] = -1;
        } else if (s != gone) {
            if (copy) a.mass_out[s] = x.mass[i];
            if (copy_pos) a.pos_out[s] = x.pos[i];
        }
    });
    if (tid == 0) a.counts[0] = n;                   // nothing is left to move
    if (!mover || gone == n) return;
    const int pt = table[gone >> p.page_shift];
    if (bad_from || (unsigned)pt >= (unsigned)p.num_pages) {
        if (tid == 0) atomicOr(p.status, KV_BAD_PAGE);
        return;
    }
    *at(pt, gone) = piece;
}

// One workgroup per (sequence, kv head). The n-th greatest key by a radix select of 11 + 11 + 10 bits, then one pass in
// slot order. Masses and positions stay in registers, so they are read once, together; what is left are LDS counters and a
// dozen barriers, which bound it: a head to a CU, 14 us at 8192 tokens, 4 of them the loads, 4 the last pass.
template <bool MOVE>
__global__ __launch_bounds__(EV_THREADS) void kv_select_kernel(const KvPool p, const KvTable tb, const KvEvict a) {
    __shared__ SelectShared sh;
    Head head(p, tb, a, blockIdx.x, blockIdx.y, blockIdx.x == 0 && threadIdx.x == 0);
    const bool one = head.len == head.n + 1;
    if (one) {
        if (head.len <= 4 * EV_THREADS) drop_one<4>(sh, p, tb, head, a.recent, blockIdx.x, blockIdx.y);
        else drop_one<EV_ROWS>(sh, p, tb, head, a.recent, blockIdx.x, blockIdx.y);
    } else if (head.len > head.n) {
        if (head.len <= 4 * EV_THREADS) select_head<4>(sh, head, a.recent);
        else select_head<EV_ROWS>(sh, head, a.recent);
    }
    keep_all(head, 0, a.side_ld);
    if constexpr (MOVE) {
        if (!one) __syncthreads();                   // the lists and counts of this workgroup
        if (blockIdx.x == 0 && threadIdx.x == 0) a.lengths_out[blockIdx.y] = head.n;
        if (!one) move_rows(p, tb, a, blockIdx.x, blockIdx.y, head.counts[0], head.n, threadIdx.x, EV_THREADS);
    }
}

// The same for tables of more slots than a workgroup holds: a workgroup per chunk, four launches. Each workgroup works out
// the head's threshold for itself from what the one before left: the chunks' newest positions, the chunks' histograms of the
// first digit, the chunks' lists of the keys that share the threshold's first digit. Sums over chunks before
// its own give it the ranks of its slots, so nothing waits for anything and no counter is shared. (32 heads of 65536 tokens:
// 5 + 5 + 8 + 17 us.)
struct ChunkWork {
    int32_t* newest;                     // [chunks]
    uint32_t* hist;                      // [chunks][2048]
    uint32_t* list;                      // [chunks][EV_CHUNK]
    __device__ __forceinline__ ChunkWork(const KvEvict& a, int64_t row, int chunks) {
        newest = a.chunk_newest + row * chunks;
        hist = a.chunk_hist + row * chunks * 2048;
        list = a.chunk_list + row * chunks * EV_CHUNK;
    }
};

// STAGE 0: newest position; 1: histogram; 2: list; 3: the outcome.
template <int STAGE>
__global__ __launch_bounds__(EV_THREADS) void kv_select_chunk_kernel(const KvPool p, const KvTable tb, const KvEvict a) {
    constexpr int R = EV_CHUNK / EV_THREADS;
    __shared__ SelectShared sh;
    const int c = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    Head head(p, tb, a, h, b, STAGE == 3 && c == 0 && h == 0 && tid == 0);
    const ChunkWork ws(a, (int64_t)b * p.heads + h, gridDim.x);
    const int slot0 = c * EV_CHUNK, chunks = (head.len + EV_CHUNK - 1) / EV_CHUNK;
    if (STAGE == 3) keep_all(head, slot0, c + 1 == (int)gridDim.x ? a.side_ld : min<int64_t>(a.side_ld, slot0 + EV_CHUNK));
    if (head.len <= head.n || c >= chunks) return;
    if (tid == 0) { sh.newest = -0x7fffffff - 1; sh.listed = 0; }
    clear_hist(sh);
    Slots<R> x;
    const int s0 = slot0 + wave * R * 64;
    x.load(head, s0 + lane, min(head.len, s0 + R * 64), R);
    __syncthreads();
    if (STAGE == 0) {
        const int newest = block_max(sh, x.newest(R));
        if (tid == 0) ws.newest[c] = newest;
        return;
    }
    if (a.recent > 0) {
        int newest = -0x7fffffff - 1;
        if (wave == 0)
            for (int i = lane; i < chunks; i += 64) newest = max(newest, ws.newest[i]);
        head.protect(block_max(sh, newest), a.recent);
    }
    x.make_keys(head, R);
    if (STAGE == 1) {
        for_rows<R>(R, [&](auto i) INLINE { count_digit(sh, x.key[i] != 0u, x.key[i] >> 21); });
        __syncthreads();
        for (int i = tid; i < 2048; i += EV_THREADS) ws.hist[(int64_t)c * 2048 + i] = sh.hist[i];
        return;
    }
    // first digit, from the sum of the chunks' histograms
    const int top = 2047 - 2 * tid;
    int c0 = 0, c1 = 0, l0 = 0, l1 = 0;              // of all chunks, and of those before this one
#pragma unroll 4
    for (int i = 0; i < chunks; ++i) {
        const uint2 x = *reinterpret_cast<const uint2*>(ws.hist + (int64_t)i * 2048 + top - 1);
        c0 += (int)x.y;
        c1 += (int)x.x;
        l0 += i < c ? (int)x.y : 0;
        l1 += i < c ? (int)x.x : 0;
    }
    pick_digit(sh, head.n, c0, c1);
    const uint32_t digit = sh.digit;
    if (STAGE == 2) {
        list_keys<R>(head, x, R, digit, ws.list + (int64_t)c * EV_CHUNK, &sh.listed);
        return;
    }
    uint32_t thr = digit << 21;
    int need = sh.left;
    const int same = sh.same;
    int gt = block_sum(sh, (top > (int)digit ? l0 : 0) + (top - 1 > (int)digit ? l1 : 0));
    // The keys that share the digit, chunk by chunk: out of LDS where they fit (chunk i's are list[i's predecessors' ..], a
    // chunk per wave at a time), else again and again out of the workspace.
    int before = 0;                                  // of them, those of chunks before this one
    if (same <= EV_LIST) {
        int sum = 0;
        for (int i0 = 0; i0 < chunks; i0 += 64) {
            const int n = i0 + lane < chunks ? (int)ws.hist[(int64_t)(i0 + lane) * 2048 + digit] : 0, inc = wave_scan(n);
            for (int i = wave; i < 64; i += EV_WAVES) {
                const int m = __builtin_amdgcn_readlane(n, i), to = sum + __builtin_amdgcn_readlane(inc - n, i);
                for (int j = lane; j < m; j += 64) sh.list[to + j] = ws.list[(int64_t)(i0 + i) * EV_CHUNK + j];
            }
            if (i0 <= c && c < i0 + 64) before = sum + __builtin_amdgcn_readlane(inc - n, c - i0);
            sum += __builtin_amdgcn_readlane(inc, 63);
        }
        __syncthreads();
    }
    auto each = [&](int upto, int upto_keys, auto f) INLINE {
        if (same <= EV_LIST) {
            for (int j = tid; j - lane < upto_keys; j += EV_THREADS) f(j < upto_keys ? sh.list[j] : 0u);
        } else {
            for (int i = 0; i < upto; ++i) {
                const int n = (int)ws.hist[(int64_t)i * 2048 + digit];
                for (int j = tid; j - lane < n; j += EV_THREADS) f(j < n ? ws.list[(int64_t)i * EV_CHUNK + j] : 0u);
            }
        }
    };
    pick_rest(sh, [&](auto f) INLINE { each(chunks, same, f); }, &thr, &need);
    int g = 0, e = 0;
    each(c, before, [&](uint32_t k) INLINE { g += k > thr; e += k == thr; });
    gt += block_sum(sh, g);
    const int eq = block_sum(sh, e);
    emit<R>(sh, head, x, R, thr, need, gt, eq);
}

// The rest of a sequence, for tables that can hold many rows to move. Nothing orders the rows: sources lie at n and beyond,
// targets below it. A copy, bound by the memory at the rate of a copy (4 x 65536 -> 8192 of 8 heads: 235 MB in 51 us).
__global__ __launch_bounds__(256) void kv_move_kernel(const KvPool p, const KvTable tb, const KvEvict a) {
    const int h = blockIdx.y, b = blockIdx.z;
    const int32_t* counts = a.counts + 2 * ((int64_t)b * p.heads + h);
    if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.lengths_out[b] = counts[1];
    move_rows(p, tb, a, h, b, counts[0], counts[1], blockIdx.x * 256 + threadIdx.x, gridDim.x * 256);
}

}  // namespace

// Compute units of a device, asked for once. (256 where the question fails, as it does without a GPU.)
static int kv_cus(int device) {
    static std::atomic<int> known[64];
    if (device < 0 || device >= 64) return 256;
    int n = known[device].load(std::memory_order_relaxed);
    if (n) return n;
    if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || n < 1) {
        (void)hipGetLastError();
        return 256;
    }
    known[device].store(n, std::memory_order_relaxed);
    return n;
}

void launch_kv_take_status(int32_t* status, int32_t* bits, hipStream_t s) { kv_take_status_kernel<<<1, 1, 0, s>>>(status, bits); }

void launch_kv_append(const KvPool& p, const KvTable& tb, const KvAppend& a, hipStream_t s) {
    const int64_t pieces = (int64_t)a.T * p.heads * ((p.dim * p.esize) >> 4);
    const bool side = a.mass || a.positions;
    kv_append_kernel<<<dim3((unsigned)((pieces + 256 * AP_ITEMS - 1) / (256 * AP_ITEMS)), tb.B, side ? 3 : 2), 256, 0, s>>>(p, tb, a);
}

// Tiles of the line if every sequence filled its table.
static int64_t attend_tiles(const KvPool& p, int B, int group, int max_pages) {
    const int tw = attend_tile(p.dtype);
    return (((int64_t)max_pages << p.page_shift) + tw - 1) / tw * B * p.heads * attend_passes(p, group);
}

bool kv_attend_fits(const KvPool& p, int B, int group, int max_pages) {
    // tiles are counted in 31 bits on the device, workgroups of 256 threads in 32
    const int64_t cap = (int64_t)max_pages << p.page_shift;
    return attend_tiles(p, B, group, max_pages) < (1ll << 30) &&
           (int64_t)B * p.heads * (group + (cap + 1023) / 1024) < (1ll << 24);
}

// Workgroups of the attention: as many as the CUs hold, or a tile for every wave where there are fewer.
static int attend_groups(const KvPool& p, int B, int group, int max_pages) {
    return (int)std::min<int64_t>((attend_tiles(p, B, group, max_pages) + AT_WAVES - 1) / AT_WAVES,
                                  attend_per_cu(p.dim) * kv_cus(p.device));
}

static bool attend_short(const KvPool& p, int B, int group, int max_pages) {
    return group <= 16 && ((int64_t)max_pages << p.page_shift) <= short_slots(p.dtype, p.dim) &&
           (int64_t)B * p.heads <= (int64_t)short_per_cu(p.dim) * kv_cus(p.device);
}

// {maximum, sum} and output of two parts per wave (the one it begins with, the one it ends with), and the scores
size_t kv_attend_ws_bytes(const KvPool& p, int B, int group, int max_pages, bool mass) {
    if (attend_short(p, B, group, max_pages)) return 0;
    const size_t parts = 2 * AT_WAVES * (size_t)attend_groups(p, B, group, max_pages), cols = (size_t)attend_columns(p, group), rows = std::min((size_t)group, cols);
    size_t n = parts * cols * sizeof(float2) + parts * rows * p.dim * sizeof(float);
    if (mass) n += (size_t)attend_tiles(p, B, group, max_pages) * rows * attend_tile(p.dtype) * sizeof(float);
    return n;
}

template <int DT, int D>
static void attend_launch(const KvPool& p, const KvTable& tb, const KvAttend& a, int W, hipStream_t s) {
    if constexpr (attend_columns(DT, D, 32) == 32) {
        if (a.group > 16) {
            if (a.mass) kv_attend_kernel<DT, D, true, 2><<<W, 64 * AT_WAVES, 0, s>>>(p, tb, a);
            else kv_attend_kernel<DT, D, false, 2><<<W, 64 * AT_WAVES, 0, s>>>(p, tb, a);
            return;
        }
    }
    if (a.mass) kv_attend_kernel<DT, D, true, 1><<<W, 64 * AT_WAVES, 0, s>>>(p, tb, a);
    else kv_attend_kernel<DT, D, false, 1><<<W, 64 * AT_WAVES, 0, s>>>(p, tb, a);
}

template <int DT, int D>
static void attend_short_launch(const KvPool& p, const KvTable& tb, const KvAttend& a, hipStream_t s) {
    const int grid = tb.B * p.heads, block = 64 * SHORT_WAVES;
    if (a.mass) kv_attend_short_kernel<DT, D, true><<<grid, block, 0, s>>>(p, tb, a);
    else kv_attend_short_kernel<DT, D, false><<<grid, block, 0, s>>>(p, tb, a);
}

template <int D>
static void attend_both(const KvPool& p, const KvTable& tb, const KvAttend& a, int W, hipStream_t s) {
    if constexpr (short_per_cu(D) > 0) {
        if (attend_short(p, tb.B, a.group, tb.max_pages)) {
            if (p.dtype == KV_F32) attend_short_launch<KV_F32, D>(p, tb, a, s);
            else if (p.dtype == KV_BF16) attend_short_launch<KV_BF16, D>(p, tb, a, s);
            else attend_short_launch<KV_F16, D>(p, tb, a, s);
            return;
        }
    }
    if (p.dtype == KV_F32) attend_launch<KV_F32, D>(p, tb, a, W, s);
    else if (p.dtype == KV_BF16) attend_launch<KV_BF16, D>(p, tb, a, W, s);
    else attend_launch<KV_F16, D>(p, tb, a, W, s);
    const int tw = attend_tile(p.dtype), waves_all = W * AT_WAVES;
    const int64_t cap = (int64_t)tb.max_pages << p.page_shift;
    if (cap <= tw && !a.mass) return;                // nothing is ever in parts
    // A wave per head where heads are in few parts, on average; a workgroup where they are in many. Longer stretches of mass
    // where there are enough of them to fill the chip. (Workgroups of some 4 us each: their number is what counts.)
    const int64_t heads = (int64_t)tb.B * p.heads * a.group, rows = (int64_t)tb.B * p.heads;
    const bool waves = waves_all <= 16 * rows * attend_passes(p, a.group);
    const int64_t joins = waves ? (heads + 3) / 4 : heads;
    const int mass_tokens = rows * ((cap + 4095) / 4096) >= 512 ? 4096 : 1024;
    const int64_t blocks = joins + (a.mass ? rows * ((cap + mass_tokens - 1) / mass_tokens) : 0);
    if (waves) kv_join_kernel<D, true><<<(unsigned)blocks, 256, 0, s>>>(p, tb, a, waves_all, tw, (int)joins, mass_tokens);
    else kv_join_kernel<D, false><<<(unsigned)blocks, 256, 0, s>>>(p, tb, a, waves_all, tw, (int)joins, mass_tokens);
}

void launch_kv_attend(const KvPool& p, const KvTable& tb, KvAttend a, void* ws, hipStream_t s) {
    const int W = attend_groups(p, tb.B, a.group, tb.max_pages), parts = 2 * W * AT_WAVES;
    a.score_rows = std::min(a.group, attend_columns(p, a.group));
    a.part_ml = (float2*)ws;
    a.part_out = (float*)(a.part_ml + (size_t)parts * attend_columns(p, a.group));
    a.scores = a.part_out + (size_t)parts * a.score_rows * p.dim;
    if (p.dim == 64) attend_both<64>(p, tb, a, W, s);
    else if (p.dim == 128) attend_both<128>(p, tb, a, W, s);
    else attend_both<256>(p, tb, a, W, s);
}

// Entries of one list: ranks of kept slots and numbers of gaps lie below n <= min(budget, capacity).
static size_t kv_evict_list(const KvPool& p, int max_pages, int budget) {
    return (size_t)std::min<int64_t>(budget, (int64_t)max_pages << p.page_shift);
}

// Chunks of the long select, 0 where a workgroup holds a head. (One launch against four: an eviction of 32 heads to half
// its tokens takes 23 us and 36 at 8192 slots, 37 and 45 at 16384; at 65536 a workgroup a head took 168 and the chunks 65.)
static int64_t kv_evict_chunks(const KvPool& p, int max_pages) {
    const int64_t cap = (int64_t)max_pages << p.page_shift;
    return cap <= EV_ROWS * EV_THREADS ? 0 : (cap + EV_CHUNK - 1) / EV_CHUNK;
}

// {kept below n, n} of every (sequence, kv head), its gaps and late kept slots, and the chunks' tables
size_t kv_evict_ws_bytes(const KvPool& p, int B, int max_pages, int budget) {
    return (size_t)B * p.heads * (2 * kv_evict_list(p, max_pages, budget) + 2 + kv_evict_chunks(p, max_pages) * (2 + 2048 + EV_CHUNK)) * 4;
}

void launch_kv_evict(const KvPool& p, const KvTable& tb, KvEvict a, void* ws, hipStream_t s) {
    const size_t rows = (size_t)tb.B * p.heads;
    const int chunks = (int)kv_evict_chunks(p, tb.max_pages);
    // 8-byte pairs of histogram bins first, everything else is read by the word
    a.chunk_hist = (uint32_t*)ws;
    a.chunk_list = a.chunk_hist + rows * chunks * 2048;
    a.counts = (int32_t*)(a.chunk_list + rows * chunks * EV_CHUNK);
    a.lists = a.counts + 2 * rows;
    a.list_ld = (int64_t)kv_evict_list(p, tb.max_pages, a.budget);
    a.chunk_newest = a.lists + 2 * rows * a.list_ld;
    if (chunks) {
        const dim3 grid(chunks, p.heads, tb.B);
        if (a.recent > 0) kv_select_chunk_kernel<0><<<grid, EV_THREADS, 0, s>>>(p, tb, a);
        kv_select_chunk_kernel<1><<<grid, EV_THREADS, 0, s>>>(p, tb, a);
        kv_select_chunk_kernel<2><<<grid, EV_THREADS, 0, s>>>(p, tb, a);
        kv_select_chunk_kernel<3><<<grid, EV_THREADS, 0, s>>>(p, tb, a);
    }
    // Few rows at most (a budget that is kept step by step) are moved by the workgroup that chose them; one launch less. Not
    // where the lengths are written over: the other heads' workgroups may still have to read them.
    const int64_t most = std::min((int64_t)a.budget, ((int64_t)tb.max_pages << p.page_shift) - a.budget);
    const int64_t vecs = std::max<int64_t>(most, 1) * ((p.dim * p.esize) >> 4);
    if (!chunks && vecs <= 2 * EV_THREADS && a.lengths_out != a.lengths) {
        kv_select_kernel<true><<<dim3(p.heads, tb.B), EV_THREADS, 0, s>>>(p, tb, a);
        return;
    }
    if (!chunks) kv_select_kernel<false><<<dim3(p.heads, tb.B), EV_THREADS, 0, s>>>(p, tb, a);
    kv_move_kernel<<<dim3((unsigned)std::min<int64_t>((vecs + 255) / 256, 64), p.heads, tb.B), 256, 0, s>>>(p, tb, a);
}

}  // namespace taco
