// The paged key-value cache of an attention decoder: append (rows into pages), attend (one new token per sequence over
// its pages) and evict (the cache cut to a budget by the attention its tokens have drawn). include/taco.h has the
// formulas. The pool holds pages of page_size tokens per kv head; a sequence names its pages in a table row, slot s of
// it lives in row s % page_size of page table[b][s / page_size].
//
// Nothing on the device trusts a length or a page id: lengths are clamped to the table's capacity, a slot whose page id
// is outside the pool is treated as masked (attend) or not written (append, evict), and either sets a bit of the pool's
// status word. Offsets into the pool and the side tables are 64-bit.
#include "kernels.h"

namespace taco {
namespace {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }   // (flushes results below 2^-126)

__device__ __forceinline__ int clamp_len(int n, int cap, int32_t* status, bool report) {
    if (n >= 0 && n <= cap) return n;
    if (report) atomicOr(status, KV_BAD_LENGTH);
    return n < 0 ? 0 : cap;
}

// Element offset of slot s (page id already checked) in a pool with strides st = {page, head, token}.
__device__ __forceinline__ int64_t slot_off(const int64_t* st, int page, int h, int in_page) {
    return (int64_t)page * st[0] + (int64_t)h * st[1] + (int64_t)in_page * st[2];
}

// ---------------------------------------------------------------------------------------
// append

// Copies 16 bytes per lane: planes 0 / 1 of the grid are K / V, (t, h, 16-byte column) with the column fastest; plane 2
// the side tables, (h, t) with t fastest. Nothing but the copy bounds it: the rows come in once and go out once.
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
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (plane == 2) {
        if (i >= (int64_t)p.heads * a.T) return;
        const int t = (int)(i % a.T), h = (int)(i / a.T);
        if (t >= count) return;
        const int64_t o = ((int64_t)b * p.heads + h) * a.side_ld + start + t;
        if (a.mass) a.mass[o] = 0.f;
        if (a.positions) a.positions[o] = (a.first ? a.first[b] : start) + t;
        return;
    }
    const int vecs = (p.dim * p.esize) >> 4;
    if (i >= (int64_t)a.T * p.heads * vecs) return;
    const int c = (int)(i % vecs);
    const int64_t th = i / vecs;
    const int h = (int)(th % p.heads), t = (int)(th / p.heads);
    if (t >= count) return;
    const int s = start + t;
    const int page = tb.table[(int64_t)b * tb.ld + (s >> p.page_shift)];
    if ((unsigned)page >= (unsigned)p.num_pages) {
        if (c == 0) atomicOr(p.status, KV_BAD_PAGE);
        return;
    }
    const int64_t* xs = plane ? a.v_st : a.k_st;
    const char* src = (const char*)(plane ? a.v : a.k) + ((int64_t)b * xs[0] + (int64_t)t * xs[1] + (int64_t)h * xs[2]) * p.esize;
    char* dst = (char*)(plane ? p.v : p.k) + slot_off(plane ? p.v_st : p.k_st, page, h, s & (p.page_size - 1)) * p.esize;
    reinterpret_cast<uint4*>(dst)[c] = reinterpret_cast<const uint4*>(src)[c];
}

// ---------------------------------------------------------------------------------------
// attend

template <typename T>
__device__ __forceinline__ float dot_row(const T* q, const T* k, int dim) {
    float s = 0.f;
    for (int d = 0; d < dim; ++d) s += (float)q[d] * (float)k[d];
    return s;
}

// Score (in units of ln 2) of query row q against slot t, or -inf where its page id is bad.
template <typename T>
__device__ __forceinline__ float slot_score(const KvPool& p, const int32_t* row, const T* q, int h, int t, float scale2,
                                            bool report) {
    const int page = row[t >> p.page_shift];
    if ((unsigned)page >= (unsigned)p.num_pages) {
        if (report) atomicOr(p.status, KV_BAD_PAGE);
        return -INFINITY;
    }
    return dot_row(q, (const T*)p.k + slot_off(p.k_st, page, h, t & (p.page_size - 1)), p.dim) * scale2;
}

// One workgroup per (sequence, query head): 256 tokens at a time, a score per thread, the running maximum and sum of the
// softmax, then a column of the output per thread.
template <typename T>
__global__ __launch_bounds__(256) void kv_attend_kernel(const KvPool p, const KvTable tb, const KvAttend a) {
    __shared__ float w[256], red[256];
    const int hq = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    const int h = hq / a.group, cap = tb.max_pages << p.page_shift;
    const int len = clamp_len(a.lengths[b], cap, p.status, hq == 0 && tid == 0);
    const int32_t* row = tb.table + (int64_t)b * tb.ld;
    const T* q = (const T*)a.q + (int64_t)b * a.q_st[0] + (int64_t)hq * a.q_st[1];
    float m = -INFINITY, l = 0.f, acc = 0.f;
    for (int t0 = 0; t0 < len; t0 += 256) {
        const int t = t0 + tid, n = min(256, len - t0);
        const float s = t < len ? slot_score(p, row, q, h, t, a.scale2, true) : -INFINITY;
        red[tid] = s;
        __syncthreads();
        float mx = m;
        for (int i = 0; i < n; ++i) mx = fmaxf(mx, red[i]);
        const float mr = mx == -INFINITY ? 0.f : mx;
        const float alpha = ex2(m - mr);
        w[tid] = ex2(s - mr);
        __syncthreads();
        // the chunk's sums first: thousands of small equal weights added to a large total one by one would all round
        // the same way
        float lc = 0.f, accc = 0.f;
        for (int i = 0; i < n; ++i) {
            lc += w[i];
            const int page = row[(t0 + i) >> p.page_shift];
            if (tid < p.dim && (unsigned)page < (unsigned)p.num_pages)
                accc += w[i] * (float)((const T*)p.v + slot_off(p.v_st, page, h, (t0 + i) & (p.page_size - 1)))[tid];
        }
        l = l * alpha + lc;
        acc = acc * alpha + accc;
        m = mx;
        __syncthreads();
    }
    // a row that saw no token, or none with a score above -inf: 0 and -inf
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (tid < p.dim) ((T*)a.out)[((int64_t)b * gridDim.x + hq) * p.dim + tid] = (T)(acc * inv);
    if (tid == 0) a.lse[(int64_t)b * gridDim.x + hq] = l == 0.f ? -INFINITY : m * LN2 + logf(l);
}

// mass[b][h][t] += sum over the query heads of kv head h of exp(score - lse): a token per thread.
template <typename T>
__global__ __launch_bounds__(256) void kv_mass_kernel(const KvPool p, const KvTable tb, const KvAttend a) {
    const int h = blockIdx.y, b = blockIdx.z, t = blockIdx.x * 256 + threadIdx.x;
    const int cap = tb.max_pages << p.page_shift;
    if (t >= clamp_len(a.lengths[b], cap, p.status, false)) return;
    const int32_t* row = tb.table + (int64_t)b * tb.ld;
    const int hq = p.heads * a.group;
    float sum = 0.f;
    for (int g = 0; g < a.group; ++g) {
        const T* q = (const T*)a.q + (int64_t)b * a.q_st[0] + (int64_t)(h * a.group + g) * a.q_st[1];
        const float lse = a.lse[(int64_t)b * hq + h * a.group + g];
        if (lse != -INFINITY) sum += ex2(slot_score(p, row, q, h, t, a.scale2, false) - lse * LOG2E);
    }
    a.mass[((int64_t)b * p.heads + h) * a.side_ld + t] += sum;
}

// ---------------------------------------------------------------------------------------
// evict

constexpr int EV_THREADS = 1024;

// Order-preserving bits of a mass: NaN above everything, -0 as +0; protected slots above that.
__device__ __forceinline__ uint32_t mass_key(float x) {
    if (x != x) return 0xfffffffeu;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Bits [shift, shift + bits) of the n-th greatest key, found from a histogram of the keys that agree with `prefix` above
// them: the digit, and how many of the n are left to find below it.
__device__ void pick_digit(const uint32_t* hist, int bins, int want, uint32_t* digit, int* left) {
    // one wave walks the bins from the top, 64 at a time
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int seen = 0;
        for (int top = bins - 1; top >= 0; top -= 64) {
            const int bin = top - lane;
            int c = bin >= 0 ? (int)hist[bin] : 0;
            int inc = c;
            for (int o = 1; o < 64; o <<= 1) {
                const int x = __shfl_up(inc, o);
                if (lane >= o) inc += x;
            }
            const unsigned long long hit = __ballot(seen + inc >= want);
            if (hit) {
                const int at = __ffsll(hit) - 1;
                if (lane == at) { *digit = (uint32_t)bin; *left = want - (seen + inc - c); }
                break;
            }
            seen += __shfl(inc, 63);
        }
    }
    __syncthreads();
}

// One workgroup per (sequence, kv head). The n-th greatest key by a radix select of 11 + 11 + 10 bits, then one pass in
// slot order with a running count of the kept: a gap below n is the (slot - kept before it)-th, a kept slot from n on
// has rank `kept before it`, so both lists come out ascending without a sort.
__global__ __launch_bounds__(EV_THREADS) void kv_select_kernel(const KvPool p, const KvTable tb, const KvEvict a) {
    __shared__ uint32_t hist[2048];
    __shared__ uint32_t digit;
    __shared__ int left, newest, kept_low;
    __shared__ int wave_gt[EV_THREADS / 64], wave_eq[EV_THREADS / 64];
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int cap = tb.max_pages << p.page_shift;
    const int len = clamp_len(a.lengths[b], cap, p.status, h == 0 && tid == 0);
    const int n = min(len, a.budget);
    const int64_t row = (int64_t)b * p.heads + h;
    const float* mass = a.mass + row * a.side_ld;
    const int32_t* pos = a.positions + row * a.side_ld;
    float* mass_out = a.mass_out + row * a.side_ld;
    int32_t* pos_out = a.positions_out + row * a.side_ld;
    int32_t* gaps = a.lists + row * 2 * a.list_ld;
    int32_t* late = gaps + a.list_ld;
    uint32_t thr = 0;            // len <= budget: every key is kept
    int need = 0;
    if (tid == 0) { newest = -0x7fffffff - 1; kept_low = n; }
    __syncthreads();
    if (len > n) {
        int mine = -0x7fffffff - 1;
        for (int s = tid; s < len; s += EV_THREADS) mine = max(mine, pos[s]);
        for (int o = 32; o; o >>= 1) mine = max(mine, __shfl_xor(mine, o));
        if (lane == 0) atomicMax(&newest, mine);
        __syncthreads();
    }
    const int64_t border = (int64_t)newest - a.recent;      // positions above it are protected
    auto key = [&](int s) { return (int64_t)pos[s] > border ? 0xffffffffu : mass_key(mass[s]); };
    if (len > n && n > 0) {
        need = n;
        int shift = 32;
        for (int bits = 11; shift > 0; ) {
            if (shift < bits) bits = shift;
            const uint32_t above = shift == 32 ? 0u : ~0u << shift;
            shift -= bits;
            for (int i = tid; i < 2048; i += EV_THREADS) hist[i] = 0;
            __syncthreads();
            for (int s = tid; s < len; s += EV_THREADS) {
                const uint32_t k = key(s);
                if ((k & above) == thr) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
            }
            __syncthreads();
            pick_digit(hist, 1 << bits, need, &digit, &left);
            thr |= digit << shift;
            need = left;
            __syncthreads();
        }
    }
    // all with a key above thr are kept, and the first `need` of those at it
    int gt0 = 0, eq0 = 0;        // before this stretch of slots
    for (int s0 = 0; s0 < a.side_ld; s0 += EV_THREADS) {
        const int s = s0 + tid;
        bool gt = false, eq = false;
        if (s < len) {
            if (len == n) gt = true;
            else if (n > 0) { const uint32_t k = key(s); gt = k > thr; eq = k == thr; }
        }
        int before = 0;
        bool keep = gt;
        if (len > n && s0 < len) {
            const unsigned long long bg = __ballot(gt), be = __ballot(eq);
            if (lane == 0) { wave_gt[wave] = __popcll(bg); wave_eq[wave] = __popcll(be); }
            __syncthreads();
            const unsigned long long low = (1ull << lane) - 1;
            int g = gt0 + __popcll(bg & low), e = eq0 + __popcll(be & low);
            for (int w = 0; w < EV_THREADS / 64; ++w) {
                if (w < wave) { g += wave_gt[w]; e += wave_eq[w]; }
                gt0 += wave_gt[w];
                eq0 += wave_eq[w];
            }
            before = g + min(e, need);
            keep = gt || (eq && e < need);
            if (s == n) kept_low = before;
            if (s < n && !keep) gaps[s - before] = s;
            if (s >= n && keep) late[before] = s;
            __syncthreads();
        }
        if (s < a.side_ld && !(keep && s >= n)) {
            // slots that stay, and slots that end up empty; gaps and the slots that fill them belong to the move
            if (s < n) { if (keep) { mass_out[s] = mass[s]; pos_out[s] = pos[s]; } }
            else { mass_out[s] = 0.f; pos_out[s] = -1; }
        }
    }
    __syncthreads();
    if (tid == 0) {
        a.counts[2 * row] = kept_low;
        a.counts[2 * row + 1] = n;
    }
}

// Row late[kept_low + i] -> row gaps[i], K and V and the side tables. Sources lie at n and beyond, targets below it.
__global__ __launch_bounds__(256) void kv_move_kernel(const KvPool p, const KvTable tb, const KvEvict a) {
    const int h = blockIdx.y, b = blockIdx.z;
    const int64_t row = (int64_t)b * p.heads + h;
    const int low = a.counts[2 * row], n = a.counts[2 * row + 1], moves = n - low;
    if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0) a.lengths_out[b] = n;
    const int32_t* gaps = a.lists + row * 2 * a.list_ld;
    const int32_t* late = gaps + a.list_ld + low;
    const int32_t* table = tb.table + (int64_t)b * tb.ld;
    const int vecs = (p.dim * p.esize) >> 4, mask = p.page_size - 1;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < (int64_t)moves * vecs; i += (int64_t)gridDim.x * 256) {
        const int c = (int)(i % vecs), r = (int)(i / vecs);
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
        const uint4 k = reinterpret_cast<const uint4*>((const char*)p.k + kf)[c];
        const uint4 v = reinterpret_cast<const uint4*>((const char*)p.v + vf)[c];
        reinterpret_cast<uint4*>((char*)p.k + kt)[c] = k;
        reinterpret_cast<uint4*>((char*)p.v + vt)[c] = v;
    }
}

}  // namespace

void launch_kv_append(const KvPool& p, const KvTable& tb, const KvAppend& a, hipStream_t s) {
    const int64_t copies = (int64_t)a.T * p.heads * ((p.dim * p.esize) >> 4);
    const bool side = a.mass || a.positions;
    kv_append_kernel<<<dim3((unsigned)((copies + 255) / 256), tb.B, side ? 3 : 2), 256, 0, s>>>(p, tb, a);
}

size_t kv_attend_ws_bytes(const KvPool&, int, int, int, bool) { return 0; }

void launch_kv_attend(const KvPool& p, const KvTable& tb, const KvAttend& a, hipStream_t s) {
    const dim3 grid(p.heads * a.group, tb.B), mgrid((((int64_t)tb.max_pages << p.page_shift) + 255) / 256, p.heads, tb.B);
    if (p.dtype == KV_F32) kv_attend_kernel<float><<<grid, 256, 0, s>>>(p, tb, a);
    else if (p.dtype == KV_BF16) kv_attend_kernel<bf16_t><<<grid, 256, 0, s>>>(p, tb, a);
    else kv_attend_kernel<f16_t><<<grid, 256, 0, s>>>(p, tb, a);
    if (!a.mass) return;
    if (p.dtype == KV_F32) kv_mass_kernel<float><<<mgrid, 256, 0, s>>>(p, tb, a);
    else if (p.dtype == KV_BF16) kv_mass_kernel<bf16_t><<<mgrid, 256, 0, s>>>(p, tb, a);
    else kv_mass_kernel<f16_t><<<mgrid, 256, 0, s>>>(p, tb, a);
}

// Entries of one list: ranks of kept slots and numbers of gaps lie below n <= min(budget, capacity).
static size_t kv_evict_list(const KvPool& p, int max_pages, int budget) {
    return (size_t)std::min<int64_t>(budget, (int64_t)max_pages << p.page_shift);
}

// gaps and late kept slots of every (sequence, kv head), and {kept below n, n}
size_t kv_evict_ws_bytes(const KvPool& p, int B, int max_pages, int budget) {
    return (size_t)B * p.heads * (2 * kv_evict_list(p, max_pages, budget) + 2) * sizeof(int32_t);
}

void launch_kv_evict(const KvPool& p, const KvTable& tb, KvEvict a, void* ws, hipStream_t s) {
    a.counts = (int32_t*)ws;
    a.lists = a.counts + (size_t)2 * tb.B * p.heads;
    a.list_ld = (int64_t)kv_evict_list(p, tb.max_pages, a.budget);
    kv_select_kernel<<<dim3(p.heads, tb.B), EV_THREADS, 0, s>>>(p, tb, a);
    const int64_t most = std::min((int64_t)a.budget, ((int64_t)tb.max_pages << p.page_shift) - a.budget);
    const int64_t vecs = std::max<int64_t>(most, 1) * ((p.dim * p.esize) >> 4);
    kv_move_kernel<<<dim3((unsigned)std::min<int64_t>((vecs + 255) / 256, 64), p.heads, tb.B), 256, 0, s>>>(p, tb, a);
}

}  // namespace taco
