// C ABI of libtaco_hip.so (include/taco.h): weight folding / re-packing at create time and the
// launch sequences of the four stages.  No arithmetic happens on the host after taco_create.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdlib>
#include <cstdio>
#include <cstring>
#include <map>
#include <mutex>
#include <string>
#include <vector>

#include "../../include/taco.h"
#include "kernels.h"

using namespace taco;

// ---------------------------------------------------------------------------------------
// errors
static thread_local char g_err[1024] = "";
static int fail(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return -1;
}
#define HIP_OK(expr)                                                                             \
    do {                                                                                         \
        hipError_t e_ = (expr);                                                                  \
        if (e_ != hipSuccess) return fail("%s failed: %s (%s:%d)", #expr, hipGetErrorString(e_), \
                                          __FILE__, __LINE__);                                   \
    } while (0)

extern "C" const char* taco_last_error(void) { return g_err; }

// ---------------------------------------------------------------------------------------
// timing
void Timing::begin(int k, hipStream_t s) {
    if (k != kind) return;
    if (used + 2 > ev.size()) {
        hipEvent_t a, b;
        (void)hipEventCreate(&a);
        (void)hipEventCreate(&b);
        ev.push_back(a);
        ev.push_back(b);
    }
    (void)hipEventRecord(ev[used], s);
}
void Timing::end(int k, hipStream_t s) {
    if (k != kind) return;
    (void)hipEventRecord(ev[used + 1], s);
    used += 2;
}

static const char* kKernelNames[KK_COUNT] = {
    "conv_gemm", "highway_combine", "embed_gather", "bigru_scan", "dec_gemm", "dec_attention",
    "dec_finalize", "decode_graph", "gl_mag", "gl_iter", "gl_ola", "dec_persistent", "dec_tile"};

// ---------------------------------------------------------------------------------------
// weights on the device
struct ConvW {
    float* W = nullptr; int ldw = 0;
    int Cin = 0, taps = 1, padl = 0, N = 0;
    float* bias = nullptr; float* scale = nullptr; float* shift = nullptr;
};
struct DecW {
    float* Wp = nullptr; float* bias = nullptr;
    int K = 0, N = 0;
};
struct CbhgW {
    int in_depth = 0, K = 0, bank_filters = 0, proj1 = 0, proj2 = 0, highway_depth = 0, n_highway = 0, gru = 0;
    int pool_width = 2;      // max-pool width (stride 1, 'same'): 2 is fused into proj_1's loader, 1 is the identity,
                             //   wider windows run maxpool_same_kernel into a buffer of their own
    std::vector<ConvW> bank;
    GemmGroup* bank_groups = nullptr;   // device table: the K bank convolutions, widest first (one grouped launch)
    ConvW p1, p2, fix;
    bool has_fix = false;
    std::vector<ConvW> hw;   // N = 2*highway_depth: [H | T]
    ConvW rnn_in;            // N = 6*gru: [fw gates | fw cand | bw gates | bw cand]
    float* Pg = nullptr;     // [2][64][512]
    float* Pc = nullptr;     // [2][32][512]
    float* Pm = nullptr;     // [2][8][96][64]: the A-operand image of bigru_scan_mfma_kernel (128 cells only)
    float* Pm4 = nullptr;    // [2][8][96][64]: the A-operand image of bigru_scan_mfma4_kernel (128 cells only)
};

struct GraphEntry {
    std::vector<uintptr_t> key;
    hipGraph_t graph = nullptr;
    hipGraphExec_t exec = nullptr;
};

struct taco_ctx {
    TacoHParams hp;
    int device = 0;
    std::vector<void*> allocs;
    char* arena = nullptr;         // all re-packed weights
    size_t arena_bytes = 0, arena_off = 0;
    float* enc_lut = nullptr;      // prenet(embedding) [num_chars, prenet2]
    CbhgW enc, post;
    ConvW mem_layer, lin_dense;
    ConvW mel_proj;                // optional "audio/mel_basis" [num_mels, num_freq] as a [ceil16(num_freq), 128] GEMM operand
    DecW pre1, pre2, att_g, att_c, query, proj, g1_g, g1_c, g2_g, g2_c, outp;
    DecW pre1_f, g1_g_f, g1_c_f;   // folded forms for the persistent decoder (Loader::dec_fold)
    DecW att_g_p, g2_g_p;          // row-reordered copies (early inputs first) for the persistent decoder
    float* attn_v = nullptr;
    float* twiddle = nullptr;
    float* window = nullptr;
    float* gl_image = nullptr;     // LDS image of gl_iter2's tables (window | twiddle tables), device
    Timing timing;
    bool timing_on = false;
    int decode_mode = 2;           // 0 eager per-stage kernels, 1 captured hipGraph of them, 2 persistent kernel
    unsigned long long* sync_words = nullptr;  // persistent decoder: per 16-utterance group {counter, abort}, 128 B apart
    int last_sync_groups = 0;                  // groups used by the last decode if it was persistent, else 0
    int last_persist_wgs = 0;                  // its grid size (for the status message)
    // Host mirror of the status words: a 32-byte device-to-host copy into pinned memory follows every persistent
    // launch on its stream, so the next taco_decode of the handle learns without a synchronisation whether the
    // previous launch aborted. persist_broken: it did; the handle uses the captured per-stage path from then on.
    unsigned* host_status = nullptr;
    hipEvent_t status_ev = nullptr;
    // Griffin-Lim of a batch as up to 4 utterance groups on streams of their own (gl_impl): created lazily, on first use
    hipStream_t gl_streams[3] = {nullptr, nullptr, nullptr};
    hipEvent_t gl_fork = nullptr, gl_join[3] = {nullptr, nullptr, nullptr};
    int gl_split = 1;              // taco_set_gl_split: utterance groups of a Griffin-Lim call on streams of their own
    int bigru_mode = 0;            // taco_set_bigru_mode: 0 = one utterance per workgroup (latency), 1 = sixteen on MFMA
    bool status_pending = false;
    bool persist_broken = false;
    unsigned long long* dbg_stamps = nullptr;  // PD_STAMPS builds: 64 s_memrealtime stamps of one step
    std::vector<GraphEntry> graphs;
};

// ---------------------------------------------------------------------------------------
// taco_griffin_lim_noalloc: the vocoder for callers that cannot allocate (include/taco.h). Its working set (the
// target magnitudes and the two ping-pong frame buffers of gl_impl) lives in this file-scope device array instead of a
// caller workspace. Every GPU the library runs on holds its own copy, at its own address, until the process ends; the
// name `scratch` is only a host-side stand-in, so the address is asked for once per device at taco_create
// (hipGetSymbolAddress with that device current) and only that pointer is ever handed to kernels.
constexpr int NOALLOC_MAX_FRAMES = 1024;    // B * T: one utterance of max_iters = 200 decoder steps x r = 5 frames
constexpr size_t NOALLOC_MAG_BYTES = ((size_t)NOALLOC_MAX_FRAMES * 1025 * 4 + 255) & ~(size_t)255;
constexpr size_t NOALLOC_FRAMES_BYTES = ((size_t)NOALLOC_MAX_FRAMES * 2048 * 4 + 255) & ~(size_t)255;   // win <= n_fft
constexpr size_t NOALLOC_SCRATCH_BYTES = NOALLOC_MAG_BYTES + 2 * NOALLOC_FRAMES_BYTES;                  // 20.0 MiB
static __device__ __align__(256) unsigned char scratch[NOALLOC_SCRATCH_BYTES];
static void* g_scratch_ptr[64] = {};        // per device, filled by taco_create
static std::mutex g_scratch_mu;

static int scratch_bind_device(int device) {
    std::lock_guard<std::mutex> lk(g_scratch_mu);
    if (device < 0 || device >= 64) return fail("device %d out of range for the static scratch table", device);
    if (g_scratch_ptr[device]) return 0;
    void* p = nullptr;
    hipError_t e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));     // (the current device is `device`)
    if (e != hipSuccess || !p)
        return fail("hipGetSymbolAddress(scratch) failed on device %d: %s", device, hipGetErrorString(e));
    g_scratch_ptr[device] = p;
    return 0;
}

namespace {

struct Loader {
    std::map<std::string, const TacoWeightEntry*> tab;
    taco_ctx* c;
    std::string err;

    const TacoWeightEntry* get(const std::string& name, std::initializer_list<int64_t> shape) {
        auto it = tab.find(name);
        if (it == tab.end()) { if (err.empty()) err = "missing weight '" + name + "'"; return nullptr; }
        const TacoWeightEntry* e = it->second;
        bool ok = e->ndim == (int)shape.size() && e->data != nullptr;
        int i = 0;
        for (int64_t d : shape) { if (ok && e->dims[i] != d) ok = false; ++i; }
        if (!ok) {
            if (err.empty()) {
                err = "weight '" + name + "' has the wrong shape (want [";
                for (int64_t d : shape) err += std::to_string(d) + ",";
                err += "])";
            }
            return nullptr;
        }
        return e;
    }
    // All device-side weights live in ONE allocation (sub-allocated at 256 B granularity): a decoder step touches
    // ~25 weight/bias arrays per step, and separate hipMallocs would put each on its own page-table fragment.
    float* upload(const std::vector<float>& h) {
        const size_t bytes = (std::max<size_t>(h.size(), 4) * sizeof(float) + 255) & ~(size_t)255;
        if (c->arena_off + bytes > c->arena_bytes) {
            if (err.empty()) err = "weight arena overflow";
            return nullptr;
        }
        char* d = c->arena + c->arena_off;
        c->arena_off += bytes;
        if (hipMemcpy(d, h.data(), h.size() * sizeof(float), hipMemcpyHostToDevice) != hipSuccess) {
            if (err.empty()) err = "hipMemcpy failed for weights";
            return nullptr;
        }
        return (float*)d;
    }
    float* upload_vec(const std::string& name, int64_t n) {
        const TacoWeightEntry* e = get(name, {n});
        if (!e) return nullptr;
        return upload(std::vector<float>(e->data, e->data + n));
    }
    // kernel [taps, Cin, N] (or [Cin, N] when taps == 0) -> zero-padded [taps*Cin, ldw]
    bool conv(ConvW& w, const std::string& kname, const std::string& bname, int taps, int Cin, int N) {
        const TacoWeightEntry* e = taps > 0 ? get(kname, {taps, Cin, N}) : get(kname, {Cin, N});
        if (!e) return false;
        const int tp = taps > 0 ? taps : 1;
        w.Cin = Cin; w.taps = tp; w.padl = (tp - 1) / 2; w.N = N;
        w.ldw = (N + 127) / 128 * 128;
        std::vector<float> h((size_t)tp * Cin * w.ldw, 0.f);
        for (size_t k = 0; k < (size_t)tp * Cin; ++k)
            memcpy(&h[k * w.ldw], e->data + k * N, (size_t)N * sizeof(float));
        w.W = upload(h);
        if (!bname.empty()) w.bias = upload_vec(bname, N);
        return w.W != nullptr && (bname.empty() || w.bias != nullptr);
    }
    // tf.layers.batch_normalization inference affine, epsilon 1e-3
    bool bn(ConvW& w, const std::string& scope) {
        const int N = w.N;
        const TacoWeightEntry* g = get(scope + "/gamma", {N});
        const TacoWeightEntry* b = get(scope + "/beta", {N});
        const TacoWeightEntry* m = get(scope + "/moving_mean", {N});
        const TacoWeightEntry* v = get(scope + "/moving_variance", {N});
        if (!g || !b || !m || !v) return false;
        std::vector<float> sc(N), sh(N);
        for (int i = 0; i < N; ++i) {
            const double inv = (double)g->data[i] / std::sqrt((double)v->data[i] + 1e-3);
            sc[i] = (float)inv;
            sh[i] = (float)((double)b->data[i] - (double)m->data[i] * inv);
        }
        w.scale = upload(sc);
        w.shift = upload(sh);
        return w.scale && w.shift;
    }
    bool cbhg(CbhgW& cb, const std::string& scope) {
        const int G = cb.gru, D = cb.highway_depth;
        cb.bank.resize(cb.K);
        for (int k = 1; k <= cb.K; ++k) {
            const std::string s = scope + "/conv_bank/conv_bank_" + std::to_string(k) + "/conv1d/";
            if (!conv(cb.bank[k - 1], s + "kernel", s + "bias", k, cb.in_depth, cb.bank_filters)) return false;
            const std::string b = scope + "/conv_bank/batch_normalization" + (k == 1 ? "" : "_" + std::to_string(k - 1));
            if (!bn(cb.bank[k - 1], b)) return false;
        }
        {
            std::vector<GemmGroup> gt;
            for (int k = cb.K; k >= 1; --k) {   // widest (most work) first
                const ConvW& w = cb.bank[k - 1];
                gt.push_back(GemmGroup{w.W, w.bias, w.scale, w.shift, w.taps, w.padl, (k - 1) * cb.bank_filters, 0});
            }
            std::vector<float> raw((gt.size() * sizeof(GemmGroup) + 3) / 4);
            memcpy(raw.data(), gt.data(), gt.size() * sizeof(GemmGroup));
            cb.bank_groups = reinterpret_cast<GemmGroup*>(upload(raw));
            if (!cb.bank_groups) return false;
        }
        std::string s = scope + "/proj_1/conv1d/";
        // proj width comes from the kernel entry itself
        auto it = tab.find(s + "kernel");
        const int pw = it != tab.end() && it->second->ndim == 3 ? (int)it->second->dims[0] : 3;
        if (!conv(cb.p1, s + "kernel", s + "bias", pw, cb.K * cb.bank_filters, cb.proj1)) return false;
        if (!bn(cb.p1, scope + "/batch_normalization")) return false;
        s = scope + "/proj_2/conv1d/";
        if (!conv(cb.p2, s + "kernel", s + "bias", pw, cb.proj1, cb.proj2)) return false;
        if (!bn(cb.p2, scope + "/batch_normalization_1")) return false;
        cb.has_fix = cb.proj2 != D;   // modules.py:83-84
        if (cb.has_fix && !conv(cb.fix, scope + "/dense/kernel", scope + "/dense/bias", 0, cb.proj2, D)) return false;
        cb.hw.resize(cb.n_highway);
        for (int i = 1; i <= cb.n_highway; ++i) {
            const std::string hs = scope + "/highway_" + std::to_string(i);
            const TacoWeightEntry* Hk = get(hs + "/H/kernel", {D, D});
            const TacoWeightEntry* Hb = get(hs + "/H/bias", {D});
            const TacoWeightEntry* Tk = get(hs + "/T/kernel", {D, D});
            const TacoWeightEntry* Tb = get(hs + "/T/bias", {D});
            if (!Hk || !Hb || !Tk || !Tb) return false;
            ConvW& w = cb.hw[i - 1];
            w.Cin = D; w.taps = 1; w.padl = 0; w.N = 2 * D; w.ldw = (2 * D + 127) / 128 * 128;
            // columns in blocks of 64 = [32 H | 32 T] of the same 32 units (ACT_HIGHWAY_FUSED, kernels.h)
            std::vector<float> h((size_t)D * w.ldw, 0.f), bias(2 * D);
            for (int u = 0; u < D; ++u) {
                const int ch = (u / 32) * 64 + (u % 32), ct = ch + 32;
                for (int k = 0; k < D; ++k) {
                    h[(size_t)k * w.ldw + ch] = Hk->data[(size_t)k * D + u];
                    h[(size_t)k * w.ldw + ct] = Tk->data[(size_t)k * D + u];
                }
                bias[ch] = Hb->data[u];
                bias[ct] = Tb->data[u];
            }
            w.W = upload(h);
            w.bias = upload(bias);
            if (!w.W || !w.bias) return false;
        }
        // BiGRU: GRUCell kernels are [in + G, 2G] / [in + G, G], rows ordered [inputs ; state] (A.5)
        const TacoWeightEntry* gk[2]; const TacoWeightEntry* gb[2]; const TacoWeightEntry* ck[2]; const TacoWeightEntry* cbias[2];
        const char* dirs[2] = {"fw", "bw"};
        for (int d = 0; d < 2; ++d) {
            const std::string rs = scope + "/bidirectional_rnn/" + dirs[d] + "/gru_cell/";
            gk[d] = get(rs + "gates/kernel", {D + G, 2 * G});
            gb[d] = get(rs + "gates/bias", {2 * G});
            ck[d] = get(rs + "candidate/kernel", {D + G, G});
            cbias[d] = get(rs + "candidate/bias", {G});
            if (!gk[d] || !gb[d] || !ck[d] || !cbias[d]) return false;
        }
        {
            ConvW& w = cb.rnn_in;
            w.Cin = D; w.taps = 1; w.padl = 0; w.N = 6 * G; w.ldw = (6 * G + 127) / 128 * 128;
            std::vector<float> h((size_t)D * w.ldw, 0.f), bias(6 * G);
            for (int d = 0; d < 2; ++d) {
                for (int k = 0; k < D; ++k) {
                    memcpy(&h[(size_t)k * w.ldw + d * 3 * G], gk[d]->data + (size_t)k * 2 * G, 2 * G * sizeof(float));
                    memcpy(&h[(size_t)k * w.ldw + d * 3 * G + 2 * G], ck[d]->data + (size_t)k * G, G * sizeof(float));
                }
                memcpy(&bias[d * 3 * G], gb[d]->data, 2 * G * sizeof(float));
                memcpy(&bias[d * 3 * G + 2 * G], cbias[d]->data, G * sizeof(float));
            }
            w.W = upload(h);
            w.bias = upload(bias);
            if (!w.W || !w.bias) return false;
        }
        if (G != BIGRU_H) {
            // recurrent halves as they are (rows D .. D+G-1 of the TF kernels), k-major: bigru_scan_generic_kernel
            std::vector<float> pg((size_t)2 * G * 2 * G), pc((size_t)2 * G * G);
            for (int d = 0; d < 2; ++d) {
                memcpy(&pg[(size_t)d * G * 2 * G], gk[d]->data + (size_t)D * 2 * G, (size_t)G * 2 * G * sizeof(float));
                memcpy(&pc[(size_t)d * G * G], ck[d]->data + (size_t)D * G, (size_t)G * G * sizeof(float));
            }
            cb.Pg = upload(pg);
            cb.Pc = upload(pc);
            if (!cb.Pg || !cb.Pc) return false;
        } else {
            // recurrent halves, one register image per thread of bigru_scan_kernel
            const int NT = BIGRU_THREADS, KG = 2 * G * G / NT, KC = G * G / NT;
            std::vector<float> pg((size_t)2 * KG * NT), pc((size_t)2 * KC * NT);
            for (int d = 0; d < 2; ++d) {
                for (int tid = 0; tid < NT; ++tid) {
                    // lane = (k-slice ks of 16 state values, output group): 4 gate outputs x 16 k, 2 candidate x 16 k
                    const int ks = tid & 7, grp = tid >> 3;
                    for (int i = 0; i < KG; ++i)
                        pg[((size_t)d * KG + i) * NT + tid] =
                            gk[d]->data[(size_t)(D + 16 * ks + (i & 15)) * 2 * G + 4 * grp + (i >> 4)];
                    for (int i = 0; i < KC; ++i)
                        pc[((size_t)d * KC + i) * NT + tid] =
                            ck[d]->data[(size_t)(D + 16 * ks + (i & 15)) * G + 2 * grp + (i >> 4)];
                }
            }
            cb.Pg = upload(pg);
            cb.Pc = upload(pc);
            if (!cb.Pg || !cb.Pc) return false;
            // ... and the A-operand image of the throughput variant: wave w owns cells 16 w .. 16 w + 15; register
            // 32 kind + 4 g + m (kind = reset / update / candidate) of lane l is W_kind[k = 16 g + 4 (l / 16) + m][cell
            // 16 w + l % 16], the k order in which the state's float4 quads reach the MFMAs (rnn.hip)
            std::vector<float> pm((size_t)2 * 8 * 96 * 64);
            for (int d = 0; d < 2; ++d)
                for (int w = 0; w < 8; ++w)
                    for (int i = 0; i < 96; ++i)
                        for (int l = 0; l < 64; ++l) {
                            const int kind = i / 32, gm = i % 32, k = 16 * (gm / 4) + 4 * (l / 16) + (gm % 4);
                            const int n = 16 * w + (l % 16);
                            pm[(((size_t)d * 8 + w) * 96 + i) * 64 + l] =
                                kind == 2 ? ck[d]->data[(size_t)(D + k) * G + n]
                                          : gk[d]->data[(size_t)(D + k) * 2 * G + (kind == 1 ? G : 0) + n];
                        }
            cb.Pm = upload(pm);
            if (!cb.Pm) return false;
            // ... and of the four-utterance variant: wave w owns cells 16 w .. 16 w + 15, lane l = (row group q = l / 16,
            // cell 16 w + l % 16); register k (< 64): the gates' W[k + 64 (q / 2)][reset (q even) / update (q odd) cell];
            // register 64 + k (k < 32): the candidate's W[32 q + k][cell]
            std::vector<float> pm4((size_t)2 * 8 * 96 * 64);
            for (int d = 0; d < 2; ++d)
                for (int w = 0; w < 8; ++w)
                    for (int i = 0; i < 96; ++i)
                        for (int l = 0; l < 64; ++l) {
                            const int n = 16 * w + (l & 15), qq = l >> 4;
                            pm4[(((size_t)d * 8 + w) * 96 + i) * 64 + l] =
                                i < 64 ? gk[d]->data[(size_t)(D + i + 64 * (qq >> 1)) * 2 * G + ((qq & 1) ? G : 0) + n]
                                       : ck[d]->data[(size_t)(D + 32 * qq + (i - 64)) * G + n];
                        }
            cb.Pm4 = upload(pm4);
            if (!cb.Pm4) return false;
        }
        return true;
    }
    // decoder-step weights: [K, N] -> Wp[N/16][K/16][64][4]  (decoder.hip)
    bool dec_pack(DecW& w, const float* data, int K, int N) {
        w.K = K; w.N = N;
        const int nt = N / 16, nk = K / 16;
        std::vector<float> h((size_t)K * N);
        for (int t = 0; t < nt; ++t)
            for (int ks = 0; ks < nk; ++ks)
                for (int lane = 0; lane < 64; ++lane)
                    for (int cc = 0; cc < 4; ++cc)
                        h[(((size_t)t * nk + ks) * 64 + lane) * 4 + cc] =
                            data[(size_t)(16 * ks + 4 * (lane >> 4) + cc) * N + 16 * t + (lane & 15)];
        w.Wp = upload(h);
        return w.Wp != nullptr;
    }
    bool dec(DecW& w, const std::string& kname, const std::string& bname, int K, int N) {
        const TacoWeightEntry* e = get(kname, {K, N});
        if (!e || !dec_pack(w, e->data, K, N)) return false;
        if (!bname.empty()) w.bias = upload_vec(bname, N);
        return bname.empty() || w.bias;
    }
    // Folded weights for the persistent decoder: a linear layer L (x -> x Wl + bl, [Kl, Nl]) feeding rows
    // [0, Nl) of the next layer's kernel Wn ([Nl + Kr, N]) is pre-multiplied into it, so that the next layer reads
    // L's INPUT and L leaves the step's dependency chain:  [x ; r] -> x (Wl Wn[0:Nl]) + r Wn[Nl:] + (bn + bl Wn[0:Nl]).
    // `lcol0` selects columns [lcol0, lcol0 + Nl) of Wl / bl (the last of the r output frames). Products in fp64.
    // `order`: row blocks (start, length) of the folded matrix [x rows ; r rows] in the order the kernel wants them
    // (inputs that arrive early first); empty = as is.
    typedef std::vector<std::pair<int, int>> RowOrder;
    static std::vector<float> reorder_rows(const std::vector<float>& h, int N, const RowOrder& order) {
        if (order.empty()) return h;
        std::vector<float> o;
        o.reserve(h.size());
        for (auto& b : order) o.insert(o.end(), h.begin() + (size_t)b.first * N, h.begin() + (size_t)(b.first + b.second) * N);
        return o;
    }
    // plain [K, N] kernel with its row blocks reordered (persistent decoder copies of unfolded layers)
    bool dec_perm(DecW& w, const std::string& kname, const DecW& bias_of, int K, int N, const RowOrder& order) {
        const TacoWeightEntry* e = get(kname, {K, N});
        if (!e) return false;
        const std::vector<float> h = reorder_rows(std::vector<float>(e->data, e->data + (size_t)K * N), N, order);
        if (h.size() != (size_t)K * N || !dec_pack(w, h.data(), K, N)) return false;
        w.bias = bias_of.bias;
        return true;
    }
    bool dec_fold(DecW& w, const TacoWeightEntry* Wl, const TacoWeightEntry* bl, int lcol0, int Nl,
                  const TacoWeightEntry* Wn, const TacoWeightEntry* bn, bool rest_first, const RowOrder& order = {}) {
        const int Kl = (int)Wl->dims[0], ldl = (int)Wl->dims[1];
        const int Kn = (int)Wn->dims[0], N = (int)Wn->dims[1], Kr = Kn - Nl;
        // rows of Wn fed by L: [0, Nl) when the layer's input is [L(x) ; r], [Kr, Kn) when it is [r ; L(x)]
        const int l0 = rest_first ? Kr : 0, r0 = rest_first ? 0 : Nl;
        std::vector<float> h((size_t)(Kl + Kr) * N);
        std::vector<double> acc(N);
        for (int k = 0; k < Kl; ++k) {
            std::fill(acc.begin(), acc.end(), 0.0);
            for (int j = 0; j < Nl; ++j) {
                const double wl = Wl->data[(size_t)k * ldl + lcol0 + j];
                const float* wn = Wn->data + (size_t)(l0 + j) * N;
                for (int n = 0; n < N; ++n) acc[n] += wl * (double)wn[n];
            }
            for (int n = 0; n < N; ++n) h[(size_t)k * N + n] = (float)acc[n];
        }
        for (int k = 0; k < Kr; ++k)
            memcpy(&h[(size_t)(Kl + k) * N], Wn->data + (size_t)(r0 + k) * N, (size_t)N * sizeof(float));
        std::vector<float> bias(N);
        for (int n = 0; n < N; ++n) {
            double a = bn ? (double)bn->data[n] : 0.0;
            if (bl)
                for (int j = 0; j < Nl; ++j) a += (double)bl->data[lcol0 + j] * (double)Wn->data[(size_t)(l0 + j) * N + n];
            bias[n] = (float)a;
        }
        const std::vector<float> hp = reorder_rows(h, N, order);
        if (hp.size() != h.size() || !dec_pack(w, hp.data(), Kl + Kr, N)) return false;
        w.bias = upload(bias);
        return w.bias != nullptr;
    }
    bool dec_gru(DecW& g, DecW& cnd, const std::string& scope, int in, int H) {
        return dec(g, scope + "gates/kernel", scope + "gates/bias", in + H, 2 * H) &&
               dec(cnd, scope + "candidate/kernel", scope + "candidate/bias", in + H, H);
    }
};

constexpr int PD_REGION_DIMS = 1024 + 512 + 512 + 256 + 128 + 768 + 768 + 256 + 256 + 256 + 256;   // 4992

struct Carver {
    char* base; size_t off = 0, cap;
    Carver(void* p, size_t n) : base((char*)p), cap(n) {}
    template <typename T>
    T* take(size_t count) {
        const size_t bytes = (count * sizeof(T) + 255) & ~(size_t)255;
        T* p = (T*)(base + off);
        off += bytes;
        return p;
    }
    bool ok() const { return off <= cap; }
};

inline size_t al(size_t bytes) { return (bytes + 255) & ~(size_t)255; }
inline int bpad16(int B) { return (B + 15) / 16 * 16; }

size_t cbhg_ws_bytes(const CbhgW& cb, size_t M) {
    size_t n = 0;
    n += al(M * cb.K * cb.bank_filters * 4);   // bank
    if (cb.pool_width > 2) n += al(M * cb.K * cb.bank_filters * 4);   // pooled bank (windows wider than the fused 2)
    n += al(M * cb.proj1 * 4);                 // proj1
    n += al(M * cb.proj2 * 4);                 // proj2 + residual
    n += 2 * al(M * cb.highway_depth * 4);     // highway ping-pong
    n += al(M * 6 * cb.gru * 4);               // rnn input projections
    const int sk = conv_gemm_pick_splitk((int)M, cb.proj1, cb.p1.taps * cb.p1.Cin / 16);
    if (sk > 1) n += al((size_t)sk * M * ((cb.proj1 + 63) / 64 * 64) * 4);   // proj_1 split-K partial sums
    return n;
}
size_t enc_ws_bytes(const taco_ctx* c, int B, int T_in) {
    const size_t M = (size_t)B * T_in;
    return al(M * c->enc.in_depth * 4) + cbhg_ws_bytes(c->enc, M);
}
size_t dec_ws_bytes(const taco_ctx* c, int B, int T_in, int S) {
    const TacoHParams& hp = c->hp;
    const size_t Bp = bpad16(B);
    const int NR = hp.num_mels * hp.outputs_per_step;
    const int Dv = 2 * hp.encoder_gru_cells;
    size_t n = 0;
    n += al((size_t)B * T_in * hp.attention_depth * 4);                     // keys
    n += al((size_t)S * NR * Bp * 4);                                        // outQ
    n += al((size_t)S * B * T_in * 4);                                       // alignS
    n += al((size_t)S * Bp * 4);                                             // nz
    n += al((size_t)S * hp.num_mels * Bp * 4);                               // teacher frames (taco_decode_teacher)
    n += al(((size_t)PD_REGION_DIMS * Bp * 2 + 4096 + (size_t)B * T_in * 2 + 64 + (size_t)S * 400 * Bp * 2) * 4) + 4096;  // persistent decoder region
    const size_t state = (size_t)(hp.num_mels + Dv + hp.attention_depth + 2 * hp.decoder_depth) * Bp * 4;
    n += al(state);
    const int mx = std::max(hp.attention_depth, hp.decoder_depth);
    n += al((size_t)hp.prenet_depth1 * Bp * 4) + al((size_t)hp.prenet_depth2 * Bp * 4) + 6 * al((size_t)mx * Bp * 4);
    return n;
}
size_t post_ws_bytes(const taco_ctx* c, int B, int T) {
    const size_t M = (size_t)B * T;
    return cbhg_ws_bytes(c->post, M) + al(M * 2 * c->post.gru * 4);
}
size_t gl_ws_bytes(const taco_ctx* c, int B, int T) {
    const size_t M = (size_t)B * T;
    return al(M * c->hp.num_freq * 4) + 2 * al(M * c->hp.win_length * 4);
}

int run_cbhg(taco_ctx* c, const CbhgW& cb, const float* x, const int32_t* lens, int B, int T, float* out,
             Carver& ws, hipStream_t s) {
    Timing* tm = c->timing_on ? &c->timing : nullptr;
    const int M = B * T;
    float* bank = ws.take<float>((size_t)M * cb.K * cb.bank_filters);
    float* pooled = cb.pool_width > 2 ? ws.take<float>((size_t)M * cb.K * cb.bank_filters) : nullptr;
    float* p1 = ws.take<float>((size_t)M * cb.proj1);
    float* p2 = ws.take<float>((size_t)M * cb.proj2);
    float* hwA = ws.take<float>((size_t)M * cb.highway_depth);
    float* hwB = ws.take<float>((size_t)M * cb.highway_depth);
    float* xp = ws.take<float>((size_t)M * 6 * cb.gru);
    const int sk = conv_gemm_pick_splitk(M, cb.proj1, cb.p1.taps * cb.p1.Cin / 16);
    float* p1part = sk > 1 ? ws.take<float>((size_t)sk * M * ((cb.proj1 + 63) / 64 * 64)) : nullptr;
    if (!ws.ok()) return fail("workspace too small (need >= %zu bytes)", ws.off);
    const int ldb = cb.K * cb.bank_filters;
    if ((size_t)M * std::max(ldb, 6 * cb.gru) * 4 >= ((size_t)1 << 31))
        return fail("B*T = %d too large for 32-bit operand offsets (row width %d)", M, ldb);
    GemmArgs g;
    // conv bank (modules.py:63-67): ReLU inside the conv, then BN; the K convolutions are one grouped launch
    {
        const ConvW& w = cb.bank[0];
        g = GemmArgs{x, cb.in_depth, M, T, w.Cin, 1, 0, nullptr, w.ldw, w.N, nullptr, nullptr, nullptr,
                     nullptr, 0, bank, ldb, ACT_RELU, 0, cb.bank_groups, cb.K, nullptr, 0};
        launch_conv_gemm(g, s, tm);
    }
    // max-pool (modules.py:70-71): the reference's width 2 is folded into proj_1's loader, width 1 is the identity,
    // wider windows are materialised first; proj_1 ReLU + BN (modules.py:74-75)
    const float* p1_in = bank;
    if (cb.pool_width > 2) {
        launch_maxpool_same(bank, pooled, M, T, ldb, cb.pool_width, s, tm);
        p1_in = pooled;
    }
    g = GemmArgs{p1_in, ldb, M, T, cb.p1.Cin, cb.p1.taps, cb.p1.padl, cb.p1.W, cb.p1.ldw, cb.p1.N, cb.p1.bias,
                 cb.p1.scale, cb.p1.shift, nullptr, 0, p1, cb.proj1, ACT_RELU, cb.pool_width == 2 ? 1 : 0, nullptr, 0,
                 p1part, sk};
    launch_conv_gemm(g, s, tm);
    // proj_2 linear + BN, + residual (modules.py:76-80)
    g = GemmArgs{p1, cb.proj1, M, T, cb.p2.Cin, cb.p2.taps, cb.p2.padl, cb.p2.W, cb.p2.ldw, cb.p2.N, cb.p2.bias,
                 cb.p2.scale, cb.p2.shift, x, cb.in_depth, p2, cb.proj2, ACT_NONE, 0};
    launch_conv_gemm(g, s, tm);
    float* h = p2;
    if (cb.has_fix) {   // modules.py:83-84
        g = GemmArgs{p2, cb.proj2, M, T, cb.fix.Cin, 1, 0, cb.fix.W, cb.fix.ldw, cb.fix.N, cb.fix.bias, nullptr,
                     nullptr, nullptr, 0, hwA, cb.highway_depth, ACT_NONE, 0};
        launch_conv_gemm(g, s, tm);
        h = hwA;
    }
    if (cb.highway_depth == 128 && cb.gru * 6 == 768 && cb.n_highway >= 0 && cb.n_highway <= 8 &&
        !getenv("TACO_NO_CBHG_TAIL")) {
        // highway layers + the BiGRU's hoisted input projections as one launch (cbhg_tail_kernel)
        CbhgTailArgs t{};
        t.X = h; t.ldx = cb.highway_depth; t.M = M;
        for (int i = 0; i < cb.n_highway; ++i) { t.Whw[i] = cb.hw[i].W; t.bhw[i] = cb.hw[i].bias; }
        t.n_hw = cb.n_highway;
        t.Wr = cb.rnn_in.W; t.br = cb.rnn_in.bias; t.ldwr = cb.rnn_in.ldw; t.Nr = cb.rnn_in.N;
        t.out = xp; t.ldo = 6 * cb.gru;
        launch_cbhg_tail(t, s, tm);
#ifndef TACO_EXP_NO_BIGRU   // (timing experiment, wrong results: what the chip does with the scan's work gone)
        if (c->bigru_mode == 1 && cb.Pm) launch_bigru_scan_mfma(xp, cb.Pm, lens, out, B, T, s, tm);
        else if (c->bigru_mode == 2 && cb.Pm4) launch_bigru_scan_mfma4(xp, cb.Pm4, lens, out, B, T, s, tm);
        else launch_bigru_scan(xp, cb.Pg, cb.Pc, lens, out, B, T, cb.gru, s, tm);
#else
        (void)hipMemsetAsync(out, 0, (size_t)M * 2 * cb.gru * sizeof(float), s);
#endif
        return 0;
    }
    // highway layers (modules.py:87-88,100-123)
    for (int i = 0; i < cb.n_highway; ++i) {
        const ConvW& w = cb.hw[i];
        // y = H*T + x*(1-T) in the GEMM's epilogue: the [H|T] matrix is never written
        float* nxt = (h == hwA) ? hwB : hwA;
        g = GemmArgs{h, cb.highway_depth, M, T, w.Cin, 1, 0, w.W, w.ldw, w.N, w.bias, nullptr, nullptr, h,
                     cb.highway_depth, nxt, cb.highway_depth, ACT_HIGHWAY_FUSED, 0};
        launch_conv_gemm(g, s, tm);
        h = nxt;
    }
    // BiGRU (modules.py:92-98): input halves as one GEMM, then the scan
    g = GemmArgs{h, cb.highway_depth, M, T, cb.rnn_in.Cin, 1, 0, cb.rnn_in.W, cb.rnn_in.ldw, cb.rnn_in.N,
                 cb.rnn_in.bias, nullptr, nullptr, nullptr, 0, xp, 6 * cb.gru, ACT_NONE, 0};
    launch_conv_gemm(g, s, tm);
    if (c->bigru_mode == 1 && cb.Pm) launch_bigru_scan_mfma(xp, cb.Pm, lens, out, B, T, s, tm);
    else if (c->bigru_mode == 2 && cb.Pm4) launch_bigru_scan_mfma4(xp, cb.Pm4, lens, out, B, T, s, tm);
    else launch_bigru_scan(xp, cb.Pg, cb.Pc, lens, out, B, T, cb.gru, s, tm);
    return 0;
}

int check_launch(const char* what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail("%s: kernel launch failed: %s", what, hipGetErrorString(e));
    return 0;
}

int check_dims(int B, int T) {
    if (B < 1 || T < 1) return fail("batch size and length must be >= 1 (got B=%d, T=%d)", B, T);
    if ((long)B * T > (1L << 30)) return fail("B*T too large");
    return 0;
}

}  // namespace

// ---------------------------------------------------------------------------------------
extern "C" int taco_create(const TacoHParams* hp, const TacoWeightEntry* weights, int32_t n_weights, int32_t device,
                           taco_handle* out) {
    if (!hp || !weights || !out) return fail("taco_create: null argument");
    *out = nullptr;
    // the first field is the size of the caller's struct: fields are only ever appended, so a mismatch means caller and
    // library were built against different headers (checked before any other field is read)
    if (hp->struct_size != sizeof(TacoHParams))
        return fail("taco_create: TacoHParams.struct_size is %u but this library's struct has %zu bytes "
                    "(caller built against another include/taco.h?)", hp->struct_size, sizeof(TacoHParams));
    // shapes the kernels are written for
    const TacoHParams& p = *hp;
    auto m16 = [](int v) { return v > 0 && v % 16 == 0; };
    if (!m16(p.embedded_depth) || !m16(p.prenet_depth1) || !m16(p.prenet_depth2) || !m16(p.encoder_bank_filters) ||
        !m16(p.encoder_proj1) || !m16(p.encoder_proj2) || !m16(p.encoder_highway_depth) || !m16(p.attention_depth) ||
        !m16(p.decoder_depth) || !m16(p.num_mels) || !m16(p.decoder_bank_filters) || !m16(p.decoder_proj1) ||
        !m16(p.decoder_proj2) || !m16(p.decoder_highway_depth))
        return fail("taco_create: every layer width must be a positive multiple of 16");
    if (p.encoder_highway_depth % 32 || p.decoder_highway_depth % 32)
        return fail("taco_create: highway depths must be multiples of 32 (fused highway epilogue)");
    if (!m16(p.encoder_gru_cells) || !m16(p.decoder_gru_cells) || p.encoder_gru_cells > 2048 || p.decoder_gru_cells > 2048)
        return fail("taco_create: *_gru_num_cells must be a positive multiple of 16 (at most 2048)");
    if (p.encoder_proj2 != p.prenet_depth2 || p.decoder_proj2 != p.num_mels)
        return fail("taco_create: the CBHG residual needs proj_num_filters[1] == input depth (modules.py:80)");
    if (p.n_fft != 2048 || p.num_freq != 1025 || p.win_length > 2048 || p.win_length < 2 || (p.win_length & 1) ||
        (p.hop_length & 1) || p.hop_length < 2 || p.hop_length > p.win_length)
        return fail("taco_create: Griffin-Lim kernel needs n_fft=2048, num_freq=1025, even hop <= even win <= 2048");
    // max-pool (hparams.py:31-32,41-42 -> modules.py:70-71): any window, stride 1 only - with another stride the
    // pooled sequence is shorter than the CBHG's input and the residual of modules.py:80 cannot be formed (the
    // reference graph does not build either)
    if (p.encoder_pooling_stride != 1 || p.decoder_pooling_stride != 1 || p.encoder_pooling_width < 1 ||
        p.decoder_pooling_width < 1 || p.encoder_pooling_width > 64 || p.decoder_pooling_width > 64)
        return fail("taco_create: max-pool needs pooling_stride 1 (the residual of modules.py:80 adds the CBHG input to a "
                    "sequence of the same length) and 1 <= pooling_width <= 64, got encoder %d/%d decoder %d/%d",
                    p.encoder_pooling_width, p.encoder_pooling_stride, p.decoder_pooling_width,
                    p.decoder_pooling_stride);
    if (p.encoder_K < 1 || p.decoder_K < 1 || p.outputs_per_step < 1 || p.num_chars < 1 || p.encoder_highways < 0 ||
        p.decoder_highways < 0)
        return fail("taco_create: bad hparams");
    int ndev = 0;
    HIP_OK(hipGetDeviceCount(&ndev));
    if (device < 0 || device >= ndev) return fail("taco_create: device %d not available (%d visible)", device, ndev);
    HIP_OK(hipSetDevice(device));
    if (scratch_bind_device(device)) return -1;
    gl_prepare_device();

    taco_ctx* c = new taco_ctx();
    c->hp = p;
    c->device = device;
    Loader L;
    L.c = c;
    size_t total = 0;
    for (int i = 0; i < n_weights; ++i) {
        if (!weights[i].name) continue;
        L.tab[weights[i].name] = &weights[i];
        size_t n = 1;
        for (int d = 0; d < weights[i].ndim && d < 4; ++d) n *= (size_t)std::max<int64_t>(weights[i].dims[d], 1);
        total += n;
    }
    // packed copies pad N to 128 columns (num_freq 1025 -> 1152) and add folded BN / tables: 2x + 16 MB is ample
    c->arena_bytes = total * sizeof(float) * 2 + (16u << 20);
    {
        void* d = nullptr;
        hipError_t e = hipMalloc(&d, c->arena_bytes);
        if (e != hipSuccess) {
            delete c;
            return fail("taco_create: hipMalloc(%zu) failed: %s", c->arena_bytes, hipGetErrorString(e));
        }
        c->arena = (char*)d;
        c->allocs.push_back(d);
    }

    const int G2 = 2 * p.encoder_gru_cells;   // encoder output depth
    const int NR = p.num_mels * p.outputs_per_step;
    const std::string DEC = "decoder/output_projection_wrapper/";
    const std::string CELL0 = DEC + "multi_rnn_cell/cell_0/output_projection_wrapper/";
    const std::string ATTW = CELL0 + "concat_output_and_attention_wrapper/attention_wrapper/";

    c->enc.in_depth = p.prenet_depth2; c->enc.K = p.encoder_K; c->enc.bank_filters = p.encoder_bank_filters;
    c->enc.proj1 = p.encoder_proj1; c->enc.proj2 = p.encoder_proj2; c->enc.highway_depth = p.encoder_highway_depth;
    c->enc.n_highway = p.encoder_highways; c->enc.gru = p.encoder_gru_cells;
    c->enc.pool_width = p.encoder_pooling_width; c->post.pool_width = p.decoder_pooling_width;
    c->post.in_depth = p.num_mels; c->post.K = p.decoder_K; c->post.bank_filters = p.decoder_bank_filters;
    c->post.proj1 = p.decoder_proj1; c->post.proj2 = p.decoder_proj2; c->post.highway_depth = p.decoder_highway_depth;
    c->post.n_highway = p.decoder_highways; c->post.gru = p.decoder_gru_cells;

    ConvW epre1, epre2;
    bool ok = true;
    ok = ok && L.conv(epre1, "prenet/prenet_dense_1/kernel", "prenet/prenet_dense_1/bias", 0, p.embedded_depth, p.prenet_depth1);
    ok = ok && L.conv(epre2, "prenet/prenet_dense_2/kernel", "prenet/prenet_dense_2/bias", 0, p.prenet_depth1, p.prenet_depth2);
    ok = ok && L.cbhg(c->enc, "encoder_cbhg");
    ok = ok && L.conv(c->mem_layer, "memory_layer/kernel", "", 0, G2, p.attention_depth);
    const std::string DP = ATTW + "decoder_prenet_wrapper/decoder_prenet/";
    ok = ok && L.dec(c->pre1, DP + "prenet_dense_1/kernel", DP + "prenet_dense_1/bias", p.num_mels + G2, p.prenet_depth1);
    ok = ok && L.dec(c->pre2, DP + "prenet_dense_2/kernel", DP + "prenet_dense_2/bias", p.prenet_depth1, p.prenet_depth2);
    ok = ok && L.dec_gru(c->att_g, c->att_c, ATTW + "decoder_prenet_wrapper/gru_cell/", p.prenet_depth2, p.attention_depth);
    ok = ok && L.dec(c->query, ATTW + "bahdanau_attention/query_layer/kernel", "", p.attention_depth, p.attention_depth);
    ok = ok && (c->attn_v = L.upload_vec(ATTW + "bahdanau_attention/attention_v", p.attention_depth)) != nullptr;
    ok = ok && L.dec(c->proj, CELL0 + "kernel", CELL0 + "bias", p.attention_depth + G2, p.decoder_depth);
    ok = ok && L.dec_gru(c->g1_g, c->g1_c, DEC + "multi_rnn_cell/cell_1/gru_cell/", p.decoder_depth, p.decoder_depth);
    ok = ok && L.dec_gru(c->g2_g, c->g2_c, DEC + "multi_rnn_cell/cell_2/gru_cell/", p.decoder_depth, p.decoder_depth);
    ok = ok && L.dec(c->outp, DEC + "kernel", DEC + "bias", p.decoder_depth, NR);
    if (ok) {
        // persistent decoder: the r-frame output projection folded into the next step's prenet-1 (input
        // [last frame ; ctx] -> [o2 ; ctx]) and the concat projection folded into GRU-1 (input [d0 ; h] / [d0 ; r.h]
        // -> [h_att ; ctx ; h] / [h_att ; ctx ; r.h])
        const int64_t D = p.decoder_depth, A = p.attention_depth;
        const TacoWeightEntry* Wo = L.get(DEC + "kernel", {D, NR});
        const TacoWeightEntry* bo = L.get(DEC + "bias", {NR});
        const TacoWeightEntry* W1 = L.get(DP + "prenet_dense_1/kernel", {p.num_mels + G2, p.prenet_depth1});
        const TacoWeightEntry* b1 = L.get(DP + "prenet_dense_1/bias", {p.prenet_depth1});
        const TacoWeightEntry* Wp = L.get(CELL0 + "kernel", {A + G2, D});
        const TacoWeightEntry* bp = L.get(CELL0 + "bias", {D});
        const std::string g1s = DEC + "multi_rnn_cell/cell_1/gru_cell/";
        const TacoWeightEntry* Wg = L.get(g1s + "gates/kernel", {2 * D, 2 * D});
        const TacoWeightEntry* bg = L.get(g1s + "gates/bias", {2 * D});
        const TacoWeightEntry* Wc = L.get(g1s + "candidate/kernel", {2 * D, D});
        const TacoWeightEntry* bc = L.get(g1s + "candidate/bias", {D});
        ok = Wo && bo && W1 && b1 && Wp && bp && Wg && bg && Wc && bc &&
             // K orders: inputs that are ready early first, the one a stage waits for last
             L.dec_fold(c->pre1_f, Wo, bo, NR - p.num_mels, p.num_mels, W1, b1, false,
                        {{(int)D, G2}, {0, (int)D}}) &&                                        // [ctx ; o2]
             L.dec_fold(c->g1_g_f, Wp, bp, 0, (int)D, Wg, bg, false,
                        {{0, (int)A}, {(int)A + G2, (int)D}, {(int)A, G2}}) &&                  // [h_att ; h1 ; ctx]
             L.dec_fold(c->g1_c_f, Wp, bp, 0, (int)D, Wc, bc, false) &&                        // [h_att ; ctx ; r.h1]
             L.dec_perm(c->att_g_p, ATTW + "decoder_prenet_wrapper/gru_cell/gates/kernel", c->att_g,
                        p.prenet_depth2 + (int)A, 2 * (int)A, {{p.prenet_depth2, (int)A}, {0, p.prenet_depth2}}) &&   // [h_att ; p2]
             L.dec_perm(c->g2_g_p, DEC + "multi_rnn_cell/cell_2/gru_cell/gates/kernel", c->g2_g, 2 * (int)D, 2 * (int)D,
                        {{(int)D, (int)D}, {0, (int)D}});                                      // [h2 ; o1]
    }
    ok = ok && L.cbhg(c->post, "post_cbhg");
    ok = ok && L.conv(c->lin_dense, "dense/kernel", "dense/bias", 0, 2 * p.decoder_gru_cells, p.num_freq);
    if (ok && L.tab.count("audio/mel_basis")) {
        // analysis side (taco_spectrogram): the mel filterbank, transposed and zero-padded in K to a multiple of 16
        const TacoWeightEntry* mb = L.get("audio/mel_basis", {p.num_mels, p.num_freq});
        ok = mb != nullptr;
        if (ok) {
            ConvW& w = c->mel_proj;
            w.Cin = (p.num_freq + 15) / 16 * 16; w.taps = 1; w.padl = 0; w.N = p.num_mels;
            w.ldw = (p.num_mels + 127) / 128 * 128;
            std::vector<float> hw((size_t)w.Cin * w.ldw, 0.f);
            for (int m = 0; m < p.num_mels; ++m)
                for (int k = 0; k < p.num_freq; ++k) hw[(size_t)k * w.ldw + m] = mb->data[(size_t)m * p.num_freq + k];
            w.W = L.upload(hw);
            ok = w.W != nullptr;
        }
    }
    const TacoWeightEntry* emb = ok ? L.get("embedding", {p.num_chars, p.embedded_depth}) : nullptr;
    ok = ok && emb;
    if (ok) {
        // FFT twiddles exp(-2 pi i j / 2048) and the periodic Hann window, from double
        std::vector<float> tw(2 * (size_t)p.n_fft), win(p.win_length);
        for (int j = 0; j < p.n_fft; ++j) {
            tw[2 * j] = (float)std::cos(2.0 * M_PI * j / p.n_fft);
            tw[2 * j + 1] = (float)-std::sin(2.0 * M_PI * j / p.n_fft);
        }
        for (int n = 0; n < p.win_length; ++n) win[n] = (float)(0.5 - 0.5 * std::cos(2.0 * M_PI * n / p.win_length));
        c->twiddle = L.upload(tw);
        c->window = L.upload(win);
        c->gl_image = L.upload(gl_lds_image(tw, win));
        c->sync_words = reinterpret_cast<unsigned long long*>(L.upload(std::vector<float>(8 * 32, 0.f)));
        ok = c->twiddle && c->window && c->gl_image && c->sync_words;
        if (ok && (hipHostMalloc(reinterpret_cast<void**>(&c->host_status), 64, hipHostMallocDefault) != hipSuccess ||
                   hipEventCreateWithFlags(&c->status_ev, hipEventDisableTiming) != hipSuccess)) {
            L.err = "cannot allocate the decoder status mirror";
            ok = false;
        }
        if (ok) memset(c->host_status, 0, 64);
    }
    if (ok) {
        // encoder prenet of every symbol, once: prenet(embedding[id]) is a pure function of the id
        // (batch.py:36-40 + encoder.py:37 with dropout = identity), computed by the same GEMM kernel.
        float* demb = L.upload(std::vector<float>(emb->data, emb->data + (size_t)p.num_chars * p.embedded_depth));
        float* t1 = L.upload(std::vector<float>((size_t)p.num_chars * p.prenet_depth1, 0.f));
        c->enc_lut = L.upload(std::vector<float>((size_t)p.num_chars * p.prenet_depth2, 0.f));
        ok = demb && t1 && c->enc_lut;
        if (ok) {
            const int M = p.num_chars;
            GemmArgs g{demb, p.embedded_depth, M, M, epre1.Cin, 1, 0, epre1.W, epre1.ldw, epre1.N, epre1.bias, nullptr,
                       nullptr, nullptr, 0, t1, p.prenet_depth1, ACT_RELU, 0};
            launch_conv_gemm(g, nullptr, nullptr);
            g = GemmArgs{t1, p.prenet_depth1, M, M, epre2.Cin, 1, 0, epre2.W, epre2.ldw, epre2.N, epre2.bias, nullptr,
                         nullptr, nullptr, 0, c->enc_lut, p.prenet_depth2, ACT_RELU, 0};
            launch_conv_gemm(g, nullptr, nullptr);
            if (hipDeviceSynchronize() != hipSuccess || hipGetLastError() != hipSuccess) {
                L.err = "prenet table kernels failed";
                ok = false;
            }
        }
    }
    if (!ok) {
        fail("taco_create: %s", L.err.empty() ? "weight upload failed" : L.err.c_str());
        taco_destroy(c);
        return -1;
    }
    *out = c;
    return 0;
}

extern "C" void taco_destroy(taco_handle h) {
    if (!h) return;
    (void)hipSetDevice(h->device);
    for (auto& g : h->graphs) {
        if (g.exec) (void)hipGraphExecDestroy(g.exec);
        if (g.graph) (void)hipGraphDestroy(g.graph);
    }
    for (hipEvent_t e : h->timing.ev) (void)hipEventDestroy(e);
    if (h->status_ev) (void)hipEventDestroy(h->status_ev);
    for (int g = 0; g < 3; ++g) {
        if (h->gl_streams[g]) (void)hipStreamDestroy(h->gl_streams[g]);
        if (h->gl_join[g]) (void)hipEventDestroy(h->gl_join[g]);
    }
    if (h->gl_fork) (void)hipEventDestroy(h->gl_fork);
    if (h->host_status) (void)hipHostFree(h->host_status);
    for (void* p : h->allocs) (void)hipFree(p);
    delete h;
}

extern "C" size_t taco_workspace_bytes(taco_handle h, int32_t B, int32_t T_in, int32_t max_iters) {
    if (!h || B < 1 || T_in < 1 || max_iters < 1) return 0;
    const int T = max_iters * h->hp.outputs_per_step;
    size_t stage = std::max(std::max(enc_ws_bytes(h, B, T_in), dec_ws_bytes(h, B, T_in, max_iters)),
                            std::max(post_ws_bytes(h, B, T), gl_ws_bytes(h, B, T)));
    return stage + al((size_t)B * T_in * 2 * h->hp.encoder_gru_cells * 4) + 4096;
}

// ---------------------------------------------------------------------------------------
static int encode_impl(taco_ctx* c, const int32_t* ids, const int32_t* lens, int B, int T_in, float* enc_out,
                       Carver& ws, hipStream_t s) {
    Timing* tm = c->timing_on ? &c->timing : nullptr;
    const int M = B * T_in;
    float* x0 = ws.take<float>((size_t)M * c->enc.in_depth);
    if (!ws.ok()) return fail("taco_encode: workspace too small");
    launch_embed_gather(ids, c->enc_lut, x0, M, c->enc.in_depth, c->hp.num_chars, s, tm);
    return run_cbhg(c, c->enc, x0, lens, B, T_in, enc_out, ws, s);
}

extern "C" int taco_encode(taco_handle h, const int32_t* ids, const int32_t* lens, int32_t B, int32_t T_in,
                           float* enc_out, void* ws, size_t ws_bytes, taco_stream_t stream) {
    if (!h || !ids || !lens || !enc_out || !ws) return fail("taco_encode: null argument");
    if (check_dims(B, T_in)) return -1;
    HIP_OK(hipSetDevice(h->device));
    Carver cv(ws, ws_bytes);
    if (encode_impl(h, ids, lens, B, T_in, enc_out, cv, (hipStream_t)stream)) return -1;
    return check_launch("taco_encode");
}

// ---------------------------------------------------------------------------------------
struct DecBufs {
    float *keys, *outQ, *alignS;
    int32_t* nz;
    float *go, *ctx, *hatt, *h1, *h2;   // zero-initialised state block (contiguous)
    size_t state_bytes;
    float *p1, *p2, *rh, *u, *q, *d0, *o1, *o2;
};

static void decode_steps(taco_ctx* c, const DecBufs& d, const float* enc_out, const float* keep, int B, int T_in,
                         int S, hipStream_t s, Timing* tm, const float* teachQ = nullptr) {
    const TacoHParams& hp = c->hp;
    const int Bp = bpad16(B);
    const int NR = hp.num_mels * hp.outputs_per_step;
    const int Dv = 2 * hp.encoder_gru_cells;
    const int A = hp.attention_depth, D = hp.decoder_depth;
    const int keep_ld = hp.prenet_depth1 + hp.prenet_depth2;
    for (int st = 0; st < S; ++st) {
        // previous frame: <GO>, then the last of the r frames just produced (helpers.py:77) or, teacher-forced, the
        // matching target frame (helpers.py:42)
        const float* prev = st == 0 ? d.go
                          : teachQ ? teachQ + (size_t)(st - 1) * hp.num_mels * Bp
                                   : d.outQ + ((size_t)(st - 1) * NR + (NR - hp.num_mels)) * Bp;
        const float* kp = keep ? keep + (size_t)st * B * keep_ld : nullptr;
        DecGemmArgs a{};
        a.B = B; a.Bpad = Bp;
        // decoder prenet on concat([prev frame, prev context]) (rnn_wrappers.py:25; AttentionWrapper cell_input_fn)
        a.src0 = prev; a.k16_0 = hp.num_mels / 16; a.src1 = d.ctx; a.k16_1 = Dv / 16;
        a.Wp = c->pre1.Wp; a.N = c->pre1.N; a.bias = c->pre1.bias; a.epi = DE_RELU; a.out = d.p1;
        a.keep = kp; a.keep_ld = keep_ld;
        launch_dec_gemm(a, s, tm);
        a = DecGemmArgs{}; a.B = B; a.Bpad = Bp;
        a.src0 = d.p1; a.k16_0 = hp.prenet_depth1 / 16;
        a.Wp = c->pre2.Wp; a.N = c->pre2.N; a.bias = c->pre2.bias; a.epi = DE_RELU; a.out = d.p2;
        a.keep = kp ? kp + hp.prenet_depth1 : nullptr; a.keep_ld = keep_ld;
        launch_dec_gemm(a, s, tm);
        // attention GRU (rnn_wrappers.py:26)
        a = DecGemmArgs{}; a.B = B; a.Bpad = Bp;
        a.src0 = d.p2; a.k16_0 = hp.prenet_depth2 / 16; a.src1 = d.hatt; a.k16_1 = A / 16;
        a.Wp = c->att_g.Wp; a.N = 2 * A; a.bias = c->att_g.bias; a.epi = DE_GATES; a.out = d.rh; a.u = d.u; a.h = d.hatt;
        launch_dec_gemm(a, s, tm);
        a.src1 = d.rh; a.Wp = c->att_c.Wp; a.N = A; a.bias = c->att_c.bias; a.epi = DE_CAND; a.out = nullptr;
        launch_dec_gemm(a, s, tm);
        // Bahdanau attention: query layer, scores, softmax, context
        a = DecGemmArgs{}; a.B = B; a.Bpad = Bp;
        a.src0 = d.hatt; a.k16_0 = A / 16; a.Wp = c->query.Wp; a.N = A; a.epi = DE_LINEAR; a.out = d.q;
        launch_dec_gemm(a, s, tm);
        DecAttnArgs at{d.q, d.keys, enc_out, c->attn_v, d.ctx, d.alignS + (size_t)st * B * T_in, B, Bp, T_in, A, Dv};
        launch_dec_attention(at, s, tm);
        // concat([cell output, context]) -> projection to decoder depth (rnn_wrappers.py:53, decoder.py:29)
        a = DecGemmArgs{}; a.B = B; a.Bpad = Bp;
        a.src0 = d.hatt; a.k16_0 = A / 16; a.src1 = d.ctx; a.k16_1 = Dv / 16;
        a.Wp = c->proj.Wp; a.N = D; a.bias = c->proj.bias; a.epi = DE_LINEAR; a.out = d.d0;
        launch_dec_gemm(a, s, tm);
        // residual GRU 1 (decoder.py:30)
        a = DecGemmArgs{}; a.B = B; a.Bpad = Bp;
        a.src0 = d.d0; a.k16_0 = D / 16; a.src1 = d.h1; a.k16_1 = D / 16;
        a.Wp = c->g1_g.Wp; a.N = 2 * D; a.bias = c->g1_g.bias; a.epi = DE_GATES; a.out = d.rh; a.u = d.u; a.h = d.h1;
        launch_dec_gemm(a, s, tm);
        a.src1 = d.rh; a.Wp = c->g1_c.Wp; a.N = D; a.bias = c->g1_c.bias; a.epi = DE_CAND; a.out = nullptr;
        a.res = d.d0; a.res_out = d.o1;
        launch_dec_gemm(a, s, tm);
        // residual GRU 2 (decoder.py:31)
        a = DecGemmArgs{}; a.B = B; a.Bpad = Bp;
        a.src0 = d.o1; a.k16_0 = D / 16; a.src1 = d.h2; a.k16_1 = D / 16;
        a.Wp = c->g2_g.Wp; a.N = 2 * D; a.bias = c->g2_g.bias; a.epi = DE_GATES; a.out = d.rh; a.u = d.u; a.h = d.h2;
        launch_dec_gemm(a, s, tm);
        a.src1 = d.rh; a.Wp = c->g2_c.Wp; a.N = D; a.bias = c->g2_c.bias; a.epi = DE_CAND; a.out = nullptr;
        a.res = d.o1; a.res_out = d.o2;
        launch_dec_gemm(a, s, tm);
        // r output frames (decoder.py:35) + TestingHelper stop test (helpers.py:75)
        a = DecGemmArgs{}; a.B = B; a.Bpad = Bp;
        a.src0 = d.o2; a.k16_0 = D / 16; a.Wp = c->outp.Wp; a.N = NR; a.bias = c->outp.bias; a.epi = DE_OUT;
        a.out = d.outQ + (size_t)st * NR * Bp; a.nz = d.nz + (size_t)st * Bp;
        launch_dec_gemm(a, s, tm);
    }
}

// Persistent decode kernels need all their workgroups resident at once (one per CU). Launches from several
// streams / handles of this process are therefore admitted against the device's CU count: a launch that would
// not fit waits (on the device, via an event) for the oldest launches still in flight.
namespace {
struct PersistSlot { hipEvent_t ev; int wgs; };
std::mutex g_persist_mu;
std::map<int, std::vector<PersistSlot>> g_persist_active;   // per device, launch order
std::map<int, int> g_persist_budget;                         // per device; absent / 0 = the CU count

int persist_admit(int device, int wgs, hipStream_t s) {
    std::lock_guard<std::mutex> lk(g_persist_mu);
    int cus = 0;
    if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || cus <= 0) cus = 256;
    if (wgs > cus) return -1;
    // taco_set_persist_budget: fewer CUs than the device has for co-resident persistent decodes, the rest stay free for
    // the GEMM / scan / vocoder kernels of the other batches in flight (a single larger decode is admitted alone)
    {
        auto it = g_persist_budget.find(device);
        const int cap = it != g_persist_budget.end() ? it->second : 0;
        if (cap > 0) cus = std::max(wgs, std::min(cus, cap));
    }
    auto& v = g_persist_active[device];
    for (size_t i = 0; i < v.size();) {
        if (hipEventQuery(v[i].ev) == hipSuccess) { (void)hipEventDestroy(v[i].ev); v.erase(v.begin() + i); }
        else ++i;
    }
    int inflight = 0;
    for (auto& p : v) inflight += p.wgs;
    for (size_t i = 0; i < v.size() && inflight + wgs > cus; ++i) {
        (void)hipStreamWaitEvent(s, v[i].ev, 0);
        inflight -= v[i].wgs;
    }
    return 0;
}
void persist_launched(int device, int wgs, hipStream_t s) {
    std::lock_guard<std::mutex> lk(g_persist_mu);
    PersistSlot p;
    if (hipEventCreateWithFlags(&p.ev, hipEventDisableTiming) != hipSuccess) return;
    (void)hipEventRecord(p.ev, s);
    p.wgs = wgs;
    g_persist_active[device].push_back(p);
}
}  // namespace

// Text for a set of status words (PD_SYNC_*) whose abort flag is set.
static int persist_fail(const unsigned* w, int wgs) {
    if (w[PD_SYNC_ABORT] == 2u)
        return fail("persistent decoder: the launch returned at once because an earlier persistent decode of this handle "
                    "had timed out; its outputs are invalid (taco_set_decode_graph(h, 2) re-arms the handle)");
    return fail("persistent decoder: a bounded inter-workgroup wait timed out; outputs are invalid "
                "(first: workgroup %u waiting for step %u stage %u; %u of %d workgroups had started%s)",
                w[PD_SYNC_WG], (w[PD_SYNC_TAG] - 1) / 13, (w[PD_SYNC_TAG] - 1) % 13, w[PD_SYNC_ARRIVED], wgs,
                (int)w[PD_SYNC_ARRIVED] < wgs ? ": the device could not hold all of them at once" : "");
}

// Looks at the pinned mirror of the previous persistent launch's status words if that launch has completed (no
// synchronisation). Returns -1 (message set) when it aborted: its outputs were invalid, and the handle leaves
// persistent mode.
static int persist_check_previous(taco_ctx* c) {
    if (!c->status_pending || hipEventQuery(c->status_ev) != hipSuccess) return 0;
    c->status_pending = false;
    if (c->host_status[PD_SYNC_ABORT] == 0u) return 0;
    c->persist_broken = true;
    return persist_fail(c->host_status, c->last_persist_wgs);
}

static int decode_impl(taco_ctx* c, const float* enc_out, int B, int T_in, int S, const float* keep, float* mel,
                       float* align, int32_t* steps_run, Carver& ws, hipStream_t s, const float* teacher = nullptr) {
    const TacoHParams& hp = c->hp;
    Timing* tm = c->timing_on ? &c->timing : nullptr;
    const int Bp = bpad16(B);
    const int NR = hp.num_mels * hp.outputs_per_step;
    const int Dv = 2 * hp.encoder_gru_cells;
    const int A = hp.attention_depth, D = hp.decoder_depth;
    if (T_in > 8192) return fail("taco_decode: T_in > 8192 not supported by the attention kernel");
    const int mx = std::max(A, D);
    DecBufs d;
    d.keys = ws.take<float>((size_t)B * T_in * A);
    d.alignS = ws.take<float>((size_t)S * B * T_in);
    d.nz = ws.take<int32_t>((size_t)S * Bp);
    unsigned long long* sync = c->sync_words;   // handle-owned (not workspace): survives later stages for taco_decode_status
    c->last_sync_groups = 0;
    // one contiguous region for everything the decoder-step kernels exchange (Q layout)
    const size_t state_floats = (size_t)(hp.num_mels + Dv + A + 2 * D) * Bp;
    const size_t e_floats = ((size_t)B * T_in + 63) & ~(size_t)63;
    const size_t region_floats = state_floats + (size_t)(hp.prenet_depth1 + hp.prenet_depth2 + 6 * mx) * Bp + e_floats +
                                 (size_t)S * NR * Bp;
    float* region = ws.take<float>(region_floats);
    if (!ws.ok()) return fail("taco_decode: workspace too small");
    float* p = region;
    d.go = p; p += (size_t)hp.num_mels * Bp;
    d.ctx = p; p += (size_t)Dv * Bp;
    d.hatt = p; p += (size_t)A * Bp;
    d.h1 = p; p += (size_t)D * Bp;
    d.h2 = p; p += (size_t)D * Bp;
    d.state_bytes = state_floats * 4;
    d.p1 = p; p += (size_t)hp.prenet_depth1 * Bp;
    d.p2 = p; p += (size_t)hp.prenet_depth2 * Bp;
    d.rh = p; p += (size_t)mx * Bp;
    d.u = p; p += (size_t)mx * Bp;
    d.q = p; p += (size_t)mx * Bp;
    d.d0 = p; p += (size_t)mx * Bp;
    d.o1 = p; p += (size_t)mx * Bp;
    d.o2 = p; p += (size_t)mx * Bp;
    p += e_floats;   // (spare)
    d.outQ = p;

    auto keys_gemm = [&](Timing* t) {
        // keys = memory_layer(enc_out), once per utterance (BahdanauAttention ctor, decoder.py:20)
        GemmArgs g{enc_out, Dv, B * T_in, T_in, c->mem_layer.Cin, 1, 0, c->mem_layer.W, c->mem_layer.ldw,
                   c->mem_layer.N, nullptr, nullptr, nullptr, nullptr, 0, d.keys, A, ACT_NONE, 0};
        launch_conv_gemm(g, s, t);
        (void)hipMemsetAsync(d.go, 0, d.state_bytes, s);   // zero_state + <GO> frame (decoder.py:36, helpers.py:80-85)
    };
    const bool fine_timing = c->timing_on && (c->timing.kind == KK_DEC_GEMM || c->timing.kind == KK_DEC_ATTN);

    // ---- mode 2: the whole loop as one persistent launch (default layer sizes, inference: no dropout replay)
    const bool default_sizes = hp.prenet_depth1 == 256 && hp.prenet_depth2 == 128 && A == 256 && D == 256 &&
                               hp.num_mels == 80 && hp.outputs_per_step == 5 && Dv == 256;
    const size_t g1 = (size_t)Bp * 2;                        // floats per unit of vector dimension, granule layout
    const size_t pe_floats = (((size_t)B * T_in * 2) + 63) & ~(size_t)63;
    // granule buffers of dec_persistent.hip: [h_att;ctx] x2, h1 x2, h2 x2, p1, p2, rh x3, u x3, q, d0, o1, o2
    const size_t pregion_floats = (size_t)PD_REGION_DIMS * g1 + pe_floats + (size_t)S * 400 * g1;
    // a caller that is capturing `s` into a graph of its own gets no host-side status plumbing (event queries and
    // the device-to-host copy stay out of its graph); taco_decode_status still works after a synchronisation
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    const bool capturing = s != nullptr && hipStreamIsCapturing(s, &cap) == hipSuccess && cap != hipStreamCaptureStatusNone;
    if (!capturing && persist_check_previous(c)) return -1;     // the PREVIOUS decode's outputs were invalid
    int dev_cus = 0;
    if (hipDeviceGetAttribute(&dev_cus, hipDeviceAttributeMultiprocessorCount, c->device) != hipSuccess || dev_cus <= 0)
        dev_cus = 256;
    // (a launch that cannot be resident as a whole - more workgroups than CUs - takes the per-stage path instead)
    if (c->decode_mode == 2 && !c->persist_broken && default_sizes && !keep && !teacher && !fine_timing && Bp / 16 <= 8 &&
        32 * (Bp / 16) <= dev_cus && pregion_floats * 4 < (size_t)1 << 31) {
        float* pregion = ws.take<float>(pregion_floats + 1024);   // + 4 KB tail for diagnostic stamps (PD_STAMPS builds)
        if (!ws.ok()) return fail("taco_decode: workspace too small");
        GemmArgs g{enc_out, Dv, B * T_in, T_in, c->mem_layer.Cin, 1, 0, c->mem_layer.W, c->mem_layer.ldw,
                   c->mem_layer.N, nullptr, nullptr, nullptr, nullptr, 0, d.keys, A, ACT_NONE, 0};
        launch_conv_gemm(g, s, tm);
        // every exchanged buffer starts as {0, tag 0}: zero_state, <GO> frame, and no stale tags of an earlier call
        (void)hipMemsetAsync(pregion, 0, (pregion_floats + 1024) * 4, s);
        c->dbg_stamps = reinterpret_cast<unsigned long long*>(pregion + pregion_floats);
        (void)hipMemsetAsync(sync, 0, 128, s);
        DecPersistArgs a{};
        const DecW* W[11] = {&c->pre1_f, &c->pre2, &c->att_g_p, &c->att_c, &c->query, &c->proj,
                             &c->g1_g_f, &c->g1_c_f, &c->g2_g_p, &c->g2_c, &c->outp};
        for (int i = 0; i < 11; ++i) { a.Wp[i] = W[i]->Wp; a.bias[i] = W[i]->bias; }
        a.bias_pre1_go = c->pre1.bias;
        a.attn_v = c->attn_v; a.keys = d.keys; a.values = enc_out;
        a.region = pregion; a.region_bytes = (unsigned)(pregion_floats * 4);
        size_t o = 0;
        auto takeg = [&](int dim) { const unsigned r = (unsigned)o; o += (size_t)dim * g1; return r; };
        a.o_hc = takeg(1024); a.o_h1 = takeg(512); a.o_h2 = takeg(512);
        a.o_p1 = takeg(256); a.o_p2 = takeg(128); a.o_rh = takeg(768); a.o_u = takeg(768); a.o_q = takeg(256);
        a.o_d0 = takeg(256); a.o_o1 = takeg(256); a.o_o2 = takeg(256);
        if (o != (size_t)PD_REGION_DIMS * g1) return fail("taco_decode: persistent region layout mismatch");
        a.o_e = (unsigned)o; o += pe_floats;
        a.o_outQ = (unsigned)o;
        a.alignS = d.alignS; a.sync = sync; a.B = B; a.Bpad = Bp; a.T_in = T_in; a.S = S;
        a.dbg = c->dbg_stamps;
        const int wgs = 32 * (Bp / 16);
        if (persist_admit(c->device, wgs, s)) return fail("taco_decode: persistent decoder does not fit the device");
        if (launch_dec_persistent(a, s, tm)) return fail("taco_decode: cannot configure the persistent decoder");
        persist_launched(c->device, wgs, s);
        c->last_sync_groups = 1;
        c->last_persist_wgs = wgs;
        if (!capturing) {
            HIP_OK(hipMemcpyAsync(c->host_status, sync, 32, hipMemcpyDeviceToHost, s));
            HIP_OK(hipEventRecord(c->status_ev, s));
            c->status_pending = true;
        }
        launch_dec_finalize(pregion + a.o_outQ, 1, d.alignS, d.nz, S, NR, B, Bp, T_in, mel, align, steps_run, s, tm);
        return 0;
    }

    // ---- mode 3: the whole loop as one launch, one workgroup per 16-utterance tile (dec_tile.hip): the throughput form
    if (c->decode_mode == 3 && default_sizes && !keep && !teacher && !fine_timing && T_in <= 2048) {
        keys_gemm(tm);
        DecTileArgs a{};
        auto stage = [&](int i, const DecW& w, int src0, int k0, int src1, int k1, int N, int epi, int out, int hh,
                         int res, int res_out) {
            a.st[i] = DecTileStage{w.Wp, w.bias, src0, k0 / 16, src1, k1 / 16, N, epi, out, hh, res, res_out};
        };
        const int P1 = hp.prenet_depth1, P2 = hp.prenet_depth2;
        stage(0, c->pre1, DTB_GO, hp.num_mels, DTB_CTX, Dv, P1, DE_RELU, DTB_P1, -1, -1, -1);       // rnn_wrappers.py:25
        stage(1, c->pre2, DTB_P1, P1, -1, 0, P2, DE_RELU, DTB_P2, -1, -1, -1);
        stage(2, c->att_g, DTB_P2, P2, DTB_HATT, A, 2 * A, DE_GATES, DTB_RH, DTB_HATT, -1, -1);     // rnn_wrappers.py:26
        stage(3, c->att_c, DTB_P2, P2, DTB_RH, A, A, DE_CAND, -1, DTB_HATT, -1, -1);
        stage(4, c->query, DTB_HATT, A, -1, 0, A, DE_LINEAR, DTB_Q, -1, -1, -1);                    // decoder.py:20
        stage(5, c->proj, DTB_HATT, A, DTB_CTX, Dv, D, DE_LINEAR, DTB_D0, -1, -1, -1);              // decoder.py:29
        stage(6, c->g1_g, DTB_D0, D, DTB_H1, D, 2 * D, DE_GATES, DTB_RH, DTB_H1, -1, -1);           // decoder.py:30
        stage(7, c->g1_c, DTB_D0, D, DTB_RH, D, D, DE_CAND, -1, DTB_H1, DTB_D0, DTB_O1);
        stage(8, c->g2_g, DTB_O1, D, DTB_H2, D, 2 * D, DE_GATES, DTB_RH, DTB_H2, -1, -1);           // decoder.py:31
        stage(9, c->g2_c, DTB_O1, D, DTB_RH, D, D, DE_CAND, -1, DTB_H2, DTB_O1, DTB_O2);
        stage(10, c->outp, DTB_O2, D, -1, 0, NR, DE_OUT, -1, -1, -1, -1);                            // decoder.py:35
        float* bufs[DTB_COUNT] = {d.go, d.ctx, d.hatt, d.h1, d.h2, d.p1, d.p2, d.rh, d.u, d.q, d.d0, d.o1, d.o2};
        for (int i = 0; i < DTB_COUNT; ++i) a.buf[i] = bufs[i];
        if (region_floats * 4 >= ((size_t)1 << 31)) return fail("taco_decode: decoder region larger than 2 GiB");
        a.region = region; a.region_bytes = (unsigned)(region_floats * 4);
        a.outQ = d.outQ; a.keys = d.keys; a.values = enc_out; a.attn_v = c->attn_v; a.alignS = d.alignS;
        a.B = B; a.Bpad = Bp; a.T_in = T_in; a.S = S; a.NR = NR; a.M = hp.num_mels;
        if (launch_dec_tile(a, s, tm)) return fail("taco_decode: cannot configure the tile decoder");
        launch_dec_finalize(d.outQ, 0, d.alignS, d.nz, S, NR, B, Bp, T_in, mel, align, steps_run, s, tm);
        return 0;
    }

    // ---- modes 0/1: one kernel per stage; eager, or captured once per shape/buffer set and replayed
    float* teachQ = nullptr;
    if (teacher) {
        teachQ = ws.take<float>((size_t)S * hp.num_mels * Bp);
        if (!ws.ok()) return fail("taco_decode: workspace too small");
    }
    auto enqueue = [&](Timing* t) {
        keys_gemm(t);
        if (teacher) launch_dec_pack_teacher(teacher, teachQ, S, hp.outputs_per_step, hp.num_mels, B, Bp, s);
        decode_steps(c, d, enc_out, keep, B, T_in, S, s, t, teachQ);
        // teacher-forced: TrainingHelper runs all its steps, there is no stop test (helpers.py:41)
        launch_dec_finalize(d.outQ, 0, d.alignS, d.nz, S, NR, B, Bp, T_in, mel, align, steps_run, s, t, !teacher);
    };
    if (c->decode_mode == 0 || teacher || s == nullptr || (c->timing_on && c->timing.kind != KK_DEC_GRAPH)) {
        enqueue(tm);
        return 0;
    }
    std::vector<uintptr_t> key = {(uintptr_t)B, (uintptr_t)T_in, (uintptr_t)S, (uintptr_t)enc_out, (uintptr_t)keep,
                                  (uintptr_t)mel, (uintptr_t)align, (uintptr_t)steps_run, (uintptr_t)ws.base};
    GraphEntry* ge = nullptr;
    for (auto& g : c->graphs)
        if (g.key == key) ge = &g;
    if (!ge) {
        if (c->graphs.size() >= 8) {
            (void)hipGraphExecDestroy(c->graphs.front().exec);
            (void)hipGraphDestroy(c->graphs.front().graph);
            c->graphs.erase(c->graphs.begin());
        }
        GraphEntry e;
        e.key = key;
        HIP_OK(hipStreamBeginCapture(s, hipStreamCaptureModeThreadLocal));
        enqueue(nullptr);
        hipError_t ce = hipStreamEndCapture(s, &e.graph);
        if (ce != hipSuccess || !e.graph) return fail("taco_decode: stream capture failed: %s", hipGetErrorString(ce));
        HIP_OK(hipGraphInstantiate(&e.exec, e.graph, nullptr, nullptr, 0));
        c->graphs.push_back(e);
        ge = &c->graphs.back();
    }
    if (tm) tm->begin(KK_DEC_GRAPH, s);
    HIP_OK(hipGraphLaunch(ge->exec, s));
    if (tm) tm->end(KK_DEC_GRAPH, s);
    return 0;
}

extern "C" int taco_decode(taco_handle h, const float* enc_out, int32_t B, int32_t T_in, int32_t max_iters,
                           const float* dropout_keep, float* mel, float* align, int32_t* steps_run, void* ws,
                           size_t ws_bytes, taco_stream_t stream) {
    if (!h || !enc_out || !mel || !align || !steps_run || !ws) return fail("taco_decode: null argument");
    if (check_dims(B, T_in) || check_dims(B, max_iters)) return -1;
    HIP_OK(hipSetDevice(h->device));
    Carver cv(ws, ws_bytes);
    if (decode_impl(h, enc_out, B, T_in, max_iters, dropout_keep, mel, align, steps_run, cv, (hipStream_t)stream))
        return -1;
    return check_launch("taco_decode");
}

extern "C" int taco_decode_teacher(taco_handle h, const float* enc_out, int32_t B, int32_t T_in, int32_t n_steps,
                                   const float* targets, const float* dropout_keep, float* mel, float* align,
                                   int32_t* steps_run, void* ws, size_t ws_bytes, taco_stream_t stream) {
    if (!h || !enc_out || !targets || !mel || !align || !steps_run || !ws)
        return fail("taco_decode_teacher: null argument");
    if (check_dims(B, T_in) || check_dims(B, n_steps)) return -1;
    HIP_OK(hipSetDevice(h->device));
    Carver cv(ws, ws_bytes);
    if (decode_impl(h, enc_out, B, T_in, n_steps, dropout_keep, mel, align, steps_run, cv, (hipStream_t)stream, targets))
        return -1;
    return check_launch("taco_decode_teacher");
}

// ---------------------------------------------------------------------------------------
static int postnet_impl(taco_ctx* c, const float* mel, int B, int T, float* linear, Carver& ws, hipStream_t s) {
    Timing* tm = c->timing_on ? &c->timing : nullptr;
    const int M = B * T;
    float* rnn = ws.take<float>((size_t)M * 2 * c->post.gru);
    if (!ws.ok()) return fail("taco_postnet: workspace too small");
    if (run_cbhg(c, c->post, mel, nullptr, B, T, rnn, ws, s)) return -1;
    const ConvW& w = c->lin_dense;   // decoder.py:57
    GemmArgs g{rnn, 2 * c->post.gru, M, T, w.Cin, 1, 0, w.W, w.ldw, w.N, w.bias, nullptr, nullptr, nullptr, 0,
               linear, w.N, ACT_NONE, 0};
    launch_conv_gemm(g, s, tm);
    return 0;
}

extern "C" int taco_postnet(taco_handle h, const float* mel, int32_t B, int32_t T, float* linear, void* ws,
                            size_t ws_bytes, taco_stream_t stream) {
    if (!h || !mel || !linear || !ws) return fail("taco_postnet: null argument");
    if (check_dims(B, T)) return -1;
    HIP_OK(hipSetDevice(h->device));
    Carver cv(ws, ws_bytes);
    if (postnet_impl(h, mel, B, T, linear, cv, (hipStream_t)stream)) return -1;
    return check_launch("taco_postnet");
}

// ---------------------------------------------------------------------------------------
static int gl_impl(taco_ctx* c, const float* linear, int B, int T, int iters, float* wav, Carver& ws, hipStream_t s) {
    Timing* tm = c->timing_on ? &c->timing : nullptr;
    const TacoHParams& hp = c->hp;
    const size_t M = (size_t)B * T;
    float* mag = ws.take<float>(M * hp.num_freq);
    float* fa = ws.take<float>(M * hp.win_length);
    float* fb = ws.take<float>(M * hp.win_length);
    if (!ws.ok()) return fail("taco_griffin_lim: workspace too small");
    GLPlan p{hp.n_fft, hp.hop_length, hp.win_length, hp.num_freq, c->twiddle, c->window, c->gl_image};
    gl_read_switches(p);                                    // (experiment switches: once per call, not per launch)
    p.prepared = true;                                      // taco_create set the kernels' attributes on this device
    launch_gl_mag(linear, mag, M * hp.num_freq, hp.min_level_db, hp.ref_level_db, hp.power, s, tm);
    int chain_rc = 0;
    auto chain = [&](int b0, int nb, hipStream_t st, Timing* t) {
        const size_t r0 = (size_t)b0 * T;
        float* a0 = fa + r0 * hp.win_length;
        float* a1 = fb + r0 * hp.win_length;
        const float* mg = mag + r0 * hp.num_freq;
        int state = 0;                                      // what `cur` holds: frames, or run records (kernels.h)
        chain_rc |= launch_gl_iter(p, a0, mg, a0, nb, T, 1, st, t, false, nullptr, &state);   // y0 = istft(mag, zero phase) (audio.py:191)
        float* cur = a0;
        float* nxt = a1;
        for (int i = 0; i < iters; ++i) {                   // audio.py:192-195
            chain_rc |= launch_gl_iter(p, cur, mg, nxt, nb, T, 0, st, t, false, nullptr, &state);
            std::swap(cur, nxt);
        }
        launch_gl_ola(p, cur, wav + (size_t)b0 * ((size_t)(T - 1) * hp.hop_length + hp.win_length), nb, T, st, t,
                      state);
    };
    // An iteration of the whole batch is one launch that has to drain before the next may start: with workgroups that
    // live for ~25 us and only four rounds of them per launch, the chip idles for a good part of every launch's last
    // round. Utterances do not depend on each other, so a large batch runs as G groups of utterances, each a chain of
    // its own on a stream of its own: the tail of one group's launch is filled by the other groups' launches.
    // (Not when the caller captures `s` or when launches are being timed on `s`.)
    // (taco_set_gl_split: worth it for a batch that has the GPU to itself, 6.2 -> 5.7 ms at B = 32; with several
    // batches in flight the tails fill with the other batches' work anyway and the extra streams cost more: default 1)
    static const int split_env = getenv("TACO_GL_SPLIT") ? atoi(getenv("TACO_GL_SPLIT")) : 0;
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    const bool capturing = s != nullptr && hipStreamIsCapturing(s, &cap) == hipSuccess && cap != hipStreamCaptureStatusNone;
    int G = std::min(std::min(split_env > 0 ? split_env : c->gl_split, 4), B / 8);
    if (capturing || tm || s == nullptr) G = 1;
    if (G > 1) {
        for (int g = 0; g < G - 1 && G > 1; ++g) {
            if (!c->gl_streams[g] && (hipStreamCreateWithFlags(&c->gl_streams[g], hipStreamNonBlocking) != hipSuccess ||
                                      hipEventCreateWithFlags(&c->gl_join[g], hipEventDisableTiming) != hipSuccess))
                G = 1;
        }
        if (!c->gl_fork && hipEventCreateWithFlags(&c->gl_fork, hipEventDisableTiming) != hipSuccess) G = 1;
    }
    const char* kStateErr = "taco_griffin_lim: internal error: run records handed to a kernel that reads frames";
    if (G <= 1) {
        chain(0, B, s, tm);
        return chain_rc ? fail("%s", kStateErr) : 0;
    }
    HIP_OK(hipEventRecord(c->gl_fork, s));
    for (int g = 1; g < G; ++g) {
        hipStream_t st = c->gl_streams[g - 1];
        HIP_OK(hipStreamWaitEvent(st, c->gl_fork, 0));
        chain((int)((long)B * g / G), (int)((long)B * (g + 1) / G - (long)B * g / G), st, nullptr);
        HIP_OK(hipEventRecord(c->gl_join[g - 1], st));
    }
    chain(0, (int)((long)B / G), s, nullptr);
    for (int g = 1; g < G; ++g) HIP_OK(hipStreamWaitEvent(s, c->gl_join[g - 1], 0));
    return chain_rc ? fail("%s", kStateErr) : 0;
}

// numpy/librosa flavour (audio.py:44-55,167-181) up to, not including, pre_emphasis_inv
static int gl_librosa_impl(taco_ctx* c, const float* linear, const float* phase_u, int B, int T, int iters, float* wav,
                           Carver& ws, hipStream_t s) {
    Timing* tm = c->timing_on ? &c->timing : nullptr;
    const TacoHParams& hp = c->hp;
    const size_t M = (size_t)B * T;
    float* mag = ws.take<float>(M * hp.num_freq);
    float* fa = ws.take<float>(M * hp.win_length);
    float* fb = ws.take<float>(M * hp.win_length);
    if (!ws.ok()) return fail("taco_griffin_lim_librosa: workspace too small");
    GLPlan p{hp.n_fft, hp.hop_length, hp.win_length, hp.num_freq, c->twiddle, c->window, c->gl_image};
    launch_gl_mag(linear, mag, M * hp.num_freq, hp.min_level_db, hp.ref_level_db, hp.power, s, tm);
    p.prepared = true;
    int rc = launch_gl_iter(p, fa, mag, fa, B, T, 1, s, tm, true, phase_u);   // y = istft(S * angles) (audio.py:175-177)
    float* cur = fa;
    float* nxt = fb;
    for (int i = 0; i < iters; ++i) {                                // audio.py:178-180
        rc |= launch_gl_iter(p, cur, mag, nxt, B, T, 0, s, tm, true, nullptr);
        std::swap(cur, nxt);
    }
    launch_gl_ola_norm(p, cur, wav, B, T, s, tm);
    return rc ? fail("taco_griffin_lim_librosa: internal error: bad vocoder state") : 0;
}

extern "C" int taco_griffin_lim_librosa(taco_handle h, const float* linear, const float* phase_u, int32_t B, int32_t T,
                                        int32_t iters, float* wav, void* ws, size_t ws_bytes, taco_stream_t stream) {
    if (!h || !linear || !wav || !ws) return fail("taco_griffin_lim_librosa: null argument");
    if (check_dims(B, T)) return -1;
    if (iters < 0) return fail("taco_griffin_lim_librosa: iters < 0");
    if ((long)h->hp.hop_length * (T - 1) <= h->hp.n_fft / 2)
        return fail("taco_griffin_lim_librosa: need hop*(T-1) > n_fft/2 samples (reflect padding of the centred STFT), "
                    "got T = %d", T);
    HIP_OK(hipSetDevice(h->device));
    Carver cv(ws, ws_bytes);
    if (gl_librosa_impl(h, linear, phase_u, B, T, iters, wav, cv, (hipStream_t)stream)) return -1;
    return check_launch("taco_griffin_lim_librosa");
}

// ---------------------------------------------------------------------------------------
extern "C" size_t taco_spectrogram_workspace_bytes(taco_handle h, int32_t B, int32_t n_samples) {
    if (!h || B < 1 || n_samples < 1) return 0;
    const size_t T = 1 + (size_t)n_samples / h->hp.hop_length;
    return al((size_t)B * T * ((h->hp.num_freq + 15) / 16 * 16) * 4) + 4096;
}

extern "C" int taco_spectrogram(taco_handle h, const float* wav, int32_t B, int32_t n_samples, float preemphasis,
                                float* linear, float* mel, void* ws, size_t ws_bytes, taco_stream_t stream) {
    if (!h || !wav || !ws || (!linear && !mel)) return fail("taco_spectrogram: null argument");
    const TacoHParams& hp = h->hp;
    if (B < 1 || n_samples <= hp.n_fft / 2)
        return fail("taco_spectrogram: need more than n_fft/2 = %d samples (reflect padding), got %d", hp.n_fft / 2,
                    n_samples);
    if (mel && !h->mel_proj.W) return fail("taco_spectrogram: no 'audio/mel_basis' was given to taco_create");
    const long T = 1 + n_samples / hp.hop_length;
    if (check_dims(B, (int)T)) return -1;
    HIP_OK(hipSetDevice(h->device));
    hipStream_t s = (hipStream_t)stream;
    Timing* tm = h->timing_on ? &h->timing : nullptr;
    Carver cv(ws, ws_bytes);
    const int ldm = (hp.num_freq + 15) / 16 * 16;
    const size_t M = (size_t)B * T;
    float* mag = cv.take<float>(M * ldm);
    if (!cv.ok()) return fail("taco_spectrogram: workspace too small");
    if (ldm != hp.num_freq) HIP_OK(hipMemsetAsync(mag, 0, M * ldm * sizeof(float), s));   // zero K padding
    GLPlan p{hp.n_fft, hp.hop_length, hp.win_length, hp.num_freq, h->twiddle, h->window, h->gl_image};
    launch_stft_center(p, wav, B, n_samples, (int)T, preemphasis, hp.ref_level_db, hp.min_level_db, mag, ldm, linear, s, tm);
    if (mel) {
        const ConvW& w = h->mel_proj;   // _linspect_to_melspect + _amp_to_db - ref + _normalize (audio.py:78-79)
        GemmArgs g{mag, ldm, (int)M, (int)T, w.Cin, 1, 0, w.W, w.ldw, w.N, nullptr, nullptr, nullptr, nullptr, 0,
                   mel, w.N, ACT_DB_NORM, 0, nullptr, 0, nullptr, 0, hp.ref_level_db, hp.min_level_db};
        launch_conv_gemm(g, s, tm);
    }
    return check_launch("taco_spectrogram");
}

extern "C" int taco_griffin_lim(taco_handle h, const float* linear, int32_t B, int32_t T, int32_t iters, float* wav,
                                void* ws, size_t ws_bytes, taco_stream_t stream) {
    if (!h || !linear || !wav || !ws) return fail("taco_griffin_lim: null argument");
    if (check_dims(B, T)) return -1;
    if (iters < 0) return fail("taco_griffin_lim: iters < 0");
    HIP_OK(hipSetDevice(h->device));
    Carver cv(ws, ws_bytes);
    if (gl_impl(h, linear, B, T, iters, wav, cv, (hipStream_t)stream)) return -1;
    return check_launch("taco_griffin_lim");
}

extern "C" int taco_griffin_lim_noalloc(taco_handle h, const float* linear, int32_t B, int32_t T, int32_t iters,
                                        float* wav, taco_stream_t stream) {
    if (!h || !linear || !wav) return fail("taco_griffin_lim_noalloc: null argument");
    if (check_dims(B, T)) return -1;
    if (iters < 0) return fail("taco_griffin_lim_noalloc: iters < 0");
    if ((long)B * T > NOALLOC_MAX_FRAMES)
        return fail("taco_griffin_lim_noalloc: B*T = %ld frames, the static scratch holds at most %d "
                    "(use taco_griffin_lim with a workspace for larger batches)", (long)B * T, NOALLOC_MAX_FRAMES);
    HIP_OK(hipSetDevice(h->device));
    void* base = h->device >= 0 && h->device < 64 ? g_scratch_ptr[h->device] : nullptr;
    if (!base) return fail("taco_griffin_lim_noalloc: no static scratch bound for device %d", h->device);
    const TacoHParams& hp = h->hp;
    hipStream_t s = (hipStream_t)stream;
    // same carve as gl_impl, out of the device's copy of `scratch`; every byte a kernel reads was written earlier in
    // this call (gl_mag fills mag, the first synthesis fills the first frame buffer), so nothing needs clearing
    Carver cv(base, NOALLOC_SCRATCH_BYTES);
    const size_t M = (size_t)B * T;
    float* mag = cv.take<float>(M * hp.num_freq);
    float* fa = cv.take<float>(M * hp.win_length);
    float* fb = cv.take<float>(M * hp.win_length);
    if (!cv.ok()) return fail("taco_griffin_lim_noalloc: static scratch too small for these hparams");
    GLPlan p{hp.n_fft, hp.hop_length, hp.win_length, hp.num_freq, h->twiddle, h->window, h->gl_image};
    gl_read_switches(p);
    p.prepared = true;             // (taco_create set the kernels' attributes on this device: no set-up call from here)
    launch_gl_mag(linear, mag, M * hp.num_freq, hp.min_level_db, hp.ref_level_db, hp.power, s, nullptr);
    int state = 0;
    int rc = launch_gl_iter(p, fa, mag, fa, B, T, 1, s, nullptr, false, nullptr, &state);
    float* cur = fa;
    float* nxt = fb;
    for (int i = 0; i < iters; ++i) {
        rc |= launch_gl_iter(p, cur, mag, nxt, B, T, 0, s, nullptr, false, nullptr, &state);
        std::swap(cur, nxt);
    }
    launch_gl_ola(p, cur, wav, B, T, s, nullptr, state);
    if (rc) return fail("taco_griffin_lim_noalloc: internal error: run records handed to a kernel that reads frames");
    return check_launch("taco_griffin_lim_noalloc");
}

// ---------------------------------------------------------------------------------------
extern "C" int taco_synthesize(taco_handle h, const int32_t* ids, const int32_t* lens, int32_t B, int32_t T_in,
                               int32_t max_iters, int32_t gl_iters, float* enc_out, float* mel, float* linear,
                               float* align, float* wav, int32_t* steps_run, void* ws, size_t ws_bytes,
                               taco_stream_t stream) {
    if (!h || !ids || !lens || !mel || !linear || !align || !steps_run || !ws)
        return fail("taco_synthesize: null argument");
    if (check_dims(B, T_in) || check_dims(B, max_iters)) return -1;
    HIP_OK(hipSetDevice(h->device));
    hipStream_t s = (hipStream_t)stream;
    Carver cv(ws, ws_bytes);
    if (!enc_out) enc_out = cv.take<float>((size_t)B * T_in * 2 * h->hp.encoder_gru_cells);
    const size_t base = cv.off;
    if (encode_impl(h, ids, lens, B, T_in, enc_out, cv, s)) return -1;
    cv.off = base;
    if (decode_impl(h, enc_out, B, T_in, max_iters, nullptr, mel, align, steps_run, cv, s)) return -1;
    // The post-net runs on all max_iters*r frames: the stop test of helpers.py:75 is an exact
    // all-zero comparison that does not fire in practice; callers that see steps_run < max_iters
    // re-run taco_postnet on the shorter mel (the Python host does).
    const int T = max_iters * h->hp.outputs_per_step;
    cv.off = base;
    if (postnet_impl(h, mel, B, T, linear, cv, s)) return -1;
    if (wav) {
        cv.off = base;
        if (gl_impl(h, linear, B, T, gl_iters, wav, cv, s)) return -1;
    }
    return check_launch("taco_synthesize");
}

// ---------------------------------------------------------------------------------------
extern "C" int taco_timing_begin(taco_handle h, int32_t kind) {
    if (!h || kind < 0 || kind >= KK_COUNT) return fail("taco_timing_begin: bad argument");
    h->timing.kind = kind;
    h->timing.used = 0;
    h->timing_on = true;
    return 0;
}

extern "C" int taco_timing_end(taco_handle h, int32_t* launches, double* total_ms) {
    if (!h || !launches || !total_ms) return fail("taco_timing_end: null argument");
    HIP_OK(hipSetDevice(h->device));
    HIP_OK(hipDeviceSynchronize());
    double tot = 0;
    for (size_t i = 0; i + 1 < h->timing.used; i += 2) {
        float ms = 0;
        HIP_OK(hipEventElapsedTime(&ms, h->timing.ev[i], h->timing.ev[i + 1]));
        tot += ms;
    }
    *launches = (int32_t)(h->timing.used / 2);
    *total_ms = tot;
    h->timing_on = false;
    h->timing.kind = -1;
    h->timing.used = 0;
    return 0;
}

extern "C" const char* taco_kernel_name(int32_t kind) { return kind >= 0 && kind < KK_COUNT ? kKernelNames[kind] : ""; }
extern "C" int32_t taco_num_kernel_kinds(void) { return KK_COUNT; }

extern "C" int taco_set_persist_budget(int32_t device, int32_t workgroups) {
    if (device < 0 || workgroups < 0) return fail("taco_set_persist_budget: negative argument");
    std::lock_guard<std::mutex> lk(g_persist_mu);
    g_persist_budget[device] = workgroups;
    return 0;
}

extern "C" int taco_set_gl_split(taco_handle h, int32_t groups) {
    if (!h) return fail("taco_set_gl_split: null handle");
    if (groups < 1 || groups > 4) return fail("taco_set_gl_split: groups must be 1..4");
    h->gl_split = groups;
    return 0;
}

extern "C" int taco_set_bigru_mode(taco_handle h, int32_t mode) {
    if (!h) return fail("taco_set_bigru_mode: null handle");
    if (mode < 0 || mode > 2) return fail("taco_set_bigru_mode: mode must be 0 (one utterance a workgroup), 1 (sixteen) or 2 (four)");
    h->bigru_mode = mode;
    return 0;
}

extern "C" int32_t taco_get_persist_budget(int32_t device) {
    std::lock_guard<std::mutex> lk(g_persist_mu);
    auto it = g_persist_budget.find(device);
    return it != g_persist_budget.end() ? it->second : 0;
}

extern "C" int taco_set_decode_graph(taco_handle h, int32_t mode) {
    if (!h) return fail("taco_set_decode_graph: null handle");
    if (mode < 0 || mode > 3) return fail("taco_set_decode_graph: mode must be 0, 1, 2 or 3");
    if (mode == 2 && h->persist_broken) {
        // explicit re-arm after a timed-out persistent decode: wait for the handle's work, clear the sticky word
        HIP_OK(hipSetDevice(h->device));
        HIP_OK(hipDeviceSynchronize());
        HIP_OK(hipMemset(reinterpret_cast<unsigned*>(h->sync_words) + PD_SYNC_STICKY, 0, 16));
        h->persist_broken = false;
        h->status_pending = false;
    }
    h->decode_mode = mode;
    return 0;
}

extern "C" int taco_decode_status(taco_handle h) {
    if (!h) return fail("taco_decode_status: null handle");
    if (!h->last_sync_groups) return 0;
    HIP_OK(hipSetDevice(h->device));
    unsigned info[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    HIP_OK(hipMemcpy(info, h->sync_words, 32, hipMemcpyDeviceToHost));
    h->status_pending = false;                 // (this read supersedes the asynchronous mirror)
#ifdef PD_PHASE_STAMPS
    {
        unsigned long long st[3];
        HIP_OK(hipMemcpy(st, reinterpret_cast<unsigned long long*>(h->sync_words) + 8, sizeof(st), hipMemcpyDeviceToHost));
        fprintf(stderr, "[pd phases] entry->step0 %.1f us, steps 1.. %.1f us\n", (st[1] - st[0]) * 0.01, (st[2] - st[1]) * 0.01);
    }
#endif
#ifdef PD_STAMPS
    if (h->dbg_stamps) {
        unsigned long long st[256];
        HIP_OK(hipMemcpy(st, h->dbg_stamps, sizeof(st), hipMemcpyDeviceToHost));
        // flags: | stage boundary, r = a poll round of wave 0 done, m = MFMAs issued, e = reduced tile ready
        fprintf(stderr, "[pd stamps, 10 ns ticks since step start]");
        const char* fl = "|rme";
        for (int i = 1; i < 256 && st[i]; ++i)
            fprintf(stderr, " %c%llu", fl[(st[i] >> 60) & 3], (st[i] & ~(15ull << 60)) - (st[0] & ~(15ull << 60)));
        fprintf(stderr, "\n");
    }
#endif
    if (info[PD_SYNC_ABORT] != 0u) {
        h->persist_broken = true;
        return persist_fail(info, h->last_persist_wgs);
    }
    return 0;
}

extern "C" int taco_debug_poison_decoder(taco_handle h) {
    if (!h) return fail("taco_debug_poison_decoder: null handle");
    HIP_OK(hipSetDevice(h->device));
    const unsigned one = 1u;
    HIP_OK(hipMemcpy(reinterpret_cast<unsigned*>(h->sync_words) + PD_SYNC_STICKY, &one, 4, hipMemcpyHostToDevice));
    return 0;
}

extern "C" int taco_debug_handoff_probe(int32_t device, int32_t rounds, double* us_per_handoff) {
    if (!us_per_handoff || rounds < 1 || rounds > (1 << 20)) return fail("taco_debug_handoff_probe: bad argument");
    HIP_OK(hipSetDevice(device));
    int cus = 0;
    HIP_OK(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device));
    if (cus < 32) return fail("taco_debug_handoff_probe: needs 32 CUs for its 32 co-resident workgroups, device has %d", cus);
    const size_t region_bytes = 2u * 32u * 256u * 4u, total = region_bytes + 256 + 128;
    char* buf = nullptr;
    HIP_OK(hipMalloc(reinterpret_cast<void**>(&buf), total));
    hipEvent_t e0 = nullptr, e1 = nullptr;
    int rc = 0;
    float ms = 0.f;
    unsigned abort_h[4] = {0, 0, 0, 0};
    auto body = [&]() -> int {
        HIP_OK(hipEventCreate(&e0));
        HIP_OK(hipEventCreate(&e1));
        for (int pass = 0; pass < 2; ++pass) {              // (first pass: code object load, clocks)
            HIP_OK(hipMemsetAsync(buf, 0, total, nullptr));
            HIP_OK(hipEventRecord(e0, nullptr));
            launch_handoff_probe(reinterpret_cast<float*>(buf), (unsigned)region_bytes, rounds,
                                 reinterpret_cast<unsigned*>(buf + region_bytes), reinterpret_cast<float*>(buf + region_bytes + 256),
                                 nullptr);
            HIP_OK(hipEventRecord(e1, nullptr));
            HIP_OK(hipEventSynchronize(e1));
            HIP_OK(hipEventElapsedTime(&ms, e0, e1));
        }
        HIP_OK(hipMemcpy(abort_h, buf + region_bytes, sizeof(abort_h), hipMemcpyDeviceToHost));
        return 0;
    };
    rc = body();
    if (e0) (void)hipEventDestroy(e0);
    if (e1) (void)hipEventDestroy(e1);
    (void)hipFree(buf);
    if (rc) return rc;
    if (abort_h[0]) return fail("taco_debug_handoff_probe: a bounded wait ran out (the 32 workgroups were not co-resident?)");
    *us_per_handoff = 1e3 * (double)ms / rounds;
    return check_launch("taco_debug_handoff_probe");
}

extern "C" int taco_debug_conv_gemm(const float* X, int32_t ldx, int32_t M, int32_t T, int32_t Cin, int32_t taps,
                                    int32_t padl, const float* W, int32_t ldw, int32_t N, const float* bias,
                                    const float* scale, const float* shift, const float* R, int32_t ldr, float* C,
                                    int32_t ldc, int32_t act, int32_t pool, taco_stream_t stream) {
    if (!X || !W || !C) return fail("taco_debug_conv_gemm: null argument");
    if (M < 1 || T < 1 || M % T || Cin < 16 || Cin % 16 || taps < 1 || ldw % 128 || N < 1 || N > ldw || ldx % 4 ||
        ldx < Cin || ldc < N || (scale == nullptr) != (shift == nullptr))
        return fail("taco_debug_conv_gemm: shapes violate the kernel's contract");
    if ((size_t)M * ldx * 4 >= ((size_t)1 << 31)) return fail("taco_debug_conv_gemm: X larger than 2 GiB");
    GemmArgs g{X, ldx, M, T, Cin, taps, padl, W, ldw, N, bias, scale, shift, R, ldr, C, ldc, act, pool};
    launch_conv_gemm(g, (hipStream_t)stream, nullptr);
    return check_launch("taco_debug_conv_gemm");
}

// ---------------------------------------------------------------------------------------
// paged key-value cache
namespace {

// The call's device for its launches; the thread's current device again afterwards. (Where there is no such device the call is
// refused: HIP's last error is cleared, or the next call would report it.)
struct DeviceScope {
    int prev = -1;
    bool ok = true;
    explicit DeviceScope(int device) {
        if (hipGetDevice(&prev) != hipSuccess) { ok = false; prev = -1; }
        else if (prev == device) prev = -1;
        else ok = hipSetDevice(device) == hipSuccess;
        if (!ok) (void)hipGetLastError();
    }
    ~DeviceScope() { if (prev >= 0) (void)hipSetDevice(prev); }
};

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int kv_pool_view(const char* what, const TacoKvPool* pool, KvPool* p) {
    if (!pool) return fail("%s: null pool", what);
    if (pool->struct_size != sizeof(TacoKvPool))
        return fail("%s: TacoKvPool.struct_size is %u, this library expects %zu", what, pool->struct_size, sizeof(TacoKvPool));
    if (!pool->k || !pool->v || !pool->status) return fail("%s: null pool tensor", what);
    if (pool->dtype < TACO_KV_F32 || pool->dtype > TACO_KV_F16) return fail("%s: dtype %d is not fp32, bf16 or fp16", what, pool->dtype);
    if (pool->device < 0) return fail("%s: device %d", what, pool->device);
    if (pool->num_pages < 1) return fail("%s: the pool needs at least one page", what);
    if (pool->kv_heads < 1 || pool->kv_heads > 1024) return fail("%s: kv_heads must be 1..1024 (got %d)", what, pool->kv_heads);
    const int ps = pool->page_size, d = pool->head_dim;
    if (ps < 8 || ps > 256 || (ps & (ps - 1))) return fail("%s: page_size must be 8, 16, 32, 64, 128 or 256 (got %d)", what, ps);
    if (d != 64 && d != 128 && d != 256) return fail("%s: head_dim must be 64, 128 or 256 (got %d)", what, d);
    const int esize = pool->dtype == TACO_KV_F32 ? 4 : 2;
    const int64_t st[6] = {pool->k_page_stride, pool->k_head_stride, pool->k_token_stride,
                           pool->v_page_stride, pool->v_head_stride, pool->v_token_stride};
    for (int64_t x : st)
        if (x < 0 || (x * esize) % 16) return fail("%s: pool strides must be non-negative multiples of 16 bytes", what);
    if (!aligned16(pool->k) || !aligned16(pool->v)) return fail("%s: the pool must start on a 16-byte boundary", what);
    p->k = pool->k;
    p->v = pool->v;
    for (int i = 0; i < 3; ++i) { p->k_st[i] = st[i]; p->v_st[i] = st[3 + i]; }
    p->device = pool->device;
    p->dtype = pool->dtype;
    p->esize = esize;
    p->num_pages = pool->num_pages;
    p->heads = pool->kv_heads;
    p->page_size = ps;
    p->page_shift = __builtin_ctz((unsigned)ps);
    p->dim = d;
    p->status = pool->status;
    return 0;
}

int kv_sizes(const char* what, const KvPool& p, int B, int max_pages) {
    if (B < 1 || B > 65535) return fail("%s: B must be 1..65535 (got %d)", what, B);
    if (max_pages < 1 || max_pages > (1 << 30) / p.page_size)
        return fail("%s: max_pages * page_size must be 1..2^30 (got %d * %d)", what, max_pages, p.page_size);
    return 0;
}

int kv_table_view(const char* what, const KvPool& p, const int32_t* table, int64_t ld, int B, int max_pages, KvTable* t) {
    if (int rc = kv_sizes(what, p, B, max_pages)) return rc;
    if (!table || ld < max_pages) return fail("%s: null page table, or rows closer than max_pages", what);
    *t = KvTable{table, ld, B, max_pages};
    return 0;
}

int kv_side(const char* what, const KvPool& p, const KvTable& t, int64_t side_ld) {
    if (side_ld < ((int64_t)t.max_pages << p.page_shift) || side_ld > (1 << 30))
        return fail("%s: side tables need a row for every slot, max_pages * page_size = %lld, and at most 2^30 (got %lld)",
                    what, (long long)t.max_pages << p.page_shift, (long long)side_ld);
    return 0;
}

int kv_heads_ok(const char* what, const KvPool& p, int B, int q_heads, int max_pages) {
    if (q_heads < 1 || q_heads > 65535 || q_heads % p.heads)
        return fail("%s: q_heads must be a multiple of kv_heads, at most 65535 (got %d over %d)", what, q_heads, p.heads);
    if (!kv_attend_fits(p, B, q_heads / p.heads, max_pages))
        return fail("%s: B * q_heads and B * kv_heads * slots are too many for one call", what);
    return 0;
}

int kv_rows(const char* what, const KvPool& p, const void* x, const int64_t* st, int n) {
    if (!x || !aligned16(x)) return fail("%s: null tensor, or one that does not start on a 16-byte boundary", what);
    for (int i = 0; i < n; ++i)
        if (st[i] < 0 || (st[i] * p.esize) % 16) return fail("%s: strides must be non-negative multiples of 16 bytes", what);
    return 0;
}

// Whether the ranges [a, a + an) and [b, b + bn) have a byte in common.
bool ranges_meet(const void* a, size_t an, const void* b, size_t bn) {
    return a && b && (uintptr_t)a < (uintptr_t)b + bn && (uintptr_t)b < (uintptr_t)a + an;
}

// Whether x meets the rows of a sequence's queries (of all heads and what lies between them), for any sequence.
bool meets_queries(const void* x, size_t n, const KvPool& p, const KvAttend& a, int B) {
    const size_t one = ((size_t)(p.heads * a.group - 1) * a.q_st[1] + p.dim) * p.esize, step = (size_t)a.q_st[0] * p.esize;
    if (!ranges_meet(x, n, a.q, (B - 1) * step + one)) return false;
    for (int b = 0; b < B; ++b)
        if (ranges_meet(x, n, (const char*)a.q + b * step, one)) return true;
    return false;
}

}  // namespace

extern "C" int taco_kv_take_status(const TacoKvPool* pool, int32_t* bits, taco_stream_t stream) {
    const char* what = "taco_kv_take_status";
    KvPool p;
    if (int rc = kv_pool_view(what, pool, &p)) return rc;
    if (!bits) return fail("%s: null argument", what);
    DeviceScope scope(pool->device);
    if (!scope.ok) return fail("%s: device %d is not available", what, pool->device);
    launch_kv_take_status(p.status, bits, (hipStream_t)stream);
    return check_launch(what);
}

extern "C" int taco_kv_append(const TacoKvPool* pool, const int32_t* table, int64_t table_ld, int32_t B, int32_t max_pages,
                              const void* k, int64_t k_batch_stride, int64_t k_token_stride, int64_t k_head_stride,
                              const void* v, int64_t v_batch_stride, int64_t v_token_stride, int64_t v_head_stride,
                              int32_t T, const int32_t* starts, const int32_t* counts, const int32_t* first, float* mass,
                              int32_t* positions, int64_t side_ld, int32_t* lengths_out, taco_stream_t stream) {
    const char* what = "taco_kv_append";
    KvPool p;
    KvTable t;
    if (int rc = kv_pool_view(what, pool, &p)) return rc;
    if (int rc = kv_table_view(what, p, table, table_ld, B, max_pages, &t)) return rc;
    KvAppend a{k, v, {k_batch_stride, k_token_stride, k_head_stride}, {v_batch_stride, v_token_stride, v_head_stride},
               T, starts, counts, first, mass, positions, side_ld, lengths_out};
    if (int rc = kv_rows(what, p, k, a.k_st, 3)) return rc;
    if (int rc = kv_rows(what, p, v, a.v_st, 3)) return rc;
    if (T < 1 || (int64_t)T * p.heads > (1 << 25)) return fail("%s: T must be at least 1 and T * kv_heads at most 2^25 (got T %d)", what, T);
    if (!starts || !lengths_out) return fail("%s: null argument", what);
    if (mass || positions)
        if (int rc = kv_side(what, p, t, side_ld)) return rc;
    // one workgroup of a sequence writes its length while others have yet to read where it starts
    const size_t ints = (size_t)B * sizeof(int32_t);
    for (const int32_t* in : {starts, counts, first})
        if (ranges_meet(lengths_out, ints, in, ints)) return fail("%s: lengths_out must not overlap starts, counts or first", what);
    DeviceScope scope(pool->device);
    if (!scope.ok) return fail("%s: device %d is not available", what, pool->device);
    launch_kv_append(p, t, a, (hipStream_t)stream);
    return check_launch(what);
}

extern "C" size_t taco_kv_attend_workspace_bytes(const TacoKvPool* pool, int32_t B, int32_t q_heads, int32_t max_pages,
                                                 int32_t with_mass) {
    const char* what = "taco_kv_attend_workspace_bytes";
    KvPool p;
    if (kv_pool_view(what, pool, &p) || kv_sizes(what, p, B, max_pages)) return 0;
    if (kv_heads_ok(what, p, B, q_heads, max_pages)) return 0;
    return std::max<size_t>(kv_attend_ws_bytes(p, B, q_heads / p.heads, max_pages, with_mass != 0), 16);
}

extern "C" int taco_kv_attend(const TacoKvPool* pool, const int32_t* table, int64_t table_ld, int32_t B,
                              int32_t max_pages, const int32_t* lengths, const void* q, int64_t q_batch_stride,
                              int64_t q_head_stride, int32_t q_heads, float scale, void* out, float* lse, float* mass,
                              int64_t side_ld, void* ws, size_t ws_bytes, taco_stream_t stream) {
    const char* what = "taco_kv_attend";
    KvPool p;
    KvTable t;
    if (int rc = kv_pool_view(what, pool, &p)) return rc;
    if (int rc = kv_table_view(what, p, table, table_ld, B, max_pages, &t)) return rc;
    if (int rc = kv_heads_ok(what, p, B, q_heads, max_pages)) return rc;
    KvAttend a{q, {q_batch_stride, q_head_stride}, q_heads / p.heads, lengths, scale * 1.4426950408889634f, out, lse, mass, side_ld,
               nullptr, nullptr, nullptr, 0};
    if (int rc = kv_rows(what, p, q, a.q_st, 2)) return rc;
    if (!lengths || !out || !lse || !aligned16(out)) return fail("%s: null argument, or out not on a 16-byte boundary", what);
    if (!std::isfinite(a.scale2)) return fail("%s: scale (and scale * log2(e)) must be finite", what);
    if (mass)
        if (int rc = kv_side(what, p, t, side_ld)) return rc;
    if (!ws || !aligned16(ws) || ws_bytes < kv_attend_ws_bytes(p, B, a.group, max_pages, mass != nullptr))
        return fail("%s: workspace too small (taco_kv_attend_workspace_bytes) or not on a 16-byte boundary", what);
    // Queries are read as a wave comes to their head, when other heads may be written already. A head's own row is written by
    // who read it, or after all have: contiguous queries may be written over in place.
    const size_t heads = (size_t)B * q_heads;
    const bool in_place = out == q && (q_heads == 1 || a.q_st[1] == p.dim) && (B == 1 || a.q_st[0] == (int64_t)q_heads * p.dim);
    if ((!in_place && meets_queries(out, heads * p.dim * p.esize, p, a, B)) || meets_queries(lse, heads * sizeof(float), p, a, B))
        return fail("%s: out must be the (contiguous) queries or not overlap them, nor may lse", what);
    DeviceScope scope(pool->device);
    if (!scope.ok) return fail("%s: device %d is not available", what, pool->device);
    launch_kv_attend(p, t, a, ws, (hipStream_t)stream);
    return check_launch(what);
}

extern "C" size_t taco_kv_evict_workspace_bytes(const TacoKvPool* pool, int32_t B, int32_t max_pages, int32_t budget) {
    const char* what = "taco_kv_evict_workspace_bytes";
    KvPool p;
    if (kv_pool_view(what, pool, &p) || kv_sizes(what, p, B, max_pages)) return 0;
    if (budget < 1) { (void)fail("%s: budget must be at least 1", what); return 0; }
    return kv_evict_ws_bytes(p, B, max_pages, budget);
}

extern "C" int taco_kv_evict(const TacoKvPool* pool, const int32_t* table, int64_t table_ld, int32_t B, int32_t max_pages,
                             const int32_t* lengths, const float* mass, const int32_t* positions, int64_t side_ld,
                             int32_t budget, int32_t recent, int32_t* lengths_out, float* mass_out,
                             int32_t* positions_out, void* ws, size_t ws_bytes, taco_stream_t stream) {
    const char* what = "taco_kv_evict";
    KvPool p;
    KvTable t;
    if (int rc = kv_pool_view(what, pool, &p)) return rc;
    if (int rc = kv_table_view(what, p, table, table_ld, B, max_pages, &t)) return rc;
    if (!lengths || !mass || !positions || !lengths_out || !mass_out || !positions_out) return fail("%s: null argument", what);
    if (int rc = kv_side(what, p, t, side_ld)) return rc;
    if (budget < 1 || recent < 0 || recent > budget)
        return fail("%s: needs 0 <= recent <= budget and budget >= 1 (got recent %d, budget %d)", what, recent, budget);
    if (!ws || !aligned16(ws) || ws_bytes < kv_evict_ws_bytes(p, B, max_pages, budget))
        return fail("%s: workspace too small (taco_kv_evict_workspace_bytes) or not on a 16-byte boundary", what);
    DeviceScope scope(pool->device);
    if (!scope.ok) return fail("%s: device %d is not available", what, pool->device);
    KvEvict a{lengths, budget, recent, mass, positions, side_ld, lengths_out, mass_out, positions_out,
              nullptr, nullptr, 0, nullptr, nullptr, nullptr};
    launch_kv_evict(p, t, a, ws, (hipStream_t)stream);
    return check_launch(what);
}
