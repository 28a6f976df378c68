// Verification of a tree of drafted tokens against the target's distributions, from given draws.
//
// Row i of the logits is the target's prediction after node i. P_i is its distribution as it is
// sampled: softmax(l / T), cut to the nucleus (the tokens in descending order of their logits, equal
// ones by index, up to the one whose running sum reaches top_p) and divided by what is left. The walk
// starts at node 0. At node i its children are tried in index order, each token c_k against its draw
// u_k in [0, 1):
//   drafts without distributions (each child a token the drafter was sure of):
//     accept c_k if u_k (1 - sum of P(c) over the tokens c rejected before) < P(c_k);
//     what is left after a rejection is P without the rejected tokens;
//   drafts sampled from Q = the draft's distribution at node i, one after the other:
//     R_0 = P, accept c_k if u_k Q(c_k) < R_k(c_k), else R_{k+1} = max(R_k - Q, 0) / its sum.
//     Unrolled, R_k = max(P - t_k Q, 0) / S_k with t_0 = 0, S_0 = 1, t_{k+1} = t_k + S_k and
//     S_k = sum max(P - t_k Q, 0): each rejection is one sum over the vocabulary.
// Either way the accepted token and, at the node where every child is rejected (or that has none),
// the next token drawn from what is left are distributed as samples of P.
//
// A token's weight is w = 2^((l - max) log2(e) / T), in 64 bits throughout (exp2_64 below): a draw falls
// on one of up to half a million borders, so sums that are off by 2^-24 would move one draw in some
// thousands. That is 16 operations a logit: 64 rows of 128,256 take 17 us with their sums and 10 without.
//
// Kernels, each with a workgroup per row and chunk of it (of 4096 or 8192 logits), but for the walk:
//   k_ver_chunks  a chunk's maximum, its index, minimum, sum of weights
//   k_ver_bins    (where top_p cuts) the weights by 512 bins; the last workgroup of a row finds the bin
//                 that the nucleus ends in
//   k_ver_cut     (where top_p cuts) that bin's tokens in a list, the weights above it; the last workgroup
//                 of a row finds the last token kept
//   k_ver_rounds  (drafts with distributions) S_1 of the rows with two or more children
//   k_ver_walk    every child's test at once, the path by its first accepted children, the draw. One
//                 workgroup where the chunks' sums serve the draw; else one a chunk of the last row, all of
//                 them walking for themselves, each summing what is left of its chunk, the last one drawing
// "The last workgroup": every workgroup sends its part past the XCDs' caches (agent-scope stores), waits for
// that, and counts itself; the one that counts all takes them in the same way. No workgroup waits for another.
//
// What bounds them (128,256 logits a row unless said): k_ver_chunks for 64 rows the reading (33 MB in 9 to 10 us;
// with the 64-bit sums the vector units, 17), for 5 its launch (5 us). k_ver_bins 18 us and k_ver_cut 15 for 64 rows,
// half of either the way from the first workgroup's parts to the last one's result (13 and 9 for 26 rows of
// 151,936). k_ver_walk 10 to 14 us, a chain of dependent rounds: nodes, their logits, the rows, the sums, the drawn
// chunk (3 to 4 us of it the draw); 24 us more for each third or later sibling tried, a whole row read by every
// workgroup. Whole calls: chain of 5 14.6 us, 64-node nucleus tree 55, 6 sampled nodes over 151,936 19.5, 26 with
// a nucleus 48 to 72.
#include <climits>

#include "dev_common.hpp"
#include "tf_internal.hpp"

namespace tfk {
namespace {

typedef unsigned long long u64_t;
constexpr int kVerThreads = 1024;
constexpr int kVerWaves = kVerThreads / kWave;
constexpr int kChunk = 4096;
constexpr int kMaxChunks = (TF_HIP_VERIFY_MAX_VOCAB + kChunk - 1) / kChunk;
// The nucleus' kernels: 16 logits a thread like the others, but half as many workgroups to count (a 64-node tree
// over 128,256 logits: 256 threads 55.1 us a call, 512 54.2, 1024 60.8).
constexpr int kCutThreads = 512, kCutChunk = 16 * kCutThreads, kBins = kCutThreads, kList = 4096, kFew = 64;
constexpr int kBinBits = 9, kIndexBits = 19;
static_assert(1 << kBinBits == kBins && 1 << kIndexBits == TF_HIP_VERIFY_MAX_VOCAB, "bits of a bin and of an index");
constexpr double kLog2e64 = 1.4426950408889634;

// Of one chunk of a row: its largest logit, that one's first index, and the weights' sum, the largest's 1.
struct VerChunk {
    double sum;
    float mx, mn;  // mn: the least that is not -inf
    int32_t arg;
};
// One row's distribution: token x with logit l has probability w(l) / z where it is kept, that is
// where l is above thr, or equal to it with x <= cut (-inf and INT_MAX: all but NaN); mx is the largest logit, first at arg.
struct VerRow {
    double z, inv_z;  // inv_z: 0 where nothing is kept
    float mx;
    float thr;
    int32_t cut;
    int32_t arg;
};
// A row on the way to its nucleus: the bin of k_ver_bins that its end lies in, the mass above that bin, the
// mass that the kept tokens reach, and the counts of workgroups that are done and of listed tokens.
struct VerCut {
    u64_t before, target;
    float mx, mn;
    int32_t bin;
    uint32_t binned, listed, done;
};
struct VerWork {
    uint32_t* arrived;  // workgroups of k_ver_walk that have their sums
    VerRow* rows;       // [n]
    VerCut* cuts;       // [n]
    VerChunk* chunks;   // [n][chunks a row]
    double* round;      // [n][chunks a row]: k_ver_rounds
    u64_t* mass;        // [n][kCutChunk chunks a row][kBins]
    u64_t* above;       // [n][kCutChunk chunks a row]: doubles
    u64_t* list;        // [n][kList]: logit, index
    u64_t* left;        // [chunks a row]: k_ver_walk's sums (doubles)
    int n_chunks, n_cuts;  // of a row, of kChunk and of kCutChunk logits
};

__device__ __forceinline__ uint32_t logit_key(float l) { return (uint32_t)(argmax_key(l, 0) >> 32); }

// 2^y for y <= 0: 2^n 2^f with |f| <= 1/2, 2^f the Taylor series of e^(f ln 2) to its 10th power (the rest is
// below 3e-13 of it). NaN, and anything below -1100, gives 0.
__device__ __forceinline__ double exp2_64(double y) {
    y = fmax(y, -1100.0);
    const double n = rint(y), x = (y - n) * 0.69314718055994531;
    double p = 1.0 / 3628800.0;
    p = fma(p, x, 1.0 / 362880.0);
    p = fma(p, x, 1.0 / 40320.0);
    p = fma(p, x, 1.0 / 5040.0);
    p = fma(p, x, 1.0 / 720.0);
    p = fma(p, x, 1.0 / 120.0);
    p = fma(p, x, 1.0 / 24.0);
    p = fma(p, x, 1.0 / 6.0);
    p = fma(p, x, 0.5);
    p = fma(p, x, 1.0);
    p = fma(p, x, 1.0);
    return __builtin_amdgcn_ldexp(p, (int)n);
}
// A logit's weight against the maximum mx; c = log2(e) / T. One equal to the maximum weighs 1 also where both
// are infinite; NaN weighs nothing.
__device__ __forceinline__ double weight(float l, float mx, double c) {
    const double w = exp2_64(((double)l - (double)mx) * c);
    return l == mx ? 1.0 : w;
}
__device__ __forceinline__ bool kept(const VerRow& r, float l, int x) { return l > r.thr || (l == r.thr && x <= r.cut); }
__device__ __forceinline__ double prob(const VerRow& r, float l, int x, double c) {
    return kept(r, l, x) ? weight(l, r.mx, c) * r.inv_z : 0.0;
}

// Folds and scans over a wave without LDS round trips: lane permutes within 16 lanes (DPP), then swaps of rows of
// 16 and of halves. Partners fold the same two values, so every lane ends with the same bits.
template <int CTRL, class T>
__device__ __forceinline__ T dpp_of(T v) {
    constexpr int kWords = sizeof(T) / 4;
    int w[kWords];
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = __builtin_amdgcn_update_dpp(0, w[i], CTRL, 0xF, 0xF, false);
    __builtin_memcpy(&v, w, sizeof(T));
    return v;
}
template <class T, class F>
__device__ __forceinline__ T wave_fold(T v, F op) {
    v = op(v, dpp_of<kDppXor1>(v));
    v = op(v, dpp_of<kDppXor2>(v));
    v = op(v, dpp_of<kDppHalfMirror>(v));
    v = op(v, dpp_of<kDppMirror>(v));
    constexpr int kWords = sizeof(T) / 4;
    uint32_t w[kWords], x[kWords], y[kWords];
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
        const auto p = __builtin_amdgcn_permlane16_swap(w[i], w[i], false, false);
        x[i] = p[0];
        y[i] = p[1];
    }
    T a, b;
    __builtin_memcpy(&a, x, sizeof(T));
    __builtin_memcpy(&b, y, sizeof(T));
    v = op(a, b);
    __builtin_memcpy(w, &v, sizeof(T));
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
        const auto p = __builtin_amdgcn_permlane32_swap(w[i], w[i], false, false);
        x[i] = p[0];
        y[i] = p[1];
    }
    __builtin_memcpy(&a, x, sizeof(T));
    __builtin_memcpy(&b, y, sizeof(T));
    return op(a, b);
}
// A 64-bit value of lane i, uniform.
template <class T>
__device__ __forceinline__ T lane_value(T v, int i) {
    static_assert(sizeof(T) == 8, "two words");
    int w[2];
    __builtin_memcpy(w, &v, 8);
    w[0] = __builtin_amdgcn_readlane(w[0], i);
    w[1] = __builtin_amdgcn_readlane(w[1], i);
    __builtin_memcpy(&v, w, 8);
    return v;
}
// The sum of the lanes up to this one.
template <class T>
__device__ __forceinline__ T wave_scan(T v) {
    v += dpp_of<0x111>(v);  // row_shr: the lane 1, 2, 4, 8 below in the row of 16, or 0
    v += dpp_of<0x112>(v);
    v += dpp_of<0x114>(v);
    v += dpp_of<0x118>(v);
    const T r0 = lane_value(v, 15), r1 = r0 + lane_value(v, 31), r2 = r1 + lane_value(v, 47);
    const int row = (int)(threadIdx.x & 63) >> 4;
    return row == 0 ? v : v + (row == 1 ? r0 : (row == 2 ? r1 : r2));
}
// Folds over the workgroup; every thread gets the result. red: a word for each wave.
template <class T, class F>
__device__ __forceinline__ T block_fold(T v, u64_t* red, F op) {
    v = wave_fold(v, op);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) ((T*)red)[threadIdx.x >> 6] = v;
    __syncthreads();
    v = ((T*)red)[0];
#pragma unroll
    for (int w = 1; w < kVerWaves; ++w) {
        if (w >= (int)(blockDim.x >> 6)) break;
        v = op(v, ((T*)red)[w]);
    }
    return v;
}
__device__ __forceinline__ double block_sum(double v, u64_t* red) {
    return block_fold(v, red, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ u64_t block_max(u64_t v, u64_t* red) {
    return block_fold(v, red, [](u64_t a, u64_t b) { return a > b ? a : b; });
}

// f(index, value) for the n floats at p, over the workgroup's threads: aligned 16-byte loads, four ahead.
template <class F>
__device__ __forceinline__ void each(const float* p, int n, F f) {
    const int tid = threadIdx.x, step = blockDim.x;
    const int head = min(n, (int)((16 - ((uintptr_t)p & 15)) & 15) >> 2), n4 = (n - head) >> 2;
    const float* b = p + head;
    if (tid < head) f(tid, p[tid]);
    auto four = [&](int i, float4 v) {
        f(head + 4 * i, v.x);
        f(head + 4 * i + 1, v.y);
        f(head + 4 * i + 2, v.z);
        f(head + 4 * i + 3, v.w);
    };
    int i = tid;
    for (; i + 3 * step < n4; i += 4 * step) {
        float4 v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = gload_f4(b + 4 * (i + k * step));
#pragma unroll
        for (int k = 0; k < 4; ++k) four(i + k * step, v[k]);
    }
    for (; i < n4; i += step) four(i, gload_f4(b + 4 * i));
    const int tail = head + 4 * n4 + tid;
    if (tail < n) f(tail, p[tail]);
}

// E values of every thread from p (n of them are there, the rest is `none`): value k of thread i is
// number place<E, RUN>(k), E i + k where RUN, else in groups of 4 that lie side by side over the threads.
template <int E, bool RUN>
__device__ __forceinline__ int place(int k) {
    const int tid = (int)threadIdx.x;
    return RUN ? E * tid + k : 4 * (tid + k / 4 * (int)blockDim.x) + k % 4;
}
template <int E, bool RUN>
__device__ __forceinline__ void take(const float* p, int n, float none, float* v) {
    const bool vec = ((uintptr_t)p & 15) == 0;
#pragma unroll
    for (int k = 0; k < E; k += 4) {
        const int at = place<E, RUN>(k);
        if (vec && at + 4 <= n) {
            const float4 x = gload_f4(p + at);
            v[k] = x.x; v[k + 1] = x.y; v[k + 2] = x.z; v[k + 3] = x.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[k + j] = at + j < n ? *gptr(p + at + j) : none;
        }
    }
}

// ---------------------------------------------------------------- rows

// Grid (chunk, row), 256 threads of 16 logits. The first workgroups ready the counts.
constexpr int kChunkEach = kChunk / kBlock;
__global__ __launch_bounds__(kBlock) void k_ver_chunks(const VerifyArgs a, const VerWork wk) {
    __shared__ u64_t red[kWavesPerBlock];
    const int row = blockIdx.y, x0 = blockIdx.x * kChunk, n = min(kChunk, a.vocab - x0);
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        if (row == 0) *wk.arrived = 0;
        wk.cuts[row].binned = wk.cuts[row].listed = wk.cuts[row].done = 0;
    }
    float v[kChunkEach];
    take<kChunkEach, false>(a.logits + (int64_t)row * a.ld + x0, n, NAN, v);
    u64_t best = 0;
    float mn = INFINITY;
#pragma unroll
    for (int k = 0; k < kChunkEach; ++k)
        if (v[k] == v[k]) {
            best = max(best, argmax_key(v[k], x0 + place<kChunkEach, false>(k)));
            if (v[k] > -INFINITY) mn = fminf(mn, v[k]);
        }
    best = block_max(best, red);
    mn = block_fold(mn, red, [](float x, float y) { return fminf(x, y); });
    const int arg = best ? (int)(0xFFFFFFFFu - (uint32_t)best) : 0;
    const uint32_t key = (uint32_t)(best >> 32);
    const float mx = best ? __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key) : -INFINITY;
    double sum = 0.0;
    if (a.temperature > 0.0f && !(a.top_p < 1.0f)) {
        const double c = kLog2e64 / (double)a.temperature;
#pragma unroll
        for (int k = 0; k < kChunkEach; ++k) sum += weight(v[k], mx, c);
        sum = block_sum(sum, red);
    }
    if (threadIdx.x == 0) wk.chunks[(int64_t)row * wk.n_chunks + blockIdx.x] = {sum, mx, mn, arg};
}

__device__ __forceinline__ double row_sum(double v) {  // over 16 lanes
    v += dpp_of<kDppXor1>(v);
    v += dpp_of<kDppXor2>(v);
    v += dpp_of<kDppHalfMirror>(v);
    v += dpp_of<kDppMirror>(v);
    return v;
}

// A row from its chunks, by each 16 lanes of a wave that ask for one (all of them get it).
__device__ __forceinline__ VerRow row_of_chunks(const VerifyArgs& a, const VerWork& wk, int row) {
    const int l16 = threadIdx.x & 15;
    const VerChunk* ch = wk.chunks + (int64_t)row * wk.n_chunks;
    constexpr int kEach = kMaxChunks / 16;
    static_assert(kMaxChunks % 16 == 0, "16 lanes take the chunks");
    VerChunk v[kEach];
    u64_t best = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        if (16 * k >= wk.n_chunks) break;
        v[k] = ch[min(l16 + 16 * k, wk.n_chunks - 1)];
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        if (16 * k >= wk.n_chunks) break;
        best = max(best, argmax_key(v[k].mx, v[k].arg));
    }
    best = max(best, dpp_of<kDppXor1>(best));
    best = max(best, dpp_of<kDppXor2>(best));
    best = max(best, dpp_of<kDppHalfMirror>(best));
    best = max(best, dpp_of<kDppMirror>(best));
    VerRow r;
    r.arg = (int32_t)(0xFFFFFFFFu - (uint32_t)best);
    const uint32_t key = (uint32_t)(best >> 32);
    r.mx = __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
    r.thr = -INFINITY;
    r.cut = INT_MAX;
    r.z = r.inv_z = 1.0;
    if (a.temperature <= 0.0f) {
        r.thr = r.mx;
        r.cut = r.arg;
    } else {
        const double c = kLog2e64 / (double)a.temperature;
        double z = 0.0;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            if (16 * k >= wk.n_chunks) break;
            if (l16 + 16 * k < wk.n_chunks && v[k].sum > 0.0) z += v[k].sum * weight(v[k].mx, r.mx, c);
        }
        z = row_sum(z);
        r.z = z;
        r.inv_z = z > 0.0 ? 1.0 / z : 0.0;
    }
    return r;
}

// The largest and the least logit of a row (but for -inf), from its chunks, in every thread.
__device__ __forceinline__ void row_range(const VerWork& wk, int row, float& mx, float& mn) {
    const int l64 = threadIdx.x & 63;
    static_assert(kMaxChunks <= 128, "two chunks a lane");
    const VerChunk* ch = wk.chunks + (int64_t)row * wk.n_chunks;
    const int i0 = min(l64, wk.n_chunks - 1), i1 = min(l64 + 64, wk.n_chunks - 1);
    mx = wave_max(fmaxf(ch[i0].mx, ch[i1].mx));
    mn = -wave_max(-fminf(ch[i0].mn, ch[i1].mn));
}

// ---------------------------------------------------------------- the nucleus
// The sums that find where it ends are of 64-bit weights as integers of 2^-44 of the largest: integers add up to
// the same in any order, so the atomics do not show. Their roundings come to 2e-8 of the total at the very most
// (half a million equal logits far below one), commonly 1e-11. 32-bit weights were 1e-9 off as a rule, which kept
// another last token in one row of some 100,000 random ones, for 49.7 us instead of 55.2 with 64 rows of 128,256.
struct Mass {
    double mx, c;  // c = log2(e) / T
    __device__ Mass(float mx, double c) : mx((double)mx), c(c) {}
    // 2^(y + 44), rounded; 0 for -inf and NaN. 2^f is the Taylor series of e^(f ln 2) to its 9th power (|f| <= 1/2:
    // the rest is below 7e-12 of it). What is added to 2^52 lies in the sum's low 52 bits.
    __device__ u64_t operator()(float l) const {
        const double y = (double)l == mx ? 0.0 : fmax(((double)l - mx) * c, -200.0), n = rint(y), f = y - n;
        double p = 1.0178086009239699e-07;
        p = fma(p, f, 1.3215486790144307e-06);
        p = fma(p, f, 1.5252733804059841e-05);
        p = fma(p, f, 1.5403530393381608e-04);
        p = fma(p, f, 1.3333558146428443e-03);
        p = fma(p, f, 9.6181291076284772e-03);
        p = fma(p, f, 5.5504108664821580e-02);
        p = fma(p, f, 2.4022650695910071e-01);
        p = fma(p, f, 6.9314718055994531e-01);
        p = fma(p, f, 1.0);
        p = __builtin_amdgcn_ldexp(p, (int)n + 44) + 0x1p52;
        return (u64_t)__double_as_longlong(p) & 0xFFFFFFFFFFFFFull;
    }
};
// kBins bins of equal width below the maximum, as far as the least logit or 24 temperatures (where a token's
// weight is 2^-34 of the largest); what is below is in the last one.
struct Bins {
    float mx, scale;  // bins for a step of 1 in the logit: 32 bits do, as the roundings keep the logits' order
    __device__ Bins(float mx, float mn, double c) : mx(mx) {
        const float span = fminf((mx - mn) * (float)c, 24.0f * (float)kLog2e64);
        scale = span > 0.0f ? (float)c * (-(float)kBins / span) : 0.0f;
    }
    // -inf and NaN are in the last one
    __device__ int operator()(float l) const { return l == mx ? 0 : (int)fminf((l - mx) * scale, (float)(kBins - 1)); }
};
__device__ __forceinline__ void send(u64_t* p, u64_t v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ u64_t receive(const u64_t* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// Counts this workgroup, whose parts every thread has sent; true in the last of n. sh: a word of LDS.
__device__ __forceinline__ bool last_of(uint32_t* count, int n, int* sh) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) *sh = (int)__hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    return *sh == n - 1;
}

// The bin whose masses reach `target` from `before` on, for kBins = blockDim.x threads with a bin each; out: the
// bin and the mass above it. red: a word for each wave.
__device__ __forceinline__ void find_bin(u64_t mass, u64_t before, u64_t target, u64_t* red, int* out_bin, u64_t* out_before) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const u64_t run = wave_scan(mass);
    __syncthreads();
    if (lane == 63) red[wave] = run;
    __syncthreads();
    u64_t at = before + run - mass;
    for (int i = 0; i < wave; ++i) at += red[i];
    if (at < target && at + mass >= target) {
        *out_bin = tid;
        *out_before = at;
    }
    __syncthreads();
}

constexpr int kCutEach = kCutChunk / kCutThreads;
__global__ __launch_bounds__(kCutThreads) void k_ver_bins(const VerifyArgs a, const VerWork wk) {
    __shared__ u64_t mass[kBins + 64], red[(kCutThreads / kWave)];  // the last 64: the last bin's, by lane
    __shared__ u64_t sh_before;
    __shared__ int sh, sh_bin;
    static_assert(kBins == kCutThreads, "a bin a thread");
    const int tid = threadIdx.x, row = blockIdx.y, x0 = blockIdx.x * kCutChunk, n = min(kCutChunk, a.vocab - x0);
    float v[kCutEach];
    take<kCutEach, false>(a.logits + (int64_t)row * a.ld + x0, n, NAN, v);
    mass[tid] = 0;
    if (tid < 64) mass[kBins + tid] = 0;
    float mx, mn;
    row_range(wk, row, mx, mn);
    __syncthreads();
    const double c = kLog2e64 / (double)a.temperature;
    const Bins bin(mx, mn, c);
    const Mass mass_of(mx, c);
    // no branches: most logits are in the last bin, and go to a place of their lane's
#pragma unroll
    for (int k = 0; k < kCutEach; ++k) {
        const int b = bin(v[k]);
        atomicAdd(&mass[b == kBins - 1 ? kBins + (tid & 63) : b], mass_of(v[k]));
    }
    __syncthreads();
    if (tid < 64) {
        const u64_t low = wave_fold(mass[kBins + tid], [](u64_t x, u64_t y) { return x + y; });
        if (tid == 0) mass[kBins - 1] = low;
    }
    __syncthreads();
    u64_t* part = wk.mass + (int64_t)row * wk.n_cuts * kBins;
    send(part + blockIdx.x * kBins + tid, mass[tid]);
    VerCut& cut = wk.cuts[row];
    if (!last_of(&cut.binned, wk.n_cuts, &sh)) return;
    u64_t m = 0;
    constexpr int kRound = 8;
    for (int i = 0; i < wk.n_cuts; i += kRound) {
        u64_t x[kRound];
#pragma unroll
        for (int j = 0; j < kRound; ++j) x[j] = receive(part + min(i + j, wk.n_cuts - 1) * kBins + tid);
#pragma unroll
        for (int j = 0; j < kRound; ++j) m += i + j < wk.n_cuts ? x[j] : 0;
    }
    const u64_t all = block_fold(m, red, [](u64_t x, u64_t y) { return x + y; });
    const double want = (double)fmaxf(a.top_p, 0.0f) * (double)all;
    u64_t target = (u64_t)want;
    if ((double)target < want) ++target;  // a token is kept while the sum before it is below top_p
    target = target < 1 ? 1 : (target > all ? all : target);
    if (tid == 0) {
        sh_bin = 0;
        sh_before = 0;
    }
    find_bin(m, 0, target, red, &sh_bin, &sh_before);
    if (tid == 0) {
        cut.before = sh_before;
        cut.target = target;
        cut.mx = mx;
        cut.mn = mn;
        cut.bin = sh_bin;
    }
}

// Which of a set of tokens the running sum ends at: `each` calls f(index, logit) for all of them (over the
// workgroup's threads), `before` is the mass above them. Narrows their keys by bins until few are left, which
// are ranked, or one logit many times over, of which the k-th in index order is the last.
struct Settle {
    u64_t mass[kBins], red[(kCutThreads / kWave)];
    uint4 few[kFew];  // key, index, mass
    u64_t before;
    uint2 end;  // of the last token kept
    uint32_t n, k_lo, k_hi;
    int bin;
};
template <class Each>
__device__ void settle(Each each_of, u64_t before, u64_t target, const Mass& weight_of, Settle& s, float& thr, int32_t& cut) {
    const int tid = threadIdx.x;
    uint32_t lo = 0, hi = 0xFFFFFFFFu;
    auto inside = [&](float l) {
        const uint32_t k = logit_key(l);
        return k >= lo && k <= hi;
    };
    for (;;) {
        __syncthreads();
        if (tid == 0) {
            s.n = 0;
            s.k_lo = 0xFFFFFFFFu;
            s.k_hi = 0;
            s.bin = 0;
            s.before = before;
            s.end = make_uint2(__float_as_uint(INFINITY), 0xFFFFFFFFu);  // none
        }
        s.mass[tid] = 0;
        __syncthreads();
        uint32_t a = 0xFFFFFFFFu, b = 0;
        each_of([&](int x, float l) {
            if (!inside(l)) return;
            const uint32_t k = logit_key(l);
            if (*(volatile uint32_t*)&s.n <= kFew) {  // past that only how many keys there are matters
                const uint32_t at = atomicAdd(&s.n, 1u);
                const u64_t w = weight_of(l);
                if (at < kFew) s.few[at] = make_uint4(k, (uint32_t)x, (uint32_t)w, (uint32_t)(w >> 32));
            }
            a = min(a, k);
            b = max(b, k);
        });
        if (a <= b) {
            atomicMin(&s.k_lo, a);
            atomicMax(&s.k_hi, b);
        }
        __syncthreads();
        if (s.n <= kFew || s.k_lo == s.k_hi) break;
        lo = s.k_lo;
        hi = s.k_hi;
        int shift = 0;
        while (((hi - lo) >> shift) >= (uint32_t)kBins) ++shift;
        each_of([&](int, float l) {
            if (inside(l)) atomicAdd(&s.mass[(hi - logit_key(l)) >> shift], weight_of(l));
        });
        __syncthreads();
        find_bin(s.mass[tid], before, target, s.red, &s.bin, &s.before);
        before = s.before;
        const uint32_t top = hi - ((uint32_t)s.bin << shift);
        lo = max(lo, top - min(top, (1u << shift) - 1));
        hi = top;
    }
    const int m = (int)s.n;
    if (m > kFew) {
        const uint32_t key = s.k_lo;
        const float l1 = __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
        const u64_t w = max(weight_of(l1), (u64_t)1), k = (target - before + w - 1) / w;
        // the index of the k-th: its bits from the highest on, kBins ranges of indices at a time
        int first = 0;
        u64_t have = 0;
        for (int shift = kIndexBits; shift > 0;) {
            const int above = shift;
            shift = max(0, shift - kBinBits);
            __syncthreads();
            s.mass[tid] = 0;
            __syncthreads();
            each_of([&](int x, float l) {
                if (logit_key(l) == key && x >> above == first >> above) atomicAdd(&s.mass[(x >> shift) & (kBins - 1)], (u64_t)1);
            });
            __syncthreads();
            find_bin(s.mass[tid], have, k, s.red, &s.bin, &s.before);
            have = s.before;
            first |= s.bin << shift;
        }
        const int a = first;
        thr = l1;
        cut = a;
        return;
    }
    __syncthreads();
    if (tid < m) {
        const uint4 me = s.few[tid];
        u64_t sum = before;
        for (int j = 0; j < m; ++j) {
            const uint4 it = s.few[j];
            if (it.x > me.x || (it.x == me.x && it.y < me.y)) sum += (u64_t)it.w << 32 | it.z;
        }
        if (sum < target && sum + ((u64_t)me.w << 32 | me.z) >= target)
            s.end = make_uint2(me.x & 0x80000000u ? me.x & 0x7FFFFFFFu : ~me.x, me.y);
    }
    __syncthreads();
    thr = __uint_as_float(s.end.x);
    cut = (int32_t)s.end.y;
}

__global__ __launch_bounds__(kCutThreads) void k_ver_cut(const VerifyArgs a, const VerWork wk) {
    __shared__ uint2 list[kList];
    __shared__ Settle s;
    __shared__ uint32_t n_here, at_here;
    __shared__ int sh;
    const int tid = threadIdx.x, row = blockIdx.y, x0 = blockIdx.x * kCutChunk, n = min(kCutChunk, a.vocab - x0);
    const float* p = a.logits + (int64_t)row * a.ld;
    float v[kCutEach];
    take<kCutEach, false>(p + x0, n, NAN, v);
    VerCut& cut = wk.cuts[row];
    const float mx = cut.mx;
    const int b0 = cut.bin;
    const double c64 = kLog2e64 / (double)a.temperature;
    const Bins bin(mx, cut.mn, c64);
    if (tid == 0) n_here = 0;
    __syncthreads();
    double above = 0.0;
#pragma unroll
    for (int k = 0; k < kCutEach; ++k) {
        const int b = v[k] <= mx ? bin(v[k]) : kBins;
        if (b == b0) {
            const uint32_t at = atomicAdd(&n_here, 1u);
            if (at < kList) list[at] = make_uint2(__float_as_uint(v[k]), (uint32_t)(x0 + place<kCutEach, false>(k)));
        }
        if (b < b0) above += weight(v[k], mx, c64);
    }
    above = block_sum(above, s.red);
    if (tid == 0) {
        send(wk.above + (int64_t)row * wk.n_cuts + blockIdx.x, (u64_t)__double_as_longlong(above));
        at_here = n_here ? __hip_atomic_fetch_add(&cut.listed, n_here, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
    }
    __syncthreads();
    for (uint32_t i = tid; i < min(n_here, (uint32_t)kList); i += kCutThreads)
        if (at_here + i < kList) send(wk.list + (int64_t)row * kList + at_here + i, (u64_t)list[i].y << 32 | list[i].x);
    if (!last_of(&cut.done, wk.n_cuts, &sh)) return;
    const uint32_t m = __hip_atomic_load(&cut.listed, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    VerRow r;
    r.mx = mx;
    r.arg = 0;
    double z = 0.0;
    for (int i = tid; i < wk.n_cuts; i += kCutThreads) z += __longlong_as_double((long long)receive(wk.above + (int64_t)row * wk.n_cuts + i));
    z = block_sum(z, s.red);
    double in = 0.0;
    auto settle_of = [&](auto each_of) {
        settle(each_of, cut.before, cut.target, Mass(mx, c64), s, r.thr, r.cut);
        each_of([&](int x, float l) {
            if (kept(r, l, x)) in += weight(l, mx, c64);
        });
    };
    if (m <= kList) {
        for (uint32_t i = tid; i < m; i += kCutThreads) {
            const u64_t e = receive(wk.list + (int64_t)row * kList + i);
            list[i] = make_uint2((uint32_t)e, (uint32_t)(e >> 32));
        }
        __syncthreads();
        settle_of([&](auto f) {
            for (uint32_t i = tid; i < m; i += kCutThreads) f((int)list[i].y, __uint_as_float(list[i].x));
        });
    } else {
        // too many for the list (one logit thousands of times over, or a bin that most logits are in): from the row
        settle_of([&](auto f) {
            each(p, a.vocab, [&](int x, float l) {
                if (l <= mx && bin(l) == b0) f(x, l);
            });
        });
    }
    r.z = z + block_sum(in, s.red);
    r.inv_z = r.z > 0.0 ? 1.0 / r.z : 0.0;
    if (tid == 0) wk.rows[row] = r;
}

// ---------------------------------------------------------------- sampled drafts: S_1

// Grid (chunk, row): the chunk's sum of max(P - Q, 0), for rows with two or more children.
__global__ __launch_bounds__(kBlock) void k_ver_rounds(const VerifyArgs a, const VerWork wk) {
    __shared__ u64_t red[kWavesPerBlock];
    __shared__ int kids;
    const int row = blockIdx.y, x0 = blockIdx.x * kChunk, n = min(kChunk, a.vocab - x0);
    if (threadIdx.x == 0) kids = 0;
    __syncthreads();
    const int j = threadIdx.x;
    static_assert(kTreeMax <= kBlock, "a thread per node");
    if (j > row && j < a.n_tree && a.parent[j] == row) atomicAdd(&kids, 1);
    __syncthreads();
    if (kids < 2) return;
    const VerRow r = a.top_p < 1.0f ? wk.rows[row] : row_of_chunks(a, wk, row);
    float l[kChunkEach], q[kChunkEach];
    take<kChunkEach, false>(a.logits + (int64_t)row * a.ld + x0, n, NAN, l);
    take<kChunkEach, false>(a.draft + (int64_t)row * a.ld_draft + x0, n, 0.0f, q);
    const double c = kLog2e64 / (double)a.temperature;
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kChunkEach; ++k)
        sum += fmax(prob(r, l[k], x0 + place<kChunkEach, false>(k), c) - (double)q[k], 0.0);
    sum = block_sum(sum, red);
    if (threadIdx.x == 0) wk.round[(int64_t)row * wk.n_chunks + blockIdx.x] = sum;
}

// ---------------------------------------------------------------- the draw

// What is left of a row: its rejected tokens or t Q taken off P (in units of 1 / z where there is no Q).
struct Left {
    VerRow r;
    const float* l;
    const float* q;    // or nullptr
    double t, c;
    const int* gone;   // the rejected tokens (LDS), where there is no Q
    int n_gone;
    // of token x, where it is kept
    __device__ double of_kept(float lx, float qx, int x) const {
        const double w = weight(lx, r.mx, c);
        if (q) return fmax(w * r.inv_z - t * (double)qx, 0.0);
        for (int i = 0; i < n_gone; ++i)
            if (gone[i] == x) return 0.0;
        return w;
    }
};

// The sum of N chunks of it (those that there are), over the workgroup's threads; every chunk's loads go first.
template <int E, int N>
__device__ __forceinline__ double left_part(const Left& f, int vocab, int chunk) {
    float l[N][E], q[N][E];
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int x0 = (chunk + i) * kChunk, n = min(kChunk, vocab - x0);
        take<E, false>(f.l + x0, n, NAN, l[i]);
        if (f.q) take<E, false>(f.q + x0, n, 0.0f, q[i]);
    }
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < E; ++k) {
            const int x = (chunk + i) * kChunk + place<E, false>(k);
            if (kept(f.r, l[i][k], x)) sum += f.of_kept(l[i][k], f.q ? q[i][k] : 0.0f, x);
        }
    return sum;
}
template <int E>
__device__ __forceinline__ double left_sum(const Left& f, int vocab, int chunk, u64_t* red) {
    return block_sum(left_part<E, 1>(f, vocab, chunk), red);
}
template <int E>
__device__ double left_row_sum(const Left& f, int vocab, int n_chunks, u64_t* red) {
    double sum = 0.0;
    for (int ch = 0; ch < n_chunks; ch += 8) sum += left_part<E, 8>(f, vocab, ch);
    return block_sum(sum, red);
}

// The first token at which the running sum exceeds u times the total, from the chunks' sums (LDS). -1 where
// nothing is left. *p_out (LDS): P of it. Inside its chunk the sums run over the threads' consecutive tokens.
template <int E>
__device__ int draw(const Left& f, int vocab, const double* sums, int n_chunks, double u, u64_t* red, int* sh, double* p_out) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __syncthreads();
    // every wave scans the chunks' sums: lane i holds those of 2 i and 2 i + 1
    static_assert(kMaxChunks <= 128, "two chunks a lane");
    const double s0 = 2 * lane < n_chunks ? sums[2 * lane] : 0.0, s1 = 2 * lane + 1 < n_chunks ? sums[2 * lane + 1] : 0.0;
    const double run = wave_scan(s0 + s1), total = lane_value(run, 63);
    if (!(total > 0.0)) return -1;
    const double target = u * total, b1 = run - s1;  // the sum up to the lane's second chunk
    // the first chunk with anything left whose running sum passes the target, else the last with anything left
    const u64_t over0 = __ballot(s0 > 0.0 && b1 > target), over1 = __ballot(s1 > 0.0 && run > target);
    const u64_t any0 = __ballot(s0 > 0.0), any1 = __ballot(s1 > 0.0);
    int chunk;
    if (over0 | over1) {
        const int i = __ffsll((unsigned long long)(over0 | over1)) - 1;
        chunk = 2 * i + (over0 >> i & 1 ? 0 : 1);
    } else {
        const int i = 63 - __clzll(any0 | any1);
        chunk = 2 * i + (any1 >> i & 1 ? 1 : 0);
    }
    chunk = __builtin_amdgcn_readfirstlane(chunk);
    const double before = lane_value(chunk & 1 ? b1 : b1 - s0, chunk >> 1);
    const int x0 = chunk * kChunk, n = min(kChunk, vocab - x0), at = E * tid;
    float l[E], q[E];
    double w[E], mine = 0.0;
    take<E, true>(f.l + x0, n, NAN, l);
    if (f.q) take<E, true>(f.q + x0, n, 0.0f, q);
#pragma unroll
    for (int k = 0; k < E; ++k) {
        w[k] = kept(f.r, l[k], x0 + at + k) ? f.of_kept(l[k], f.q ? q[k] : 0.0f, x0 + at + k) : 0.0;
        mine += w[k];
    }
    const double up = wave_scan(mine);
    if (lane == 63) ((double*)red)[wave] = up;
    if (tid == 0) {
        sh[0] = INT_MAX;
        sh[1] = -1;
    }
    __syncthreads();
    double cum = before + up - mine;
#pragma unroll
    for (int i = 0; i < kVerWaves; ++i) cum += i < wave ? ((double*)red)[i] : 0.0;
    int hit = INT_MAX, last = -1;
#pragma unroll
    for (int k = 0; k < E; ++k) {
        cum += w[k];
        if (w[k] > 0.0) {
            if (cum > target) hit = min(hit, at + k);
            last = at + k;
        }
    }
    // a wave's first hit is its first such lane's, its last token its last such lane's
    const u64_t hits = __ballot(hit != INT_MAX), lasts = __ballot(last >= 0);
    if (hits && lane == __ffsll((unsigned long long)hits) - 1) atomicMin(&sh[0], hit);
    if (lasts && lane == 63 - __clzll(lasts)) atomicMax(&sh[1], last);
    __syncthreads();
    const int tok = sh[0] == INT_MAX ? sh[1] : sh[0];  // past the sums' rounding: the last token that is left
#pragma unroll
    for (int k = 0; k < E; ++k)
        if (at + k == tok) *p_out = weight(l[k], f.r.mx, f.c) * f.r.inv_z;
    __syncthreads();
    return x0 + tok;
}

__device__ __forceinline__ void put_next(const VerifyArgs& a, int tok, double p) {
    if (threadIdx.x) return;
    a.result[1] = tok;
    if (a.probs) a.probs[0] = (float)p;
}

// ---------------------------------------------------------------- the walk
constexpr int kWalkEach = kChunk / kVerThreads;
__global__ __launch_bounds__(kVerThreads) void k_ver_walk(const VerifyArgs a, const VerWork wk) {
    __shared__ VerRow rows[kTreeMax];
    __shared__ __align__(16) int parent[kTreeMax];
    __shared__ int token[kTreeMax], first[kTreeMax], gone[kTreeMax];
    __shared__ float gone_l[kTreeMax];
    __shared__ double pc[kTreeMax], qc[kTreeMax], draws[kTreeMax], s1[kTreeMax], sums[kMaxChunks];
    __shared__ u64_t red[kVerWaves];
    __shared__ int sh[4];
    __shared__ double p_next;
    const int tid = threadIdx.x, n = a.n_tree, V = a.vocab;
    const bool greedy = a.temperature <= 0.0f, cut = !greedy && a.top_p < 1.0f, sampled = a.draft && !greedy;
    const bool leader = blockIdx.x == 0;  // writes what all workgroups find alike
    const double c = greedy ? 0.0 : kLog2e64 / (double)a.temperature;
    float lt = NAN, qt = 0.0f;
    if (tid < kTreeMax) parent[tid] = -1;
    if (tid < n) {
        // a parent that does not come before its child, or a token that is none: never accepted
        int up = tid ? a.parent[tid] : -1;
        const int x = a.tokens[tid];
        if (up < 0 || up >= tid) up = -1;
        parent[tid] = up;
        token[tid] = x;
        first[tid] = INT_MAX;
        draws[tid] = (double)a.draws[tid];
        if (up >= 0 && x >= 0 && x < V) {
            lt = a.logits[(int64_t)up * a.ld + x];
            if (sampled) qt = a.draft[(int64_t)up * a.ld_draft + x];
        }
    }
    if (tid == 0) sh[2] = 0;
    for (int i = tid >> 4; i < n; i += kVerThreads / 16) {
        const VerRow r = cut ? wk.rows[i] : row_of_chunks(a, wk, i);
        if ((tid & 15) == 0) rows[i] = r;
        if (sampled) {
            double s = 0.0;
            for (int k = tid & 15; k < wk.n_chunks; k += 16) s += wk.round[(int64_t)i * wk.n_chunks + k];
            s = row_sum(s);
            if ((tid & 15) == 0) s1[i] = s;  // of rows with fewer than two children: not written, and not used
        }
    }
    __syncthreads();
    // the children's probabilities; of siblings with one token the first has it (drafts without distributions)
    const int up = tid < n ? parent[tid] : -1;
    uint32_t elder[kTreeMax / 32];  // elder siblings, a bit a node
    int k = 0;
    if (tid < n) {
        const double p = lt == lt && up >= 0 ? prob(rows[up], lt, token[tid], c) : 0.0;
        bool again = false;
#pragma unroll
        for (int w = 0; w < kTreeMax / 32; ++w) {
            elder[w] = 0;
            if (32 * w >= tid || up < 0) continue;
#pragma unroll
            for (int i = 0; i < 32; i += 4) {
                const int4 q = *(const int4*)&parent[32 * w + i];
                elder[w] |= (uint32_t)(q.x == up) << i | (uint32_t)(q.y == up) << (i + 1) | (uint32_t)(q.z == up) << (i + 2) |
                            (uint32_t)(q.w == up) << (i + 3);
            }
            if (tid < 32 * w + 32) elder[w] &= (1u << (tid - 32 * w)) - 1;
            k += __popc(elder[w]);
            for (uint32_t e = elder[w]; e; e &= e - 1) again |= token[32 * w + __ffs((int)e) - 1] == token[tid];
        }
        pc[tid] = sampled || !again ? p : 0.0;
        qc[tid] = (double)qt;
        if (tid && a.probs && leader) a.probs[tid] = (float)p;
    }
    __syncthreads();
    // every child's test, as if its parent were on the path and its elder siblings rejected
    if (up >= 0) {
        const double p = pc[tid];
        bool take = p > 0.0;
        if (sampled) {
            const double left = p - (k ? 1.0 : 0.0) * qc[tid];
            take = k < 2 && left > 0.0 && draws[tid] * qc[tid] * (k ? s1[up] : 1.0) < left;
        } else if (!greedy) {
            double before = 0.0;
#pragma unroll
            for (int w = 0; w < kTreeMax / 32; ++w)
                for (uint32_t e = elder[w]; e; e &= e - 1) before += pc[32 * w + __ffs((int)e) - 1];
            take = take && draws[tid] * (1.0 - before) < p;
        }
        if (take) atomicMin(&first[up], tid);
    }
    __syncthreads();
    int at = 0, count = 1;
    if (tid == 0 && leader) a.path[0] = 0;
    double t = 0.0;
    for (;;) {
        int next = first[at];
        t = 0.0;
        if (sampled && next == INT_MAX) {
            // the children past the second, one sum over the row after another
            int kids = 0;
            for (int j = at + 1; j < n; ++j) {
                if (parent[j] != at) continue;
                double S = kids ? s1[at] : 1.0;
                if (kids >= 2) {
                    const Left f = {rows[at], a.logits + (int64_t)at * a.ld, a.draft + (int64_t)at * a.ld_draft, t, c, nullptr, 0};
                    S = left_row_sum<kWalkEach>(f, V, wk.n_chunks, red);
                    const double left = pc[j] - t * qc[j];
                    if (left > 0.0 && draws[j] * qc[j] * S < left) {
                        next = j;
                        break;
                    }
                }
                t += S;
                ++kids;
            }
        }
        if (next == INT_MAX) break;
        at = next;
        if (tid == 0 && leader) a.path[count] = at;
        ++count;
    }
    const VerRow r = rows[at];
    const float* l = a.logits + (int64_t)at * a.ld;
    if (leader) {
        for (int i = count + tid; i < n; i += kVerThreads) a.path[i] = -1;
        if (tid == 0) a.result[0] = count;
    }
    if (greedy) {
        put_next(a, r.arg, 1.0);
        return;
    }
    // the next token, from what is left of row `at`
    if (!sampled && up == at) {
        gone[k] = token[tid];
        gone_l[k] = lt;
        atomicMax(&sh[2], k + 1);
    }
    __syncthreads();
    const int n_gone = sh[2];
    Left f = {r, l, sampled && t > 0.0 ? a.draft + (int64_t)at * a.ld_draft : nullptr, t, c, gone, n_gone};
    auto chunk_sums = [&]() {  // P's own, from k_ver_chunks
        for (int i = tid; i < wk.n_chunks; i += kVerThreads) {
            const VerChunk ch = wk.chunks[(int64_t)at * wk.n_chunks + i];
            sums[i] = ch.sum > 0.0 ? ch.sum * weight(ch.mx, r.mx, c) : 0.0;
        }
        __syncthreads();
    };
    if (cut || sampled) {
        const double mine = left_sum<kWalkEach>(f, V, blockIdx.x, red);
        if (tid == 0) send(&wk.left[blockIdx.x], (u64_t)__double_as_longlong(mine));
        if (!last_of(wk.arrived, wk.n_chunks, &sh[3])) return;
        for (int i = tid; i < wk.n_chunks; i += kVerThreads) sums[i] = __longlong_as_double((long long)receive(&wk.left[i]));
    } else {
        // without the rejected tokens; a chunk that they were nearly all of is summed again
        chunk_sums();
        for (int i = 0; i < n_gone; ++i) {
            const int x = gone[i];
            bool again = x < 0 || x >= V;
            for (int j = 0; j < i; ++j) again |= gone[j] == x;
            if (again) continue;
            const int ch = x / kChunk;
            const double old = sums[ch];
            double now = old - weight(gone_l[i], r.mx, c);
            if (!(now > old * 0x1p-16)) now = left_sum<kWalkEach>(f, V, ch, red);
            __syncthreads();
            if (tid == 0) sums[ch] = now;
            __syncthreads();
        }
    }
    int tok = draw<kWalkEach>(f, V, sums, wk.n_chunks, draws[0], red, sh, &p_next);
    if (tok < 0) {  // nothing is left: from P itself
        f.q = nullptr;
        f.n_gone = 0;
        __syncthreads();
        if (cut) {
            for (int ch = 0; ch < wk.n_chunks; ++ch) {
                const double s = left_sum<kWalkEach>(f, V, ch, red);
                if (tid == 0) sums[ch] = s;
            }
        } else {
            chunk_sums();
        }
        tok = draw<kWalkEach>(f, V, sums, wk.n_chunks, draws[0], red, sh, &p_next);
    }
    put_next(a, tok < 0 ? r.arg : tok, tok < 0 ? 0.0 : p_next);
}

VerWork work_of(int n_tree, int vocab, void* ws, size_t* bytes) {
    VerWork w{};
    w.n_chunks = (vocab + kChunk - 1) / kChunk;
    char* p = (char*)ws;
    auto part = [&](size_t n) {
        char* at = p;
        p += (n + 63) / 64 * 64;
        return at;
    };
    w.arrived = (uint32_t*)part(sizeof(uint32_t));
    const size_t n = (size_t)n_tree, all = n * w.n_chunks;
    w.rows = (VerRow*)part(n * sizeof(VerRow));
    w.cuts = (VerCut*)part(n * sizeof(VerCut));
    w.chunks = (VerChunk*)part(all * sizeof(VerChunk));
    w.round = (double*)part(all * sizeof(double));
    w.n_cuts = (vocab + kCutChunk - 1) / kCutChunk;
    w.mass = (u64_t*)part(n * w.n_cuts * kBins * sizeof(u64_t));
    w.above = (u64_t*)part(n * w.n_cuts * sizeof(u64_t));
    w.list = (u64_t*)part(n * kList * sizeof(u64_t));
    w.left = (u64_t*)part((size_t)w.n_chunks * sizeof(u64_t));
    if (bytes) *bytes = (size_t)(p - (char*)ws);
    return w;
}

}  // namespace

size_t verify_ws_bytes(int n_tree, int vocab) {
    size_t bytes = 0;
    (void)work_of(n_tree, vocab, nullptr, &bytes);
    return bytes;
}

hipError_t launch_verify(const VerifyArgs& a, void* ws, hipStream_t st) {
    const VerWork wk = work_of(a.n_tree, a.vocab, ws, nullptr);
    const bool greedy = a.temperature <= 0.0f, cut = !greedy && a.top_p < 1.0f, sampled = !greedy && a.draft;
    const dim3 grid((unsigned)wk.n_chunks, (unsigned)a.n_tree);
    auto launch = [&](void (*k)(VerifyArgs, VerWork), dim3 g, int threads) {
        return launch_kernel(k, g, dim3(threads), st, a, wk);
    };
    hipError_t e = launch(k_ver_chunks, grid, kBlock);
    const dim3 cuts((unsigned)wk.n_cuts, (unsigned)a.n_tree);
    if (e == hipSuccess && cut) e = launch(k_ver_bins, cuts, kCutThreads);
    if (e == hipSuccess && cut) e = launch(k_ver_cut, cuts, kCutThreads);
    if (e == hipSuccess && sampled) e = launch(k_ver_rounds, grid, kBlock);
    if (e == hipSuccess) e = launch(k_ver_walk, dim3(cut || sampled ? (unsigned)wk.n_chunks : 1u), kVerThreads);
    return e;
}

}  // namespace tfk
