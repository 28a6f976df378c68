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
// thousands. At 16 operations a logit that costs less than reading the logits does.
//
//   k_ver_chunks   a workgroup per row and 4096 logits: maximum, its index, sum of weights
//   k_ver_nucleus  (instead, where top_p cuts) a workgroup per row: the kept tokens and their sum
//   k_ver_rounds   (drafts with distributions) S_1 of the rows with two or more children
//   k_ver_walk     one workgroup: every child's test at once, the path by its first accepted children,
//                  and the draw where the chunks' sums serve it
//   k_ver_draw     (else) the sums of what is left of the last row, and the draw by the workgroup that
//                  ends last
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
constexpr double kLog2e64 = 1.4426950408889634;

// Of one chunk of a row: its largest logit, that one's first index, and the weights' sum, the largest's 1.
struct VerChunk {
    double sum;
    float mx;
    int32_t arg;
};
// One row's distribution: token x with logit l has probability w(l) / z where it is kept, that is
// where its key is above thr, or equal to it with x <= cut; mx is the largest logit, first at arg.
struct VerRow {
    double z;
    float mx;
    uint32_t thr;
    int32_t cut;
    int32_t arg;
};
// What the draw takes from: row `at`, P without its children's tokens (drafts without distributions)
// or max(P - t Q, 0).
struct VerState {
    double t;
    int32_t at;
    uint32_t arrived; // workgroups of k_ver_draw that have their sums
};
struct VerWork {
    VerState* state;
    VerRow* rows;       // [n]
    VerChunk* chunks;   // [n][chunks a row]
    double* round;      // [n][chunks a row]: k_ver_rounds
    u64_t* left;        // [chunks a row]: k_ver_draw's sums (doubles)
    int n_chunks;
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
__device__ __forceinline__ bool kept(const VerRow& r, float l, int x) {
    const uint32_t k = logit_key(l);
    return k > r.thr || (k == r.thr && x <= r.cut);
}
__device__ __forceinline__ double prob(const VerRow& r, float l, int x, double c) {
    return kept(r, l, x) && r.z > 0.0 ? weight(l, r.mx, c) / r.z : 0.0;
}

// Folds over the workgroup; every thread gets the result. red: a word for each wave.
template <class T, class F>
__device__ __forceinline__ T block_fold(T v, u64_t* red, F op) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) ((T*)red)[threadIdx.x >> 6] = v;
    __syncthreads();
    v = ((T*)red)[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v = op(v, ((T*)red)[w]);
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
    return RUN ? E * tid + k : 4 * (tid + k / 4 * (kChunk / E)) + k % 4;
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

// Grid (chunk, row), 256 threads of 16 logits. The first workgroup readies the state.
constexpr int kChunkEach = kChunk / kBlock;
__global__ __launch_bounds__(kBlock) void k_ver_chunks(const VerifyArgs a, const VerWork wk) {
    __shared__ u64_t red[kWavesPerBlock];
    const int row = blockIdx.y, x0 = blockIdx.x * kChunk, n = min(kChunk, a.vocab - x0);
    if (row == 0 && blockIdx.x == 0 && threadIdx.x == 0) wk.state->arrived = 0;
    float v[kChunkEach];
    take<kChunkEach, false>(a.logits + (int64_t)row * a.ld + x0, n, NAN, v);
    u64_t best = 0;
#pragma unroll
    for (int k = 0; k < kChunkEach; ++k)
        if (v[k] == v[k]) best = max(best, argmax_key(v[k], x0 + place<kChunkEach, false>(k)));
    best = block_max(best, red);
    const int arg = best ? (int)(0xFFFFFFFFu - (uint32_t)best) : 0;
    const uint32_t key = (uint32_t)(best >> 32);
    const float mx = best ? __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key) : -INFINITY;
    double sum = 0.0;
    if (a.temperature > 0.0f) {
        const double c = kLog2e64 / (double)a.temperature;
#pragma unroll
        for (int k = 0; k < kChunkEach; ++k) sum += weight(v[k], mx, c);
        sum = block_sum(sum, red);
    }
    if (threadIdx.x == 0) wk.chunks[(int64_t)row * wk.n_chunks + blockIdx.x] = {sum, mx, arg};
}

// ---------------------------------------------------------------- the nucleus
// The sums that find where it ends are of 32-bit weights (the last token's place is off only where the
// running sum comes within 1e-7 of top_p), as integers of 2^-44 of the largest: integers add up to the
// same in any order, so the atomics do not show. What is kept is summed in 64 bits.
constexpr int kBins = 2048, kList = 2048;
struct Nucleus {
    u64_t mass[kBins];
    uint2 list[kList];  // logit, index
    u64_t red[kVerWaves];
    u64_t before;       // the mass above the interval
    uint32_t n_list, bin, k_lo, k_hi;
};

__device__ __forceinline__ u64_t weight_fix(float l, float mx, float c) {
    const float w = l == mx ? 1.0f : __builtin_amdgcn_exp2f((l - mx) * c);
    return (u64_t)(w * 17592186044416.0f);  // 2^44
}

// The bin whose masses reach `target` from s.before on; s.before grows by those above it.
__device__ void find_bin(Nucleus& s, u64_t target) {
    const int tid = threadIdx.x;
    __syncthreads();
    if (tid < 64) {
        constexpr int kEach = kBins / 64;
        u64_t sum = 0;
        for (int i = 0; i < kEach; ++i) sum += s.mass[tid * kEach + i];
        u64_t run = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const u64_t up = __shfl_up(run, o);
            if (tid >= o) run += up;
        }
        u64_t at = s.before + run - sum;
        if (at < target && at + sum >= target) {
            int b = tid * kEach;
            while (at + s.mass[b] < target) at += s.mass[b++];
            s.bin = b;
            s.before = at;  // every lane of this wave has read it
        }
    }
    __syncthreads();
}

// r.thr, r.cut and r.z of the tokens up to the one whose running sum reaches top_p. First the row's
// logits in kBins bins of equal width below the maximum (as far as 24 temperatures, where a token's
// weight is 2^-34 of the largest), then the elements of the bin that the sum ends in: few of them are
// ranked directly; many are binned again by their keys, until few or one key is left.
__device__ void nucleus(const float* p, int n, double c64, float top_p, float mn, VerRow& r, Nucleus& s) {
    const int tid = threadIdx.x;
    const float mx = r.mx, c = (float)c64;
    const float span = fminf(mx - mn, 24.0f * (float)kLog2e64 / c);
    const float inv = span > 0.0f && span < INFINITY ? (float)kBins / span : 0.0f;
    auto bin_of = [&](float l) {
        const float d = (mx - l) * inv;
        return l == mx ? 0 : (d < (float)(kBins - 1) ? (int)d : kBins - 1);
    };
    for (int i = tid; i < kBins; i += kVerThreads) s.mass[i] = 0;
    if (tid == 0) s.before = 0;
    __syncthreads();
    u64_t part = 0, low = 0;
    each(p, n, [&](int, float l) {
        if (!(l <= mx)) return;
        const u64_t w = weight_fix(l, mx, c);
        const int b = bin_of(l);
        part += w;
        if (b == kBins - 1)
            low += w;
        else
            atomicAdd(&s.mass[b], w);
    });
    atomicAdd(&s.mass[kBins - 1], low);
    const u64_t all = block_fold(part, s.red, [](u64_t a, u64_t b) { return a + b; });
    top_p = fmaxf(top_p, 0.0f);
    u64_t target = (u64_t)((double)top_p * (double)all);
    // a token is kept while the sum before it is below top_p
    if ((double)target < (double)top_p * (double)all) ++target;
    target = target < 1 ? 1 : (target > all ? all : target);
    find_bin(s, target);
    const int b0 = s.bin;
    uint32_t lo = 0, hi = 0xFFFFFFFFu;  // keys of the interval
    auto inside = [&](float l) {
        const uint32_t k = logit_key(l);
        return l <= mx && bin_of(l) == b0 && k >= lo && k <= hi;
    };
    auto above = [&](float l) { return l <= mx && (bin_of(l) < b0 || (bin_of(l) == b0 && logit_key(l) > hi)); };
    bool one_key = false;
    double z = 0.0;
    // the interval's elements, if they fit, and the weight above it
    auto gather = [&]() {
        __syncthreads();
        if (tid == 0) s.n_list = 0;
        __syncthreads();
        z = 0.0;
        each(p, n, [&](int x, float l) {
            if (inside(l)) {
                const uint32_t at = atomicAdd(&s.n_list, 1u);
                if (at < kList) s.list[at] = make_uint2(__float_as_uint(l), (uint32_t)x);
            }
            if (above(l)) z += weight(l, mx, c64);
        });
        __syncthreads();
        return s.n_list;
    };
    while (gather() > kList) {
        __syncthreads();
        if (tid == 0) {
            s.k_lo = 0xFFFFFFFFu;
            s.k_hi = 0;
        }
        for (int i = tid; i < kBins; i += kVerThreads) s.mass[i] = 0;
        __syncthreads();
        uint32_t a = 0xFFFFFFFFu, b = 0;
        each(p, n, [&](int, float l) {
            if (inside(l)) {
                const uint32_t k = logit_key(l);
                a = min(a, k);
                b = max(b, k);
            }
        });
        atomicMin(&s.k_lo, a);
        atomicMax(&s.k_hi, b);
        __syncthreads();
        lo = s.k_lo;
        hi = s.k_hi;
        if (lo == hi) {  // one logit many times over
            one_key = true;
            break;
        }
        int shift = 0;
        while (((hi - lo) >> shift) >= (uint32_t)kBins) ++shift;
        each(p, n, [&](int, float l) {
            if (inside(l)) atomicAdd(&s.mass[(hi - logit_key(l)) >> shift], weight_fix(l, mx, c));
        });
        find_bin(s, target);
        const uint32_t top = hi - (s.bin << shift);
        lo = max(lo, top - min(top, (1u << shift) - 1));
        hi = top;
    }
    z = block_sum(z, s.red);
    const u64_t before = s.before;
    if (one_key) {
        // the sum reaches the target at the k-th of them, in index order
        const uint32_t bits = lo & 0x80000000u ? lo & 0x7FFFFFFFu : ~lo;
        const float l1 = __uint_as_float(bits);
        const u64_t w = weight_fix(l1, mx, c), k = (target - before + w - 1) / w;  // w > 0: the target lies here
        int a = 0, b = n - 1;  // its index: halve the range by counts
        while (a < b) {
            const int mid = a + (b - a) / 2;
            u64_t c0 = 0;
            each(p, n, [&](int x, float l) { c0 += x <= mid && inside(l) ? 1 : 0; });
            c0 = block_fold(c0, s.red, [](u64_t x, u64_t y) { return x + y; });
            if (c0 >= k)
                b = mid;
            else
                a = mid + 1;
        }
        r.thr = lo;
        r.cut = a;
        r.z = z + (double)k * weight(l1, mx, c64);
        return;
    }
    const int m = (int)s.n_list;
    for (int i = tid; i < m; i += kVerThreads) {
        const float l = __uint_as_float(s.list[i].x);
        const uint32_t k = logit_key(l), x = s.list[i].y;
        u64_t sum = before;
        for (int j = 0; j < m; ++j) {
            const float lj = __uint_as_float(s.list[j].x);
            const uint32_t kj = logit_key(lj);
            if (kj > k || (kj == k && s.list[j].y < x)) sum += weight_fix(lj, mx, c);
        }
        if (sum < target && sum + weight_fix(l, mx, c) >= target) {
            s.k_lo = k;
            s.k_hi = x;
        }
    }
    __syncthreads();
    r.thr = s.k_lo;
    r.cut = (int32_t)s.k_hi;
    double in = 0.0;
    for (int i = tid; i < m; i += kVerThreads) {
        const float l = __uint_as_float(s.list[i].x);
        if (kept(r, l, (int)s.list[i].y)) in += weight(l, mx, c64);
    }
    r.z = z + block_sum(in, s.red);
}

__global__ __launch_bounds__(kVerThreads) void k_ver_nucleus(const VerifyArgs a, const VerWork wk) {
    __shared__ Nucleus s;
    const int i = blockIdx.x, n = a.vocab;
    const float* p = a.logits + (int64_t)i * a.ld;
    if (i == 0 && threadIdx.x == 0) wk.state->arrived = 0;
    u64_t best = 0;
    float mn = INFINITY;
    each(p, n, [&](int x, float l) {
        if (l == l) {
            best = max(best, argmax_key(l, x));
            if (l > -INFINITY) mn = fminf(mn, l);
        }
    });
    best = block_max(best, s.red);
    mn = block_fold(mn, s.red, [](float x, float y) { return fminf(x, y); });
    VerRow r;
    r.arg = best ? (int32_t)(0xFFFFFFFFu - (uint32_t)best) : 0;
    r.mx = best ? p[r.arg] : -INFINITY;
    r.thr = 0;
    r.cut = INT_MAX;
    r.z = 0.0;
    if (best) nucleus(p, n, kLog2e64 / (double)a.temperature, a.top_p, mn, r, s);
    if (threadIdx.x == 0) wk.rows[i] = r;
}

// A row from its chunks, by one wave (every lane gets it).
__device__ __forceinline__ VerRow row_of_chunks(const VerifyArgs& a, const VerWork& wk, int row) {
    const int lane = threadIdx.x & 63;
    const VerChunk* ch = wk.chunks + (int64_t)row * wk.n_chunks;
    constexpr int kEach = (kMaxChunks + 63) / 64;
    VerChunk v[kEach];
    u64_t best = 0;
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
        const bool on = lane + 64 * k < wk.n_chunks;
        v[k] = on ? ch[lane + 64 * k] : VerChunk{0.0, -INFINITY, INT_MAX};
        if (on) best = max(best, argmax_key(v[k].mx, v[k].arg));
    }
    best = wave_max_u64(best);
    VerRow r;
    r.arg = (int32_t)(0xFFFFFFFFu - (uint32_t)best);
    const uint32_t key = (uint32_t)(best >> 32);
    r.mx = __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
    r.thr = 0;
    r.cut = INT_MAX;
    r.z = 1.0;
    if (a.temperature <= 0.0f) {
        r.thr = key;
        r.cut = r.arg;
    } else {
        const double c = kLog2e64 / (double)a.temperature;
        double z = 0.0;
#pragma unroll
        for (int k = 0; k < kEach; ++k)
            if (v[k].sum > 0.0) z += v[k].sum * weight(v[k].mx, r.mx, c);
        r.z = wave_sum_d(z);
    }
    return r;
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
    __device__ double operator()(float lx, float qx, int x) const {
        if (!kept(r, lx, x)) return 0.0;
        const double w = weight(lx, r.mx, c);
        if (q) return r.z > 0.0 ? fmax(w / r.z - t * (double)qx, 0.0) : 0.0;
        for (int i = 0; i < n_gone; ++i)
            if (gone[i] == x) return 0.0;
        return w;
    }
};

// The sum of a chunk of it, over the workgroup.
template <int E>
__device__ __forceinline__ double left_sum(const Left& f, int vocab, int chunk, u64_t* red) {
    const int x0 = chunk * kChunk, n = min(kChunk, vocab - x0);
    float l[E], q[E];
    take<E, false>(f.l + x0, n, NAN, l);
    if (f.q) take<E, false>(f.q + x0, n, 0.0f, q);
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < E; ++k) sum += f(l[k], f.q ? q[k] : 0.0f, x0 + place<E, false>(k));
    return block_sum(sum, red);
}

// The first token at which the running sum exceeds u times the total, from the chunks' sums (LDS). -1 where
// nothing is left. Inside its chunk the sums run over the threads' consecutive tokens.
template <int E>
__device__ int draw(const Left& f, int vocab, const double* sums, int n_chunks, double u, u64_t* red, int* sh) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __syncthreads();
    double total = 0.0, before = 0.0;
    for (int i = 0; i < n_chunks; ++i) total += sums[i];
    if (!(total > 0.0)) return -1;
    const double target = u * total;
    int chunk = -1;
    double run = 0.0;
    for (int i = 0; i < n_chunks; ++i) {
        if (sums[i] > 0.0 && (chunk < 0 || run <= target)) {  // up to the first that passes it, else the last
            chunk = i;
            before = run;
        }
        run += sums[i];
    }
    const int x0 = chunk * kChunk, n = min(kChunk, vocab - x0), at = E * tid;
    float l[E], q[E];
    double w[E], mine = 0.0;
    take<E, true>(f.l + x0, n, NAN, l);
    if (f.q) take<E, true>(f.q + x0, n, 0.0f, q);
#pragma unroll
    for (int k = 0; k < E; ++k) {
        w[k] = f(l[k], f.q ? q[k] : 0.0f, x0 + at + k);
        mine += w[k];
    }
    double up = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const double x = __shfl_up(up, o);
        if (lane >= o) up += x;
    }
    if (lane == 63) ((double*)red)[wave] = up;
    if (tid == 0) {
        sh[0] = INT_MAX;
        sh[1] = -1;
    }
    __syncthreads();
    double cum = before + up - mine;
    for (int i = 0; i < wave; ++i) cum += ((double*)red)[i];
    int hit = INT_MAX, last = -1;
#pragma unroll
    for (int k = 0; k < E; ++k) {
        cum += w[k];
        if (w[k] > 0.0) {
            if (cum > target) hit = min(hit, at + k);
            last = at + k;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        hit = min(hit, __shfl_xor(hit, o));
        last = max(last, __shfl_xor(last, o));
    }
    if (lane == 0) {
        atomicMin(&sh[0], hit);
        atomicMax(&sh[1], last);
    }
    __syncthreads();
    return x0 + (sh[0] == INT_MAX ? sh[1] : sh[0]);  // past the sums' rounding: the last token that is left
}

__device__ __forceinline__ void put_next(const VerifyArgs& a, const VerRow& r, const float* l, int tok, double c) {
    if (threadIdx.x) return;
    a.result[1] = tok;
    if (a.probs) a.probs[0] = (float)(a.temperature <= 0.0f ? 1.0 : prob(r, l[tok], tok, c));
}

// ---------------------------------------------------------------- the walk
__global__ __launch_bounds__(kVerThreads) void k_ver_walk(const VerifyArgs a, const VerWork wk) {
    __shared__ VerRow rows[kTreeMax];
    __shared__ int parent[kTreeMax], token[kTreeMax], first[kTreeMax], gone[kTreeMax];
    __shared__ double pc[kTreeMax], qc[kTreeMax], draws[kTreeMax], s1[kTreeMax], sums[kMaxChunks];
    __shared__ u64_t red[kVerWaves];
    __shared__ int sh[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n_tree, V = a.vocab;
    const bool greedy = a.temperature <= 0.0f, cut = !greedy && a.top_p < 1.0f;
    const double c = greedy ? 0.0 : kLog2e64 / (double)a.temperature;
    float lt = 0.0f, qt = 0.0f;
    if (tid < n) {
        // a parent that does not come before its child, or a token that is none: never accepted
        int up = tid ? a.parent[tid] : -1;
        const int x = a.tokens[tid];
        if (up < 0 || up >= tid) up = -1;
        parent[tid] = up;
        token[tid] = x;
        first[tid] = INT_MAX;
        draws[tid] = (double)a.draws[tid];
        const bool known = up >= 0 && x >= 0 && x < V;
        lt = known ? a.logits[(int64_t)up * a.ld + x] : NAN;
        qt = known && a.draft ? a.draft[(int64_t)up * a.ld_draft + x] : 0.0f;
    }
    for (int i = wave; i < n; i += kVerWaves) {
        const VerRow r = cut ? wk.rows[i] : row_of_chunks(a, wk, i);
        if (lane == 0) rows[i] = r;
        if (a.draft && !greedy) {
            double s = 0.0;
            for (int k = lane; k < wk.n_chunks; k += 64) s += wk.round[(int64_t)i * wk.n_chunks + k];
            s = wave_sum_d(s);
            if (lane == 0) s1[i] = s;  // of rows with fewer than two children: not written, and not used
        }
    }
    __syncthreads();
    if (tid < n) {
        const int up = parent[tid], x = token[tid];
        const double p = lt == lt && up >= 0 ? prob(rows[up], lt, x, c) : 0.0;
        pc[tid] = p;
        qc[tid] = (double)qt;
        if (tid && a.probs) a.probs[tid] = (float)p;
    }
    __syncthreads();
    // every child's test, as if its parent were on the path and its elder siblings rejected
    const bool sampled = a.draft && !greedy;
    if (tid > 0 && tid < n && parent[tid] >= 0) {
        const int up = parent[tid], x = token[tid];
        int k = 0;
        double before = 0.0, p = pc[tid];
        for (int j = up + 1; j < tid; ++j) {
            if (parent[j] != up) continue;
            ++k;
            if (sampled || greedy) continue;
            bool again = false;  // a token counts once
            for (int i = up + 1; i < j; ++i) again |= parent[i] == up && token[i] == token[j];
            before += again ? 0.0 : pc[j];
            if (token[j] == x) p = 0.0;
        }
        bool take = p > 0.0;
        if (sampled) {
            const double t = k ? 1.0 : 0.0, left = p - t * qc[tid];
            take = k < 2 && left > 0.0 && draws[tid] * qc[tid] * (k ? s1[up] : 1.0) < left;
        } else if (!greedy) {
            take = take && draws[tid] * (1.0 - before) < p;
        }
        if (take) atomicMin(&first[up], tid);
    }
    __syncthreads();
    int at = 0, count = 1;
    if (tid == 0) a.path[0] = 0;
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
                    S = 0.0;
                    for (int ch = 0; ch < wk.n_chunks; ++ch) S += left_sum<kChunk / kVerThreads>(f, V, ch, red);
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
        if (tid == 0) a.path[count] = at;
        ++count;
    }
    for (int i = count + tid; i < n; i += kVerThreads) a.path[i] = -1;
    const VerRow r = rows[at];
    const float* l = a.logits + (int64_t)at * a.ld;
    if (tid == 0) {
        a.result[0] = count;
        wk.state->at = at;
        wk.state->t = t;
    }
    if (greedy) {
        put_next(a, r, l, r.arg, c);
        return;
    }
    if (cut || sampled) return;  // k_ver_draw
    // the chunks' sums without the rejected tokens; a chunk that they were nearly all of is summed again
    if (tid == 0) sh[2] = 0;
    __syncthreads();
    if (tid > at && tid < n && parent[tid] == at) gone[atomicAdd(&sh[2], 1)] = token[tid];
    for (int i = tid; i < wk.n_chunks; i += kVerThreads) {
        const VerChunk ch = wk.chunks[(int64_t)at * wk.n_chunks + i];
        sums[i] = ch.sum > 0.0 ? ch.sum * weight(ch.mx, r.mx, c) : 0.0;
    }
    __syncthreads();
    const int n_gone = sh[2];
    const Left f = {r, l, nullptr, 0.0, c, gone, n_gone};
    for (int i = 0; i < n_gone; ++i) {
        const int x = gone[i];
        bool again = x < 0 || x >= V;
        for (int k = 0; k < i; ++k) again |= gone[k] == x;
        if (again) continue;
        const int ch = x / kChunk;
        const double w = weight(l[x], r.mx, c), old = sums[ch];
        double now = old - w;
        if (!(now > old * 0x1p-16)) now = left_sum<kChunk / kVerThreads>(f, V, ch, red);
        __syncthreads();
        if (tid == 0) sums[ch] = now;
        __syncthreads();
    }
    int tok = draw<kChunk / kVerThreads>(f, V, sums, wk.n_chunks, draws[0], red, sh);
    if (tok < 0) {  // nothing is left: from P itself
        __syncthreads();
        for (int i = tid; i < wk.n_chunks; i += kVerThreads) {
            const VerChunk ch = wk.chunks[(int64_t)at * wk.n_chunks + i];
            sums[i] = ch.sum > 0.0 ? ch.sum * weight(ch.mx, r.mx, c) : 0.0;
        }
        const Left g = {r, l, nullptr, 0.0, c, gone, 0};
        tok = draw<kChunk / kVerThreads>(g, V, sums, wk.n_chunks, draws[0], red, sh);
    }
    put_next(a, r, l, tok < 0 ? r.arg : tok, c);
}

// A workgroup per chunk of the last row; the one that ends last draws. Sums go out and come in past the
// XCDs' caches (agent scope), each before its workgroup is counted.
__global__ __launch_bounds__(kBlock) void k_ver_draw(const VerifyArgs a, const VerWork wk) {
    __shared__ double sums[kMaxChunks];
    __shared__ u64_t red[kWavesPerBlock];
    __shared__ int gone[kTreeMax], sh[4];
    const int tid = threadIdx.x;
    const VerState st = *wk.state;
    const double c = kLog2e64 / (double)a.temperature;
    if (tid == 0) sh[2] = 0;
    __syncthreads();
    if (!a.draft && tid > st.at && tid < a.n_tree && a.parent[tid] == st.at) gone[atomicAdd(&sh[2], 1)] = a.tokens[tid];
    const VerRow r = a.top_p < 1.0f ? wk.rows[st.at] : row_of_chunks(a, wk, st.at);
    __syncthreads();
    Left f = {r, a.logits + (int64_t)st.at * a.ld, a.draft && st.t > 0.0 ? a.draft + (int64_t)st.at * a.ld_draft : nullptr,
              st.t, c, gone, sh[2]};
    const double mine = left_sum<kChunkEach>(f, a.vocab, blockIdx.x, red);
    if (tid == 0) {
        __hip_atomic_store(&wk.left[blockIdx.x], (u64_t)__double_as_longlong(mine), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        sh[3] = (int)__hip_atomic_fetch_add(&wk.state->arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (sh[3] != wk.n_chunks - 1) return;
    for (int i = tid; i < wk.n_chunks; i += kBlock)
        sums[i] = __longlong_as_double((long long)__hip_atomic_load(&wk.left[i], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
    const double u = (double)a.draws[0];
    int tok = draw<kChunkEach>(f, a.vocab, sums, wk.n_chunks, u, red, sh);
    if (tok < 0) {  // nothing is left: from P itself
        f.q = nullptr;
        f.n_gone = 0;
        for (int ch = 0; ch < wk.n_chunks; ++ch) {
            const double s = left_sum<kChunkEach>(f, a.vocab, ch, red);
            __syncthreads();
            if (tid == 0) sums[ch] = s;
        }
        tok = draw<kChunkEach>(f, a.vocab, sums, wk.n_chunks, u, red, sh);
    }
    put_next(a, r, f.l, tok < 0 ? r.arg : tok, c);
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
    w.state = (VerState*)part(sizeof(VerState));
    w.rows = (VerRow*)part((size_t)n_tree * sizeof(VerRow));
    w.chunks = (VerChunk*)part((size_t)n_tree * w.n_chunks * sizeof(VerChunk));
    w.round = (double*)part((size_t)n_tree * w.n_chunks * sizeof(double));
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
    hipError_t e;
    if (cut)
        hipLaunchKernelGGL(k_ver_nucleus, dim3((unsigned)a.n_tree), dim3(kVerThreads), 0, st, a, wk);
    else
        hipLaunchKernelGGL(k_ver_chunks, grid, dim3(kBlock), 0, st, a, wk);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    if (sampled) {
        hipLaunchKernelGGL(k_ver_rounds, grid, dim3(kBlock), 0, st, a, wk);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    hipLaunchKernelGGL(k_ver_walk, dim3(1), dim3(kVerThreads), 0, st, a, wk);
    if ((e = hipGetLastError()) != hipSuccess || !(cut || sampled)) return e;
    hipLaunchKernelGGL(k_ver_draw, dim3((unsigned)wk.n_chunks), dim3(kBlock), 0, st, a, wk);
    return hipGetLastError();
}

}  // namespace tfk
