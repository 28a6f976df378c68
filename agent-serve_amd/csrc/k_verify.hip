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
// Arithmetic: a token's weight is e^((l - max) / T). The tests and the draw take it in 64 bits, so
// that a comparison falls as it would with exact numbers unless it is within 1e-7 of its border;
// the rows' sums take 32-bit exponentials (each within 2^-22 or so of its value) added in 64 bits.
// The nucleus adds them as integers, 2^-44 of the largest to one unit: their sums are the same in
// any order, so the atomics that form them do not show.
#include <cfloat>
#include <climits>

#include "dev_common.hpp"
#include "tf_internal.hpp"

namespace tfk {
namespace {

constexpr int kVerThreads = 1024;
constexpr int kVerWaves = kVerThreads / kWave;
constexpr float kLog2e = 1.44269504088896341f;

// One row's distribution: token x with logit l has probability w(l) / z where it is kept, that is
// where its key is above thr, or equal to it with x <= cut; mx is the largest logit.
struct VerRow {
    double z;
    float mx;
    uint32_t thr;
    int32_t cut;
    int32_t arg;  // the first largest logit's index
};

__device__ __forceinline__ uint32_t logit_key(float l) { return (uint32_t)(argmax_key(l, 0) >> 32); }

// 2^x for the row sums. A token equal to the maximum weighs 1 also where both are infinite; one that
// is not below it (NaN) weighs nothing.
__device__ __forceinline__ float weight32(float l, float mx, float c) {
    return l == mx ? 1.0f : (l < mx ? __builtin_amdgcn_exp2f((l - mx) * c) : 0.0f);
}
__device__ __forceinline__ double weight64(float l, float mx, double inv_t) {
    return l == mx ? 1.0 : (l < mx ? exp(((double)l - (double)mx) * inv_t) : 0.0);
}
__device__ __forceinline__ bool kept(const VerRow& r, float l, int x) {
    const uint32_t k = logit_key(l);
    return k > r.thr || (k == r.thr && x <= r.cut);
}
__device__ __forceinline__ double prob64(const VerRow& r, float l, int x, double inv_t) {
    return kept(r, l, x) && r.z > 0.0 ? weight64(l, r.mx, inv_t) / r.z : 0.0;
}

// f(index, value) for the n floats at p, over the workgroup's threads.
template <class F>
__device__ __forceinline__ void each(const float* p, int n, F f) {
    const int tid = threadIdx.x, step = blockDim.x;
    const int head = min(n, (int)((16 - ((uintptr_t)p & 15)) & 15) >> 2), n4 = (n - head) >> 2;
    if (tid < head) f(tid, p[tid]);
    for (int i = tid; i < n4; i += step) {
        const float4 v = gload_f4(p + head + 4 * i);
        f(head + 4 * i, v.x);
        f(head + 4 * i + 1, v.y);
        f(head + 4 * i + 2, v.z);
        f(head + 4 * i + 3, v.w);
    }
    const int tail = head + 4 * n4 + tid;
    if (tail < n) f(tail, p[tail]);
}

// Sums and maxima over the workgroup; every thread gets the result. red: kVerWaves words.
template <class T, class F>
__device__ __forceinline__ T block_fold(T v, T* red, F op) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = op(v, __shfl_xor(v, o));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < (int)(blockDim.x >> 6); ++w) v = op(v, red[w]);
    return v;
}
typedef unsigned long long u64_t;
__device__ __forceinline__ double block_sum(double v, u64_t* red) {
    return block_fold(v, (double*)red, [](double a, double b) { return a + b; });
}
__device__ __forceinline__ u64_t block_max(u64_t v, u64_t* red) {
    return block_fold(v, red, [](u64_t a, u64_t b) { return a > b ? a : b; });
}

// ---------------------------------------------------------------- the nucleus of one row
constexpr int kBins = 2048, kList = 2048;
struct Nucleus {
    u64_t mass[kBins];
    uint32_t count[kBins];
    uint2 list[kList];  // key, index
    u64_t red[kVerWaves];
    u64_t before;       // the mass above the interval
    uint32_t n_list, bin, k_lo, k_hi;
};

__device__ __forceinline__ u64_t weight_fix(float l, float mx, float c) {
    return (u64_t)(weight32(l, mx, c) * 17592186044416.0f);  // 2^44
}

// The bin whose masses reach `target` from s.before on; s.before grows by those above it. One wave.
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
            s.before = at;  // read above by every lane of this wave already
        }
    }
    __syncthreads();
}

// r.thr, r.cut and r.z of the tokens up to the one whose running sum reaches top_p. First the row's
// logits in kBins bins of equal width below the maximum (as far as 24 temperatures, where a token's
// weight is 2^-34 of the largest), then the elements of the bin that the sum ends in: few of them are
// ranked directly; many are binned again by their keys, until few or one key is left.
__device__ void nucleus(const float* p, int n, float c, float top_p, float mn, VerRow& r, Nucleus& s) {
    const int tid = threadIdx.x;
    const float mx = r.mx;
    const float span = fminf(mx - mn, 24.0f * kLog2e / c);
    const float inv = span > 0.0f && span < INFINITY ? (float)kBins / span : 0.0f;
    auto bin_of = [&](float l) {
        const float d = (mx - l) * inv;
        return l == mx ? 0 : (d < (float)(kBins - 1) ? (int)d : kBins - 1);
    };
    for (int i = tid; i < kBins; i += kVerThreads) {
        s.mass[i] = 0;
        s.count[i] = 0;
    }
    if (tid == 0) s.before = 0;
    __syncthreads();
    u64_t part = 0;
    each(p, n, [&](int, float l) {
        if (!(l <= mx)) return;
        const u64_t w = weight_fix(l, mx, c);
        const int b = bin_of(l);
        part += w;
        atomicAdd(&s.mass[b], w);
        atomicAdd(&s.count[b], 1u);
    });
    const u64_t all = block_fold(part, s.red, [](u64_t a, u64_t b) { return a + b; });
    top_p = fmaxf(top_p, 0.0f);
    u64_t target = (u64_t)((double)top_p * (double)all);
    // the exact product may lie above: a token is kept while the sum before it is below top_p
    if ((double)target < (double)top_p * (double)all) ++target;
    target = target < 1 ? 1 : (target > all ? all : target);
    find_bin(s, target);
    const int b0 = s.bin;
    uint32_t in_bin = s.count[b0];
    uint32_t lo = 0, hi = 0xFFFFFFFFu;  // keys of the interval
    auto inside = [&](float l) {
        const uint32_t k = logit_key(l);
        return l <= mx && bin_of(l) == b0 && k >= lo && k <= hi;
    };
    while (in_bin > kList) {
        __syncthreads();
        if (tid == 0) {
            s.k_lo = 0xFFFFFFFFu;
            s.k_hi = 0;
        }
        for (int i = tid; i < kBins; i += kVerThreads) {
            s.mass[i] = 0;
            s.count[i] = 0;
        }
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
        if (lo == hi) break;  // one logit many times over
        int shift = 0;
        while (((hi - lo) >> shift) >= (uint32_t)kBins) ++shift;
        each(p, n, [&](int, float l) {
            if (inside(l)) {
                const int b = (int)((hi - logit_key(l)) >> shift);
                atomicAdd(&s.mass[b], weight_fix(l, mx, c));
                atomicAdd(&s.count[b], 1u);
            }
        });
        find_bin(s, target);
        in_bin = s.count[s.bin];
        const uint32_t top = hi - ((uint32_t)s.bin << shift);
        lo = max(lo, top - min(top, (1u << shift) - 1));
        hi = top;
    }
    __syncthreads();
    if (in_bin > kList) {
        // ties of one logit: the sum reaches the target at the k-th of them, in index order
        u64_t w = 0;
        each(p, n, [&](int, float l) {
            if (inside(l)) w = weight_fix(l, mx, c);
        });
        w = block_max(w, s.red);
        const u64_t before = s.before;
        const u64_t k = (target - before + w - 1) / w;  // w > 0: the masses reach the target here
        // its index: count, then halve the range of indices
        int a = 0, b = n - 1;
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
        r.z = (double)(before + k * w) / 17592186044416.0;
        return;
    }
    if (tid == 0) s.n_list = 0;
    __syncthreads();
    each(p, n, [&](int x, float l) {
        if (inside(l)) {
            const uint32_t at = atomicAdd(&s.n_list, 1u);
            s.list[at] = make_uint2(__float_as_uint(l), (uint32_t)x);
        }
    });
    __syncthreads();
    const int m = (int)s.n_list;
    const u64_t before = s.before;
    u64_t end = 0;
    for (int i = tid; i < m; i += kVerThreads) {
        const float l = __uint_as_float(s.list[i].x);
        const uint32_t k = logit_key(l), x = s.list[i].y;
        u64_t sum = before;
        for (int j = 0; j < m; ++j) {
            const float lj = __uint_as_float(s.list[j].x);
            const uint32_t kj = logit_key(lj);
            if (kj > k || (kj == k && s.list[j].y < x)) sum += weight_fix(lj, mx, c);
        }
        const u64_t with = sum + weight_fix(l, mx, c);
        if (sum < target && with >= target) {
            s.k_lo = k;
            s.k_hi = x;
            end = with;
        }
    }
    end = block_max(end, s.red);
    r.thr = s.k_lo;
    r.cut = (int32_t)s.k_hi;
    r.z = (double)end / 17592186044416.0;
}

// A workgroup per row: its maximum, its kept tokens and their sum.
__global__ __launch_bounds__(kVerThreads) void k_ver_rows(const VerifyArgs a, VerRow* rows) {
    __shared__ Nucleus s;
    const int i = blockIdx.x, n = a.vocab;
    const float* p = a.logits + (int64_t)i * a.ld;
    u64_t best = 0;
    float mn = INFINITY;
    each(p, n, [&](int x, float l) {
        if (l == l) {
            const u64_t k = argmax_key(l, x);
            best = k > best ? k : best;
            if (l > -INFINITY) mn = fminf(mn, l);
        }
    });
    best = block_max(best, s.red);
    mn = block_fold(mn, (float*)s.red, [](float x, float y) { return fminf(x, y); });
    VerRow r;
    r.arg = best ? (int32_t)(0xFFFFFFFFu - (uint32_t)best) : 0;
    r.mx = best ? p[r.arg] : -INFINITY;
    r.thr = 0;
    r.cut = INT_MAX;
    r.z = best ? 1.0 : 0.0;
    if (a.temperature <= 0.0f) {
        r.thr = logit_key(r.mx);
        r.cut = r.arg;
    } else if (best) {
        const float c = kLog2e / a.temperature;
        if (a.top_p < 1.0f) {
            nucleus(p, n, c, a.top_p, mn, r, s);
        } else {
            double z = 0.0;
            each(p, n, [&](int, float l) { z += (double)weight32(l, r.mx, c); });
            r.z = block_sum(z, s.red);
        }
    }
    if (threadIdx.x == 0) rows[i] = r;
}

// One workgroup: the children's tests, the walk, and the draw of the next token.
__global__ __launch_bounds__(kVerThreads) void k_ver_walk(const VerifyArgs a, const VerRow* rows) {
    __shared__ int parent[kTreeMax], token[kTreeMax];
    __shared__ double pc[kTreeMax];
    __shared__ u64_t red[kVerWaves];
    __shared__ double wave_total[kVerWaves];
    __shared__ int found[kVerWaves], last_pos[kVerWaves];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n_tree, V = a.vocab;
    const bool greedy = a.temperature <= 0.0f;
    const double inv_t = greedy ? 0.0 : 1.0 / (double)a.temperature;
    if (tid < n) {
        // a parent that does not come before its child, or a token that is none: never accepted
        int up = tid ? a.parent[tid] : -1;
        const int x = a.tokens[tid];
        if (up < 0 || up >= tid) up = -1;
        parent[tid] = up;
        token[tid] = x;
        double p = 0.0;
        if (up >= 0 && x >= 0 && x < V) p = prob64(rows[up], a.logits[(int64_t)up * a.ld + x], x, inv_t);
        pc[tid] = p;
        if (tid && a.probs) a.probs[tid] = (float)p;
    }
    __syncthreads();
    int at = 0, count = 1;
    if (tid == 0) a.path[0] = 0;
    double t = 0.0, S = 1.0;
    for (;;) {
        const VerRow r = rows[at];
        const float* lp = a.logits + (int64_t)at * a.ld;
        const float* qp = a.draft ? a.draft + (int64_t)at * a.ld_draft : nullptr;
        t = 0.0;
        S = 1.0;
        int next = -1;
        double gone = 0.0;
        for (int j = at + 1; j < n && next < 0; ++j) {
            if (parent[j] != at) continue;
            const int x = token[j];
            if (greedy) {
                if (pc[j] > 0.0) next = j;
                continue;
            }
            if (!qp) {
                bool again = false;
                for (int k = at + 1; k < j; ++k) again |= parent[k] == at && token[k] == x;
                const double p = again ? 0.0 : pc[j];
                if (p > 0.0 && (double)a.draws[j] * (1.0 - gone) < p) next = j;
                gone += p;
                continue;
            }
            const double q = x >= 0 && x < V ? (double)qp[x] : 0.0;
            const double left = pc[j] - t * q;
            if (left > 0.0 && (double)a.draws[j] * q * S < left) {
                next = j;
                continue;
            }
            t += S;
            double sum = 0.0;
            each(lp, V, [&](int y, float l) { sum += fmax(prob64(r, l, y, inv_t) - t * (double)qp[y], 0.0); });
            S = block_sum(sum, red);
        }
        if (next < 0) break;
        at = next;
        if (tid == 0) a.path[count] = at;
        ++count;
    }
    for (int i = count + tid; i < n; i += kVerThreads) a.path[i] = -1;
    // the next token, from what is left of row `at`: P without its children's tokens, or max(P - t Q, 0)
    const VerRow r = rows[at];
    const float* lp = a.logits + (int64_t)at * a.ld;
    const float* qp = a.draft && t > 0.0 ? a.draft + (int64_t)at * a.ld_draft : nullptr;
    int tok = r.arg;
    if (!greedy) {
        const int each_wave = (V + kVerWaves - 1) / kVerWaves, x0 = wave * each_wave, x1 = min(V, x0 + each_wave);
        for (int whole = 0; whole < 2; ++whole) {  // where nothing is left, from P itself
            auto weight = [&](int x) {
                double w = prob64(r, lp[x], x, inv_t);
                if (whole) return w;
                if (qp) return fmax(w - t * (double)qp[x], 0.0);
                if (!a.draft)
                    for (int j = at + 1; j < n; ++j)
                        if (parent[j] == at && token[j] == x) w = 0.0;
                return w;
            };
            double sum = 0.0;
            for (int x = x0 + lane; x < x1; x += 64) sum += weight(x);
            sum = wave_sum_d(sum);
            __syncthreads();
            if (lane == 0) wave_total[wave] = sum;
            __syncthreads();
            double total = 0.0, run = 0.0;
            for (int w = 0; w < kVerWaves; ++w) {
                if (w == wave) run = total;
                total += wave_total[w];
            }
            if (!(total > 0.0)) continue;
            const double target = (double)a.draws[0] * total;
            int hit = INT_MAX, last = -1;
            for (int x = x0; x < x1; x += 64) {
                const double w = x + lane < x1 ? weight(x + lane) : 0.0;
                double inc = w;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const double up = __shfl_up(inc, o);
                    if (lane >= o) inc += up;
                }
                const u64_t over = __ballot(w > 0.0 && run + inc > target), pos = __ballot(w > 0.0);
                if (pos) last = x + 63 - __clzll(pos);
                if (over) {
                    hit = x + __ffsll((unsigned long long)over) - 1;
                    break;
                }
                run += __shfl(inc, 63);
            }
            if (lane == 0) {
                found[wave] = hit;
                last_pos[wave] = last;
            }
            __syncthreads();
            tok = INT_MAX;
            int end = 0;
            for (int w = 0; w < kVerWaves; ++w) {
                tok = min(tok, found[w]);
                end = max(end, last_pos[w]);
            }
            if (tok == INT_MAX) tok = end;  // the draw is past the sums' rounding
            break;
        }
    }
    if (tid == 0) {
        a.result[0] = count;
        a.result[1] = tok;
        if (a.probs) a.probs[0] = (float)prob64(r, lp[tok], tok, inv_t);
    }
}

}  // namespace

size_t verify_ws_bytes(int n_tree, int) { return (size_t)n_tree * sizeof(VerRow); }

hipError_t launch_verify(const VerifyArgs& a, void* ws, hipStream_t st) {
    VerRow* rows = (VerRow*)ws;
    hipLaunchKernelGGL(k_ver_rows, dim3((unsigned)a.n_tree), dim3(kVerThreads), 0, st, a, rows);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_ver_walk, dim3(1), dim3(kVerThreads), 0, st, a, rows);
    return hipGetLastError();
}

}  // namespace tfk
