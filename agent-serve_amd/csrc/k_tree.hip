// Attention of a tree of drafted tokens over a cache, and the move of the accepted nodes' rows.
//
// Node i of the tree has its key and value at cache position n_past + i. Its query sees every
// position below n_past and, of the tree, the nodes whose bit its mask sets:
//   s_j = q_i . k_j / sqrt(hd),   o_i = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   m = max_j s_j
// over the positions j that it sees; a row that sees none is zero.
//
// The n_rep query heads of a kv head times the nodes are the rows of two matrix products over the
// positions, S^T = K Q^T and O^T = V^T P^T, on v_mfma_f32_16x16x32_f16 with an online softmax
// between. fp32 operands enter as fp16 pairs hi + lo (22 significant bits): x y = hi_x hi_y +
// hi_x lo_y + lo_x hi_y, the rest being 2^-22 of the product; fp16 caches are operands as they
// are, so only q and p are pairs. Numbers are scaled by powers of two, exactly taken out again:
//   a query row by its largest element; the 8 or 16 keys that a wave loads by their largest, the values
//   that it does likewise (all in [2^14, 2^15): fp16 pairs hold 22 bits down to 2^-18 of that, and 2^-40 of
//   it below);
//   a weight by 2^14, so that weights down to 2^-18 of the row's largest keep 22 bits.
// The softmax's running reference is the score's maximum in units of log2, rounded up to a whole
// number: rescaling by 2^(old - new) is exact, and it is needed only when the maximum passes one.
//
// A workgroup of NW waves takes 16 QS rows of one kv head a wave and one split of the positions, 32 at a
// time (a step): the step's keys and values lie in LDS in fragment order (a record), and every wave runs its
// rows over them. Half of the threads load, scale and store keys, half values, one step ahead of the
// products; the next step's loads are under way meanwhile. Splits are merged by k_tree_merge; one split
// writes the output itself.
//
// What bounds it. Few positions: the launch and three dependent memory rounds (one query over 7 positions,
// 5.2 us of kernel). A middling call: the same and the merge's launch (8 queries of 32 heads over 1,000 fp32
// positions 6 + 4 us; 37 of 14 heads over 2,029 10.3 + 4.5). Many rows over long caches: the matrix pipes
// and, beside them, the softmax and the splitting of numbers (64 queries of 64 heads of 128 over 32,768 fp16
// positions 146 us, the merge's 8 among them: 138 GFLOP of matrix work at 1,000 TFLOP/s, a large library product
// reaching 1,205; the matrix pipes are busy 38 % of the cycles; 46 % issue to them or the vector units).
#include <algorithm>
#include <type_traits>

#include "dev_common.hpp"
#include "tf_internal.hpp"

namespace tfk {
namespace {

constexpr float kLog2e = 1.44269504088896341f;
constexpr int kRec = 32;  // positions of a record
constexpr int kWeightExp = 14;

// 2^e for e in [-126, 127]
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// The power of two that takes amax into [2^14, 2^15); 126 for 0 (a tile of zeros, exact in any scale).
__device__ __forceinline__ int scale_exp(float amax) {
    const int e = amax > 0.0f ? 15 - __builtin_amdgcn_frexp_expf(amax) : 126;
    return min(max(e, -126), 126);
}

// Where a V^T fragment's (dim, key group) entry lies among its 64: dims of one group in an order that
// leaves 8 consecutive lanes on 8 different 16-byte banks, for the reader (dims 0..7 or 8..15) and for
// writers that hold 1, 2, 4 or 8 consecutive dims each.
__device__ __forceinline__ int v_entry(int dim, int dt, int kg) {
    const int b3 = dim >> 3 & 1;
    return 16 * kg + 8 * b3 + ((dim & 7) ^ b3 ^ (dt << 1 & 6));
}

// Eight numbers x(j), times sc in the second form, as fp16 pairs. The rest of a number is one mixed-precision
// fma (number x 1 - its half); written out, the compiler widens the half first.
template <class X>
__device__ __forceinline__ void split8(X x, h8_t& hi, h8_t& lo) {
    typedef float f2_t __attribute__((ext_vector_type(2)));
    typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
    uint32_t h[4], l[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const f2_t y = {x(2 * j), x(2 * j + 1)};
        h[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(y, h2_t));
        f2_t r;
        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel_hi:[0,0,1]" : "=v"(r.x) : "v"(y.x), "v"(h[j]));
        asm("v_fma_mix_f32 %0, %1, 1.0, -%2 op_sel:[0,0,1] op_sel_hi:[0,0,1]" : "=v"(r.y) : "v"(y.y), "v"(h[j]));
        l[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(r, h2_t));
    }
    __builtin_memcpy(&hi, h, 16);
    __builtin_memcpy(&lo, l, 16);
}
template <class X>
__device__ __forceinline__ void split8(X x, float sc, h8_t& hi, h8_t& lo) {
    split8([&](int j) { return x(j) * sc; }, hi, lo);
}

template <class T, int HP, int NW, int QS, bool EXACT>
__global__ __launch_bounds__(64 * NW) void k_tree_attn(const TreeAttnArgs a) {
    constexpr bool kPair = sizeof(T) == 4;
    constexpr int NC = HP / 32, NT = HP / 16, kE = (int)sizeof(T);
    // Keys: a wave takes kWaveKeys positions of a step, kLanes lanes a position, 64 / kLanes positions a unit.
    constexpr int kHalf = NW / 2, kWaveKeys = kRec / kHalf, kLanes = HP / 8, kUnits = kWaveKeys * kLanes / 64;
    // dims of 8 values each a thread loads per step: at least a word of them (then some threads load none)
    constexpr int DV = HP / NW / 8 > 4 / kE ? HP / NW / 8 : 4 / kE;
    constexpr int kWords = (kUnits > DV ? kUnits : DV) * 8 * kE / 4;
    constexpr int kFrag = kPair ? 2048 : 1024;  // bytes of a fragment: hi, then lo
    constexpr int kKeys = 2 * NC * kFrag, REC = kKeys + NT * kFrag;
    constexpr int kBufs = 2;
    static_assert(NW % 2 == 0 && HP / NW >= 8, "half of the waves load keys, half values");
    __shared__ __align__(16) unsigned char lds[kBufs * REC];
    __shared__ int scale_of[2][NW];  // the exponents of a step's key waves and value waves, by step mod 2
    __shared__ uint32_t bad[3];  // positions of a record with an infinity or NaN, by step mod 3

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = lane & 15, gq = lane >> 4;
    const int hd = EXACT ? HP : a.hd, rep = a.H / a.G, rows = a.n_tree * rep;
    // A span of keys is a kv head's split (kv head fastest); a span's row blocks are a.group workgroups apart.
    const int blocks = (rows + 16 * QS * NW - 1) / (16 * QS * NW);
    const int span = blockIdx.x / (a.group * blocks) * a.group + blockIdx.x % a.group, blk = blockIdx.x / a.group % blocks;
    if (span >= a.G * a.S) return;
    const int g = span % a.G, split = span / a.G;
    const int end = a.n_past + a.n_tree;
    const int units = (end + kRec - 1) / kRec, per = (units + a.S - 1) / a.S;
    const int u0 = split * per, steps = min(units - u0, per);
    const int stride = a.layout == TF_HIP_KV_HEAD_MAJOR ? hd : a.G * hd;  // elements a position
    const int64_t base = kv_offset(a.layout, a.G, a.max_seq, hd, g, 0);

    // ---- loads
    // Keys: lane = (position lane / kLanes of a unit, 8 dims); they are entry 16 ch + (position ^ 2 ch ^ c mod 2)
    // of the fragment of their half and chunk c (ch: their place among its 4 times 8 dims), which leaves 8
    // consecutive lanes on 8 different 16-byte banks. Values: a thread holds the 8 positions of a key group
    // (4 kg + 0..3 and 16 + 4 kg + 0..3, as the weights lie in the lanes) of DV dims.
    const bool key_wave = wave < kHalf;
    const int tv = tid - 64 * kHalf;  // value threads
    const int v_d = DV * (tv % (HP / DV)), v_kg = tv / (HP / DV);
    const char* src = (const char*)((const T*)(key_wave ? a.kc : a.vc) + base);
    uint32_t raw[kWords];
    auto element = [&](int i) __attribute__((always_inline)) -> float {
        if constexpr (kPair)
            return __uint_as_float(raw[i]);
        else
            return h2f(i & 1 ? raw[i / 2] >> 16 : raw[i / 2] & 0xFFFFu);
    };
    // The thread's first place in a step; its others are uniform distances away. Dims past the head's are loaded
    // from dim 0 and zeros take their place. Every offset is from a row's start and not negative.
    const int k_pos = wave * kWaveKeys + lane / kLanes;  // its unit 0's position
    const int my_pos = key_wave ? k_pos : 4 * v_kg, my_dim = key_wave ? 8 * (lane % kLanes) : v_d;
    const int row_bytes = stride * kE;
    auto words = [&](const char* q, uint32_t* to, auto n) __attribute__((always_inline)) {
        if constexpr (n() >= 4) {
#pragma unroll
            for (int i = 0; i < n(); i += 4) {
                const uint4 x = gload_u4(q + 4 * i);
                to[i] = x.x; to[i + 1] = x.y; to[i + 2] = x.z; to[i + 3] = x.w;
            }
        } else if constexpr (n() == 2) {
            const uint2 x = gload_u2(q);
            to[0] = x.x; to[1] = x.y;
        } else {
            to[0] = *(const TF_GLOBAL uint32_t*)q;
        }
    };
    auto load_as = [&](auto FULL, int step) __attribute__((always_inline)) {
        const int p = kRec * (u0 + step), last = end - 1 - p;  // last: the end's position in the step
        const char* at = src + (int64_t)p * row_bytes;
        // place `row` rows below the thread's first; past the end the last row repeats
        const int dim = EXACT || my_dim < hd ? my_dim : 0;
        const uint32_t mine = (uint32_t)(my_pos * row_bytes + dim * kE);
        auto place = [&](int row) __attribute__((always_inline)) -> const char* {
            if constexpr (FULL()) return at + row * row_bytes + mine;
            return at + (uint32_t)(min(my_pos + row, last) * row_bytes + dim * kE);
        };
        if (key_wave) {
#pragma unroll
            for (int u = 0; u < kUnits; ++u) words(place(u * (64 / kLanes)), raw + u * 2 * kE, std::integral_constant<int, 2 * kE>());
        } else if (v_kg < 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j) words(place(j < 4 ? j : 12 + j), raw + j * DV * kE / 4, std::integral_constant<int, DV * kE / 4>());
        }
        if (!EXACT && my_dim >= hd)
#pragma unroll
            for (int i = 0; i < kWords; ++i) raw[i] = 0;
    };
    auto load = [&](int step) __attribute__((always_inline)) {
        if (kRec * (u0 + step + 1) <= end)
            load_as(std::true_type(), step);
        else
            load_as(std::false_type(), step);
    };
    // the power of two that this wave's elements are scaled by, from the largest finite one
    auto scale = [&]() __attribute__((always_inline)) -> int {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < kWords; ++i) m = fmaxf(m, fabsf(__uint_as_float(raw[i])));
        if (!(m < INFINITY)) {
            m = 0.0f;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                const float x = fabsf(__uint_as_float(raw[i]));
                if (x < INFINITY) m = fmaxf(m, x);
            }
        }
        return scale_exp(wave_max(m));
    };
    // Infinities and NaN among `n` elements from i are taken out; whether there were any.
    auto clean = [&](int i, int n) __attribute__((always_inline)) {
        bool odd = false;
#pragma unroll
        for (int k = i; k < i + n; ++k) {
            if (fabsf(element(k)) < INFINITY) continue;
            odd = true;
            if constexpr (kPair)
                raw[k] = 0;
            else
                raw[k / 2] &= k & 1 ? 0xFFFFu : 0xFFFF0000u;
        }
        return odd;
    };
    // The loaded step as records. A step that reaches into the tree takes its infinities and NaN out and
    // notes their positions: a zero weight times one of them would be NaN in the rows that do not see it.
    auto store = [&](int step) __attribute__((always_inline)) {
        unsigned char* buf = lds + (step & 1) * REC;
        const bool tree = kRec * (u0 + step + 1) > a.n_past;
        float sc = 1.0f;
        if constexpr (kPair) {
            const int e = scale();
            sc = pow2f(e);
            if (lane == 0) scale_of[step & 1][wave] = e;
        }
        if (key_wave) {
            const int c = lane % kLanes >> 2, ch = lane & 3;
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
                const int pos = k_pos + u * (64 / kLanes);
                if (tree && clean(8 * u, 8)) atomicOr(&bad[step % 3], 1u << pos);
                unsigned char* to = buf + ((pos >> 4) * NC + c) * kFrag + 16 * (16 * ch + ((pos & 15) ^ (2 * ch) ^ (c & 1)));
                if constexpr (kPair) {
                    h8_t hi, lo;
                    split8([&](int j) { return __uint_as_float(raw[8 * u + j]); }, sc, hi, lo);
                    *(h8_t*)to = hi;
                    *(h8_t*)(to + 1024) = lo;
                } else {
                    *(uint4*)to = make_uint4(raw[4 * u], raw[4 * u + 1], raw[4 * u + 2], raw[4 * u + 3]);
                }
            }
        } else if (v_kg < 4) {
            if (tree)
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (clean(j * DV, DV)) atomicOr(&bad[step % 3], 1u << (4 * v_kg + (j < 4 ? j : 12 + j)));
#pragma unroll
            for (int i = 0; i < DV; ++i) {
                const int d = v_d + i, dt = d >> 4;
                unsigned char* to = buf + kKeys + dt * kFrag + 16 * v_entry(d & 15, dt, v_kg);
                if constexpr (kPair) {
                    h8_t hi, lo;
                    split8([&](int j) { return __uint_as_float(raw[j * DV + i]); }, sc, hi, lo);
                    *(h8_t*)to = hi;
                    *(h8_t*)(to + 1024) = lo;
                } else {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j)  // halves i of positions 2 j and 2 j + 1
                        w[j] = __builtin_amdgcn_perm(raw[((2 * j + 1) * DV + i) / 2], raw[(2 * j * DV + i) / 2], i & 1 ? 0x07060302u : 0x05040100u);
                    *(uint4*)to = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    };

#pragma unroll
    for (int i = 0; i < kWords; ++i) raw[i] = 0;
    if (tid < 3) bad[tid] = 0;
    __syncthreads();  // before store(0) sets bits of it
    load(0);

    // ---- the wave's queries: lane l holds row l % 16 of each subtile, dims 32 c + 8 (l / 16) ..
    h8_t qh[QS][NC], ql[QS][NC];
    float fq[QS];
    int row[QS];
#pragma unroll
    for (int qs = 0; qs < QS; ++qs) {
        row[qs] = (blk * NW + wave) * 16 * QS + 16 * qs + l16;
        const int r = min(row[qs], rows - 1);
        const float* qr = a.q + (int64_t)(r / rep) * a.ldq + (int64_t)(g * rep + r % rep) * hd;
        float v[NC][8], m = 0.0f;
        const bool vec = (((uintptr_t)a.q | (uint64_t)a.ldq * 4) & 15) == 0;
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d = 32 * c + 8 * gq;
            if (!EXACT && d >= hd) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] = 0.0f;
            } else if (vec) {
                const float4 x = gload_f4(qr + d), y = gload_f4(qr + d + 4);
                v[c][0] = x.x; v[c][1] = x.y; v[c][2] = x.z; v[c][3] = x.w;
                v[c][4] = y.x; v[c][5] = y.y; v[c][6] = y.z; v[c][7] = y.w;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[c][j] = *gptr(qr + d + j);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[c][j]));
        }
        const int e = scale_exp(quad_max(m));
        fq[qs] = ldexpf(kLog2e / sqrtf((float)hd), -e);  // scores in units of log2
#pragma unroll
        for (int c = 0; c < NC; ++c) split8([&](int j) { return v[c][j]; }, pow2f(e), qh[qs][c], ql[qs][c]);
    }
    f4_t acc[QS][NT];  // O 2^(unit + 14)
    float m_run[QS], l_run[QS];  // l of this lane's positions
    int unit = kPair ? 126 : 0;
#pragma unroll
    for (int qs = 0; qs < QS; ++qs) {
        m_run[qs] = -INFINITY;
        l_run[qs] = 0.0f;
#pragma unroll
        for (int d = 0; d < NT; ++d) acc[qs][d] = (f4_t){0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int k_at[2] = {16 * (16 * gq + (l16 ^ (2 * gq))), 16 * (16 * gq + (l16 ^ (2 * gq) ^ 1))};
    int v_at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v_at[i] = 16 * v_entry(l16, i, gq);

    // ---- one record; TREE: it reaches into the tree
    auto record = [&](auto TREE, int step) __attribute__((always_inline)) {
        const unsigned char* rec = lds + (step & 1) * REC;
        const int p = kRec * (u0 + step);
        f4_t s[QS][2];
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) s[qs][0] = s[qs][1] = (f4_t){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const unsigned char* f = rec + (half * NC + c) * kFrag + k_at[c & 1];
                const h8_t kh = *(const h8_t*)f;
#pragma unroll
                for (int qs = 0; qs < QS; ++qs) s[qs][half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qh[qs][c], s[qs][half], 0, 0, 0);
#pragma unroll
                for (int qs = 0; qs < QS; ++qs) s[qs][half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, ql[qs][c], s[qs][half], 0, 0, 0);
                if constexpr (kPair) {
                    const h8_t kl = *(const h8_t*)(f + 1024);
#pragma unroll
                    for (int qs = 0; qs < QS; ++qs) s[qs][half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kl, qh[qs][c], s[qs][half], 0, 0, 0);
                }
            }
        __builtin_amdgcn_s_setprio(0);
        // the values are read ahead of the softmax, whose branches they would otherwise wait behind
        h8_t vh[NT];
#pragma unroll
        for (int d = 0; d < NT; ++d) vh[d] = *(const h8_t*)(rec + kKeys + d * kFrag + v_at[d & 3]);
#pragma unroll
        for (int d = 0; d < NT; ++d) asm volatile("" : "+v"(vh[d]));
        uint32_t bits[QS], odd = 0;
        if constexpr (TREE()) {
            // bit b: the row sees position p + b
            odd = bad[step % 3];
            const int off = p - a.n_past, left = end - p;
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) {
                const uint64_t* m = a.masks + (int64_t)(min(row[qs], rows - 1) / rep) * a.mask_words;
                uint64_t x = ~0ull;
                if (off <= -kRec) {
                } else if (off < 0) {
                    x = (m[0] << -off) | ((1ull << -off) - 1);
                } else {
                    const int w = off >> 6, sh = off & 63;
                    x = m[w] >> sh;
                    if (sh && w + 1 < a.mask_words) x |= m[w + 1] << (64 - sh);
                }
                bits[qs] = (uint32_t)x & (left >= 32 ? 0xFFFFFFFFu : (1u << left) - 1);
            }
        }
        // The scales of the lane's keys (its first four positions, its last four) and values, and the output's unit:
        // the least of the values' scales so far. Values of a greater one have their weights shrunk by as much.
        int ke[2] = {0, 0}, e = 0;
        float shrink = 1.0f;
        if constexpr (kPair) {
            const int* of = scale_of[step & 1];
            e = unit;
#pragma unroll
            for (int w = 0; w < kHalf; ++w) e = min(e, of[kHalf + w]);
            e = __builtin_amdgcn_readfirstlane(e);
            ke[0] = of[4 * gq / kWaveKeys];
            ke[1] = of[(16 + 4 * gq) / kWaveKeys];
            shrink = pow2f(max(e - of[kHalf + gq * kHalf / 4], -126));
        }
        const int de = e - unit;
        unit = e;
        h8_t ph[QS], pl[QS];
        float resc[QS];
        bool scaled = false;
#pragma unroll
        for (int qs = 0; qs < QS; ++qs) {
            float f[2], x[8], mt[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 2; ++i) f[i] = fmaxf(kPair ? ldexpf(fq[qs], -ke[i]) : fq[qs], 1e-37f);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = s[qs][j >> 2][j & 3];
            if constexpr (TREE()) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int b = 4 * gq + (j < 4 ? j : 12 + j);
                    if (odd >> b & 1) x[j] = NAN;
                    if (!(bits[qs] >> b & 1)) x[j] = -INFINITY;
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) mt[j >> 2] = fmaxf(mt[j >> 2], x[j]);
            const float top = quad_max(kPair ? fmaxf(mt[0] * f[0], mt[1] * f[1]) : fmaxf(mt[0], mt[1]) * f[0]);
            const float m_new = fmaxf(m_run[qs], ceilf(top));
            const float m_ref = m_new == -INFINITY ? 0.0f : m_new;
            const float alpha = __builtin_amdgcn_exp2f(m_run[qs] - m_ref);
            const float sh = (float)kWeightExp - m_ref;
            float ls = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = __builtin_amdgcn_exp2f(fmaf(x[j], f[kPair ? j >> 2 : 0], sh));
                ls += x[j];
            }
            if constexpr (kPair)
                split8([&](int j) { return x[j]; }, shrink, ph[qs], pl[qs]);
            else
                split8([&](int j) { return x[j]; }, ph[qs], pl[qs]);
            l_run[qs] = fmaf(l_run[qs], alpha, ls * pow2f(-kWeightExp));
            m_run[qs] = m_new;
            resc[qs] = kPair ? ldexpf(alpha, de) : alpha;
            scaled = scaled || resc[qs] != 1.0f;
        }
        if (__builtin_amdgcn_ballot_w64(scaled) != 0)
#pragma unroll
            for (int qs = 0; qs < QS; ++qs)
#pragma unroll
                for (int d = 0; d < NT; ++d) acc[qs][d] = acc[qs][d] * resc[qs];
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int d = 0; d < NT; ++d) {
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) acc[qs][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[d], ph[qs], acc[qs][d], 0, 0, 0);
#pragma unroll
            for (int qs = 0; qs < QS; ++qs) acc[qs][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vh[d], pl[qs], acc[qs][d], 0, 0, 0);
            if constexpr (kPair) {
                const h8_t vl = *(const h8_t*)(rec + kKeys + d * kFrag + v_at[d & 3] + 1024);
#pragma unroll
                for (int qs = 0; qs < QS; ++qs) acc[qs][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vl, ph[qs], acc[qs][d], 0, 0, 0);
            }
        }
        __builtin_amdgcn_s_setprio(0);
    };

    // every wave's LDS writes are done; loads under way stay so, which __syncthreads would wait for
    auto barrier = [&]() __attribute__((always_inline)) { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    store(0);
    if (steps > 1) load(1);
    barrier();
    // step t: its record is complete, the loads of t + 1 are there or under way. The next step's stores go first:
    // the waves leave the barrier together, and those on the vector units keep out of the way of the matrix ones
    // (after the record 2.3 us more, of 25.3, for 64 queries of 32 heads over 8,191 fp16 positions).
    auto step = [&](auto TREE, int t) __attribute__((always_inline)) {
        if (t + 1 < steps) store(t + 1);
        if (tid == 0) bad[(t + 2) % 3] = 0;
        if (t + 2 < steps) load(t + 2);
        record(TREE, t);
        if (t + 1 < steps) barrier();
    };
    const int plain = max(0, min(steps, a.n_past / kRec - u0));  // steps below n_past
    int t = 0;
    for (; t < plain; ++t) step(std::false_type(), t);
    for (; t < steps; ++t) step(std::true_type(), t);

    // ---- the row's 4 lanes
#pragma unroll
    for (int qs = 0; qs < QS; ++qs) {
        l_run[qs] = quad_sum(l_run[qs]);
        if constexpr (kPair)
#pragma unroll
            for (int i = 0; i < 4 * NT; ++i) acc[qs][i >> 2][i & 3] = ldexpf(acc[qs][i >> 2][i & 3], -unit);
    }
#pragma unroll
    for (int qs = 0; qs < QS; ++qs) {
        if (row[qs] >= rows) continue;
        const int t = row[qs] / rep, h = g * rep + row[qs] % rep;
        if (a.S == 1) {
            const float inv = l_run[qs] == 0.0f ? 0.0f : pow2f(-kWeightExp) / l_run[qs];
            float* o = a.out + (int64_t)t * a.ldo + (int64_t)h * hd + 4 * gq;
            const bool vec = (((uintptr_t)a.out | (uint64_t)a.ldo * 4) & 15) == 0;
#pragma unroll
            for (int d = 0; d < NT; ++d) {
                if (!EXACT && 16 * d + 4 * gq >= hd) continue;
                const f4_t x = acc[qs][d] * inv;
                if (vec)
                    *(f4_t*)(o + 16 * d) = x;
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[16 * d + i] = x[i];
            }
        } else {
            const int64_t part = ((int64_t)t * a.H + h) * a.S + split;
#pragma unroll
            for (int d = 0; d < NT; ++d)
                if (EXACT || 16 * d + 4 * gq < hd) *(f4_t*)(a.part_o + part * hd + 16 * d + 4 * gq) = acc[qs][d] * pow2f(-kWeightExp);
            if (gq == 0) *(float2*)(a.part_ml + 2 * part) = make_float2(m_run[qs], l_run[qs]);
        }
    }
}

// Merges the splits: o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s (the weights are powers of two).
// tpr threads a row, in groups of hd / 4: a thread takes 4 dims of every (tpr / (hd / 4))-th split in one
// round of loads, and the groups meet in LDS. Bound by its launch and that round.
__global__ __launch_bounds__(kBlock) void k_tree_merge(const TreeAttnArgs a, int tpr) {
    __shared__ f4_t part[kBlock];
    __shared__ float2 mls[kBlock];
    const int per = a.hd >> 2, groups = tpr / per, in = threadIdx.x % tpr, grp = in / per, d = 4 * (in % per);
    const int64_t row = (int64_t)blockIdx.x * (kBlock / tpr) + threadIdx.x / tpr;
    const bool on = grp < groups && row < (int64_t)a.n_tree * a.H;
    float M = -INFINITY, L = 0.0f;
    f4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
    if (on) {
        const float2* ml = (const float2*)a.part_ml + row * a.S;
        const float* po = a.part_o + row * a.S * a.hd + d;
        constexpr int kRound = 8;
        for (int s0 = grp; s0 < a.S; s0 += kRound * groups) {
            float2 x[kRound];
            f4_t y[kRound];
#pragma unroll
            for (int k = 0; k < kRound; ++k) {
                const int s = min(s0 + k * groups, a.S - 1);
                x[k] = ml[s];
                y[k] = *(const f4_t*)(po + (int64_t)s * a.hd);
            }
            float top = M;
#pragma unroll
            for (int k = 0; k < kRound; ++k) top = fmaxf(top, x[k].x);
            const float ref = top == -INFINITY ? 0.0f : top, f = __builtin_amdgcn_exp2f(M - ref);
            L *= f;
            o *= f;
            M = top;
#pragma unroll
            for (int k = 0; k < kRound; ++k) {
                if (s0 + k * groups >= a.S) continue;
                const float w = __builtin_amdgcn_exp2f(x[k].x - ref);
                L = fmaf(w, x[k].y, L);
                o += w * y[k];
            }
        }
    }
    part[threadIdx.x] = o;
    mls[threadIdx.x] = make_float2(M, L);
    __syncthreads();
    if (!on || grp) return;
    for (int k = 1; k < groups; ++k) {
        const float2 x = mls[threadIdx.x + k * per];
        const float top = fmaxf(M, x.x), ref = top == -INFINITY ? 0.0f : top;
        const float f = __builtin_amdgcn_exp2f(M - ref), w = __builtin_amdgcn_exp2f(x.x - ref);
        L = fmaf(w, x.y, L * f);
        o = o * f + w * part[threadIdx.x + k * per];
        M = top;
    }
    o *= L == 0.0f ? 0.0f : 1.0f / L;
    float* out = a.out + row / a.H * a.ldo + row % a.H * a.hd + d;
#pragma unroll
    for (int k = 0; k < 4; ++k) out[k] = o[k];
}

// Row n_past + path[i] of every layer, K and V, moves to row n_past + i, for i up to the path's length or
// up to the first entry that does not name a node past the one before. A thread owns 16 bytes of a row's
// place and walks the path in order: path[i] >= i, so a row is read before an earlier entry's write could
// reach it (that entry wrote a lower row). Bound by its launch and one dependent round a moved row: 3.5 us for 4
// rows of 16 layers, 5.2 for 9 of 28 (1 MB read and written); a whole call is 7.9 us, the host's launch.
__global__ __launch_bounds__(kBlock) void k_keep_path(const KeepArgs a) {
    const int64_t per_layer = (int64_t)a.G * a.row16;  // 16-byte pieces of one position
    const int64_t i = (int64_t)blockIdx.x * kBlock + threadIdx.x;
    if (i >= per_layer * a.n_layer) return;
    const int layer = (int)(i / per_layer), g = (int)(i % per_layer / a.row16), c = (int)(i % a.row16);
    uint4* base = (uint4*)(blockIdx.y ? a.vc : a.kc) + (int64_t)layer * per_layer * a.max_seq;
    const int n = min(*a.n_path, a.n_tree);
    int last = -1;
    for (int k = 0; k < n; ++k) {
        const int node = a.path[k];
        if (node <= last || node >= a.n_tree) break;
        last = node;
        if (node == k) continue;
        base[kv_offset(a.layout, a.G, a.max_seq, a.row16, g, a.n_past + k) + c] =
            base[kv_offset(a.layout, a.G, a.max_seq, a.row16, g, a.n_past + node) + c];
    }
}

}  // namespace

namespace {

// Rows of a workgroup, positions of a step and splits for a call. See launch_tree_attn.
struct TreePlan {
    int hp, bm, blocks, splits;
};

TreePlan tree_plan(int n_tree, int H, int G, int hd, int n_past, int size) {  // size: bytes of an element
    TreePlan p{};
    const int rows = n_tree * (H / G);
    p.hp = hd <= 64 ? 64 : (hd <= 128 ? 128 : 256);
    // Workgroups of 256 rows (head sizes up to 128) read keys and values fewest times and run two row subtiles on
    // every fragment, but fill the chip only where there is enough (more than 128 rows): 16 steps for each of 256
    // workgroups. Below that, 64 rows and about two workgroups a CU. (With an earlier merge, 64 queries of 64 heads
    // of 128 over 32,768 fp16 positions took 178 us, by 64 rows 213; of 32 heads of 64 over 8,191 31.0 and 29.3.)
    const int64_t units = ((int64_t)n_past + n_tree + kRec - 1) / kRec;
    const bool big = p.hp <= 128 && rows > 128 && (int64_t)G * ((rows + 255) / 256) * units >= 16 * 256;
    p.bm = big ? 256 : 64;
    p.blocks = (rows + p.bm - 1) / p.bm;
    const int64_t want = std::min(units, std::max<int64_t>(1, (big ? 256 : 512) / ((int64_t)G * p.blocks)));
    // Few steps run one after the other without a merge: they cost less than the second launch (1.3 us a step of fp32
    // rows of 64, half that for fp16, 1.9 and 0.95 for rows of 128; the merge 3 us and its launch): 101 positions of 8
    // fp32 heads of 64 take 9.0 us a call in one split and 11.0 in four, 161 take 11.9 and 10.9.
    const int64_t per = units * p.hp * size <= 1024 ? units : (units + want - 1) / want;
    p.splits = (int)((units + per - 1) / per);
    return p;
}

template <class T, int HP, int NW, int QS>
hipError_t launch_tree(const TreeAttnArgs& a, const TreePlan& p, hipStream_t st) {
    static_assert(HP == 256 || NW * QS == 4 || NW * QS == 16, "the plan's rows");
    const dim3 grid((unsigned)((a.G * a.S + a.group - 1) / a.group * a.group * p.blocks)), block(64 * NW);
    return launch_kernel(a.hd == HP ? k_tree_attn<T, HP, NW, QS, true> : k_tree_attn<T, HP, NW, QS, false>, grid, block, st, a);
}

template <class T>
hipError_t launch_tree_type(const TreeAttnArgs& a, const TreePlan& p, hipStream_t st) {
    if (p.hp == 256) return launch_tree<T, 256, 4, 1>(a, p, st);
    if (p.hp == 128) return p.bm == 64 ? launch_tree<T, 128, 4, 1>(a, p, st) : launch_tree<T, 128, 8, 2>(a, p, st);
    return p.bm == 64 ? launch_tree<T, 64, 4, 1>(a, p, st) : launch_tree<T, 64, 8, 2>(a, p, st);
}

}  // namespace

size_t tree_attn_ws_bytes(int n_tree, int H, int G, int hd, int n_past) {
    const int S = std::max(tree_plan(n_tree, H, G, hd, n_past, 4).splits, tree_plan(n_tree, H, G, hd, n_past, 2).splits);
    return S == 1 ? 0 : (size_t)n_tree * H * S * (hd + 2) * 4;
}

hipError_t launch_tree_attn(const TreeAttnArgs& args, void* ws, hipStream_t st) {
    TreeAttnArgs a = args;
    const TreePlan p = tree_plan(a.n_tree, a.H, a.G, a.hd, a.n_past, a.kv_type == TF_HIP_TYPE_F32 ? 4 : 2);
    a.mask_words = (a.n_tree + 63) / 64;
    a.S = p.splits;
    // Workgroups go to the 8 XCDs in turn: with a span's row blocks 8 apart they meet in one L2 (26 queries of 12 heads
    // of 128 over 4,096 fp32 positions read 9.5 MB instead of 26.4 and take 19.3 us a call instead of 19.9). Few spans
    // that are no multiple of 8 would leave XCDs idle: all spans' first blocks, then all second ones.
    const int spans = a.G * a.S;
    a.group = p.blocks > 1 && (spans >= 64 || spans % 8 == 0) ? 8 : spans;
    a.part_o = (float*)ws;
    a.part_ml = a.part_o + (size_t)a.n_tree * a.H * a.S * a.hd;
    const hipError_t e = a.kv_type == TF_HIP_TYPE_F32 ? launch_tree_type<float>(a, p, st) : launch_tree_type<_Float16>(a, p, st);
    if (e != hipSuccess || a.S == 1) return e;
    // a wave a row while that leaves a thread 16 splits, two rounds of loads, else four waves: a call over 8,191 fp16
    // positions (16 splits of 64 dims) takes 25.3 us so and 27.7 by four, over 4,096 of 128 dims (65 splits) 21.4 and 18.9
    const int tpr = a.S * (a.hd >> 2) <= 64 * 16 ? 64 : kBlock, rows = a.n_tree * a.H, per = kBlock / tpr;
    return launch_kernel(k_tree_merge, dim3((unsigned)((rows + per - 1) / per)), dim3(kBlock), st, a, tpr);
}

hipError_t launch_keep_path(const KeepArgs& a, hipStream_t st) {
    const int64_t pieces = (int64_t)a.n_layer * a.G * a.row16;
    return launch_kernel(k_keep_path, dim3((unsigned)((pieces + kBlock - 1) / kBlock), 2), dim3(kBlock), st, a);
}

}  // namespace tfk
