// Attention of a tree of drafted tokens over a cache, and the move of the accepted nodes' rows.
//
// Node i of the tree has its key and value at cache position n_past + i. Its query sees every
// position below n_past and, of the tree, the nodes whose bit its mask sets:
//   s_j = q_i . k_j / sqrt(hd),   o_i = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m),   m = max_j s_j
// over the positions j that it sees; a row that sees none is zero. The positions are cut into
// splits, each with its own m and l = sum_j e^(s_j - m); the merge adds them as
// sum_s e^(m_s - M) o_s / sum_s e^(m_s - M) l_s.
#include "dev_common.hpp"
#include "tf_internal.hpp"

namespace tfk {
namespace {

constexpr float kLog2e = 1.44269504088896341f;

template <class T>
__device__ __forceinline__ float cache_value(const T* p) {
    return (float)*p;
}

// Grid (row t H + h, split), 4 waves: wave w takes the split's positions w, w + 4, ...; a lane holds the
// dims lane, lane + 64, ... of its query and of its wave's output.
template <class T>
__global__ __launch_bounds__(kBlock) void k_tree_attn(const TreeAttnArgs a) {
    constexpr int kDims = 4;  // hd <= 256
    __shared__ float mo[kWavesPerBlock][kDims * 64], ml[kWavesPerBlock][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int t = blockIdx.x / a.H, h = blockIdx.x % a.H, g = h / (a.H / a.G), s = blockIdx.y;
    const int end = a.n_past + a.n_tree;
    const int p0 = (int)((int64_t)end * s / a.S), p1 = (int)((int64_t)end * (s + 1) / a.S);
    const float* q = a.q + (int64_t)t * a.ldq + (int64_t)h * a.hd;
    float qv[kDims], o[kDims];
#pragma unroll
    for (int i = 0; i < kDims; ++i) {
        qv[i] = lane + 64 * i < a.hd ? q[lane + 64 * i] : 0.0f;
        o[i] = 0.0f;
    }
    const float scale = kLog2e / sqrtf((float)a.hd);
    float m = -INFINITY, l = 0.0f;
    for (int p = p0 + wave; p < p1; p += kWavesPerBlock) {
        const int j = p - a.n_past;
        if (j >= 0 && !(a.masks[(int64_t)t * a.mask_words + (j >> 6)] >> (j & 63) & 1)) continue;
        const int64_t at = kv_offset(a.layout, a.G, a.max_seq, a.hd, g, p);
        const T *k = (const T*)a.kc + at, *v = (const T*)a.vc + at;
        float x = 0.0f;
#pragma unroll
        for (int i = 0; i < kDims; ++i)
            if (lane + 64 * i < a.hd) x = fmaf(qv[i], cache_value(k + lane + 64 * i), x);
        x = wave_sum(x) * scale;
        const float m_new = x != x ? x : fmaxf(m, x);  // a NaN score stays in m or in l
        const float alpha = m_new == m ? 1.0f : exp2f(m - m_new), w = x == m_new ? 1.0f : exp2f(x - m_new);
        l = l * alpha + w;
        m = m_new;
#pragma unroll
        for (int i = 0; i < kDims; ++i)
            if (lane + 64 * i < a.hd) o[i] = fmaf(w, cache_value(v + lane + 64 * i), o[i] * alpha);
    }
#pragma unroll
    for (int i = 0; i < kDims; ++i) mo[wave][lane + 64 * i] = o[i];
    if (lane == 0) {
        ml[wave][0] = m;
        ml[wave][1] = l;
    }
    __syncthreads();
    float M = -INFINITY, L = 0.0f, sum = 0.0f;
    for (int w = 0; w < kWavesPerBlock; ++w) M = fmaxf(M, ml[w][0]);
    for (int w = 0; w < kWavesPerBlock; ++w) {
        const float f = ml[w][0] == -INFINITY ? 0.0f : exp2f(ml[w][0] - M);
        L += f * ml[w][1];
        if (f > 0.0f) sum = fmaf(f, mo[w][tid], sum);
    }
    const int64_t part = (int64_t)blockIdx.x * a.S + s;
    if (tid < a.hd) a.part_o[part * a.hd + tid] = sum;
    if (tid == 0) {
        a.part_ml[2 * part] = L == L ? M : L;
        a.part_ml[2 * part + 1] = L;
    }
}

// Merges the splits of row blockIdx.x.
__global__ __launch_bounds__(kBlock) void k_tree_merge(const TreeAttnArgs a) {
    const int t = blockIdx.x / a.H, h = blockIdx.x % a.H, d = threadIdx.x;
    const int64_t part = (int64_t)blockIdx.x * a.S;
    float M = -INFINITY, L = 0.0f, sum = 0.0f;
    for (int s = 0; s < a.S; ++s) M = fmaxf(M, a.part_ml[2 * (part + s)]);
    for (int s = 0; s < a.S; ++s) {
        const float m = a.part_ml[2 * (part + s)];
        if (m == -INFINITY) continue;
        const float f = exp2f(m - M);
        L = fmaf(f, a.part_ml[2 * (part + s) + 1], L);
        if (d < a.hd) sum = fmaf(f, a.part_o[(part + s) * a.hd + d], sum);
    }
    if (d < a.hd) a.out[(int64_t)t * a.ldo + (int64_t)h * a.hd + d] = L == 0.0f ? 0.0f : sum / L;
}

// Row n_past + path[i] of every layer, K and V, moves to row n_past + i, for i up to the path's length or
// up to the first entry that does not name a node past the one before. A thread owns 16 bytes of a row's
// place and walks the path in order: path[i] >= i, so a row is read before an earlier entry's write could
// reach it (that entry wrote a lower row).
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

int tree_attn_splits(int n_tree, int H, int G, int hd, int n_past) {
    const int by_len = (n_past + n_tree + 63) / 64, by_rows = 2048 / (n_tree * H) + 1;
    return by_len < by_rows ? by_len : by_rows;
}

size_t tree_attn_ws_bytes(int n_tree, int H, int G, int hd, int n_past) {
    return (size_t)n_tree * H * tree_attn_splits(n_tree, H, G, hd, n_past) * (hd + 2) * 4;
}

hipError_t launch_tree_attn(const TreeAttnArgs& args, void* ws, hipStream_t st) {
    TreeAttnArgs a = args;
    a.mask_words = (a.n_tree + 63) / 64;
    a.S = tree_attn_splits(a.n_tree, a.H, a.G, a.hd, a.n_past);
    a.part_o = (float*)ws;
    a.part_ml = a.part_o + (size_t)a.n_tree * a.H * a.S * a.hd;
    const dim3 grid((unsigned)(a.n_tree * a.H), (unsigned)a.S);
    if (a.kv_type == TF_HIP_TYPE_F32)
        hipLaunchKernelGGL(k_tree_attn<float>, grid, dim3(kBlock), 0, st, a);
    else
        hipLaunchKernelGGL(k_tree_attn<_Float16>, grid, dim3(kBlock), 0, st, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_tree_merge, dim3((unsigned)(a.n_tree * a.H)), dim3(kBlock), 0, st, a);
    return hipGetLastError();
}

hipError_t launch_keep_path(const KeepArgs& a, hipStream_t st) {
    const int64_t pieces = (int64_t)a.n_layer * a.G * a.row16;
    hipLaunchKernelGGL(k_keep_path, dim3((unsigned)((pieces + kBlock - 1) / kBlock), 2), dim3(kBlock), 0, st, a);
    return hipGetLastError();
}

}  // namespace tfk
