// Attention of drafted tokens (a tree, a chain, or one token) over the paged cache, for sequences whose
// lengths and block tables stay on the GPU.
//
// Sequence s has ctx live rows and `len` drafted ones behind them, all in the cache (K stored rotated).
// Token t sees every live row and the drafted rows j whose bit is set in its mask (no masks: j <= t):
//   S = scale * rot(Q_t) . K,  O = softmax(S) V,  LSE = max + ln sum exp(S - max).
// A row that sees nothing, and the rows t >= len, get O = 0 and LSE = -inf. So does a sequence whose
// lengths do not fit its table, and a token whose position the (cos, sin) table does not have; keys on
// pages outside the pool are as if masked. No counterpart in the reference, whose decode takes one
// query a sequence and host tables (src/wgpu_paged_decode.rs:300).
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace fa {

template <typename T>
__device__ __forceinline__ float element(const void* p, int64_t i) {
    if constexpr (std::is_same<T, float>::value) return ((const float*)p)[i];
    else return Half<T>::lo(((const uint16_t*)p)[i]);
}
template <typename T>
__device__ __forceinline__ void put(void* p, int64_t i, float x) {
    if constexpr (std::is_same<T, float>::value) ((float*)p)[i] = x;
    else ((uint16_t*)p)[i] = (uint16_t)Half<T>::pack(x, 0.0f);
}

// One wave a row (sequence, token, head): a key per lane for the scores, two dims per lane for P.V.
template <typename T>
__global__ __launch_bounds__(64) void tree_rows(TreeArgs a, FastDiv ps) {
    __shared__ float qv[128];
    const int lane = threadIdx.x, D = a.head_dim;
    const int hq = blockIdx.x % a.q_heads, r = blockIdx.x / a.q_heads;
    const int s = r / a.max_tokens, t = r % a.max_tokens;
    const int ctx = a.ctx_lens[s], len = a.tree_lens[s];
    bool live = ctx >= 0 && len >= 0 && len <= a.max_tokens && t < len &&
                (int64_t)ctx + len <= (int64_t)a.max_pages * a.page_size;
    int64_t pos = 0;
    if (live && a.rope_table) {
        pos = a.positions ? a.positions[r] : ctx + t;
        live = pos >= 0 && pos < a.rope_positions;
    }
    const int64_t q0 = ((int64_t)r * a.q_heads + hq) * D;
    if (live) {
        for (int d = 2 * lane; d < D; d += 128) {
            float e = element<T>(a.q, q0 + d), o = element<T>(a.q, q0 + d + 1);
            if (a.rope_table) {
                const float2 cs = a.rope_table[(pos + a.rope_offset) * (D / 2) + d / 2];
                rope_pair(e, o, cs.x, cs.y);
            }
            qv[d] = e;
            qv[d + 1] = o;
        }
    }
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
    const int n = live ? ctx + len : 0;
    const int64_t width = (int64_t)a.kv_heads * D, head = (int64_t)(hq / a.group) * D;
    for (int base = 0; base < n; base += 64) {
        const int key = base + lane, j = key - ctx;
        bool seen = key < n;
        int64_t row = -1;
        if (seen && j >= 0)
            seen = a.masks ? (a.masks[(int64_t)r * a.words + (j >> 6)] >> (j & 63)) & 1 : j <= t;
        if (seen) {
            const int lp = (int)ps.div((uint32_t)key);
            const int page = a.block_tables[(int64_t)s * a.max_pages + lp];
            if ((unsigned)page < (unsigned)a.physical_pages)
                row = (int64_t)page * a.page_size + (key - lp * a.page_size);
        }
        float sc = -INFINITY;
        if (row >= 0) {
            float x = 0.0f;
            for (int d = 0; d < D; ++d) x = fmaf(qv[d], element<T>(a.k_pool, row * width + head + d), x);
            sc = x * a.scale;
        }
        float mt = sc;
        for (int k = 32; k; k >>= 1) mt = fmaxf(mt, shfl_xor(mt, k));
        if (mt == -INFINITY) continue;
        const float mn = fmaxf(m, mt), keep = fast_exp2((m - mn) * kLog2e);
        const float p = fast_exp2((sc - mn) * kLog2e);
        m = mn;
        l = l * keep + p;
        o0 *= keep;
        o1 *= keep;
        for (int k = 0; k < 64; ++k) {
            const float pk = __shfl(p, k, 64);
            const int64_t rk = __shfl((long long)row, k, 64);
            if (pk == 0.0f) continue;
            if (lane < D) o0 = fmaf(pk, element<T>(a.v_pool, rk * width + head + lane), o0);
            if (lane + 64 < D) o1 = fmaf(pk, element<T>(a.v_pool, rk * width + head + lane + 64), o1);
        }
    }
    for (int k = 32; k; k >>= 1) l += shfl_xor(l, k);
    const float inv = l > 0.0f ? 1.0f / l : 0.0f;
    if (lane < D) put<T>(a.o, q0 + lane, o0 * inv);
    if (lane + 64 < D) put<T>(a.o, q0 + lane + 64, o1 * inv);
    if (lane == 0) a.lse[((int64_t)s * a.q_heads + hq) * a.max_tokens + t] =
        l > 0.0f ? m + logf(l) : -INFINITY;
}

void launch_tree_attention(Dtype dt, const TreeArgs& a, hipStream_t s, unsigned grid[3],
                           unsigned* block, unsigned* dispatches) {
    const FastDiv ps((uint32_t)a.page_size);
    grid[0] = (unsigned)((int64_t)a.n_seqs * a.max_tokens * a.q_heads);
    grid[1] = grid[2] = 1;
    *block = 64;
    *dispatches = 1;
    switch (dt) {
        case Dtype::BF16: tree_rows<bf16_t><<<grid[0], 64, 0, s>>>(a, ps); break;
        case Dtype::F16: tree_rows<f16_t><<<grid[0], 64, 0, s>>>(a, ps); break;
        default: tree_rows<float><<<grid[0], 64, 0, s>>>(a, ps); break;
    }
}

}  // namespace fa
