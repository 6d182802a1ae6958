// What the attention kernels of the device-resident batch share: a sequence's live rows, which steps of
// keys it reads, and which keys of a block a token sees.
#pragma once

#include "common.hpp"
#include "kernels.hpp"

namespace fa {

// Division of numbers below 2^31 by a constant of the launch, in 32 bits: with s = ceil(log2 d) and
// m = floor(2^(31 + s) / d) + 1, m d - 2^(31 + s) <= 2^s, so n m / 2^(31 + s) is off by less than 1 / d.
struct SmallDiv {
    uint32_t m, s;
    __host__ SmallDiv() : m(0), s(0) {}
    __host__ explicit SmallDiv(uint32_t d) {
        for (s = 0; (1ull << s) < d; ++s) {
        }
        m = (uint32_t)((1ull << (31 + s)) / d + 1);
    }
    __device__ __forceinline__ int div(int n) const { return (int)(__umulhi((uint32_t)n << 1, m) >> s); }
};

// Live rows of a sequence, drafted ones included; 0: it has no part in this call.
__device__ __forceinline__ int tree_rows_of(const TreeArgs& a, int s) {
    const int ctx = a.ctx_lens[s], len = a.tree_lens[s];
    const bool ok = ctx >= 0 && len > 0 && len <= a.max_tokens &&
                    (int64_t)ctx + len <= (int64_t)a.max_pages * a.page_size;
    return ok ? ctx + len : 0;
}

// Inclusive prefix sum over a wave (row shifts by 1, 2, 4, 8, then the last lane of each row of 16 to
// the next row, and of the first half to the second).
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

// With a window the steps (of kt keys) between the sinks and the first key that token 0 sees are left out:
// how many, behind the first `*before` ones. 0: every step is read.
__device__ __forceinline__ int tree_skip(const TreeArgs& a, int rows, int len, int kt, int* before) {
    const int low = max(0, rows - len + 1 - a.window) / kt;  // step of that key
    const int sinks = (min(a.sinks, low * kt) + kt - 1) / kt;
    *before = sinks;
    return low - sinks;
}

// Bit i: key key0 + i (of 32) is seen by the token at row pos, by position alone.
__device__ __forceinline__ uint32_t causal_word(int pos, int key0) {
    const int last = pos - key0;
    return last >= 31 ? 0xffffffffu : last >= 0 ? (2u << last) - 1u : 0u;
}
__device__ __forceinline__ uint32_t window_word(const TreeArgs& a, int pos, int key0) {
    const int first = pos - key0 - a.window + 1, sinks = a.sinks - key0;
    const uint32_t near = first <= 0 ? 0xffffffffu : first < 32 ? 0xffffffffu << first : 0u;
    const uint32_t begin = sinks >= 32 ? 0xffffffffu : sinks > 0 ? (1u << sinks) - 1u : 0u;
    return causal_word(pos, key0) & (near | begin);
}
// The same from a token's mask: j0 = key0 - ctx is the drafted token of the first key. mask0: the mask of
// a tree of up to 64 tokens.
__device__ __forceinline__ uint32_t mask_word(const TreeArgs& a, bool row_ok, int tok, uint64_t mask0,
                                              int j0) {
    const uint64_t* const m = a.masks + (int64_t)tok * a.words;
    const int at64 = j0 >= 0 ? j0 >> 6 : 0, sh = j0 & 63;
    uint64_t w0 = mask0, w1 = 0;
    if (a.words > 1) {
        w0 = row_ok && at64 < a.words ? m[at64] : 0;
        w1 = row_ok && j0 >= 0 && at64 + 1 < a.words ? m[at64 + 1] : 0;
    } else if (at64 > 0) {
        w0 = 0;
    }
    if (j0 >= 0) return (uint32_t)((w0 >> sh) | (sh ? w1 << (64 - sh) : 0));
    if (j0 > -32) return (uint32_t)(w0 << -j0 | ((1u << -j0) - 1u));
    return 0xffffffffu;
}

}  // namespace fa
