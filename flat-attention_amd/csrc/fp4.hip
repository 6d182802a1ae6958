// The paged cache in 4 bits a value: rows into it and out of it, and attention of new tokens over it.
//
// A row (one token) holds the e2m1 codes of all kv heads and one e8m0 scale for every 32 values of a head:
// value = code * 2^e, code one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives. No counterpart in the
// reference.
#include <algorithm>
#include <type_traits>

#include "tree.hpp"

namespace fa {

// ------------------------------------------------------------------ rows
// The scale of 32 values of largest magnitude `top` (its bits): the least e, -127 .. 125, with top < 7 * 2^e,
// as e + 127. 7 = 1.75 * 2^2, so adding a quarter of the exponent's step carries at a mantissa of 1.75. (Up to
// 125: 6 * 2^126 is no f32 number; larger values are cut to 6 * 2^125.) 255 where one is infinite or NaN.
__device__ __forceinline__ int fp4_scale(uint32_t top) {
    if (top >= 0x7f800000u) return 255;
    return min(max((int)((top + 0x200000u) >> 23) - 2, 0), 252);
}

// Nearest code of x / scale, ties to the even one.
__device__ __forceinline__ uint32_t fp4_code(float x, float inv) {
    const float a = fabsf(x) * inv;
    uint32_t c = a > 0.25f;
    c += a >= 0.75f;
    c += a > 1.25f;
    c += a >= 1.75f;
    c += a > 2.5f;
    c += a >= 3.5f;
    c += a > 5.0f;
    return c | (__float_as_uint(x) >> 31 << 3);
}

// Eight values of piece c of a row, as f32.
template <typename T>
__device__ __forceinline__ void load8(const void* src, int64_t piece, float (&x)[8]) {
    if constexpr (std::is_same<T, float>::value) {
        const f32x4_t a = ((const f32x4_t*)src)[2 * piece], b = ((const f32x4_t*)src)[2 * piece + 1];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[j] = a[j];
            x[4 + j] = b[j];
        }
    } else {
        const u32x4_t a = ((const u32x4_t*)src)[piece];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = Half<T>::lo(a[j]);
            x[2 * j + 1] = Half<T>::hi(a[j]);
        }
    }
}

// One thread: eight values of K and of V of a row; four neighbouring threads share a scale.
template <typename T>
__global__ __launch_bounds__(256) void append_fp4(SlotAppendArgs a, FastDiv per_row, FastDiv per_seq,
                                                  FastDiv per_head, int row_bytes) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const bool in = i < (int64_t)a.n_rows * per_row.d;
    const uint32_t at = in ? (uint32_t)i : 0u;
    const int r = (int)per_row.div(at), c = (int)(at - (uint32_t)r * per_row.d);
    const int slot = a.slots[r];
    bool ok = in && (unsigned)slot < (unsigned)a.pool_rows;
    float k[8], v[8];
    load8<T>(a.k_src, (int64_t)r * per_row.d + c, k);
    load8<T>(a.v_src, (int64_t)r * per_row.d + c, v);
    if (a.rope_table) {
        const int s = (int)per_seq.div((uint32_t)r);
        const int64_t pos = a.positions ? (int64_t)a.positions[r]
                                        : (int64_t)a.ctx_lens[s] + (r - s * (int)per_seq.d);
        if (pos < 0 || pos >= a.rope_positions) ok = false;
        const int d0 = (c - (int)(per_head.div((uint32_t)c) * per_head.d)) * 8;
        const float2* cs = a.rope_table + ((ok ? pos : 0) + a.rope_offset) * (a.head_dim / 2) + d0 / 2;
        const f32x4_t t0 = ((const f32x4_t*)cs)[0], t1 = ((const f32x4_t*)cs)[1];
        const float c8[8] = {t0[0], t0[1], t0[2], t0[3], t1[0], t1[1], t1[2], t1[3]};
        rope4(k, c8);
    }
    const int codes = (int)per_row.d * 4;  // bytes of the codes of a row
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const float (&x)[8] = n ? v : k;
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(x[j]) & 0x7fffffffu);
        top = max(top, (uint32_t)__shfl_xor((int)top, 1, 64));
        top = max(top, (uint32_t)__shfl_xor((int)top, 2, 64));
        const int scale = fp4_scale(top);
        const float inv = __uint_as_float((uint32_t)(254 - min(scale, 253)) << 23);
        uint32_t w = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) w |= fp4_code(x[j], inv) << (4 * j);
        if (!ok) continue;
        uint8_t* const row = (uint8_t*)(n ? a.v_pool : a.k_pool) + (int64_t)slot * row_bytes;
        *(uint32_t*)(row + 4 * c) = scale == 255 ? 0u : w;
        if ((c & 3) == 0) row[codes + c / 4] = (uint8_t)scale;
        // (zeros behind the scales)
        if (c == 0)
            for (int p = codes + codes / 16; p < row_bytes; ++p) row[p] = 0;
    }
}

// value of code `c` (4 bits) as f32: 1.0 and above are sign, two exponent bits, one of the mantissa
__device__ __forceinline__ float fp4_value(uint32_t c) {
    const uint32_t m = c & 7;
    const float x = m < 2 ? 0.5f * (float)m : __uint_as_float(0x3f800000u + ((m - 2) << 22));
    return c & 8 ? -x : x;
}
__device__ __forceinline__ float fp4_scale_value(uint32_t b) {
    return __uint_as_float(b == 255 ? 0x7fc00000u : b == 0 ? 0x400000u : b << 23);
}

template <typename T>
__global__ __launch_bounds__(256) void read_fp4(SlotAppendArgs a, FastDiv per_row, int row_bytes) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.n_rows * per_row.d) return;
    const int r = (int)per_row.div((uint32_t)i), c = (int)((uint32_t)i - (uint32_t)r * per_row.d);
    const int slot = a.slots[r], codes = (int)per_row.d * 4;
    const bool ok = (unsigned)slot < (unsigned)a.pool_rows;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const uint8_t* const row = (const uint8_t*)(n ? a.v_pool : a.k_pool) + (int64_t)(ok ? slot : 0) * row_bytes;
        const uint32_t w = ok ? *(const uint32_t*)(row + 4 * c) : 0u;
        const float s = ok ? fp4_scale_value(row[codes + c / 4]) : 0.0f;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = fp4_value((w >> (4 * j)) & 15u) * s;
        void* const to = const_cast<void*>(n ? a.v_src : a.k_src);
        if constexpr (std::is_same<T, float>::value) {
            ((f32x4_t*)to)[2 * i] = f32x4_t{x[0], x[1], x[2], x[3]};
            ((f32x4_t*)to)[2 * i + 1] = f32x4_t{x[4], x[5], x[6], x[7]};
        } else {
            ((u32x4_t*)to)[i] = u32x4_t{Half<T>::pack(x[0], x[1]), Half<T>::pack(x[2], x[3]),
                                        Half<T>::pack(x[4], x[5]), Half<T>::pack(x[6], x[7])};
        }
    }
}

static unsigned fp4_grid(const SlotAppendArgs& a, unsigned grid[3]) {
    const int64_t per_row = (int64_t)a.kv_heads * a.head_dim / 8;
    grid[0] = (unsigned)((a.n_rows * per_row + 255) / 256);
    grid[1] = grid[2] = 1;
    return grid[0];
}
void launch_append_fp4(Dtype dt, const SlotAppendArgs& a, hipStream_t s, unsigned grid[3]) {
    const FastDiv per_row((uint32_t)(a.kv_heads * a.head_dim / 8)), per_seq((uint32_t)a.max_new),
        per_head((uint32_t)(a.head_dim / 8));
    const unsigned g = fp4_grid(a, grid);
    const int rb = fp4_row_bytes(a.kv_heads, a.head_dim);
    switch (dt) {
        case Dtype::BF16: append_fp4<bf16_t><<<g, 256, 0, s>>>(a, per_row, per_seq, per_head, rb); break;
        case Dtype::F16: append_fp4<f16_t><<<g, 256, 0, s>>>(a, per_row, per_seq, per_head, rb); break;
        default: append_fp4<float><<<g, 256, 0, s>>>(a, per_row, per_seq, per_head, rb); break;
    }
}
void launch_read_fp4(Dtype dt, const SlotAppendArgs& a, hipStream_t s, unsigned grid[3]) {
    const FastDiv per_row((uint32_t)(a.kv_heads * a.head_dim / 8));
    const unsigned g = fp4_grid(a, grid);
    const int rb = fp4_row_bytes(a.kv_heads, a.head_dim);
    switch (dt) {
        case Dtype::BF16: read_fp4<bf16_t><<<g, 256, 0, s>>>(a, per_row, rb); break;
        case Dtype::F16: read_fp4<f16_t><<<g, 256, 0, s>>>(a, per_row, rb); break;
        default: read_fp4<float><<<g, 256, 0, s>>>(a, per_row, rb); break;
    }
}

// ------------------------------------------------------------------ attention
// What is seen, and what rows that see nothing get, as in tree.hip. A wave works by itself: 16 NB rows of a
// (sequence, kv head), flattened as row = t * group + head, over a range of keys. Per 32 keys
//   S^T[32 keys x 16 rows] = K . Q^T     K's codes from memory into registers, converted there (v_cvt_scalef32_pk_bf16_fp4:
//                                        every 4-bit value is a bf16 number)
//   P^T = exp2((S - m) scale log2 e)     two lane exchanges for a row's maximum
//   O^T[dims x 16 rows]   += V^T . P^T   V converted, through LDS (8 KiB of the wave's own), read transposed
// The products are 16x16x32 bf16 MFMAs with exact K and V. Q is carried as bf16 parts of its f32 value (two;
// f32 storage three), so scores and LSE have f32 accuracy; P as one for bf16, two for f16 and three for f32.
// Lane (r, j) = (lane & 15, lane >> 4) holds, of key r of a 16-key block, the dims from j DP / 4 on (a 16- or
// 8-byte piece of the codes, which lies in one group of 32, one scale), and of S^T row r, keys 4 j .. 4 j + 3
// of each block: the order of the dims and of the keys in a product is free, so Q and V are taken in these.
// The codes of the next 32 keys, and the table entries of those behind, are on their way meanwhile.
constexpr int kFp4Start = 4;  // steps that the start of a unit counts for in the split

template <typename T, int DP, int NB>
struct Fp4Cfg {
    static constexpr bool F32 = std::is_same<T, float>::value;
    static constexpr int NQ = F32 ? 3 : 2;                                            // parts of Q
    static constexpr int NP = F32 ? 3 : std::is_same<T, f16_t>::value ? 2 : 1;  // of P
    static constexpr int KS = DP / 32;                                                 // steps of Q.K^T
    static constexpr int DB = DP / 16;                                                 // 16-dim blocks of O^T
    static constexpr int CB = DP / 8;                // bytes of codes a lane reads of a row
    static constexpr int CPR = DP / 8;               // 16-byte pieces of a row of V in LDS
    static constexpr int VB = 32 * DP * 2;           // bytes of a wave's V
    static constexpr int QUADS = NB * DB * 64;       // f32 quads of a partial
};
constexpr int kFp4Waves = 4;    // of a workgroup
constexpr int kFp4PerCu = 2;    // workgroups

struct Fp4KArgs {
    TreeArgs a;
    SmallDiv ps, grp;
    FastDiv ranges, row_blocks;
    int row_bytes;
};

// Which 16-byte column a piece of a V row is kept in: piece ^ fp4_swizzle(row). Sixteen rows of one piece (the
// stores), and sixteen rows of two pieces (the transposing reads), lie in all columns alike.
template <int CPR>
__device__ __forceinline__ int fp4_swizzle(int row) {
    if constexpr (CPR == 16) return ((row & 3) << 2) | ((row >> 2) & 3);
    else return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

// Maximum (sum) over the lanes that hold the same row: lane ^ 16, lane ^ 32.
__device__ __forceinline__ float max_rows(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_rows(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Two codes (byte B of w) times the scale whose exponent `s` has, as a pair of bf16.
template <int B>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float s) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, s, B));
}
__device__ __forceinline__ u32x4_t fp4_eight(uint32_t w, float s) {
    return u32x4_t{fp4_pair<0>(w, s), fp4_pair<1>(w, s), fp4_pair<2>(w, s), fp4_pair<3>(w, s)};
}

// The bf16 parts of eight values: part n is the rounding of what the parts before leave.
template <int N>
__device__ __forceinline__ void bf16_parts(float (&x)[8], u32x4_t (&out)[N]) {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t p = pack_bf16(x[2 * j], x[2 * j + 1]);
            out[n][j] = p;
            if (n + 1 < N) {
                x[2 * j] -= bf16_lo(p);
                x[2 * j + 1] -= bf16_hi(p);
            }
        }
}

// Four dims of a finished row, as in tree.hip.
template <typename T>
__device__ __forceinline__ void fp4_write(const TreeArgs& a, int s, int kvh, int row, int d, f32x4_t o,
                                          float m, float l, const SmallDiv& grp) {
    const int t = grp.div(row), hq = kvh * a.group + row - t * a.group;
    const bool none = l == 0.0f;
    const float inv = none ? 0.0f : 1.0f / l;
    const int64_t at = (((int64_t)s * a.max_tokens + t) * a.q_heads + hq) * a.head_dim + d;
    if (none) o = f32x4_t{0.f, 0.f, 0.f, 0.f};
    if constexpr (std::is_same<T, float>::value)
        *(f32x4_t*)((float*)a.o + at) = o * inv;
    else
        *(u32x2_t*)((uint16_t*)a.o + at) = u32x2_t{Half<T>::pack(o[0] * inv, o[1] * inv),
                                                   Half<T>::pack(o[2] * inv, o[3] * inv)};
    if (d == 0)
        a.lse[((int64_t)s * a.q_heads + hq) * a.max_tokens + t] = none ? -INFINITY : m * a.scale + logf(l);
}

// Steps of 32 keys that sequence s reads.
__device__ __forceinline__ int fp4_steps(const TreeArgs& a, int rows, int len) {
    int n = (rows + 31) / 32, before;
    if (a.window) n -= tree_skip(a, rows, len, 32, &before);
    return n;
}

template <typename T, int DP, int NB, int HW>
__global__ __launch_bounds__(64 * kFp4Waves, NB == 1 ? 2 : 1) void fp4_split(Fp4KArgs ka) {
    using C = Fp4Cfg<T, DP, NB>;
    constexpr int KS = C::KS, DB = C::DB, NQ = C::NQ, NP = C::NP;
    constexpr int KG = kFp4Waves / HW;  // ranges of a workgroup
    __shared__ __attribute__((aligned(1024))) uint8_t smem[kFp4Waves * C::VB];
    const TreeArgs& a = ka.a;
    const int lane = threadIdx.x & 63, r16 = lane & 15, j4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int hd = wave % HW;
    uint8_t* const vlds = smem + wave * C::VB;
    const int D = a.head_dim;
    const int logical = xcd_remap(blockIdx.x, gridDim.x);
    const int wg = __builtin_amdgcn_readfirstlane((int)ka.row_blocks.div((uint32_t)logical));
    const int rb = logical - wg * (int)ka.row_blocks.d;
    const int range = wg * KG + wave / HW;
    const int units = a.kv_heads / HW;  // of a sequence

    // ---- this wave's range of steps [pos, end), and the sequence that holds the first (as in tree.hip)
    auto rows_of = [&](int i) { return i < a.n_seqs ? tree_rows_of(a, i) : 0; };
    auto len_of = [&](int i) { return a.tree_lens[min(i, a.n_seqs - 1)]; };
    int mine = 0, count = 0;
    for (int i = lane; i < a.n_seqs; i += 64) {
        const int rows = rows_of(i), n = rows ? fp4_steps(a, rows, len_of(i)) : 0;
        mine += units * n;
        count += n ? units : 0;
    }
    const int n_steps = __builtin_amdgcn_readlane(wave_scan(mine), 63);
    const int n_units = __builtin_amdgcn_readlane(wave_scan(count), 63);
    const int ov = min(kFp4Start, (int)ka.ranges.div((uint32_t)n_steps) / 2);
    const int total = n_steps + n_units * ov;
    auto length_of = [&](int rows, int len) { return rows ? fp4_steps(a, rows, len) + ov : 0; };  // of a unit
    const int share = max(1, (int)ka.ranges.div((uint32_t)total + ka.ranges.d - 1));
    int64_t pos = (int64_t)range * share;
    const int64_t end = pos + share < total ? pos + share : total;
    const bool plans = logical == 0 && wave == 0;  // writes what fp4_combine needs
    if (plans && lane == 0) {
        a.plan[a.n_seqs] = share;
        a.plan[a.n_seqs + 1] = ov;
    }
    int s = 0, first = 0, rows_s = 0, len = 0;
    bool found = pos >= end;
    for (int base = 0, carry = 0; base < a.n_seqs && (plans || !found); base += 64) {
        const int rows = rows_of(base + lane), ln = len_of(base + lane), v = units * length_of(rows, ln);
        const int upto = carry + wave_scan(v);
        if (plans && base + lane < a.n_seqs) a.plan[base + lane] = upto - v;
        const uint64_t past = __ballot(upto > pos);
        if (!found && past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            s = base + l;
            first = __builtin_amdgcn_readlane(upto - v, l);
            rows_s = __builtin_amdgcn_readlane(rows, l);
            len = __builtin_amdgcn_readlane(ln, l);
            found = true;
        }
        carry = __builtin_amdgcn_readlane(upto, 63);
    }
    if (pos >= end) return;
    s = __builtin_amdgcn_readfirstlane(s);

    // ---- lane constants
    const int d_lane = j4 * (DP / 4);                       // first dim of this lane's piece of a row
    const bool d_ok = d_lane < D;
    const int dl = d_ok ? d_lane : 0;
    const int codes = a.kv_heads * D / 2;
    const float c2 = a.scale * kLog2e;
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s lds_v4s;

    while (pos < end) {
        while (pos >= (int64_t)first + units * length_of(rows_s, len)) {
            first += units * length_of(rows_s, len);
            ++s;
            rows_s = __builtin_amdgcn_readfirstlane(tree_rows_of(a, s));
            len = __builtin_amdgcn_readfirstlane(a.tree_lens[s]);
        }
        const int steps = fp4_steps(a, rows_s, len);
        const int in_seq = (int)(pos - first);
        const int unit = __builtin_amdgcn_readfirstlane(in_seq / (steps + ov)), kvh = unit * HW + hd;
        const int from = in_seq - unit * (steps + ov);
        const int to = (int)min((int64_t)steps + ov, from + (end - pos));
        pos += to - from;
        const int st0 = max(0, from - ov), st1 = to - ov;
        if (st1 <= st0) continue;
        const int ctx = rows_s - len;
        const int rows_total = len * a.group, r0 = rb * 16 * NB;
        if (r0 >= rows_total) continue;
        int before = 0, skip = 0;
        if (a.window) skip = tree_skip(a, rows_s, len, 32, &before);
        // steps [open0, open1) (real ones) hold keys that every row sees
        const int open1 = ctx / 32, open0 = a.window ? (max(0, rows_s - a.window) + 31) / 32 : 0;

        // ---- this lane's query rows: row 16 nb + r16 of the block
        int tok[NB], t_of[NB];
        bool row_ok[NB];
        uint64_t mask0[NB];
        u32x4_t qop[NB][KS][NQ];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int row = r0 + 16 * nb + r16, rq = min(row, rows_total - 1), t = ka.grp.div(rq);
            row_ok[nb] = row < rows_total;
            t_of[nb] = t;
            tok[nb] = s * a.max_tokens + t;
            mask0[nb] = 0;
            if (row_ok[nb] && a.masks && a.words == 1) mask0[nb] = a.masks[tok[nb]];
            int rope_pos = 0;
            if (a.rope_table) {
                rope_pos = a.positions ? a.positions[tok[nb]] : ctx + t;
                row_ok[nb] = row_ok[nb] && rope_pos >= 0 && rope_pos < a.rope_positions;
            }
            const int64_t q0 = ((int64_t)tok[nb] * a.q_heads + kvh * a.group + rq - t * a.group) * D + dl;
            const float2* const cs =
                a.rope_table + ((int64_t)(row_ok[nb] ? rope_pos : 0) + a.rope_offset) * (D >> 1) + dl / 2;
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                float x[8];
                if constexpr (C::F32) load8<T>((const float*)a.q + q0 + 8 * c, 0, x);
                else load8<T>((const uint16_t*)a.q + q0 + 8 * c, 0, x);
                if (a.rope_table) {
                    const f32x4_t w0 = *(const f32x4_t*)(cs + 4 * c), w1 = *(const f32x4_t*)(cs + 4 * c + 2);
                    const float c8[8] = {w0[0], w0[1], w0[2], w0[3], w1[0], w1[1], w1[2], w1[3]};
                    rope4(x, c8);
                }
                const bool ok = row_ok[nb] && d_ok;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = ok ? x[e] : 0.0f;
                bf16_parts<NQ>(x, qop[nb][c]);
            }
        }
        f32x4_t oacc[NB][DB];
        float m_run[NB], l_run[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m_run[nb] = -INFINITY;
            l_run[nb] = 0.0f;
#pragma unroll
            for (int db = 0; db < DB; ++db) oacc[nb][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
        const int* const table = a.block_tables + (int64_t)s * a.max_pages;
        const int head_codes = (kvh * D + dl) / 2, head_scales = codes + (kvh * D + dl) / 32;

        auto real = [&](int step) { return a.window && step >= before ? step + skip : step; };
        // table entries of the two keys of this lane in a step, -1 outside the pool
        auto pages_of = [&](int step, int (&page)[2]) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int key = min(real(step) * 32 + 16 * b + r16, rows_s - 1);
                page[b] = table[ka.ps.div(key)];
            }
        };
        // their codes and scales (those of row 0 of the pool for a page outside it)
        typedef uint32_t piece_t __attribute__((ext_vector_type(C::CB / 4)));
        struct Tile {
            piece_t k[2], v[2];
            uint32_t ks[2], vs[2];
            uint32_t there;  // bit i: key i of the 32 is there
        };
        auto load_tile = [&](int step, const int (&page)[2], Tile& t) {
            t.there = 0;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int key_raw = real(step) * 32 + 16 * b + r16, key = min(key_raw, rows_s - 1);
                const int lp = ka.ps.div(key);
                const bool in = (unsigned)page[b] < (unsigned)a.physical_pages;
                const int64_t row = in ? (int64_t)page[b] * a.page_size + key - lp * a.page_size : 0;
                const uint8_t* const kp = (const uint8_t*)a.k_pool + row * ka.row_bytes;
                const uint8_t* const vp = (const uint8_t*)a.v_pool + row * ka.row_bytes;
                t.k[b] = __builtin_nontemporal_load((const piece_t*)(kp + head_codes));
                t.v[b] = __builtin_nontemporal_load((const piece_t*)(vp + head_codes));
                t.ks[b] = kp[head_scales];
                t.vs[b] = vp[head_scales];
                t.there |= ((uint32_t)__ballot(in && key_raw < rows_s) & 0xffffu) << (16 * b);
            }
        };

        int page[2];
        Tile next;
        pages_of(st0, page);
        load_tile(st0, page, next);
        if (st0 + 1 < st1) pages_of(st0 + 1, page);
#pragma unroll 1
        for (int step = st0; step < st1; ++step) {
            const Tile cur = next;
            if (step + 1 < st1) {
                load_tile(step + 1, page, next);
                if (step + 2 < st1) pages_of(step + 2, page);
            }
            const int rs = real(step), key0 = rs * 32;
            // ---- V into LDS: row 16 b + r16, dims d_lane ..; without NaN (the score has it then)
            uint32_t v_nan = 0;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const bool nan = cur.vs[b] == 255u && d_ok;
                const uint64_t any = __ballot(nan);
                v_nan |= (uint32_t)((any | any >> 16 | any >> 32 | any >> 48) & 0xffffu) << (16 * b);
                const float sc = __uint_as_float(nan ? 0u : cur.vs[b] << 23);
                const int row = 16 * b + r16;
#pragma unroll
                for (int c = 0; c < C::CB / 4; ++c) {
                    const uint32_t w = nan || !d_ok ? 0u : cur.v[b][c];
                    const int piece = d_lane / 8 + c;
                    *(u32x4_t*)(vlds + row * (2 * DP) + ((piece ^ fp4_swizzle<C::CPR>(row)) << 4)) =
                        fp4_eight(w, sc);
                }
            }
            // ---- K operands
            u32x4_t kop[2][KS];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const float sc = __uint_as_float(cur.ks[b] << 23);
#pragma unroll
                for (int c = 0; c < KS; ++c) kop[b][c] = fp4_eight(d_ok ? cur.k[b][c] : 0u, d_ok ? sc : 1.0f);
            }
            const bool masked = rs < open0 || rs >= open1 || cur.there != 0xffffffffu || v_nan;
            u32x4_t pop[NB][NP];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                f32x4_t sc[2] = {f32x4_t{0.f, 0.f, 0.f, 0.f}, f32x4_t{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
                for (int c = 0; c < KS; ++c)
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int b = 0; b < 2; ++b)
                            sc[b] = Half<bf16_t>::mfma16(kop[b][c], qop[nb][c][n], sc[b]);
                wait_mfma(sc[0]);
                wait_mfma(sc[1]);
                if (masked) {
                    uint32_t w;
                    if (a.window) w = window_word(a, ctx + t_of[nb], key0);
                    else if (a.masks) w = mask_word(a, row_ok[nb], tok[nb], mask0[nb], key0 - ctx);
                    else w = causal_word(ctx + t_of[nb], key0);
                    const uint32_t see = (w & cur.there) >> (4 * j4), bad = v_nan >> (4 * j4);
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if ((bad >> (16 * b + i)) & 1) sc[b][i] = __uint_as_float(0x7fc00000u);
                            if (!((see >> (16 * b + i)) & 1)) sc[b][i] = -INFINITY;
                        }
                }
                float mt = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                                 fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
                mt = max_rows(mt);
                // (the running maximum moves when a step's exceeds it by more than 2^8 in probability)
                const bool need = mt * c2 > m_run[nb] * c2 + 8.0f;
                if (__any(need)) {
                    const float m_use = need ? mt : m_run[nb];
                    const float alpha = m_run[nb] == m_use ? 1.0f : fast_exp2((m_run[nb] - m_use) * c2);
                    l_run[nb] *= alpha;
#pragma unroll
                    for (int db = 0; db < DB; ++db) oacc[nb][db] *= alpha;
                    m_run[nb] = m_use;
                }
                const float neg = m_run[nb] == -INFINITY ? 0.0f : -m_run[nb] * c2;
                float p[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    p[i] = fast_exp2(fmaf(sc[i >> 2][i & 3], c2, neg));
                    l_run[nb] += p[i];
                }
                bf16_parts<NP>(p, pop[nb]);
            }
            // ---- O^T += V^T . P^T: dims 16 db + r16 of the keys 4 j4 .. and 16 + 4 j4 ..
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                u32x4_t vop;
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int row = 16 * b + 4 * j4 + (r16 >> 2), piece = 2 * db + ((r16 & 3) >> 1);
                    const uint8_t* const src = vlds + row * (2 * DP) +
                                               ((piece ^ fp4_swizzle<C::CPR>(row)) << 4) + 8 * (r16 & 1);
                    const u32x2_t x = __builtin_bit_cast(
                        u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)src));
                    vop[2 * b] = x[0];
                    vop[2 * b + 1] = x[1];
                }
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int n = 0; n < NP; ++n)
                        oacc[nb][db] = Half<bf16_t>::mfma16(vop, pop[nb][n], oacc[nb][db]);
            }
        }

        // ---- finished rows to O and LSE, partial ones to their slot
        const bool whole = st0 == 0 && st1 == steps;
        const int64_t slot =
            ((2 * ((int64_t)range * ka.row_blocks.d + rb) + (st0 == 0 ? 1 : 0)) * HW + hd);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float l = sum_rows(l_run[nb]);
            if (!row_ok[nb]) l = 0.0f;
            const int row = r0 + 16 * nb + r16;
            if (whole) {
                if (row < rows_total)
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        const int d = 16 * db + 4 * j4;
                        if (d < D) fp4_write<T>(a, s, kvh, row, d, oacc[nb][db], m_run[nb], l, ka.grp);
                    }
            } else {
                f32x4_t* const out = (f32x4_t*)a.part_o + slot * C::QUADS + nb * DB * 64 + lane;
#pragma unroll
                for (int db = 0; db < DB; ++db) out[db * 64] = oacc[nb][db];
                if (j4 == 0) a.part_ml[slot * 16 * NB + 16 * nb + r16] = make_float2(m_run[nb], l);
            }
        }
    }
}

// Merges the partials of the units that several ranges share, in their order, and writes the rows past each
// sequence's tokens. A thread ends with one quad: dims 16 db + 4 j4 .. of a row.
template <typename T, int DP>
__global__ __launch_bounds__(256) void fp4_combine(Fp4KArgs ka, int hw, int nb_rows, int blocks) {
    const TreeArgs& a = ka.a;
    constexpr int DB = DP / 16, PER = DB * 64 / 256;  // quads of 16 rows for a thread of 256
    const int D = a.head_dim, tid = threadIdx.x;
    int id = blockIdx.x;
    const int part = id % PER;
    id /= PER;
    const int b16 = id % blocks, sh = id / blocks, kvh = sh % a.kv_heads, s = sh / a.kv_heads;
    const int lane = tid & 63, db = part * 4 + (tid >> 6);
    const int row = b16 * 16 + (lane & 15), d = 16 * db + 4 * (lane >> 4);
    const int rows_all = a.max_tokens * a.group;
    const int rows_s = tree_rows_of(a, s), len = rows_s ? a.tree_lens[s] : 0;
    const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
    if (row < rows_all && row >= len * a.group && d < D)
        fp4_write<T>(a, s, kvh, row, d, zero, 0.0f, 0.0f, ka.grp);
    if (b16 * 16 >= len * a.group) return;
    const int share = a.plan[a.n_seqs], ov = a.plan[a.n_seqs + 1];
    const int steps = fp4_steps(a, rows_s, len);
    const uint32_t u0 = (uint32_t)a.plan[s] + (uint32_t)(kvh / hw) * (uint32_t)(steps + ov) + (uint32_t)ov;
    const int g0 = (int)(u0 / (uint32_t)share), g1 = (int)((u0 + steps - 1) / (uint32_t)share);
    if (g0 == g1) return;  // finished by the range that covers it
    const int rb = b16 / nb_rows, in = b16 - rb * nb_rows, nrb = (int)ka.row_blocks.d;
    const float c2 = a.scale * kLog2e;
    float M = -INFINITY, L = 0.0f;
    f32x4_t o = zero;
    constexpr int UN = 4;
    for (int g = g0; g <= g1; g += UN) {
        float2 ml[UN];
        f32x4_t x[UN];
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            const int at = min(g + i, g1);
            const int64_t slot = (2 * ((int64_t)at * nrb + rb) + (at == g0 ? 1 : 0)) * hw + kvh % hw;
            ml[i] = a.part_ml[slot * 16 * nb_rows + in * 16 + (lane & 15)];
            x[i] = ((const f32x4_t*)a.part_o)[(slot * nb_rows + in) * (DB * 64) + db * 64 + lane];
        }
#pragma unroll
        for (int i = 0; i < UN; ++i) {
            if (g + i > g1 || ml[i].y == 0.0f) continue;  // (it saw nothing)
            const float mx = fmaxf(M, ml[i].x);
            const float w0 = L == 0.0f ? 0.0f : fast_exp2((M - mx) * c2);
            const float w1 = fast_exp2((ml[i].x - mx) * c2);
            M = mx;
            L = fmaf(ml[i].y, w1, L * w0);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(x[i][e], w1, o[e] * w0);
        }
    }
    if (row < len * a.group && d < D) fp4_write<T>(a, s, kvh, row, d, o, M, L, ka.grp);
}

struct Fp4Shape {
    int nb, hw, row_blocks, ranges, workgroups;
};
static Fp4Shape fp4_shape(const TreeArgs& a) {
    Fp4Shape s;
    const int rows = a.max_tokens * a.group;
    s.nb = rows <= 16 ? 1 : 2;
    s.hw = a.kv_heads % 4 == 0 ? 4 : a.kv_heads % 2 == 0 ? 2 : 1;
    s.row_blocks = (rows + 16 * s.nb - 1) / (16 * s.nb);
    const int wgs = std::max(1, kFp4PerCu * device_cus() / s.row_blocks);
    s.ranges = wgs * (kFp4Waves / s.hw);
    s.workgroups = wgs * s.row_blocks;
    return s;
}

// (one size for every shape, as tree_workspace: two partials a wave of at most 32 rows of 128 dims)
size_t fp4_workspace(Dtype, const TreeArgs& a, size_t* ml_offset, size_t* plan_offset) {
    const size_t waves = std::max<size_t>((size_t)kFp4PerCu * device_cus(), fp4_shape(a).workgroups) * kFp4Waves;
    *ml_offset = waves * 2 * 32 * 128 * 4;
    *plan_offset = *ml_offset + waves * 2 * 32 * 8;
    return *plan_offset + ((size_t)a.n_seqs + 2) * 4;
}

template <typename T, int DP>
static void fp4_launch(Fp4KArgs& ka, const Fp4Shape& sh, hipStream_t st, void (*between)(void*), void* user) {
    const TreeArgs& a = ka.a;
    auto split = [&](auto nb, auto hw) {
        fp4_split<T, DP, decltype(nb)::value, decltype(hw)::value>
            <<<sh.workgroups, 64 * kFp4Waves, 0, st>>>(ka);
    };
    auto heads = [&](auto nb) {
        if (sh.hw == 4) split(nb, std::integral_constant<int, 4>{});
        else if (sh.hw == 2) split(nb, std::integral_constant<int, 2>{});
        else split(nb, std::integral_constant<int, 1>{});
    };
    if (sh.nb == 1) heads(std::integral_constant<int, 1>{});
    else heads(std::integral_constant<int, 2>{});
    if (between) between(user);
    const int blocks = (a.max_tokens * a.group + 15) / 16;
    const unsigned g = (unsigned)((int64_t)a.n_seqs * a.kv_heads * blocks * (DP / 64));
    fp4_combine<T, DP><<<g, 256, 0, st>>>(ka, sh.hw, sh.nb, blocks);
}

void launch_fp4_attention(Dtype dt, const TreeArgs& a, hipStream_t s, unsigned grid[3],
                          unsigned* block, unsigned* rows, void (*between)(void*), void* user) {
    const Fp4Shape sh = fp4_shape(a);
    Fp4KArgs ka;
    ka.a = a;
    ka.ps = SmallDiv((uint32_t)a.page_size);
    ka.grp = SmallDiv((uint32_t)a.group);
    ka.ranges = FastDiv((uint32_t)sh.ranges);
    ka.row_blocks = FastDiv((uint32_t)sh.row_blocks);
    ka.row_bytes = fp4_row_bytes(a.kv_heads, a.head_dim);
    grid[0] = (unsigned)sh.workgroups;
    grid[1] = grid[2] = 1;
    *block = 64 * kFp4Waves;
    *rows = (unsigned)(16 * sh.nb);
    auto go = [&](auto tag) {
        using T = decltype(tag);
        if (a.head_dim <= 64) fp4_launch<T, 64>(ka, sh, s, between, user);
        else fp4_launch<T, 128>(ka, sh, s, between, user);
    };
    switch (dt) {
        case Dtype::BF16: go(bf16_t{}); break;
        case Dtype::F16: go(f16_t{}); break;
        default: go(float{}); break;
    }
}

}  // namespace fa
