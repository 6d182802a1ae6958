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

// Nearest codes of eight values over the scale whose exponent `s` has, ties to the even ones, past 6 the largest
// (v_cvt_scalef32_pk_fp4_f32 does just that; with comparisons the append of 48 x 512 bf16 rows took 29 us, not 19).
__device__ __forceinline__ uint32_t fp4_codes(const float (&x)[8], float s) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], s, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], s, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], s, 3);
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

// One thread: eight values of K and of V of a row; four neighbouring threads share a scale. Memory bounds it: bf16
// rows of 8 heads of 128, 48 sequences of up to 512, 19 us; 16-byte loads, 4-byte stores.
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
        const uint32_t w = fp4_codes(x, __uint_as_float((uint32_t)scale << 23));
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

// As append_fp4, the other way: 20 us for the same rows.
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
//   S^T[32 keys x 16 rows] = K . Q^T     K's codes are converted in registers (v_cvt_scalef32_pk_bf16_fp4:
//                                        every 4-bit value is a bf16 number)
//   P^T = exp2((S - m) scale log2 e)     two lane exchanges for a row's maximum
//   O^T[dims x 16 rows]   += V^T . P^T   V converted, through LDS (4 KiB of the wave's own), read transposed
// The products are 16x16x32 bf16 MFMAs with exact K and V. Q is carried as bf16 parts of its f32 value (two;
// f32 storage three), so scores and LSE have f32 accuracy; P as one for bf16, two for f16 and three for f32.
// Lane (r, j) = (lane & 15, lane >> 4) holds, of key r of a 16-key block, the dims from j DP / 4 on (a 16- or
// 8-byte piece of the codes, which lies in one group of 32, one scale), and of S^T row r, keys 4 j .. 4 j + 3
// of each block: the order of the dims and of the keys in a product is free, so Q and V are taken in these.
// Where the head count is a multiple of four, a workgroup's waves take a head each over the same keys and move
// the rows of the four into LDS together, 16 bytes a lane in the order of the row (global_load_lds), three steps
// deep with one barrier a step. With another count a wave loads its own codes into registers, two steps deep;
// its loads then touch 64 bytes of a row each, and their addresses are what bounds it (64 contexts of 512 to 8192
// tokens, 8 heads of 128, single tokens: 119 us that way, 78 together; with the eight heads in one workgroup a CU,
// 83). More than 16 rows of up to 64 dims are the exception: what they compute bounds them, and the waves do it
// better apart (16 contexts of up to 6000 tokens, trees of 24, 8 heads of 64: 48 us apart, 53 together; of 128:
// 80 and 73).
constexpr int kFp4Start = 4;  // steps that the start of a unit counts for in the split

template <typename T, int DP, int NB, int HW>
struct Fp4Cfg {
    static constexpr bool F32 = std::is_same<T, float>::value;
    static constexpr bool COOP = HW == 4;
    static constexpr int NW = 4;                                                       // waves
    static constexpr int NQ = F32 ? 3 : 2;                                            // parts of Q
    static constexpr int NP = F32 ? 3 : std::is_same<T, f16_t>::value ? 2 : 1;  // of P
    static constexpr int KS = DP / 32;                                                 // steps of Q.K^T
    static constexpr int DB = DP / 16;                                                 // 16-dim blocks of O^T
    static constexpr int CB = DP / 8;                // bytes of codes a lane reads of a row
    static constexpr int VB = 32 * 128;              // bytes of a wave's V: 64 dims of 32 keys
    static constexpr int VP = DP / 64;               // such parts
    // of them, read before the softmax, as the registers allow
    static constexpr int VEARLY = VP == 2 && NB == 1 && !F32 ? 2 : VP == 2 && NB == 2 && !F32 && COOP ? 0 : 1;
    static constexpr int QUADS = NB * DB * 64;       // f32 quads of a partial
    // the rows are loaded while the first keys are on their way, as the registers allow
    static constexpr bool LATE = F32 || NB == 1 || DP == 64;
    // waves a SIMD, as the registers allow
    static constexpr int WAVES = NB == 2 && DP == 128 && (F32 || !COOP) ? 1 : 2;
    // COOP: 16-byte pieces of a row segment in LDS (an odd number: sixteen rows of one column lie in all
    // banks), which is also the number of transfer instructions of a step (K and V); those of a wave
    static constexpr int RP = (HW * DP / 2 + HW * DP / 32 + 15) / 16 | 1;
    static constexpr int NI = (RP + NW - 1) / NW;
    static constexpr int STAGE = RP * 1024;
    static constexpr int NST = 3;
    static constexpr int SMEM = NW * VB + (COOP ? NST * STAGE : 0);
};
constexpr int kFp4Pages = 256;  // block-table entries that a wave (COOP: the workgroup) holds in LDS at a time

struct Fp4KArgs {
    TreeArgs a;
    SmallDiv ps, grp;
    FastDiv ranges, row_blocks;
    int row_bytes;
};

// Which 16-byte column (of 8) a piece of a V row is kept in: piece ^ fp4_swizzle(row), so that eight rows of one
// piece (a store's clock) and the two neighbouring pieces of eight rows (half a transposing read) lie in all banks.
__device__ __forceinline__ int fp4_swizzle(int row) { return row & 7; }

__device__ __forceinline__ void fp4_to_lds16(const void* p, uint32_t lds) {
    asm volatile("global_load_lds_dwordx4 %0, off" : : "v"(p), "{m0}"(lds));
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
__global__ __launch_bounds__((64 * Fp4Cfg<T, DP, NB, HW>::NW), (Fp4Cfg<T, DP, NB, HW>::WAVES))
void fp4_split(Fp4KArgs ka) {
    using C = Fp4Cfg<T, DP, NB, HW>;
    constexpr int KS = C::KS, DB = C::DB, NQ = C::NQ, NP = C::NP;
    constexpr bool COOP = C::COOP;
    constexpr int NW = C::NW, KG = NW / HW;  // waves, and ranges, of a workgroup
    __shared__ __attribute__((aligned(1024))) uint8_t smem[C::SMEM];
    __shared__ int bt_lds[COOP ? 1 : NW][kFp4Pages];
    __shared__ int bad_lds[NW];
    __shared__ uint64_t row_lds[COOP ? NW : 1][32];  // byte offset of each row of the step to come
    const TreeArgs& a = ka.a;
    const int lane = threadIdx.x & 63, r16 = lane & 15, j4 = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int hd = wave % HW;
    uint8_t* const vlds = smem + wave * C::VB;
    int* const bt = bt_lds[COOP ? 0 : wave];
    const int D = a.head_dim;
    const int logical = xcd_remap(blockIdx.x, gridDim.x);
    const int wg = __builtin_amdgcn_readfirstlane((int)ka.row_blocks.div((uint32_t)logical));
    const int rb = logical - wg * (int)ka.row_blocks.d;
    const int range = wg * KG + wave / HW;
    const int units = a.kv_heads / HW;  // of a sequence

    // ---- this wave's range of steps [pos, end), and the sequence that holds the first (as in tree.hip)
    auto rows_of = [&](int i, int& len) {
        const int at = min(i, a.n_seqs - 1);
        len = a.tree_lens[at];
        const int rows = tree_rows_of(a, at);
        return i < a.n_seqs ? rows : 0;
    };
    int mine = 0, count = 0, len0;
    const int rows0 = rows_of(lane, len0);  // (of the first 64 sequences: not asked for again)
    for (int i = lane; i < a.n_seqs; i += 64) {
        int rows = rows0, ln = len0;
        if (i != lane) rows = rows_of(i, ln);
        const int n = rows ? fp4_steps(a, rows, ln) : 0;
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
        int rows = rows0, ln = len0;
        if (base) rows = rows_of(base + lane, ln);
        const int v = units * length_of(rows, ln);
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
    const bool d_ok = d_lane < D;  // (else: any codes times a Q of zeros, and dims of O that do not exist)
    const int dl = d_ok ? d_lane : 0;
    const int codes = a.kv_heads * D / 2;
    const float c2 = a.scale * kLog2e;
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    const uint32_t stage0 = (uint32_t)(uintptr_t)(lds_void_t*)smem + NW * C::VB;
    const int n_ins = COOP ? (C::RP - wave + NW - 1) / NW : 0;

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
        auto load_rows = [&] {
            int dq = dl;
            asm volatile("" : "+v"(dq));  // (addresses made of it are not held, or spilled, from unit to unit)
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
                const int64_t q0 = ((int64_t)tok[nb] * a.q_heads + kvh * a.group + rq - t * a.group) * D + dq;
                const float2* const cs =
                    a.rope_table + ((int64_t)(row_ok[nb] ? rope_pos : 0) + a.rope_offset) * (D >> 1) + dq / 2;
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
        };
        if constexpr (COOP && !C::LATE) load_rows();
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
        // (this lane's scale is a byte of an aligned word of its row, which is a multiple of 16 bytes)
        const int scale_byte = (kvh * D + dl) / 32, scale_at = 8 * (scale_byte & 3);
        const int head_codes = (kvh * D + dl) / 2, head_scales = codes + (scale_byte & ~3);

        // COOP: this lane's piece in each of its wave's transfers, as its address in row 0 and its row. Pieces of a
        // step are numbered through the rows of K, then of V; the last ones of a row may not exist (the last that
        // does is fetched again).
        const uint8_t* piece_base[COOP ? C::NI : 1];
        int piece_row[COOP ? C::NI : 1];
        if constexpr (COOP) {
            // pieces of codes; of scales, whose HW D / 32 bytes (16 at most) need not begin with one
            const int cp = HW * D / 32, sp = 16 % cp == 0 ? 1 : 2;
            const int seg_codes = unit * (HW * D / 2), seg_scales = codes + (unit * (HW * D / 32) & ~15);
            int ln = lane;
            asm volatile("" : "+v"(ln));  // (as dq)
#pragma unroll
            for (int i = 0; i < C::NI; ++i) {
                const int p = min((wave + i * NW) * 64 + ln, 64 * C::RP - 1);
                const int r = p / C::RP, c = min(p - r * C::RP, cp + sp - 1);
                // (of two pieces of scales the second may lie past the row, and is not needed then)
                const int at = c < cp ? seg_codes + 16 * c : min(seg_scales + 16 * (c - cp), ka.row_bytes - 16);
                piece_row[i] = r & 31;
                piece_base[i] = (const uint8_t*)(r < 32 ? a.k_pool : a.v_pool) + at;
            }
        }
        // (with a window, `skip` steps behind the first `before` are left out: a part of the loop ends there)
        for (int at0 = st0; at0 < st1;) {
        const int shift = at0 >= before ? skip : 0, c0 = at0 + shift;
        const int part = at0 < before && skip > 0 ? min(st1, before) : st1 + shift;
        // ---- table entries of as many steps as they cover: first pool row of each page, -1 outside the pool
        const int p0 = ka.ps.div(c0 * 32);
        const int64_t reach = ((int64_t)p0 + kFp4Pages) * a.page_size;  // keys below are covered
        const int c1 = (int)min((int64_t)part, max((int64_t)c0 + 1, reach / 32));
        const int k_end = min(c1 * 32, rows_s);
        const int n_pages = ka.ps.div(k_end - 1) - p0 + 1;
        bool bad = false;
        if constexpr (COOP) __syncthreads();  // (the entries and stages before have been read)
        for (int i = COOP ? (int)threadIdx.x : lane; i < n_pages; i += COOP ? 64 * NW : 64) {
            const int page = table[p0 + i];
            const bool in = (unsigned)page < (unsigned)a.physical_pages;
            bt[i] = in ? page * a.page_size : -1;
            bad |= !in;
        }
        bad = __any(bad);
        if constexpr (COOP) {
            if (lane == 0) bad_lds[wave] = bad;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < NW; ++w) bad |= bad_lds[w] != 0;
            bad = __builtin_amdgcn_readfirstlane(bad);
        }
        // codes and scales of this lane's two keys of a step (those of row 0 for a page outside the pool)
        typedef uint32_t piece_t __attribute__((ext_vector_type(C::CB / 4)));
        struct Tile {
            piece_t k[2], v[2];
            uint32_t ks[2], vs[2];  // the word that holds the scale (COOP: the scale)
        };
        auto load_tile = [&](int step, Tile& t) {
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const int key = min(step * 32 + 16 * b + r16, k_end - 1);
                const int lp = ka.ps.div(key);
                const uint64_t row = (uint64_t)(uint32_t)(max(bt[lp - p0], 0) + key - lp * a.page_size) *
                                     (uint32_t)ka.row_bytes;
                const uint8_t* const kp = (const uint8_t*)a.k_pool + row;
                const uint8_t* const vp = (const uint8_t*)a.v_pool + row;
                t.k[b] = *(const piece_t*)(kp + head_codes);
                t.v[b] = *(const piece_t*)(vp + head_codes);
                t.ks[b] = *(const uint32_t*)(kp + head_scales);
                t.vs[b] = *(const uint32_t*)(vp + head_scales);
            }
        };
        auto scale_of = [&](uint32_t w) { return COOP ? w : (w >> scale_at) & 255u; };

        // COOP: a step's rows on their way into a stage
        auto transfer = [&](int step, int stage) {
            if (lane < 32) {
                const int key = min(step * 32 + lane, k_end - 1), lp = ka.ps.div(key);
                row_lds[wave][lane] = (uint64_t)(uint32_t)(max(bt[lp - p0], 0) + key - lp * a.page_size) *
                                      (uint32_t)ka.row_bytes;
            }
#pragma unroll
            for (int i = 0; i < C::NI; ++i) {
                if (i >= n_ins) break;
                const uint8_t* const p = piece_base[i] + row_lds[wave][piece_row[i]];
                fp4_to_lds16(p, stage0 + stage * C::STAGE + (wave + i * NW) * 1024);
            }
        };
        // a step's codes from its stage
        auto fetch = [&](int stage, Tile& t) {
            const uint8_t* const at = smem + NW * C::VB + stage * C::STAGE;
            const int cd = hd * D / 2 + dl / 2;
            const int sb = HW * D / 2 + (unit * (HW * D / 32) & 15) + (hd * D + dl) / 32;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint8_t* const k = at + (16 * b + r16) * (C::RP * 16);
                t.k[b] = *(const piece_t*)(k + cd);
                t.ks[b] = k[sb];
                const uint8_t* const v = k + 32 * C::RP * 16;
                t.v[b] = *(const piece_t*)(v + cd);
                t.vs[b] = v[sb];
            }
        };

        // One step. Not COOP: its codes are used up before the softmax, and those of the step after the next
        // take their place. (Near the end the last step's again: a branch here would have every load waited for.)
        const auto process = [&](Tile& cur, int step) {
            const int key0 = step * 32;
            // ---- V into LDS, without NaN (the score has it then), 64 dims at a time: of part t the dims
            // d_lane + 16 t .. of row 16 b + r16 in pieces 2 j4, 2 j4 + 1
            bool nan[2];
            float vsc[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint32_t e = scale_of(cur.vs[b]);
                nan[b] = e == 255u && d_ok;
                vsc[b] = __uint_as_float(e == 255u ? 0u : e << 23);
            }
            const bool any_nan = __any(nan[0] || nan[1]);
            piece_t vc[2] = {cur.v[0], cur.v[1]};
            auto write_v = [&](int t) {
#pragma unroll
                for (int b = 0; b < 2; ++b)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int row = 16 * b + r16;
                        *(u32x4_t*)(vlds + row * 128 + (((2 * j4 + c) ^ fp4_swizzle(row)) << 4)) =
                            fp4_eight(vc[b][2 * t + c], vsc[b]);
                    }
            };
            // and back transposed: dims 16 g + r16 of it (of O: block VP g + t) of the keys 4 j4 .. and 16 + 4 j4 ..
            u32x4_t vop[4 * (C::VEARLY ? C::VEARLY : 1)];
            auto read_v = [&](int to) {
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        const int row = 16 * b + 4 * j4 + (r16 >> 2), piece = 2 * g + ((r16 & 3) >> 1);
                        const uint8_t* const src =
                            vlds + row * 128 + ((piece ^ fp4_swizzle(row)) << 4) + 8 * (r16 & 1);
                        const u32x2_t x = __builtin_bit_cast(
                            u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)src));
                        vop[4 * to + g][2 * b] = x[0];
                        vop[4 * to + g][2 * b + 1] = x[1];
                    }
            };
            if constexpr (C::VEARLY > 0) write_v(0);
            // ---- scores; K's operands are converted as they are multiplied
            float ksc[2];
#pragma unroll
            for (int b = 0; b < 2; ++b) ksc[b] = __uint_as_float(d_ok ? scale_of(cur.ks[b]) << 23 : 0x3f800000u);
            f32x4_t sall[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int b = 0; b < 2; ++b) sall[nb][b] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                u32x4_t kop[2];
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    kop[b] = fp4_eight(cur.k[b][c], ksc[b]);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int b = 0; b < 2; ++b)
                            sall[nb][b] = Half<bf16_t>::mfma16(kop[b], qop[nb][c][n], sall[nb][b]);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (!COOP) load_tile(min(step + 2, c1 - 1), cur);
            // V's operands are on their way while the softmax runs
            if constexpr (C::VEARLY > 0) read_v(0);
            if constexpr (C::VEARLY == 2) {
                write_v(1);
                read_v(1);
            }
            __builtin_amdgcn_sched_barrier(0);
            const bool masked = step < open0 || step >= open1 || bad || any_nan;
            // keys that are there, and those whose V has a NaN (masked steps only)
            uint32_t there = 0, v_nan = 0;
            if (masked) {
                const int key_raw = key0 + (lane & 31), key = min(key_raw, k_end - 1);
                there = (uint32_t)__ballot(bt[ka.ps.div(key) - p0] >= 0 && key_raw < k_end);
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const uint64_t any = __ballot(nan[b]);
                    v_nan |= (uint32_t)((any | any >> 16 | any >> 32 | any >> 48) & 0xffffu) << (16 * b);
                }
            }
            u32x4_t pop[NB][NP];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                f32x4_t (&sc)[2] = sall[nb];
                wait_mfma(sc[0]);
                wait_mfma(sc[1]);
                if (masked) {
                    uint32_t w;
                    if (a.window) w = window_word(a, ctx + t_of[nb], key0);
                    else if (a.masks) w = mask_word(a, row_ok[nb], tok[nb], mask0[nb], key0 - ctx);
                    else w = causal_word(ctx + t_of[nb], key0);
                    const uint32_t see = (w & there) >> (4 * j4), odd = v_nan >> (4 * j4);
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if ((odd >> (16 * b + i)) & 1) sc[b][i] = __uint_as_float(0x7fc00000u);
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
            // ---- O^T += V^T . P^T
#pragma unroll
            for (int t = 0; t < C::VP; ++t) {
                if (t >= C::VEARLY) {
                    write_v(t);
                    read_v(0);
                }
#pragma unroll
                for (int g = 0; g < 4; ++g)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int n = 0; n < NP; ++n)
                            oacc[nb][C::VP * g + t] = Half<bf16_t>::mfma16(
                                vop[4 * (t < C::VEARLY ? t : 0) + g], pop[nb][n], oacc[nb][C::VP * g + t]);
            }
        };
        if constexpr (COOP) {
            static_assert(C::NST == 3, "two steps ahead");
            transfer(c0, 0);
            if (c0 + 1 < c1) transfer(c0 + 1, 1);
            if (C::LATE && at0 == st0) load_rows();  // (while the first keys are on their way)
            int stage = 0;
#pragma unroll 1
            for (int step = c0; step < c1; ++step) {
                // (transfers complete in order: those of the next step may be on their way)
                if (step + 1 < c1) {
                    if (n_ins == C::NI) wait_vmcnt<C::NI>();
                    else wait_vmcnt<C::NI - 1>();
                } else {
                    wait_dma();
                }
                __syncthreads();
                const int ahead = stage == 0 ? 2 : stage - 1;
                if (step + 2 < c1) transfer(step + 2, ahead);
                Tile t;
                fetch(stage, t);
                process(t, step);
                stage = stage == 2 ? 0 : stage + 1;
            }
        } else {
        Tile even, odd;
        load_tile(c0, even);
        load_tile(min(c0 + 1, c1 - 1), odd);
        if (at0 == st0) load_rows();
#pragma unroll 1
        for (int step = c0; step < c1; step += 2) {
            process(even, step);
            if (step + 1 < c1) process(odd, step + 1);
        }
        }
        at0 = c1 - shift;
        }

        // ---- finished rows to O and LSE, partial ones to their slot
        int ln = lane;
        asm volatile("" : "+v"(ln));  // (as dq)
        const bool whole = st0 == 0 && st1 == steps;
        const int64_t slot =
            ((2 * ((int64_t)range * ka.row_blocks.d + rb) + (st0 == 0 ? 1 : 0)) * HW + hd);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            float l = sum_rows(l_run[nb]);
            if (!row_ok[nb]) l = 0.0f;
            const int row = r0 + 16 * nb + (ln & 15);
            if (whole) {
                if (row < rows_total)
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        const int d = 16 * db + 4 * (ln >> 4);
                        if (d < D) fp4_write<T>(a, s, kvh, row, d, oacc[nb][db], m_run[nb], l, ka.grp);
                    }
            } else if (row < rows_total) {  // (few rows: the others are a good part of the traffic)
                f32x4_t* const out = (f32x4_t*)a.part_o + slot * C::QUADS + nb * DB * 64 + ln;
#pragma unroll
                for (int db = 0; db < DB; ++db) out[db * 64] = oacc[nb][db];
                if (j4 == 0) a.part_ml[slot * 16 * NB + 16 * nb + (ln & 15)] = make_float2(m_run[nb], l);
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
    // (all asked for together)
    const int share = a.plan[a.n_seqs], ov = a.plan[a.n_seqs + 1], before = a.plan[s], len_s = a.tree_lens[s];
    const int rows_s = tree_rows_of(a, s), len = rows_s ? len_s : 0;
    const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
    if (row < rows_all && row >= len * a.group && d < D)
        fp4_write<T>(a, s, kvh, row, d, zero, 0.0f, 0.0f, ka.grp);
    if (b16 * 16 >= len * a.group) return;
    const int steps = fp4_steps(a, rows_s, len);
    const uint32_t u0 = (uint32_t)before + (uint32_t)(kvh / hw) * (uint32_t)(steps + ov) + (uint32_t)ov;
    const int g0 = (int)(u0 / (uint32_t)share), g1 = (int)((u0 + steps - 1) / (uint32_t)share);
    if (g0 == g1) return;  // finished by the range that covers it
    if (row >= len * a.group) return;
    const int rb = b16 / nb_rows, in = b16 - rb * nb_rows, nrb = (int)ka.row_blocks.d;
    const float c2 = a.scale * kLog2e;
    float M = -INFINITY, L = 0.0f;
    f32x4_t o = zero;
    constexpr int UN = 8;
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
    if (d < D) fp4_write<T>(a, s, kvh, row, d, o, M, L, ka.grp);
}

struct Fp4Shape {
    int nb, hw, nw, row_blocks, ranges, workgroups;
};
// Calls f with the 16-row blocks a wave and the heads of a launch as constants.
template <typename T, int DP, typename F>
static auto fp4_dispatch(const TreeArgs& a, F f) {
    using std::integral_constant;
    auto heads = [&](auto nb) {
        if constexpr (DP == 128 || decltype(nb)::value == 1)
            if (a.kv_heads % 4 == 0) return f(nb, integral_constant<int, 4>{});
        if (a.kv_heads % 2 == 0) return f(nb, integral_constant<int, 2>{});
        return f(nb, integral_constant<int, 1>{});
    };
    return a.max_tokens * a.group <= 16 ? heads(integral_constant<int, 1>{}) : heads(integral_constant<int, 2>{});
}
template <typename T, int DP>
static Fp4Shape fp4_shape_t(const TreeArgs& a) {
    return fp4_dispatch<T, DP>(a, [&](auto nb, auto hw) {
        using C = Fp4Cfg<T, DP, decltype(nb)::value, decltype(hw)::value>;
        Fp4Shape s;
        s.nb = decltype(nb)::value;
        s.hw = decltype(hw)::value;
        s.nw = C::NW;
        s.row_blocks = (a.max_tokens * a.group + 16 * s.nb - 1) / (16 * s.nb);
        // one round of workgroups
        const int wgs = std::max(1, C::WAVES * 4 / C::NW * device_cus() / s.row_blocks);
        s.ranges = wgs * (C::NW / s.hw);
        s.workgroups = wgs * s.row_blocks;
        return s;
    });
}
static Fp4Shape fp4_shape(Dtype dt, const TreeArgs& a) {
    if (a.head_dim <= 64) return dt == Dtype::F32 ? fp4_shape_t<float, 64>(a) : fp4_shape_t<bf16_t, 64>(a);
    return dt == Dtype::F32 ? fp4_shape_t<float, 128>(a) : fp4_shape_t<bf16_t, 128>(a);
}

// (one size for every shape, as tree_workspace: two partials a wave, at most 64 rows of 128 dims of them on a
// CU; a single range, which more row blocks than workgroups have, leaves some with fewer than four heads)
size_t fp4_workspace(Dtype dt, const TreeArgs& a, size_t* ml_offset, size_t* plan_offset) {
    const size_t rows = std::max<size_t>((size_t)device_cus() * 2, (size_t)fp4_shape(dt, a).row_blocks * 2) *
                        32 * 4 * 2;
    *ml_offset = rows * 128 * 4;
    *plan_offset = *ml_offset + rows * 8;
    return *plan_offset + ((size_t)a.n_seqs + 2) * 4;
}

template <typename T, int DP>
static void fp4_launch(Fp4KArgs& ka, const Fp4Shape& sh, hipStream_t st, void (*between)(void*), void* user) {
    const TreeArgs& a = ka.a;
    fp4_dispatch<T, DP>(a, [&](auto nb, auto hw) {
        fp4_split<T, DP, decltype(nb)::value, decltype(hw)::value><<<sh.workgroups, 64 * sh.nw, 0, st>>>(ka);
    });
    if (between) between(user);
    const int blocks = (a.max_tokens * a.group + 15) / 16;
    const unsigned g = (unsigned)((int64_t)a.n_seqs * a.kv_heads * blocks * (DP / 64));
    fp4_combine<T, DP><<<g, 256, 0, st>>>(ka, sh.hw, sh.nb, blocks);
}

void launch_fp4_attention(Dtype dt, const TreeArgs& a, hipStream_t s, unsigned grid[3],
                          unsigned* block, unsigned* rows, void (*between)(void*), void* user) {
    const Fp4Shape sh = fp4_shape(dt, a);
    Fp4KArgs ka;
    ka.a = a;
    ka.ps = SmallDiv((uint32_t)a.page_size);
    ka.grp = SmallDiv((uint32_t)a.group);
    ka.ranges = FastDiv((uint32_t)sh.ranges);
    ka.row_blocks = FastDiv((uint32_t)sh.row_blocks);
    ka.row_bytes = fp4_row_bytes(a.kv_heads, a.head_dim);
    grid[0] = (unsigned)sh.workgroups;
    grid[1] = grid[2] = 1;
    *block = (unsigned)(64 * sh.nw);
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
