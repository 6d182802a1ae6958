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

#include "tree.hpp"

namespace fa {

// Rows of one (sequence, kv head) are flattened as row = t * group + head, so every K/V byte read
// serves all of them. A workgroup holds RW blocks of 32 rows; its waves are RW row blocks times HW kv
// heads times KW key groups. Per 32 keys and wave, the products transposed so that a lane owns one query
// row:
//   S^T[32 keys x 32 rows] = K . Q^T     K from LDS (A operand), Q in registers (B)
//   P^T = exp2((S - m) scale log2 e)     one lane exchange (lane ^ 32) for the row maximum
//   O^T[dims x 32 rows]   += V^T . P^T   V read transposed from LDS; the S^T accumulator is the P^T
//                                        operand as it stands, V's keys are taken in its order
// K and V rows go straight from memory into LDS, 16 bytes a lane, one to three tiles ahead; the LDS column
// of a piece is XORed with its row so that both operand reads are free of bank conflicts without padding
// (none counted). Rows that do not exist, and dims past head_dim, are fetched from 16 zero bytes.
// 16-bit storage: the rotated Q is kept as a 16-bit high part and the rounding of its residual, two
// MFMAs a step, so that scores and LSE carry f32 accuracy; P is rounded once to the storage type (its
// sum is taken before), an error of the size of O's own rounding. f16 has no normal numbers below 2^-14 and
// nothing below 2^-25: its P is kept 2^7 times as large (at most 2^15, as the running maximum may lag by
// 2^8), so that a key loses 2^-32 of the largest one's weight at most, and 10^5 small ones beside a large
// one 2^-15 of O.
//
// The lengths are known on the GPU only, so the launch has a fixed number of workgroups; each finds its
// share by a prefix sum over the sequences: the steps (KT keys) of all (sequence, kv head) units laid
// end to end, with a few steps' worth before each for its start, are cut into equal ranges. A unit that
// one range covers is finished there; the others leave partial (O, m, l), at most two a workgroup, that
// tree_combine merges in their order.
//
// What bounds it (both launches, Hq32 Hkv8 D128 bf16, pages of 16 rows, contexts of 512..8192):
//   64 sequences, one token: 1.16 GB in 192 us, 6.0 TB/s; memory (a copy reaches 5.16 TB/s here, loads
//     alone 6.75). What is left is each unit's start, while its workgroup does not stream.
//   24 sequences, 16 / 32 / 64 tokens each: 92 / 103 / 163..178 us (by the box). 64 tokens fill 256
//     rows: the matrix cores are busy 0.47 of the CUs' busy cycles, 0.51 over contexts of 16384 (trees of 32
//     to 64 tokens leave a fifth of the waves without rows; two waves a SIMD, whose softmax and products
//     overlap only in part), and a unit's start (its lengths, table entries, Q with its angles, first tile,
//     masked blocks, end) takes as long as six steps.
//   One sequence, 5 tokens, 1000 keys, Hq16 Hkv4 D64: 12.9 us, the latency of two launches (8 and 5) and of
//     four dependent loads in the first (lengths; table entries; Q; tile). Its 32 steps are one range each,
//     and consecutive ranges run on one XCD, here all on the first.
// The simplest kernel of this layout (operands read by each lane from memory, no stages) took 7254, 20521
// and 205 us for the first, the 64-token and the last of these.

// Sixteen zero bytes: what rows and dims that do not exist are fetched from.
__device__ __attribute__((aligned(16))) uint32_t tree_zero[4];

// Scheduling groups (LLVM sched_group_barrier masks: 0x2 VALU, 0x8 MFMA, 0x100 DS read, 0x400 transcendental).
#define FA_SG(mask, n) __builtin_amdgcn_sched_group_barrier(mask, n, 0)

constexpr int kTreePages = 1024;  // block-table entries held in LDS at a time
// Steps that the start of a unit counts for in the split (its table entries, Q, first tile, masked keys and
// end take as long), but at most half of a range's steps: with few steps a range the split would be uneven.
// 24 trees of 64 tokens over 512..8192 bf16 keys, Hq32 Hkv8: 198 us with 0, 189 / 182 / 184 / 192 with 3 / 6
// / 9 / 14; 64 single tokens 212 / 209 / 210 / 213 / 212. (Measured at these two shapes of 128 dims; other
// types and row counts, whose steps are shorter or longer, take the same.)
constexpr int kTreeStart = 6;

// RW row blocks of 32 rows, HW kv heads side by side: NW / RW groups of waves, of which HW KW = NW / RW
// with KW key groups a head.
template <typename T, int DPAD, int RW, int HW>
struct TreeCfg {
    static constexpr bool F32 = std::is_same<T, float>::value;
    static constexpr int EB = F32 ? 4 : 2;
    static constexpr int NW = F32 && RW == 2 ? 2 : RW == 8 ? 8 : 4;  // waves
    static constexpr int GR = NW / RW;                              // groups
    static constexpr int KW = GR / HW;                              // key groups
    static constexpr int BN = !F32 && RW == 8 ? 64 : 32;            // keys of a group's tile
    static constexpr int KT = KW * BN;                              // keys of a step
    static constexpr int ROWB = DPAD * EB;                          // bytes of an LDS row
    static constexpr int CPR = ROWB / 16;                           // 16-byte pieces of it
    static constexpr int TILE = BN * ROWB;
    static constexpr int STAGE = 2 * TILE;  // K and V of a group
    // f32 rows of one block: one stage, whose K is replaced once the scores have it and whose V once P.V
    // has it, so that LDS holds the tiles of four waves (16 single tokens over 512..4096 keys, Hq32 Hkv8
    // D128: 92 us; two waves with two stages 120). 16-bit: 218 us against 212 for the 64 tokens above.
    static constexpr bool ONE = F32 && RW == 1;
    static constexpr int NST = ONE ? 1 : F32 || RW < 4 ? 2 : 4;  // stages: NST - 1 tiles are on their way
    static constexpr int SMEM_KV = GR * NST * STAGE;
    static constexpr int MROW = DPAD * 4 + 16;  // row of the O exchange
    static constexpr int SMEM_O = KW > 1 ? NW * 32 * MROW : 0;
    static constexpr int SMEM = SMEM_KV > SMEM_O ? SMEM_KV : SMEM_O;
    static constexpr int ROWS = 32 * RW;
    // transfer instructions (64 pieces each) of K (or V) a wave issues per tile
    static constexpr int NI = BN * CPR / 64 / RW;
    // the scores of the next block are computed beside the softmax of this one: its tile has to be there
    static constexpr bool PIPE = !F32 && NST > 2;
    // waves a SIMD (three at 64 dims and four row blocks: 24 drafted tokens for 16 sequences, Hq32 Hkv8 f16,
    // 55 us against 57 with two; at two row blocks 45 against 42), and workgroups a CU (with 5 KiB of LDS
    // besides the stages, 160 KiB in all)
    static constexpr int WAVES = (SMEM > 72 * 1024 && NW < 8) || (F32 && DPAD > 64) ? 1
                                 : !F32 && DPAD == 64 && RW == 4                   ? 3
                                                                                   : 2;
    static constexpr int BY_LDS = 160 / (SMEM / 1024 + 5), BY_WAVES = 4 * WAVES / NW;
    static constexpr int PER_CU = BY_LDS < BY_WAVES ? BY_LDS : BY_WAVES;
    // f32 quads of a 32-row block in a partial, in the order that the waves hold them
    static constexpr int QUADS = 8 * DPAD;
};

// The power of two by which P and its sum are kept larger.
template <typename T> constexpr int kTreeLift = std::is_same<T, f16_t>::value ? 7 : 0;
// What is added to a score's c2-fold before exp2.
template <typename T>
__device__ __forceinline__ float exponent_of(float m, float c2) {
    return kTreeLift<T> ? fmaf(-m, c2, (float)kTreeLift<T>) : -m * c2;
}

// Which column a piece of an LDS row is kept in: piece ^ swizzle(row). 16 columns of 16 bytes are the 64
// banks. K is read one row a lane (8 rows at a time have to lie in different columns), V with four rows
// times four neighbouring pieces (16-bit) or eight pieces of two rows four apart (f32) at a time.
template <int CPR, bool F32>
__device__ __forceinline__ int swizzle(int row) {
    if constexpr (F32) return (((row >> 2) & 1) << 3) | ((row & 3) << 1) | ((row >> 3) & 1);
    else if constexpr (CPR == 16) return ((row & 3) << 2) | ((row >> 2) & 3);
    else return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
}

// Non-temporal: the cache is read once, or by the row blocks of one range at about the same time. 64 single
// bf16 tokens over 512..8192 keys (Hq32 Hkv8 D128) 212 against 229 us, 16 drafted tokens for 24 sequences
// 95 against 105; one sequence of 8192 whose rows were still in the caches 36 against 34.
__device__ __forceinline__ void global_to_lds16(const void* p, uint32_t lds) {
    asm volatile("global_load_lds_dwordx4 %0, off nt" : : "v"(p), "{m0}"(lds));
}

struct TreeKArgs {
    TreeArgs a;
    SmallDiv ps, grp;
    FastDiv ranges, row_blocks;
};

// Bits of a word's values (one f32, two 16-bit) that are infinite or NaN.
template <typename T>
__device__ __forceinline__ uint32_t not_finite(uint32_t w) {
    if constexpr (std::is_same<T, float>::value) return (w & 0x7f800000u) == 0x7f800000u ? ~0u : 0u;
    constexpr uint32_t e = std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;
    return ((w & e) == e ? 0xffffu : 0u) | ((w & (e << 16)) == (e << 16) ? 0xffff0000u : 0u);
}

// Wait for the result of a 32x32 MFMA, written out because branches come between the last product and
// its readers (see wait_mfma).
template <bool F32>
__device__ __forceinline__ void wait_mfma32(f32x16_t& v) {
    if constexpr (F32) asm volatile("s_nop 15\n\ts_nop 3" : "+v"(v));
    else asm volatile("s_nop 11" : "+v"(v));
}

// V operands of P.V from the stage: dims 32 mb + (lane & 31) of the keys that the lane's half of S^T
// holds. 16-bit: eight keys, in S^T's order, transposed on the way; f32: the key of accumulator i.
template <int DPAD>
__device__ __forceinline__ u32x4_t tree_v16(const uint8_t* smem, int va0, int k2, int mb) {
    typedef short v4s __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) v4s lds_v4s;
    // column bits: mb in 6 and up (two rows share 256 bytes at 64 dims), e in 5
    const int x0 = va0 ^ (mb << 6), x1 = va0 ^ (mb << 6) ^ (1 << 5);
    const u32x2_t a = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                      (lds_v4s*)(smem + x0 + 16 * k2 * DPAD * 2)));
    const u32x2_t b = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                                      (lds_v4s*)(smem + x1 + (16 * k2 + 8) * DPAD * 2)));
    return u32x4_t{a[0], a[1], b[0], b[1]};
}
template <int DPAD>
__device__ __forceinline__ float tree_v32(const uint8_t* smem, int va0, int i, int mb) {
    const int col = ((i & 3) << 1 | ((i >> 2) & 1)) << 4;  // swizzle of the row's part in i
    return *(const float*)(smem + (va0 ^ (mb << 7) ^ col) + (8 * (i / 4) + i % 4) * DPAD * 4);
}

// Four dims of a finished row: O / l and, with the first dims, LSE. l = 0: the row saw no key, 0 and
// -inf. (A row whose keys are all NaN has m = -inf too, but l = NaN.)
template <typename T>
__device__ __forceinline__ void write_row4(const TreeArgs& a, int s, int kvh, int row, int d, f32x4_t o,
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
        a.lse[((int64_t)s * a.q_heads + hq) * a.max_tokens + t] =
            none ? -INFINITY : m * a.scale + logf(l * (1.0f / (1 << kTreeLift<T>)));
}

// WIN: the steps between the sinks and the first key that a sequence's first token sees are left out; steps that hold
// an edge run masked. 64 single tokens, window 1024, 4 sinks, Hkv8 D128 bf16 (269 MB): 60 us and 5 for the combine.
template <typename T, int DPAD, int RW, int HW, bool SPLIT, bool WIN = false>
__global__ __launch_bounds__((64 * TreeCfg<T, DPAD, RW, HW>::NW),
                             (TreeCfg<T, DPAD, RW, HW>::WAVES))
void tree_split(TreeKArgs ka) {
    using C = TreeCfg<T, DPAD, RW, HW>;
    constexpr bool F32 = C::F32;
    constexpr int MB = DPAD / 32;                   // 32-dim blocks of O^T
    constexpr int KS = F32 ? DPAD / 8 : DPAD / 16;  // K pieces a lane reads per 32 keys
    constexpr int NT = 64 * C::NW;
    constexpr int E = 16 / C::EB;                   // elements of a piece
    __shared__ __attribute__((aligned(1024))) uint8_t smem[C::SMEM];
    __shared__ int bt_lds[kTreePages];
    __shared__ int vote_lds[C::NW];
    __shared__ float2 ml_lds[C::NW * 32];
    __shared__ int odd_lds[C::NW];  // this wave took infinities or NaN out of V (2: on any key, 1: behind ctx)
    const TreeArgs& a = ka.a;
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rw = wave % RW, gi = wave / RW, kg = gi % C::KW, hd = gi / C::KW;
    const int D = a.head_dim;
    const int logical = xcd_remap(blockIdx.x, gridDim.x);
    const int range = __builtin_amdgcn_readfirstlane((int)ka.row_blocks.div((uint32_t)logical));
    const int rb = logical - range * (int)ka.row_blocks.d;
    const int units = a.kv_heads / HW;  // of a sequence

    // ---- this workgroup's range of steps [pos, end), and the sequence that holds the first; every wave
    // for itself, without a barrier
    auto steps_of = [&](int rows, int len) {
        int n = (rows + C::KT - 1) / C::KT, before;
        if constexpr (WIN) n -= tree_skip(a, rows, len, C::KT, &before);
        return n;
    };
    auto rows_of = [&](int i) { return i < a.n_seqs ? tree_rows_of(a, i) : 0; };
    auto len_of = [&](int i) { return WIN ? a.tree_lens[min(i, a.n_seqs - 1)] : 0; };
    int mine = 0, count = 0;  // steps, and units that have any
    for (int i = lane; i < a.n_seqs; i += 64) {
        const int n = steps_of(rows_of(i), len_of(i));
        mine += units * n;
        count += n ? units : 0;
    }
    const int n_steps = __builtin_amdgcn_readlane(wave_scan(mine), 63);
    const int n_units = __builtin_amdgcn_readlane(wave_scan(count), 63);
    const int ov = min(kTreeStart, (int)ka.ranges.div((uint32_t)n_steps) / 2);
    const int total = n_steps + n_units * ov;
    auto length_of = [&](int rows, int len) { return rows ? steps_of(rows, len) + ov : 0; };  // of a unit
    const int share = max(1, (int)ka.ranges.div((uint32_t)total + ka.ranges.d - 1));
    int64_t pos = (int64_t)range * share;
    const int64_t end = pos + share < total ? pos + share : total;
    const bool plans = logical == 0 && wave == 0;  // writes what tree_combine needs
    if (plans && lane == 0) {
        a.plan[a.n_seqs] = share;
        a.plan[a.n_seqs + 1] = ov;
    }
    int s = 0, first = 0, rows_s = 0, len = 0;  // the sequence, its first step, its rows, the drafted ones
    bool found = pos >= end;
    for (int base = 0, carry = 0; base < a.n_seqs && (plans || !found); base += 64) {
        const int rows = rows_of(base + lane), v = units * length_of(rows, len_of(base + lane));
        const int upto = carry + wave_scan(v);
        if (plans && base + lane < a.n_seqs) a.plan[base + lane] = upto - v;
        const uint64_t past = __ballot(upto > pos);
        if (!found && past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            s = base + l;
            first = __builtin_amdgcn_readlane(upto - v, l);
            rows_s = __builtin_amdgcn_readlane(rows, l);
            len = __builtin_amdgcn_readlane(a.tree_lens[min(base + lane, a.n_seqs - 1)], l);
            found = true;
        }
        carry = __builtin_amdgcn_readlane(upto, 63);
    }
    if (pos >= end) return;
    s = __builtin_amdgcn_readfirstlane(s);
    if (lane == 0) odd_lds[wave] = 0;

    // ---- lane constants
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_void_t*)smem;
    const int group_base = gi * C::NST * C::STAGE;
    const int n16 = lane & 15;
    // K operand: row lane & 31, piece 2 c + h: the column's XOR takes c by itself
    const int kbase = group_base + (lane & 31) * C::ROWB +
                      ((h ^ swizzle<C::CPR, F32>(lane & 31)) << 4);
    // V operand. 16-bit: rows 16 k2 + 8 e + 4 h + (n16 >> 2), pieces 4 mb + 2 (lane >> 4 & 1) +
    // ((n16 & 3) >> 1); e and mb enter the column by XOR. f32: row 8 (i / 4) + 4 h + i % 4, piece
    // 8 mb + (lane & 31) / 4.
    int vbase;
    if constexpr (F32) {
        vbase = group_base + C::TILE + 4 * h * C::ROWB + ((((lane & 31) >> 2) ^ (h << 3)) << 4) +
                4 * (lane & 3);
    } else {
        const int r = 4 * h + (n16 >> 2), p = 2 * ((lane >> 4) & 1) + ((n16 & 3) >> 1);
        vbase = group_base + C::TILE + r * C::ROWB + ((p ^ swizzle<C::CPR, F32>(r)) << 4) +
                8 * (n16 & 1);
    }
    const uint32_t row_bytes = (uint32_t)(a.kv_heads * D) * C::EB;
    const float c2 = a.scale * kLog2e;
    const int page_size = a.page_size;

    while (pos < end) {
        // ---- the unit that holds step pos and this range's part of it
        while (pos >= (int64_t)first + units * length_of(rows_s, len)) {
            first += units * length_of(rows_s, len);
            ++s;
            rows_s = __builtin_amdgcn_readfirstlane(tree_rows_of(a, s));
            len = __builtin_amdgcn_readfirstlane(a.tree_lens[s]);
        }
        const int steps = steps_of(rows_s, len);
        const int in_seq = (int)(pos - first);
        const int unit = __builtin_amdgcn_readfirstlane(in_seq / (steps + ov)), kvh = unit * HW + hd;
        const int from = in_seq - unit * (steps + ov);
        const int to = (int)min((int64_t)steps + ov, from + (end - pos));
        pos += to - from;
        const int st0 = max(0, from - ov), st1 = to - ov;
        if (st1 <= st0) continue;
        const int ctx = rows_s - len;
        const int rows_total = len * a.group, r0 = rb * C::ROWS;
        if (r0 >= rows_total) continue;

        // ---- this lane's query row
        const int row = r0 + rw * 32 + (lane & 31);
        const int t = ka.grp.div(row);
        bool row_ok = row < rows_total;
        const bool live = r0 + rw * 32 < rows_total;  // this wave has rows at all
        const int tok = s * a.max_tokens + t;
        int rope_pos = 0;
        // the mask of a tree of up to 64 tokens: one word
        uint64_t mask0 = 0;
        if (row_ok && a.masks && a.words == 1) mask0 = a.masks[tok];
        if (row_ok && a.rope_table) {
            rope_pos = a.positions ? a.positions[tok] : ctx + t;
            row_ok = rope_pos >= 0 && rope_pos < a.rope_positions;
        }
        // (without branches: a row that does not exist reads another one, and is set to zero)
        u32x4_t qop[KS], qlo[SPLIT ? KS : 1];
        auto load_q = [&]() {
            int hh = h;
            asm volatile("" : "+v"(hh));  // (no address is kept past this)
            const int rq = min(row, a.max_tokens * a.group - 1), tq = ka.grp.div(rq);
            const int hr = s * a.max_tokens + tq;
            const uint8_t* const qrow = (const uint8_t*)a.q + ((int64_t)hr * a.q_heads + kvh * a.group +
                                                               rq - tq * a.group) * (D * C::EB);
            const float2* const cs =
                a.rope_table + (int64_t)((row_ok ? rope_pos : 0) + a.rope_offset) * (D >> 1);
#pragma unroll
            for (int c = 0; c < KS; ++c) {
                // (four pieces and their angles at a time: all of them do not fit the registers)
                if (c % 4 == 0) __builtin_amdgcn_sched_barrier(0);
                const int d0 = (2 * c + hh) * E, dl = min(d0, D - E);
                u32x4_t raw = *(const u32x4_t*)(qrow + dl * C::EB), lo = {0u, 0u, 0u, 0u};
                if constexpr (F32) {
                    if (a.rope_table) {
                        const f32x4_t w = *(const f32x4_t*)(cs + dl / 2);
                        float x[4] = {__uint_as_float(raw[0]), __uint_as_float(raw[1]),
                                      __uint_as_float(raw[2]), __uint_as_float(raw[3])};
                        rope_pair(x[0], x[1], w[0], w[1]);
                        rope_pair(x[2], x[3], w[2], w[3]);
#pragma unroll
                        for (int j = 0; j < 4; ++j) raw[j] = __float_as_uint(x[j]);
                    }
                } else if constexpr (SPLIT) {
                    const f32x4_t w0 = *(const f32x4_t*)(cs + dl / 2);
                    const f32x4_t w1 = *(const f32x4_t*)(cs + dl / 2 + 2);
                    const float c8[8] = {w0[0], w0[1], w0[2], w0[3], w1[0], w1[1], w1[2], w1[3]};
                    float x[8];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        x[2 * j] = Half<T>::lo(raw[j]);
                        x[2 * j + 1] = Half<T>::hi(raw[j]);
                    }
                    rope4(x, c8);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        raw[j] = Half<T>::pack(x[2 * j], x[2 * j + 1]);
                        lo[j] = Half<T>::pack(x[2 * j] - Half<T>::lo(raw[j]),
                                              x[2 * j + 1] - Half<T>::hi(raw[j]));
                    }
                }
                const bool ok = row_ok && d0 < D;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    qop[c][j] = ok ? raw[j] : 0u;
                    if constexpr (SPLIT) qlo[c][j] = ok ? lo[j] : 0u;
                }
            }
        };

        load_q();  // (ahead of the first transfers: behind them it waits for their tiles)
        f32x16_t oacc[MB];
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
            for (int i = 0; i < 16; ++i) oacc[mb][i] = 0.0f;
        float m_run = -INFINITY, l_run = 0.0f;
        const uint8_t* const kpool = (const uint8_t*)a.k_pool + (int64_t)kvh * D * C::EB;
        const uint8_t* const vpool = (const uint8_t*)a.v_pool + (int64_t)kvh * D * C::EB;
        const int* const table = a.block_tables + (int64_t)s * a.max_pages;

        // (WIN: behind the first `before` steps `skip` are left out, and a part of the loop ends there)
        int before = 0, skip = 0;
        if constexpr (WIN) skip = tree_skip(a, rows_s, len, C::KT, &before);
        for (int at0 = st0; at0 < st1;) {
            const int shift = WIN && at0 >= before ? skip : 0, c0 = at0 + shift;
            const int part = WIN && at0 < before && skip > 0 ? min(st1, before) : st1 + shift;
            // ---- table entries of as many steps as they cover: first pool row of each page, -1 where
            // the id lies outside the pool
            const int p0 = ka.ps.div(c0 * C::KT);
            const int64_t reach = ((int64_t)p0 + kTreePages) * page_size;  // keys below are covered
            const int c1 = (int)min((int64_t)part, max((int64_t)c0 + 1, reach / C::KT));
            const int k_end = min(c1 * C::KT, rows_s);
            const int n_pages = ka.ps.div(k_end - 1) - p0 + 1;
            bool bad = false;
            __syncthreads();  // (the stages and entries before have been read)
            for (int i = tid; i < n_pages; i += NT) {
                const int page = table[p0 + i];
                const bool in = (unsigned)page < (unsigned)a.physical_pages;
                bt_lds[i] = in ? page * page_size : -1;
                bad |= !in;
            }
            // (a vote of its own: __syncthreads_or goes by the block's three dimensions, registers that
            // are missed later)
            bad = __any(bad);
            if (lane == 0) vote_lds[wave] = bad;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < C::NW; ++w) bad |= vote_lds[w] != 0;
            bad = __builtin_amdgcn_readfirstlane(bad);

            constexpr std::true_type yes{};
            constexpr std::false_type no{};
            // ---- one tile of this wave's key group into a stage: its K, its V
            auto transfer = [&](int step, int stage, auto k_c, auto v_c) {
                const int tile = step * C::KT + kg * C::BN;
                if (tile >= k_end) return;
                uint32_t ln = lane, zero;
                asm volatile("" : "+v"(ln));  // (what depends on the lane alone is not kept)
                // (left to itself the compiler takes the zeros above 32-bit offsets from a vector of 16)
                asm volatile("v_mov_b32 %0, 0" : "=v"(zero));
                constexpr int RPI = 64 / C::CPR;  // rows of an instruction
                const int r1 = (int)(ln / C::CPR), col = (int)(ln % C::CPR);
#pragma unroll
                for (int i = 0; i < C::NI; ++i) {
                    const int r = (rw * C::NI + i) * RPI + r1;
                    const int piece = col ^ swizzle<C::CPR, F32>(r);
                    const int key = min(tile + r, k_end - 1);
                    const int lp = ka.ps.div(key), base = bt_lds[lp - p0];
                    const bool there = tile + r < k_end && base >= 0 && piece * E < D;
                    const uint64_t off = (uint64_t)(uint32_t)(base + key - lp * page_size) * row_bytes +
                                         ((uint64_t)zero << 32 | (uint32_t)piece * 16);
                    const uint8_t* const kp = there ? kpool + off : (const uint8_t*)tree_zero;
                    const uint8_t* const vp = there ? vpool + off : (const uint8_t*)tree_zero;
                    const uint32_t dst = lds0 + group_base + stage + (rw * C::NI + i) * 1024;
                    if constexpr (decltype(k_c)::value) global_to_lds16(kp, dst);
                    if constexpr (decltype(v_c)::value) global_to_lds16(vp, dst + C::TILE);
                }
            };

            // ---- 32 keys from `key0` at `at` of a stage: scores, softmax, P.V. MASKED: blocks in which
            // some row may not see some key.
            // `next` (ONE): the step whose K and V follow into the stage, -1: none.
            auto block = [&](int key0, int at, auto masked_c, int next) {
                constexpr bool MASKED = decltype(masked_c)::value;
                const int ka0 = kbase + at, va0 = vbase + at;
                f32x16_t sc;
#pragma unroll
                for (int i = 0; i < 16; ++i) sc[i] = 0.0f;
                // all K pieces are asked for before the first product (f32: half of them)
                constexpr int KH = F32 ? KS / 2 : KS;
#pragma unroll
                for (int c0k = 0; c0k < KS; c0k += KH) {
                    u32x4_t kf[KH];
#pragma unroll
                    for (int c = 0; c < KH; ++c)
                        kf[c] = *(const u32x4_t*)(smem + (ka0 ^ ((c0k + c) << 5)));
                    if constexpr (C::ONE)
                        if (c0k + KH == KS) {
                            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                            if (next >= 0) transfer(next, 0, yes, no);
                        }
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int c = 0; c < KH; ++c) {
                        if constexpr (F32) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                sc = __builtin_amdgcn_mfma_f32_32x32x2f32(
                                    __uint_as_float(kf[c][j]), __uint_as_float(qop[c0k + c][j]), sc, 0,
                                    0, 0);
                        } else {
                            sc = Half<T>::mfma32(kf[c], qop[c], sc);
                            if constexpr (SPLIT) sc = Half<T>::mfma32(kf[c], qlo[c], sc);
                        }
                    }
                }
                // 16-bit: V's operands are on their way while the softmax runs
                u32x4_t vf[F32 ? 1 : 2][F32 ? 1 : MB];
                if constexpr (!F32 && !MASKED) {
#pragma unroll
                    for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                        for (int mb = 0; mb < MB; ++mb) vf[k2][mb] = tree_v16<DPAD>(smem, va0, k2, mb);
                }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (MASKED) {
                    wait_mfma32<F32>(sc);
                    const int j0 = key0 - ctx;  // drafted token of the first key
                    uint32_t w;
                    if constexpr (WIN) w = window_word(a, ctx + t, key0);
                    else if (a.masks) w = mask_word(a, row_ok, tok, mask0, j0);
                    else w = causal_word(t, j0);
                    // keys past the live rows, and on pages that are not there
                    const int left = k_end - key0;
                    uint32_t there = left >= 32 ? 0xffffffffu : (1u << left) - 1u;
                    if (bad) {
                        const int key = min(key0 + (lane & 31), k_end - 1);
                        const int lp = ka.ps.div(key);
                        there &= (uint32_t)__ballot(bt_lds[lp - p0] >= 0);
                    }
                    const uint32_t see = (w & there) >> (4 * h);  // this row sees these keys
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!((see >> (8 * (i / 4) + i % 4)) & 1)) sc[i] = -INFINITY;
                }
                float mt = sc[0];
#pragma unroll
                for (int i = 1; i < 16; ++i) mt = fmaxf(mt, sc[i]);
                mt = fmaxf(mt, xor32(mt));
                // the running maximum only moves when a block's exceeds it by more than 2^8 in
                // probability, so O is rarely rescaled
                const bool need = mt * c2 > m_run * c2 + 8.0f;
                if (__any(need)) {
                    const float m_use = need ? mt : m_run;
                    const float alpha = m_run == m_use ? 1.0f : fast_exp2((m_run - m_use) * c2);
                    l_run *= alpha;
#pragma unroll
                    for (int mb = 0; mb < MB; ++mb) oacc[mb] *= alpha;
                    m_run = m_use;
                }
                // (MASKED: maybe no key seen yet)
                const float neg = MASKED && m_run == -INFINITY ? 0.0f : exponent_of<T>(m_run, c2);
                float ls = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    sc[i] = fast_exp2(fmaf(sc[i], c2, neg));
                    ls += sc[i];
                }
                l_run += ls;
                // MASKED: a key that some row does not see may hold infinities and NaN, and 0 * inf would
                // bring them to that row. V is taken without them; tree_combine adds what is missing.
                uint32_t off = 0;
                if constexpr (F32) {
                    if constexpr (C::ONE) {
                        if (next >= 0) wait_vmcnt<C::NI>();  // (K of the next tile may be on its way)
                        else wait_dma();
                    }
#pragma unroll
                    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float v = tree_v32<DPAD>(smem, va0, i, mb);
                            if constexpr (MASKED) {
                                const uint32_t x = not_finite<T>(__float_as_uint(v));
                                off |= x;
                                v = x ? 0.0f : v;
                            }
                            oacc[mb] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, sc[i], oacc[mb], 0, 0, 0);
                        }
                    if constexpr (C::ONE) {
                        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                        if (next >= 0) transfer(next, 0, no, yes);
                    }
                } else {
                    if constexpr (MASKED) {
                        typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
                        u16x2 top = {0, 0};  // largest magnitude, sign off
#pragma unroll
                        for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                            for (int mb = 0; mb < MB; ++mb) {
                                vf[k2][mb] = tree_v16<DPAD>(smem, va0, k2, mb);
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    top = __builtin_elementwise_max(
                                        top, __builtin_bit_cast(u16x2, vf[k2][mb][j] & 0x7fff7fffu));
                            }
                        off = not_finite<T>(__builtin_bit_cast(uint32_t, top));
                        if (__any(off != 0)) {
#pragma unroll
                            for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                                for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                                    for (int j = 0; j < 4; ++j)
                                        vf[k2][mb][j] &= ~not_finite<T>(vf[k2][mb][j]);
                        }
                    }
#pragma unroll
                    for (int k2 = 0; k2 < 2; ++k2) {
                        u32x4_t pb;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            pb[j] = Half<T>::pack(sc[8 * k2 + 2 * j], sc[8 * k2 + 2 * j + 1]);
#pragma unroll
                        for (int mb = 0; mb < MB; ++mb) {
                            oacc[mb] = Half<T>::mfma32(vf[k2][mb], pb, oacc[mb]);
                        }
                    }
                }
                // (the larger one of all units and parts of this range)
                if constexpr (MASKED)
                    if (__any(off != 0) && lane == 0) odd_lds[wave] = max(odd_lds[wave], WIN || bad ? 2 : 1);
            };

            // ---- the steps, NST - 1 transfers ahead: first those whose keys every row sees
#pragma unroll
            for (int i = 0; i < C::NST - 1; ++i)
                if (c0 + i < c1) transfer(c0 + i, i * C::STAGE, yes, yes);
            if constexpr (C::ONE) {
                transfer(c0, 0, yes, no);
                transfer(c0, 0, no, yes);
            }
            int stage = 0;
            auto run = [&](int from, int to, auto masked_c) {
                if constexpr (C::ONE) {
#pragma unroll 1
                    for (int step = from; step < to; ++step) {
                        const int tile = step * C::KT + kg * C::BN;
                        if (tile >= k_end) continue;
                        wait_vmcnt<C::NI>();  // (V may be on its way)
                        block(tile, 0, masked_c, step + 1 < c1 && tile + C::KT < k_end ? step + 1 : -1);
                    }
                    return;
                }
#pragma unroll 1
                for (int step = from; step < to; ++step) {
                    // (transfers complete in order: those of the NST - 2 tiles behind this one may be
                    // on their way; near the end there are fewer)
                    if (C::NST > 2 && step + C::NST - 2 < c1 - 1)
                        wait_vmcnt<(C::NST - 2) * 2 * C::NI>();
                    else
                        wait_dma();
                    if constexpr (RW > 1) __syncthreads();
                    else asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    const int ahead = stage == 0 ? (C::NST - 1) * C::STAGE : stage - C::STAGE;
                    if (step + C::NST - 1 < c1) transfer(step + C::NST - 1, ahead, yes, yes);
                    const int tile = step * C::KT + kg * C::BN;
#pragma unroll 1
                    for (int kb = 0; kb < C::BN; kb += 32)
                        if (live && (!decltype(masked_c)::value || tile + kb < k_end))
                            block(tile + kb, stage + kb * C::ROWB, masked_c, -1);
                    stage = stage == (C::NST - 1) * C::STAGE ? 0 : stage + C::STAGE;
                }
            };
            // The same for blocks that every row sees, as a pipeline: Q.K^T of the next block is issued
            // among the softmax of this one (the matrix core runs while the vector unit works), so a
            // step's transfers have to be complete one step earlier.
            auto run_pipe = [&](int from, int to) {
                if constexpr (C::PIPE) {
                f32x16_t sc;
                const auto scores = [&](int at, f32x16_t& out) {
                    const int ka0 = kbase + at;
                    u32x4_t kf[KS];
#pragma unroll
                    for (int c = 0; c < KS; ++c) kf[c] = *(const u32x4_t*)(smem + (ka0 ^ (c << 5)));
                    f32x16_t x;
#pragma unroll
                    for (int i = 0; i < 16; ++i) x[i] = 0.0f;
#pragma unroll
                    for (int c = 0; c < KS; ++c) {
                        x = Half<T>::mfma32(kf[c], qop[c], x);
                        if constexpr (SPLIT) x = Half<T>::mfma32(kf[c], qlo[c], x);
                    }
                    out = x;
                };
#pragma unroll 1
                for (int step = from; step < to; ++step) {
                    if (step + C::NST - 2 < c1 - 1) wait_vmcnt<(C::NST - 3) * 2 * C::NI>();
                    else wait_dma();
                    __syncthreads();
                    const int ahead = stage == 0 ? (C::NST - 1) * C::STAGE : stage - C::STAGE;
                    if (step + C::NST - 1 < c1) transfer(step + C::NST - 1, ahead, yes, yes);
                    const int next = stage == (C::NST - 1) * C::STAGE ? 0 : stage + C::STAGE;
                    if (live) {
                        if (step == from) scores(stage, sc);
#pragma unroll  // (two blocks: the scores change places without copies)
                        for (int kb = 0; kb < C::BN; kb += 32) {
                            const int at = stage + kb * C::ROWB;
                            // (behind the last block of the run its own scores again, not used)
                            const int at_next = kb + 32 < C::BN ? at + 32 * C::ROWB : step + 1 < to ? next : at;
                            f32x16_t sn;
                            scores(at_next, sn);
                            u32x4_t vf[2][MB];  // (the second half is read after the first products)
#pragma unroll
                            for (int mb = 0; mb < MB; ++mb) vf[0][mb] = tree_v16<DPAD>(smem, vbase + at, 0, mb);
                            float mt = sc[0];
#pragma unroll
                            for (int i = 1; i < 16; ++i) mt = fmaxf(mt, sc[i]);
                            mt = fmaxf(mt, xor32(mt));
                            const bool need = mt * c2 > m_run * c2 + 8.0f;
                            const float m_use = need ? mt : m_run;
                            const float neg = exponent_of<T>(m_use, c2);
                            float ls = 0.0f;
                            u32x4_t pb[2];
#pragma unroll
                            for (int i = 0; i < 16; i += 2) {
                                const float p0 = fast_exp2(fmaf(sc[i], c2, neg));
                                const float p1 = fast_exp2(fmaf(sc[i + 1], c2, neg));
                                ls += p0 + p1;
                                pb[i / 8][i % 8 / 2] = Half<T>::pack(p0, p1);
                            }
                            // (here, not behind the branch)
                            asm volatile("" : "+v"(pb[0]), "+v"(pb[1]), "+v"(ls));
                            // issue order: K reads, the maximum, then a product with some of the rest
                            FA_SG(0x100, KS);
                            FA_SG(0x402, 14);
#pragma unroll
                            for (int i = 0; i < (SPLIT ? 2 : 1) * KS; ++i) {
                                FA_SG(0x008, 1);
                                FA_SG(0x100, (SPLIT ? 2 : 4) * MB / KS);
                                FA_SG(0x402, SPLIT ? 5 : 9);
                            }
                            if (__any(need)) {
                                const float alpha = need ? fast_exp2((m_run - m_use) * c2) : 1.0f;
                                l_run *= alpha;
#pragma unroll
                                for (int mb = 0; mb < MB; ++mb) oacc[mb] *= alpha;
                                m_run = m_use;
                            }
                            l_run += ls;
                            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                            for (int mb = 0; mb < MB; ++mb) vf[1][mb] = tree_v16<DPAD>(smem, vbase + at, 1, mb);
#pragma unroll
                            for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                                for (int mb = 0; mb < MB; ++mb)
                                    oacc[mb] = Half<T>::mfma32(vf[k2][mb], pb[k2], oacc[mb]);
                            sc = sn;
                        }
                    }
                    stage = next;
                }
                }
            };
            int cm = bad ? c0 : max(c0, min(c1, ctx / C::KT));
            if constexpr (WIN) {
                // steps before ca hold keys that the last token's window does not reach (or sinks)
                const int reached = (max(0, rows_s - a.window) + C::KT - 1) / C::KT;
                const int ca = bad ? c1 : max(c0, min(c1, reached));
                run(c0, ca, std::true_type{});
                cm = max(ca, cm);
                if constexpr (C::PIPE) run_pipe(ca, cm);
                else run(ca, cm, std::false_type{});
            } else if constexpr (C::PIPE) run_pipe(c0, cm);
            else run(c0, cm, std::false_type{});
            run(cm, c1, std::true_type{});
            at0 = c1 - shift;
        }

        // ---- finished rows to O and LSE, partial ones to their slot: per 32-row block the quads (four
        // dims of a row) in the order that the waves hold them, 1 KiB a store
        l_run += xor32(l_run);
        if (!row_ok) l_run = 0.0f;  // (a token without a position has run with Q = 0: as if it saw nothing)
        int te = tid;
        asm volatile("" : "+v"(te));  // (no address is kept from unit to unit)
        const int le = te & 63, he = le >> 5;
        const bool whole = st0 == 0 && st1 == steps;
        const int64_t slot = 2 * ((int64_t)range * ka.row_blocks.d + rb) + (st0 == 0 ? 1 : 0);
        if constexpr (C::KW == 1) {
            const int64_t blk = (slot * HW + hd) * RW + rw;
            if (live && whole) {
                if (row < rows_total) {
#pragma unroll
                    for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int d = 32 * mb + 8 * i + 4 * he;
                            if (d < D)
                                write_row4<T>(a, s, kvh, row, d,
                                              f32x4_t{oacc[mb][4 * i], oacc[mb][4 * i + 1],
                                                      oacc[mb][4 * i + 2], oacc[mb][4 * i + 3]},
                                              m_run, l_run, ka.grp);
                        }
                }
            } else if (live) {
                f32x4_t* const to = (f32x4_t*)a.part_o + blk * C::QUADS + le;
#pragma unroll
                for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        to[(4 * mb + i) * 64] = f32x4_t{oacc[mb][4 * i], oacc[mb][4 * i + 1],
                                                        oacc[mb][4 * i + 2], oacc[mb][4 * i + 3]};
                if (he == 0) a.part_ml[blk * 32 + le] = make_float2(m_run, l_run);
            }
        } else {  // the key groups are merged in LDS
            if (he == 0) ml_lds[wave * 32 + le] = make_float2(m_run, l_run);
            __syncthreads();  // (every stage has been read)
#pragma unroll
            for (int mb = 0; mb < MB; ++mb)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *(f32x4_t*)(smem + (wave * 32 + (le & 31)) * C::MROW + (32 * mb + 8 * i + 4 * he) * 4) =
                        f32x4_t{oacc[mb][4 * i], oacc[mb][4 * i + 1], oacc[mb][4 * i + 2],
                                oacc[mb][4 * i + 3]};
            __syncthreads();
            // quads of a thread, UN on their way (one after the other: 6 single tokens 29 us against 27)
            constexpr int N = HW * RW * C::QUADS / NT, UN = N < 4 ? N : 4;
            static_assert(N * NT == HW * RW * C::QUADS && N % UN == 0, "every quad has one thread");
            for (int n0 = 0; n0 < N; n0 += UN) {
                f32x4_t o[UN];
                float M[UN], L[UN];
#pragma unroll
                for (int n = 0; n < UN; ++n) {
                    const int i = te + (n0 + n) * NT, blk = i / C::QUADS, q = i % C::QUADS;
                    const int r = q & 31, d = q / 64 * 8 + 4 * ((q >> 5) & 1);
                    // (block = head * RW + row block)
                    const int at = (blk / RW * C::KW) * C::ROWS + blk % RW * 32 + r;
                    float2 ml[C::KW];
                    f32x4_t x[C::KW];
#pragma unroll
                    for (int g = 0; g < C::KW; ++g) {
                        ml[g] = ml_lds[at + g * C::ROWS];
                        x[g] = *(const f32x4_t*)(smem + (at + g * C::ROWS) * C::MROW + 4 * d);
                    }
                    M[n] = ml[0].x;
#pragma unroll
                    for (int g = 1; g < C::KW; ++g) M[n] = fmaxf(M[n], ml[g].x);
                    L[n] = 0.0f;
                    o[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int g = 0; g < C::KW; ++g) {
                        const bool seen = ml[g].y != 0.0f;  // (else it saw nothing)
                        const float w = seen ? fast_exp2((ml[g].x - M[n]) * c2) : 0.0f;
                        L[n] = seen ? fmaf(ml[g].y, w, L[n]) : L[n];
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[n][j] = seen ? fmaf(x[g][j], w, o[n][j]) : o[n][j];
                    }
                }
#pragma unroll
                for (int n = 0; n < UN; ++n) {
                    const int i = te + (n0 + n) * NT, blk = i / C::QUADS, q = i % C::QUADS;
                    const int r = q & 31, d = q / 64 * 8 + 4 * ((q >> 5) & 1);
                    const int rr = blk % RW * 32 + r, hh = blk / RW;
                    if (r0 + rr >= rows_total || d >= D) continue;
                    if (whole) {
                        write_row4<T>(a, s, unit * HW + hh, r0 + rr, d, o[n], M[n], L[n], ka.grp);
                    } else {
                        const int64_t b = slot * (HW * RW) + blk;
                        ((f32x4_t*)a.part_o)[b * C::QUADS + q] = o[n];
                        if (d == 0) a.part_ml[b * 32 + r] = make_float2(M[n], L[n]);
                    }
                }
            }
        }
    }
    __syncthreads();
    if (tid == 0) {
        int odd = 0;
#pragma unroll
        for (int w = 0; w < C::NW; ++w) odd = max(odd, odd_lds[w]);
        a.odd[logical] = odd;
    }
}

// Merges the partials of the units that several ranges share, and writes the rows past each tree. A
// thread ends with one row and a quad of dims in each of N 32-dim blocks.
// Not WIDE: a workgroup per 32 rows of a (sequence, kv head), which merges their partials in their order,
// several loads ahead. WIDE, where those do not fill the chip: one per 32 dims of them; its waves take every
// fourth partial each and are merged in LDS, in their order (256 ranges, one sequence of 8192 keys, 16 tokens,
// Hkv8: 14 us against 37; the chain of 5 over 1000 keys 8 against 13; 24 trees of 64 tokens 24 against 15).
// Partials are f32: of the 24 trees they are 60 MB, 14 us at 4.4 TB/s.
template <typename T, int DPAD, bool WIDE>
__global__ __launch_bounds__(256) void tree_combine(TreeKArgs ka, int kt, int rw, int hw, int blocks) {
    const TreeArgs& a = ka.a;
    constexpr int N = WIDE ? 1 : DPAD / 32;
    constexpr int NQ = WIDE ? 4 : N;      // quads of a thread while merging
    constexpr int UN = 4;                 // partials on their way
    constexpr int STEP = WIDE ? 4 : 1;
    const int D = a.head_dim, tid = threadIdx.x, wave = tid >> 6;
    int id = blockIdx.x, mb0 = 0;
    if constexpr (WIDE) {
        mb0 = id % (DPAD / 32);
        id /= DPAD / 32;
    }
    const int b32 = id % blocks, sh = id / blocks;
    const int kvh = sh % a.kv_heads, s = sh / a.kv_heads;
    const int row = b32 * 32 + (tid & 31), rows_all = a.max_tokens * a.group;
    const int share = a.plan[a.n_seqs], ov = a.plan[a.n_seqs + 1], before = a.plan[s];  // (asked for with the lengths)
    const int rows_s = tree_rows_of(a, s);
    const int len = rows_s ? a.tree_lens[s] : 0;
    const int d0 = 32 * mb0 + 8 * wave + 4 * ((tid >> 5) & 1);  // dims d0 + 32 n .. + 3
    const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
    if (row < rows_all && row >= len * a.group) {
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (d0 + 32 * n < D) write_row4<T>(a, s, kvh, row, d0 + 32 * n, zero, 0.0f, 0.0f, ka.grp);
    }
    if (b32 * 32 >= len * a.group) return;
    int before_skip, steps = (rows_s + kt - 1) / kt;
    if (a.window) steps -= tree_skip(a, rows_s, len, kt, &before_skip);
    const uint32_t u0 = (uint32_t)before + (uint32_t)(kvh / hw) * (uint32_t)(steps + ov) + (uint32_t)ov;
    const int g0 = (int)(u0 / (uint32_t)share), g1 = (int)((u0 + steps - 1) / (uint32_t)share);
    const int rb = b32 / rw, in = b32 - rb * rw;
    const int nrb = (int)ka.row_blocks.d;
    const float c2 = a.scale * kLog2e;
    int odd = 0;
    float M = -INFINITY, L = 0.0f;
    f32x4_t o[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n) o[n] = zero;
    // another part (m, l, x) into (M, L, o); l = 0: it saw nothing
    const auto merge = [&](float2 ml, const f32x4_t (&x)[NQ]) {
        if (ml.y == 0.0f) return;
        const float mx = fmaxf(M, ml.x);
        const float w0 = L == 0.0f ? 0.0f : fast_exp2((M - mx) * c2);
        const float w1 = fast_exp2((ml.x - mx) * c2);
        M = mx;
        L = fmaf(ml.y, w1, L * w0);
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int j = 0; j < 4; ++j) o[n][j] = fmaf(x[n][j], w1, o[n][j] * w0);
    };
    if (g0 == g1) {
        odd = a.odd[g0 * nrb + rb];
        if (!odd) return;  // finished by the range that covers it
    } else {
        for (int g = g0 + (WIDE ? wave : 0); g <= g1; g += UN * STEP) {
            float2 ml[UN];
            f32x4_t x[UN][NQ];
            int od[UN];
#pragma unroll
            for (int i = 0; i < UN; ++i) {  // (past the end: the last partial again, not counted)
                const int at = min(g + i * STEP, g1);
                const int64_t blk = ((2 * ((int64_t)at * nrb + rb) + (at == g0 ? 1 : 0)) * hw + kvh % hw) * rw + in;
                const f32x4_t* const from = (const f32x4_t*)a.part_o + blk * (8 * DPAD);
                od[i] = a.odd[at * nrb + rb];
                ml[i] = a.part_ml[blk * 32 + (tid & 31)];
#pragma unroll
                for (int n = 0; n < NQ; ++n)
                    x[i][n] = WIDE ? from[(4 * mb0 + n) * 64 + (tid & 63)] : from[n * 256 + tid];
            }
#pragma unroll
            for (int i = 0; i < UN; ++i) {
                odd = max(odd, od[i]);
                if (g + i * STEP <= g1) merge(ml[i], x[i]);
            }
        }
        if constexpr (WIDE) {
            __shared__ f32x4_t o_lds[4][NQ][64];
            __shared__ float2 ml_lds[4][32];
            __shared__ int odd_lds[4];
            if ((tid & 63) < 32) ml_lds[wave][tid & 31] = make_float2(M, L);
            if ((tid & 63) == 0) odd_lds[wave] = odd;
#pragma unroll
            for (int n = 0; n < NQ; ++n) o_lds[wave][n][tid & 63] = o[n];
            __syncthreads();
            M = -INFINITY;
            L = 0.0f;
            f32x4_t x[NQ];
#pragma unroll
            for (int n = 0; n < NQ; ++n) o[n] = x[n] = zero;
#pragma unroll
            for (int w = 0; w < 4; ++w) {
                odd = max(odd, odd_lds[w]);
                x[0] = o_lds[w][wave][tid & 63];
                merge(ml_lds[w][tid & 31], x);
            }
        }
    }
    if (row >= len * a.group) return;
    if (g0 < g1) {
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (d0 + 32 * n < D) write_row4<T>(a, s, kvh, row, d0 + 32 * n, o[n], M, L, ka.grp);
    }
    if (!odd) return;
    // ---- V held infinities or NaN where rows do not see every key: the values that this row sees
    const int ctx = rows_s - len, t = ka.grp.div(row);
    const int hq = kvh * a.group + row - t * a.group;
    if (g0 == g1) L = a.lse[((int64_t)s * a.q_heads + hq) * a.max_tokens + t] == -INFINITY ? 0.0f : 1.0f;
    if (L == 0.0f) return;  // (sees nothing)
#pragma unroll 1
    for (int n = 0; n < N; ++n) {
        const int d = d0 + 32 * n;
        if (d >= D) break;
        f32x4_t add = zero;
        for (int key = odd > 1 ? 0 : ctx / kt * kt; key < rows_s; ++key) {
            const int j = key - ctx;
            const bool seen = a.window ? j <= t && (t - j < a.window || key < a.sinks)
                              : j < 0  ? true
                              : a.masks
                                  ? (a.masks[((int64_t)s * a.max_tokens + t) * a.words + (j >> 6)] >> (j & 63)) & 1
                                  : j <= t;
            if (!seen) continue;
            const int lp = ka.ps.div(key), page = a.block_tables[(int64_t)s * a.max_pages + lp];
            if ((unsigned)page >= (unsigned)a.physical_pages) continue;
            const int64_t at =
                (((int64_t)page * a.page_size + key - lp * a.page_size) * a.kv_heads + kvh) * D + d;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v;
                if constexpr (std::is_same<T, float>::value) v = ((const float*)a.v_pool)[at + e];
                else v = Half<T>::lo(((const uint16_t*)a.v_pool)[at + e]);
                if (!(fabsf(v) < INFINITY)) add[e] += v;
            }
        }
        const int64_t to = (((int64_t)s * a.max_tokens + t) * a.q_heads + hq) * D + d;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            if (add[e] == 0.0f) continue;
            if constexpr (std::is_same<T, float>::value) ((float*)a.o)[to + e] += add[e];
            else
                ((uint16_t*)a.o)[to + e] = (uint16_t)Half<T>::pack(
                    Half<T>::lo(((const uint16_t*)a.o)[to + e]) + add[e], 0.0f);
        }
    }
}

// The shape of a launch. Rows: as few row blocks of 32 as hold every row of a (sequence, kv head), at
// most 8 (f32: 4), since K and V are read once for each 32 RW rows (24 trees of 64 tokens, 256 rows: 175 us
// with 8 blocks and 64 keys a step, 202 with 4 that read K and V twice). Waves left over take two kv heads
// side by side and two key groups; the key groups alone where the head count is odd, the heads alone where
// two groups are left. Four heads / two and two / four key groups: 64 single bf16 tokens over 512..8192 keys
// 210 / 195 / 194 us, 200 over 16..600 72 / 80 / 100, 8 drafted tokens for 16 sequences of 16 heads 75 / 71 /
// 75. f32 takes four heads: 16 single tokens 85 us, four key groups 97.
struct TreeShape {
    int rw, hw, kt, row_blocks, ranges, threads;
};
template <typename T, int DPAD, int RW, int HW>
static TreeShape shape_of(const TreeArgs& a) {
    using C = TreeCfg<T, DPAD, RW, HW>;
    TreeShape s;
    s.rw = RW;
    s.hw = HW;
    s.kt = C::KT;
    s.row_blocks = (a.max_tokens * a.group + C::ROWS - 1) / C::ROWS;
    // one round of workgroups: as many a CU as LDS and registers hold
    s.ranges = std::max(1, C::PER_CU * device_cus() / s.row_blocks);
    s.threads = 64 * C::NW;
    return s;
}
// Calls f with the row waves and heads of a launch as constants.
template <typename T, typename F>
static auto tree_dispatch(const TreeArgs& a, F f) {
    using std::integral_constant;
    constexpr bool F32 = std::is_same<T, float>::value;
    const int rows = a.max_tokens * a.group;
    auto go = [&](auto dpad) {
        constexpr int DP = decltype(dpad)::value;
        auto run = [&](auto rw, auto hw) { return f(integral_constant<int, DP>{}, rw, hw); };
        using One = integral_constant<int, 1>;
        using Two = integral_constant<int, 2>;
        using Four = integral_constant<int, 4>;
        if (rows <= 32) {
            if constexpr (F32)
                if (a.kv_heads % 4 == 0) return run(One{}, Four{});
            return a.kv_heads % 2 == 0 ? run(One{}, Two{}) : run(One{}, One{});
        }
        if (rows <= 64) {
            if constexpr (!F32)
                if (a.kv_heads % 2 == 0) return run(Two{}, Two{});
            return run(Two{}, One{});
        }
        if constexpr (!F32)
            if (rows > 128) return run(integral_constant<int, 8>{}, One{});
        return run(Four{}, One{});
    };
    return a.head_dim <= 64 ? go(integral_constant<int, 64>{}) : go(integral_constant<int, 128>{});
}
template <typename T>
static TreeShape shape_t(const TreeArgs& a) {
    return tree_dispatch<T>(a, [&](auto dpad, auto rw, auto hw) {
        return shape_of<T, decltype(dpad)::value, decltype(rw)::value, decltype(hw)::value>(a);
    });
}
static TreeShape tree_shape(Dtype dt, const TreeArgs& a) {
    return dt == Dtype::F32 ? shape_t<float>(a) : shape_t<bf16_t>(a);  // (the 16-bit types alike)
}

// What the partials of a launch take on one CU: rows (with hw heads of rw row blocks), bytes of O, workgroups.
// The most of any shape that tree_dispatch chooses.
struct TreeMost {
    int rows, bytes, groups;
};
template <typename T, int DPAD, int RW, int HW>
static constexpr TreeMost most_of(TreeMost m) {
    using C = TreeCfg<T, DPAD, RW, HW>;
    constexpr int rows = C::PER_CU * C::ROWS * HW;
    return {std::max(m.rows, rows), std::max(m.bytes, rows * DPAD * 4), std::max(m.groups, C::PER_CU)};
}
template <int DPAD>
static constexpr TreeMost most_with(TreeMost m) {
    m = most_of<bf16_t, DPAD, 1, 1>(most_of<bf16_t, DPAD, 1, 2>(m));
    m = most_of<bf16_t, DPAD, 2, 1>(most_of<bf16_t, DPAD, 2, 2>(m));
    m = most_of<bf16_t, DPAD, 4, 1>(most_of<bf16_t, DPAD, 8, 1>(m));
    m = most_of<float, DPAD, 1, 1>(most_of<float, DPAD, 1, 2>(most_of<float, DPAD, 1, 4>(m)));
    return most_of<float, DPAD, 2, 1>(most_of<float, DPAD, 4, 1>(m));
}

// The same partials for every shape and type (69 MB on 256 CUs), so that no later call of up to as many
// sequences has to allocate: a shape's own need is not monotone in it (65 to 128 16-bit rows of 64 dims have
// more workgroups than 256 rows, and row blocks that do not divide the workgroups leave some out). A single
// range, which more row blocks than workgroups have, leaves no partials.
size_t tree_workspace(Dtype dt, const TreeArgs& a, size_t* ml_offset, size_t* plan_offset,
                      size_t* odd_offset) {
    constexpr TreeMost most = most_with<64>(most_with<128>({0, 0, 0}));
    const size_t cus = (size_t)device_cus();
    *ml_offset = 2 * cus * most.bytes;
    *plan_offset = *ml_offset + 2 * cus * most.rows * 8;
    *odd_offset = *plan_offset + ((size_t)a.n_seqs + 2) * 4;
    return *odd_offset + std::max<size_t>(cus * most.groups, tree_shape(dt, a).row_blocks) * 4;
}

template <typename T>
static void launch_t(TreeKArgs& ka, hipStream_t st, unsigned grid[3], unsigned* block, unsigned* rows,
                     void (*between)(void*), void* user) {
    const TreeArgs& a = ka.a;
    const TreeShape s = shape_t<T>(a);
    ka.ranges = FastDiv((uint32_t)s.ranges);
    ka.row_blocks = FastDiv((uint32_t)s.row_blocks);
    grid[0] = (unsigned)(s.ranges * s.row_blocks);
    grid[1] = grid[2] = 1;
    *block = (unsigned)s.threads;
    *rows = (unsigned)(32 * s.rw);
    tree_dispatch<T>(a, [&](auto dpad, auto rw, auto hw) {
        constexpr int DP = decltype(dpad)::value, RW = decltype(rw)::value, HW = decltype(hw)::value;
        const auto split = [&](auto win) {
            constexpr bool WIN = decltype(win)::value;
            if constexpr (!std::is_same<T, float>::value) {
                if (a.rope_table) {
                    tree_split<T, DP, RW, HW, true, WIN><<<grid[0], s.threads, 0, st>>>(ka);
                    return;
                }
            }
            tree_split<T, DP, RW, HW, false, WIN><<<grid[0], s.threads, 0, st>>>(ka);
        };
        if (a.window) split(std::true_type{});
        else split(std::false_type{});
    });
    if (between) between(user);
    const int blocks = (a.max_tokens * a.group + 31) / 32;
    auto combine = [&](auto dpad) {
        constexpr int DP = decltype(dpad)::value;
        const unsigned g = (unsigned)((int64_t)a.n_seqs * a.kv_heads * blocks);
        if (g <= (unsigned)device_cus())
            tree_combine<T, DP, true><<<g * (DP / 32), 256, 0, st>>>(ka, s.kt, s.rw, s.hw, blocks);
        else
            tree_combine<T, DP, false><<<g, 256, 0, st>>>(ka, s.kt, s.rw, s.hw, blocks);
    };
    if (a.head_dim <= 64) combine(std::integral_constant<int, 64>{});
    else combine(std::integral_constant<int, 128>{});
}

void launch_tree_attention(Dtype dt, const TreeArgs& a, hipStream_t s, unsigned grid[3],
                           unsigned* block, unsigned* rows, void (*between)(void*), void* user) {
    TreeKArgs ka;
    ka.a = a;
    ka.ps = SmallDiv((uint32_t)a.page_size);
    ka.grp = SmallDiv((uint32_t)a.group);
    switch (dt) {
        case Dtype::BF16: launch_t<bf16_t>(ka, s, grid, block, rows, between, user); break;
        case Dtype::F16: launch_t<f16_t>(ka, s, grid, block, rows, between, user); break;
        default: launch_t<float>(ka, s, grid, block, rows, between, user); break;
    }
}

}  // namespace fa
