// A batch's page tables and cache rows kept on the GPU: slots reserved from request lengths, the
// masks and positions of drafted trees, rows appended by slot, accepted rows moved into place.
//
// No counterpart in the reference, whose tables are host metadata (src/paged_kv.rs:76): a serving
// step that knows its lengths only on the GPU (how many drafted tokens were accepted) would wait for
// them to reach the host. Everything here reads its lengths on the device, writes each output once
// from one thread, and uses no atomics, so a replayed graph gives the same results.
//
// Lengths, page ids, slots and parents come from device memory that the host cannot check: every one
// is compared with its range before it addresses anything, and what does not fit takes no part.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace fa {

// ---------------------------------------------------------------------------- slot reservation
//
// need_s = max(0, ceil((ctx_s + new_s) / page) - mapped_s) pages, taken from the top of the free stack
// in sequence order: with the exclusive prefix sum x_s, page j of sequence s is
// free[avail - 1 - (x_s + j)], avail = free_count + the pages that ended sequences put back first. A
// sequence whose inclusive sum passes avail gets nothing (nor does any later one that needs a page).
// A few integers a sequence: bound by the launch and two dependent loads. One workgroup does the
// prefix sum (a wave scan and one exchange between the waves); it also writes tables and slots where
// they are few (reserve_fused), otherwise reserve_fill does from the plan it leaves.
// One sequence 4.7 us, the smallest a call takes; 256 of up to 2048 tokens, 24 ended, 11.0 (17.8 with four
// slots a thread and each wave putting back the pages of its own ended sequences).

// What reserve_fill has to know of a sequence: pages that stay, tokens granted, the exclusive prefix sum of
// the pages taken, and how many it takes.
struct ReservePlan {
    int kept, granted, first, taken;
};

struct ReserveKArgs {
    ReserveArgs a;
    FastDiv ps;
};

// Inclusive prefix sum over the workgroup of two counts below 2^31 in one 64-bit value; *total is the
// workgroup's sum. `sums` holds one value per wave.
__device__ __forceinline__ uint64_t block_scan(uint64_t v, uint64_t* sums, uint64_t* total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t up = __shfl_up((unsigned long long)v, o, 64);
        if (lane >= o) v += up;
    }
    __syncthreads();  // (the values of an earlier scan have been read)
    if (lane == 63) sums[wave] = v;
    __syncthreads();
    uint64_t all = 0, before = 0;
#pragma unroll
    for (int w = 0; w < 16; ++w) {  // (16 loads at once; those of waves that are not there are dropped)
        const uint64_t x = sums[w];
        if (w == wave) before = all;
        all += w < waves ? x : 0;
    }
    *total = all;
    return v + before;
}

// Page ids, tables and slots of one sequence for tokens [t0, t1); `lanes` consecutive threads, `lane`
// among them. Pages the table already has are read, the others come from the free stack.
__device__ __forceinline__ void fill_sequence(const ReserveKArgs& ka, int s, const ReservePlan& p,
                                              int ctx, int avail, int t0, int t1, int lane,
                                              int lanes) {
    const ReserveArgs& a = ka.a;
    int* const row = a.block_tables + (int64_t)s * a.max_pages;
    auto fresh = [&](int j) { return a.free_pages[avail - 1 - (p.first + j)]; };
    // the new entries belong to the part that starts at token 0
    if (t0 == 0)
        for (int j = lane; j < p.taken; j += lanes) row[p.kept + j] = fresh(j);
    int* const slots = a.slots + (int64_t)s * a.max_new;
    for (int t = t0 + lane; t < t1; t += lanes) {
        int slot = -1;
        if (t < p.granted) {
            const int logical = ctx + t;
            const int lp = (int)ka.ps.div((uint32_t)logical);
            const int page = lp < p.kept ? row[lp] : fresh(lp - p.kept);
            if ((unsigned)page < (unsigned)a.physical_pages)
                slot = page * a.page_size + (logical - lp * a.page_size);
        }
        slots[t] = slot;
    }
}

__global__ __launch_bounds__(1024) void reserve_plan(ReserveKArgs ka, int fused) {
    const ReserveArgs& a = ka.a;
    __shared__ uint64_t sums[16];
    __shared__ ReservePlan plans[1024];
    __shared__ int ctxs[1024];
    __shared__ int2 backs[1024];  // of an ended sequence: its pages, and how many go on the stack before
    __shared__ uint64_t ends[16];
    const int tid = threadIdx.x, threads = blockDim.x;
    const int count = min(max(a.free_count[0], 0), a.free_capacity);
    auto kept_of = [&](int s) { return min(max(a.mapped[s], 0), a.max_pages); };
    // pages put back: known after the scan itself where one pass covers the batch
    int64_t back_all = 0;
    if (a.n_seqs > threads) {
        uint64_t mine = 0;
        for (int s = tid; s < a.n_seqs; s += threads)
            if (a.new_lens[s] < 0) mine += (uint64_t)kept_of(s);
        uint64_t total;
        block_scan(mine, sums, &total);
        back_all = (int64_t)total;
    }
    uint64_t carry = 0;  // (pages back << 32 | pages needed) of the sequences before this pass
    uint64_t taken = 0;  // pages taken by the batch
    int avail = 0;
    for (int base = 0; base < a.n_seqs; base += threads) {
        const int s = base + tid;
        int ctx = 0, fresh = 0, kept = 0;
        if (s < a.n_seqs) {
            ctx = a.ctx_lens[s];
            fresh = a.new_lens[s];
            kept = kept_of(s);
        }
        const bool ended = s < a.n_seqs && fresh < 0;
        const int64_t tokens = (int64_t)ctx + fresh;
        const bool valid = ctx >= 0 && fresh > 0 && fresh <= a.max_new &&
                           tokens <= (int64_t)a.max_pages * a.page_size;
        const int pages = valid ? (int)ka.ps.div((uint32_t)(tokens + a.page_size - 1)) : 0;
        const int need = max(0, pages - kept);
        const uint64_t mine = (uint64_t)(ended ? kept : 0) << 32 | (uint32_t)(valid ? need : 0);
        uint64_t total;
        const uint64_t upto = carry + block_scan(mine, sums, &total);
        if (a.n_seqs <= threads) back_all = (int64_t)(total >> 32);
        avail = (int)min((int64_t)count + back_all, (int64_t)a.free_capacity);
        const int64_t need_upto = (int64_t)(upto & 0xffffffffu);
        const bool ok = valid && (need == 0 || need_upto <= avail);
        const int got = ok ? need : 0;
        if (got > 0) taken = (uint64_t)need_upto;
        if (s < a.n_seqs) {
            a.granted[s] = ok ? fresh : 0;
            a.mapped_out[s] = ended ? 0 : kept + got;
            const ReservePlan p = {kept, ok ? fresh : 0, (int)(need_upto - need), got};
            if (fused) {
                plans[tid] = p;
                ctxs[tid] = ctx;
            } else {
                a.plan[s] = make_int4(p.kept, p.granted, p.first, p.taken);
            }
        }
        // the pages of ended sequences, dealt out to the waves: they are on the stack before any is taken
        if (ended) backs[tid] = make_int2(kept, (int)((upto >> 32) - kept));
        const uint64_t mine_end = __ballot(ended);
        if ((tid & 63) == 0) ends[tid >> 6] = mine_end;
        __syncthreads();
        const int waves = threads >> 6, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const uint64_t all_ends = ends[tid & (waves - 1)];  // (1, 4 or 16 waves)
        int turn = 0;
        for (int w = 0; w < waves; ++w)
            for (uint64_t left = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(all_ends >> 32), w) << 32 |
                                 (uint32_t)__builtin_amdgcn_readlane((int)all_ends, w);
                 left; left &= left - 1) {
                if ((turn++ & (waves - 1)) != wave) continue;
                const int l = w * 64 + __ffsll((unsigned long long)left) - 1;
                const int n = backs[l].x;
                const int64_t at = (int64_t)count + backs[l].y;
                const int* const row = a.block_tables + (int64_t)(base + l) * a.max_pages;
                for (int j0 = tid & 63; j0 < n; j0 += 256) {
                    int page[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) page[i] = row[min(j0 + 64 * i, n - 1)];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (j0 + 64 * i < n && at + j0 + 64 * i < a.free_capacity)
                            a.free_pages[at + j0 + 64 * i] = page[i];
                }
            }
        if (ended) a.ctx_lens[s] = 0;
        carry += total;
    }
    // most pages any granted sequence reached = the pages taken (a refused one is followed by no
    // sequence that takes any)
    for (int o = 32; o; o >>= 1) {
        const uint64_t other = __shfl_xor((unsigned long long)taken, o, 64);
        taken = other > taken ? other : taken;
    }
    __syncthreads();
    if ((tid & 63) == 0) sums[tid >> 6] = taken;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 1; w < 16; ++w) {
            const uint64_t x = sums[w];
            if (w < (threads >> 6)) taken = x > taken ? x : taken;
        }
        a.free_count_out[0] = avail - (int)taken;
        if (!fused) a.plan[a.n_seqs] = make_int4(avail, 0, 0, 0);
    }
    if (!fused) return;
    __threadfence_block();
    __syncthreads();
    // few slots: threads in groups of 16 to 64, a sequence each
    const int lanes = a.max_new <= 16 ? 16 : 64;
    for (int s = tid / lanes; s < a.n_seqs; s += threads / lanes)
        fill_sequence(ka, s, plans[s], ctxs[s], avail, 0, a.max_new, tid % lanes, lanes);
}

constexpr int kFillTokens = 256;  // slots per workgroup of reserve_fill, one a thread: two loads in a row

__global__ __launch_bounds__(256) void reserve_fill(ReserveKArgs ka, int parts) {
    const int s = blockIdx.x / parts, t0 = blockIdx.x % parts * kFillTokens;
    const int4 p = ka.a.plan[s];
    fill_sequence(ka, s, ReservePlan{p.x, p.y, p.z, p.w}, ka.a.ctx_lens[s], ka.a.plan[ka.a.n_seqs].x,
                  t0, min(t0 + kFillTokens, ka.a.max_new), threadIdx.x, 256);
}

// One workgroup writes everything up to here: beyond it a second launch over the whole chip. Fused / not
// (us): 16 sequences of 16 tokens 5.0 / 8.8, 64 of 16 7.1 / 8.8, 64 of 64 8.6 / 8.9, 256 of 16 10.0 / 10.3,
// 256 of 32 15.3 / 10.5; 8 of 512 7.9 / 8.0, 1 of 2048 (a sequence has 64 threads) 9.4 / 8.0.
static bool reserve_fused(int n_seqs, int max_new) {
    return n_seqs <= 1024 && max_new <= 512 && (int64_t)n_seqs * max_new <= 4096;
}

void launch_reserve(const ReserveArgs& a, hipStream_t s, unsigned grid[3], unsigned* block,
                    unsigned* dispatches) {
    ReserveKArgs ka;
    ka.a = a;
    ka.ps = FastDiv((uint32_t)a.page_size);
    const bool fused = reserve_fused(a.n_seqs, a.max_new);
    const int64_t work = fused ? std::max<int64_t>((int64_t)a.n_seqs * std::min(a.max_new, 64), a.n_seqs)
                               : a.n_seqs;
    // (not fused: the waves share the pages of ended sequences)
    const int threads = fused && work <= 64 ? 64 : fused && work <= 256 ? 256 : 1024;
    reserve_plan<<<1, threads, 0, s>>>(ka, fused ? 1 : 0);
    grid[0] = 1;
    grid[1] = grid[2] = 1;
    *block = (unsigned)threads;
    *dispatches = 1;
    if (!fused) {
        const int parts = (a.max_new + kFillTokens - 1) / kFillTokens;
        reserve_fill<<<(unsigned)(a.n_seqs * parts), 256, 0, s>>>(ka, parts);
        grid[0] = (unsigned)(a.n_seqs * parts);
        *block = 256;
        *dispatches = 2;
    }
}

// ---------------------------------------------------------------------------- tree masks
//
// mask_t = the bits of token t and its ancestors, position = ctx + number of ancestors. With p the
// parent, mask_t = bit t | mask_p(t): log2(depth) rounds of pointer doubling (mask |= mask[jump],
// jump = jump[jump]) instead of a walk as long as the tree is deep. One workgroup a sequence, masks in
// LDS, bound by launch and round latency: 4 trees of 24 tokens 4.2 us, 192 of 256 6.3 (7.9 with the number
// of words a variable, which costs a division an item and round).
// A parent that is neither -1 nor an earlier token ends in -2, which every descendant inherits: those
// tokens get an empty mask and position -1.
template <int W>  // words of a mask
__global__ __launch_bounds__(1024) void tree_masks(TreeMaskArgs a) {
    __shared__ uint64_t m[64 * W * W];
    __shared__ int jump[64 * W];
    const int s = blockIdx.x, tid = threadIdx.x, threads = blockDim.x;
    const int ctx = a.ctx_lens[s], len = a.tree_lens[s];
    const int n = ctx >= 0 && len >= 0 && len <= a.max_tokens ? len : 0;
    constexpr int kItems = (64 * W * W + 1023) / 1024;  // words a thread may hold
    for (int t = tid; t < n; t += threads) {
        const int p = a.parents[(int64_t)s * a.max_tokens + t];
        jump[t] = p < -1 || p >= t ? -2 : p;
    }
    for (int i = tid; i < n * W; i += threads) {
        const int t = i / W, w = i - t * W;
        m[i] = (t >> 6) == w ? 1ull << (t & 63) : 0ull;
    }
    __syncthreads();
    while (true) {
        uint64_t add[kItems];
        int next[kItems];
        int more = 0;
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const int i = tid + k * threads;
            add[k] = 0;
            next[k] = -1;
            if (i < n * W) {
                const int t = i / W, j = jump[t];
                next[k] = j;
                if (j >= 0) {
                    add[k] = m[j * W + (i - t * W)];
                    next[k] = jump[j];
                    more = 1;
                }
            }
        }
        if (!__syncthreads_or(more)) break;
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const int i = tid + k * threads;
            if (i < n * W) {
                const int t = i / W;
                m[i] |= add[k];
                if (i == t * W) jump[t] = next[k];
            }
        }
        __syncthreads();
    }
    uint64_t* const out = a.masks + (int64_t)s * a.max_tokens * W;
    for (int i = tid; i < a.max_tokens * W; i += threads) {
        const int t = i / W;
        out[i] = t < n && jump[t] != -2 ? m[i] : 0ull;
    }
    for (int t = tid; t < a.max_tokens; t += threads) {
        int64_t pos = -1;
        if (t < n && jump[t] != -2) {
            int bits = 0;
            for (int w = 0; w < W; ++w) bits += __popcll((unsigned long long)m[t * W + w]);
            pos = (int64_t)ctx + bits - 1;
            if (pos > 0x7fffffff) pos = -1;
        }
        a.positions[(int64_t)s * a.max_tokens + t] = (int)pos;
    }
}

void launch_tree_masks(const TreeMaskArgs& a, hipStream_t s, unsigned grid[3], unsigned* block) {
    const int items = a.max_tokens * a.words;
    const int threads = items >= 1024 ? 1024 : (items + 63) / 64 * 64;
    const unsigned g = (unsigned)a.n_seqs;
    switch (a.words) {
        case 1: tree_masks<1><<<g, threads, 0, s>>>(a); break;
        case 2: tree_masks<2><<<g, threads, 0, s>>>(a); break;
        case 3: tree_masks<3><<<g, threads, 0, s>>>(a); break;
        case 4: tree_masks<4><<<g, threads, 0, s>>>(a); break;
        case 5: tree_masks<5><<<g, threads, 0, s>>>(a); break;
        case 6: tree_masks<6><<<g, threads, 0, s>>>(a); break;
        case 7: tree_masks<7><<<g, threads, 0, s>>>(a); break;
        default: tree_masks<8><<<g, threads, 0, s>>>(a); break;
    }
    grid[0] = (unsigned)a.n_seqs;
    grid[1] = grid[2] = 1;
    *block = (unsigned)threads;
}

// ---------------------------------------------------------------------------- append by slot
//
// Pool row slots[r] = source row r, K rotated at its position on the way (one rounding to the storage
// type, after the rotation in f32). Bound by memory: a 16-byte piece of K and one of V per thread; 48
// sequences of up to 512 bf16 rows of 8 heads of 128 (99 MB): 20.3 us, 4.86 TB/s, a copy's rate 5.16.
// Rows without a slot, and rows whose position the (cos, sin) table does not have, are left out.
template <typename T>
__global__ __launch_bounds__(256) void append_slots(SlotAppendArgs a, FastDiv per_row, FastDiv per_seq,
                                                    FastDiv per_head) {
    constexpr bool F32 = std::is_same<T, float>::value;
    constexpr int E = F32 ? 4 : 8;  // elements of a 16-byte piece
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= (int64_t)a.n_rows * per_row.d) return;
    const int r = (int)per_row.div((uint32_t)i), c = (int)((uint32_t)i - (uint32_t)r * per_row.d);
    const int slot = a.slots[r];
    if ((unsigned)slot >= (unsigned)a.pool_rows) return;
    const int64_t from = (int64_t)r * per_row.d + c, to = (int64_t)slot * per_row.d + c;
    u32x4_t k = ((const u32x4_t*)a.k_src)[from];
    const u32x4_t v = ((const u32x4_t*)a.v_src)[from];
    if (a.rope_table) {
        const int s = (int)per_seq.div((uint32_t)r);
        const int64_t pos = a.positions ? (int64_t)a.positions[r]
                                        : (int64_t)a.ctx_lens[s] + (r - s * (int)per_seq.d);
        if (pos < 0 || pos >= a.rope_positions) return;
        const int d0 = (c - (int)(per_head.div((uint32_t)c) * per_head.d)) * E;
        const float2* cs = a.rope_table + (pos + a.rope_offset) * (a.head_dim / 2) + d0 / 2;
        if constexpr (F32) {
            const f32x4_t t = *(const f32x4_t*)cs;
            float x[4] = {__uint_as_float(k[0]), __uint_as_float(k[1]), __uint_as_float(k[2]),
                          __uint_as_float(k[3])};
            rope_pair(x[0], x[1], t[0], t[1]);
            rope_pair(x[2], x[3], t[2], t[3]);
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = __float_as_uint(x[j]);
        } else {
            const f32x4_t t0 = ((const f32x4_t*)cs)[0], t1 = ((const f32x4_t*)cs)[1];
            float x[8];
            const float c8[8] = {t0[0], t0[1], t0[2], t0[3], t1[0], t1[1], t1[2], t1[3]};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[2 * j] = Half<T>::lo(k[j]);
                x[2 * j + 1] = Half<T>::hi(k[j]);
            }
            rope4(x, c8);
#pragma unroll
            for (int j = 0; j < 4; ++j) k[j] = Half<T>::pack(x[2 * j], x[2 * j + 1]);
        }
    }
    ((u32x4_t*)a.k_pool)[to] = k;
    ((u32x4_t*)a.v_pool)[to] = v;
}

void launch_append_slots(Dtype dt, const SlotAppendArgs& a, hipStream_t s, unsigned grid[3]) {
    const int e = dt == Dtype::F32 ? 4 : 8;
    const FastDiv per_row((uint32_t)(a.kv_heads * a.head_dim / e)), per_seq((uint32_t)a.max_new),
        per_head((uint32_t)(a.head_dim / e));
    grid[0] = (unsigned)(((int64_t)a.n_rows * per_row.d + 255) / 256);
    grid[1] = grid[2] = 1;
    switch (dt) {
        case Dtype::BF16: append_slots<bf16_t><<<grid[0], 256, 0, s>>>(a, per_row, per_seq, per_head); break;
        case Dtype::F16: append_slots<f16_t><<<grid[0], 256, 0, s>>>(a, per_row, per_seq, per_head); break;
        default: append_slots<float><<<grid[0], 256, 0, s>>>(a, per_row, per_seq, per_head); break;
    }
}

// ---------------------------------------------------------------------------- accepted rows
//
// Row ctx + path[i] -> row ctx + i for the `accepted` tokens of a path through the tree, and the new
// length ctx + accepted. A path is strictly increasing (parents come before children), so path[i] >= i
// and no row is overwritten before it is read if they are moved in order; a thread moves one 16-byte
// column of every row, kAcceptRows loads ahead of their stores (a store goes to a row at or before the
// loads of its round). Bound by latency: the table lookups of all rows at once, then a round of loads; 2
// sequences 4.8 us, 128 with up to 16 rows of 4 KiB (8.4 MB) 4.9.
// A path that is not strictly increasing inside the tree, or that meets an entry outside the pool,
// moves nothing and leaves the length. One workgroup a sequence: it reads the length before any thread
// writes it, so both may be the same array.
constexpr int kAcceptRows = 8;

__global__ __launch_bounds__(1024) void accept_rows(AcceptArgs a, FastDiv ps) {
    __shared__ int from[kTreeTokens], to[kTreeTokens];
    const int s = blockIdx.x, tid = threadIdx.x, threads = blockDim.x;
    const int ctx = a.ctx_lens[s], n_all = a.accepted[s];
    const int len = a.tree_lens[s];
    const bool fits = ctx >= 0 && len >= 0 && len <= a.max_tokens && n_all >= 0 && n_all <= len &&
                      n_all <= a.max_accept &&
                      (int64_t)ctx + len <= (int64_t)a.max_pages * a.page_size;
    const int n = fits ? n_all : 0;
    const int* const path = a.paths + (int64_t)s * a.max_accept;
    const int* const row = a.block_tables + (int64_t)s * a.max_pages;
    auto pool_row = [&](int logical) {
        const int lp = (int)ps.div((uint32_t)logical), page = row[lp];
        return (unsigned)page < (unsigned)a.physical_pages
                   ? page * a.page_size + (logical - lp * a.page_size)
                   : -1;
    };
    int bad = 0;
    for (int i = tid; i < n; i += threads) {
        const int p = path[i];
        if (p < i || p >= len || (i > 0 && path[i - 1] >= p)) {
            bad = 1;
        } else {
            const int f = pool_row(ctx + p), t = pool_row(ctx + i);
            bad |= f < 0 || t < 0;
            from[i] = f;
            to[i] = t;
        }
    }
    bad = __syncthreads_or(bad);
    if (tid == 0) a.ctx_lens_out[s] = fits && !bad ? ctx + n : ctx;
    if (bad || n == 0) return;
    for (int c = tid; c < 2 * a.row_pieces; c += threads) {
        const bool second = c >= a.row_pieces;
        u32x4_t* const pool = (u32x4_t*)(second ? a.v_pool : a.k_pool) + (second ? c - a.row_pieces : c);
        for (int i0 = 0; i0 < n; i0 += kAcceptRows) {
            u32x4_t v[kAcceptRows];
#pragma unroll
            for (int k = 0; k < kAcceptRows; ++k)
                v[k] = pool[(int64_t)from[min(i0 + k, n - 1)] * a.row_pieces];
#pragma unroll
            for (int k = 0; k < kAcceptRows; ++k)
                if (i0 + k < n && to[i0 + k] != from[i0 + k])
                    pool[(int64_t)to[i0 + k] * a.row_pieces] = v[k];
        }
    }
}

void launch_accept(const AcceptArgs& a, hipStream_t s, unsigned grid[3], unsigned* block) {
    const int items = 2 * a.row_pieces;
    const int threads = items >= 1024 ? 1024 : (items + 63) / 64 * 64;
    accept_rows<<<(unsigned)a.n_seqs, threads, 0, s>>>(a, FastDiv((uint32_t)a.page_size));
    grid[0] = (unsigned)a.n_seqs;
    grid[1] = grid[2] = 1;
    *block = (unsigned)threads;
}

}  // namespace fa
