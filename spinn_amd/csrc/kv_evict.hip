// kv_evict.hip - eviction from a paged key-value cache by accumulated attention weight.
//
// Per (sequence, kv head): of n slots the `budget` of the highest (key, lowest slot) stay, key
// ordering safe tokens before all others and those by weight. Two launches:
//  * one workgroup per row finds the budget-th key by radix selection (11, 11 and 10 bits, counts in
//    LDS), then numbers the places below the budget that fall free and the kept slots behind
//    it; the n-th of these goes to the n-th of those. A source is never below the
//    budget and a destination always is, so nothing is read after it was overwritten, and no more
//    rows move than have to. Up to 8192 slots a thread holds 8 neighbouring keys in registers and
//    each numbering is one prefix sum; longer rows walk through memory in steps of 1024;
//  * the rows are moved, 16 lanes per row of K and V.
// Bound: the rows' moves by memory (256-byte rows at random), the selection by its dozen dependent steps.
// 16 sequences of 3000 to 8000 slots, 8 heads of 128 bf16, cut to 2000: selection 13 us, moves 47 us (3.8 TB/s).
// (Counts added up by a wave's ballots before they go to LDS: selection 36 us, the vector units of the one CU.)
#include "decode.h"

namespace spinn {
namespace {

typedef int32_t i32x4 __attribute__((ext_vector_type(4)));

constexpr int kPick = 1024;      // threads of a selecting workgroup, at most
constexpr int kHeld = 8;         // keys that a thread holds in registers
constexpr int kMovesPer = 64;    // moves per workgroup of the second launch
constexpr int kMoveGroups = 1 << 20; // workgroups of it at once

struct EvictArgs {
    const int32_t *table, *lengths, *next_pos, *pos;
    const float *acc;
    float *acc_out;
    int32_t *pos_out, *lengths_out;
    int32_t *left;      // [seqs] slots left
    int32_t *n_moves;   // [rows]
    int32_t *from, *to; // [rows][most]
    int64_t acc_stride, page_stride, head_stride, slot_stride;
    int32_t kv_heads, page_size, n_pages, max_pages, budget, recent, sinks, max_len, most;
    int32_t runs; // rows of acc and pos, in and out, start at multiples of 16 bytes
};

// Order of slots as unsigned numbers: NaN 0, then -inf .. +inf, safe tokens last.
__device__ __forceinline__ uint32_t key_of(const EvictArgs &a, float w, int pos, int64_t first_recent) {
    if (pos < a.sinks || (int64_t)pos >= first_recent) return 0xffffffffu;
    if (w != w) return 0u;
    const uint32_t b = __builtin_bit_cast(uint32_t, w == 0.f ? 0.f : w); // both zeros are equal
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive prefix sum of v over the W waves of the workgroup, in thread order; total in `all`. Two barriers.
template <int W>
__device__ __forceinline__ int prefix(int v, int *waves, int &all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int o = __shfl_up(s, off);
        if (lane >= off) s += o;
    }
    __syncthreads(); // the last call's readers are done
    if (lane == 63) waves[wave] = s;
    __syncthreads();
    int before = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        const int c = waves[w];
        if (w < wave) before += c;
        all += c;
    }
    return before + s - v;
}

// The want-th largest of the workgroup's keys, by 11, 11 and 10 bits: on return keys above `found` are higher, and
// `want` of those equal to it belong to the want highest. Ends early where all keys that share the bits found so
// far do: `found` is then the least number with those bits, less 1.
// count(high, found, shift, hist) adds the keys that share found's upper bits to hist.
constexpr int kBins = 2048;
template <int W, class F>
__device__ __forceinline__ void select_key(uint32_t &found, int &want, int *hist, int *waves, F count) {
    __shared__ uint32_t s_found;
    __shared__ int s_want, s_in;
    constexpr int kPer = kBins / (64 * W);
    const int tid = threadIdx.x;
    found = 0;
    uint32_t high = 0;
    for (int shift = 21; shift >= 0; shift = shift == 21 ? 10 : shift == 10 ? 0 : -1) {
#pragma unroll
        for (int j = 0; j < kPer; ++j) hist[tid + j * 64 * W] = 0;
        __syncthreads();
        count(high, found, shift, hist);
        __syncthreads();
        // thread t: kPer bins from the top (in the last pass the highest of the 11 bits is one found before)
        int c[kPer], sum = 0;
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            c[j] = hist[kBins - 1 - kPer * tid - j];
            sum += c[j];
        }
        int all;
        int above = prefix<W>(sum, waves, all);
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
            if (above < want && want <= above + c[j]) {
                s_found = found | (uint32_t)(kBins - 1 - kPer * tid - j) << shift;
                s_want = want - above;
                s_in = c[j];
            }
            above += c[j];
        }
        __syncthreads();
        found = s_found;
        want = s_want;
        high = 0xffffffffu << shift;
        if (want == s_in && found != 0) { // (a found of 0 has no number below it; the next passes end there too)
            found -= 1;
            want = 0;
            return;
        }
    }
}

// TH threads; HELD: rows of up to TH * kHeld slots, else of any length.
template <int TH, bool HELD>
__global__ __launch_bounds__(TH) void evict_pick_kernel(EvictArgs a) {
    const int row = blockIdx.x, seq = row / a.kv_heads, tid = threadIdx.x;
    const int n = min(max(a.lengths[seq], 0), a.max_len);
    const int left = min(n, a.budget);
    const float *acc = a.acc + (int64_t)row * a.acc_stride;
    const int32_t *pos = a.pos + (int64_t)row * a.acc_stride;
    float *acc_out = a.acc_out + (int64_t)row * a.acc_stride;
    int32_t *pos_out = a.pos_out + (int64_t)row * a.acc_stride;
    if (row == seq * a.kv_heads && tid == 0) a.left[seq] = left;
    if (left == n || left == 0) { // everything stays, or nothing
        if (tid == 0) a.n_moves[row] = 0;
        for (int i = tid; i < left; i += TH) {
            acc_out[i] = acc[i];
            pos_out[i] = pos[i];
        }
        return;
    }
    const int64_t first_recent = (int64_t)a.next_pos[seq] - a.recent;
    constexpr int W = TH / 64;
    __shared__ int waves[W], hist[kBins];
    int32_t *from = a.from + (int64_t)row * a.most, *to = a.to + (int64_t)row * a.most;
    uint32_t found;
    int want = left, moves;
    if constexpr (HELD) {
        // the thread's slots: kHeld neighbours, so that one prefix sum over threads numbers them all
        const int first = tid * kHeld;
        float w[kHeld];
        int p[kHeld];
        uint32_t key[kHeld];
        if (a.runs && first + kHeld <= n) {
#pragma unroll
            for (int j = 0; j < kHeld; j += 4) {
                const f32x4 wv = *reinterpret_cast<const f32x4 *>(acc + first + j);
                const i32x4 pv = *reinterpret_cast<const i32x4 *>(pos + first + j);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[j + i] = wv[i];
                    p[j + i] = pv[i];
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < kHeld; ++j) {
                w[j] = first + j < n ? acc[first + j] : 0.f;
                p[j] = first + j < n ? pos[first + j] : 0;
            }
        }
#pragma unroll
        for (int j = 0; j < kHeld; ++j) key[j] = key_of(a, w[j], p[j], first_recent);
        select_key<W>(found, want, hist, waves, [&](uint32_t high, uint32_t found, int shift, int *hist) {
#pragma unroll
            for (int j = 0; j < kHeld; ++j)
                if (first + j < n && (key[j] & high) == found) atomicAdd(&hist[key[j] >> shift & (kBins - 1)], 1);
        });
        int equal = 0, all;
#pragma unroll
        for (int j = 0; j < kHeld; ++j) equal += first + j < n && key[j] == found;
        equal = prefix<W>(equal, waves, all);
        uint32_t kept = 0;
        int holes = 0, movers = 0;
#pragma unroll
        for (int j = 0; j < kHeld; ++j) {
            const int i = first + j;
            const bool eq = key[j] == found;
            const bool keep = i < n && (key[j] > found || (eq && equal < want));
            equal += eq;
            kept |= (uint32_t)keep << j;
            holes += i < left && !keep;
            movers += i >= left && keep;
        }
        // both in one sum: at most 8192 of each
        int at = prefix<W>(holes | movers << 16, waves, all);
        int hole = at & 0xffff, mover = at >> 16;
        moves = all >> 16;
        // a mover leaves its slot and what goes with it by its number, the hole of that number fetches them
        __shared__ int32_t slot_by[TH * kHeld / 2];
        __shared__ float acc_by[TH * kHeld / 2];
        __shared__ int32_t pos_by[TH * kHeld / 2];
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (first + j >= left && kept >> j & 1) {
                slot_by[mover] = first + j;
                acc_by[mover] = w[j];
                pos_by[mover] = p[j];
                ++mover;
            }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kHeld; ++j)
            if (first + j < left && !(kept >> j & 1)) {
                w[j] = acc_by[hole];
                p[j] = pos_by[hole];
                from[hole] = slot_by[hole];
                to[hole] = first + j;
                ++hole;
            }
        if (a.runs && first + kHeld <= left) {
#pragma unroll
            for (int j = 0; j < kHeld; j += 4) {
                *reinterpret_cast<f32x4 *>(acc_out + first + j) = (f32x4){w[j], w[j + 1], w[j + 2], w[j + 3]};
                *reinterpret_cast<i32x4 *>(pos_out + first + j) = (i32x4){p[j], p[j + 1], p[j + 2], p[j + 3]};
            }
        } else {
#pragma unroll
            for (int j = 0; j < kHeld; ++j)
                if (first + j < left) {
                    acc_out[first + j] = w[j];
                    pos_out[first + j] = p[j];
                }
        }
    } else {
        select_key<W>(found, want, hist, waves, [&](uint32_t high, uint32_t found, int shift, int *hist) {
#pragma unroll 4
            for (int i = tid; i < n; i += TH) {
                const uint32_t k = key_of(a, acc[i], pos[i], first_recent);
                if ((k & high) == found) atomicAdd(&hist[k >> shift & (kBins - 1)], 1);
            }
        });
        int equal_before = 0, free_before = 0, moved_before = 0;
        for (int base = 0; base < n; base += TH) {
            const int i = base + tid;
            const uint32_t k = i < n ? key_of(a, acc[i], pos[i], first_recent) : 0u;
            const bool eq = i < n && k == found;
            int all;
            const int eq_rank = equal_before + prefix<W>(eq, waves, all);
            equal_before += all;
            const bool kept = i < n && (k > found || (eq && eq_rank < want));
            const bool hole = i < left && !kept, mover = i >= left && kept;
            // one sum for both: at most TH of each per step
            const int both = prefix<W>((int)hole | (int)mover << 16, waves, all);
            if (hole) to[free_before + (both & 0xffff)] = i;
            if (mover) from[moved_before + (both >> 16)] = i;
            free_before += all & 0xffff;
            moved_before += all >> 16;
        }
        moves = moved_before;
        if (acc_out != acc || pos_out != pos)
            for (int i = tid; i < left; i += TH) {
                if (acc_out != acc) acc_out[i] = acc[i];
                if (pos_out != pos) pos_out[i] = pos[i];
            }
        __syncthreads();
        for (int i = tid; i < moves; i += TH) {
            acc_out[to[i]] = acc[from[i]];
            pos_out[to[i]] = pos[from[i]];
        }
    }
    // as many holes as movers: both are `left` less the kept slots below the budget
    if (tid == 0) a.n_moves[row] = moves;
}

// 16 lanes per move, `U` the unit of copying. `chunks` workgroups a row, from the first-th share of its moves on.
template <class U>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a, U *k, U *v, int units, int chunks, int first) {
    const int row = blockIdx.x / chunks, chunk = first + (int)blockIdx.x - row * chunks;
    const int seq = row / a.kv_heads, head = row - seq * a.kv_heads;
    if (chunk == 0 && head == 0 && threadIdx.x == 0) a.lengths_out[seq] = a.left[seq];
    const int n = a.n_moves[row];
    const int32_t *table = a.table + (int64_t)seq * a.max_pages;
    const int l = threadIdx.x & 15;
    // a lane's moves, all their reads in flight before the first write
    constexpr int M = kMovesPer / 16;
    const U *src_k[M], *src_v[M];
    int64_t dst[M];
    int moves = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) {
        const int at = chunk * kMovesPer + i * 16 + (threadIdx.x >> 4);
        dst[i] = -1;
        src_k[i] = k;
        src_v[i] = v;
        if (at < n) {
            const int from = a.from[(int64_t)row * a.most + at], to = a.to[(int64_t)row * a.most + at];
            const int fp = from / a.page_size, tp = to / a.page_size;
            const int from_page = table[fp], to_page = table[tp];
            if ((unsigned)from_page < (unsigned)a.n_pages && (unsigned)to_page < (unsigned)a.n_pages) {
                const int64_t s = (int64_t)from_page * a.page_stride + (int64_t)head * a.head_stride +
                                  (int64_t)(from - fp * a.page_size) * a.slot_stride;
                dst[i] = (int64_t)to_page * a.page_stride + (int64_t)head * a.head_stride +
                         (int64_t)(to - tp * a.page_size) * a.slot_stride;
                src_k[i] = k + s;
                src_v[i] = v + s;
                ++moves;
            }
        }
    }
    if (moves == 0) return;
    for (int u = l; u < units; u += 16) {
        U kk[M], vv[M];
#pragma unroll
        for (int i = 0; i < M; ++i)
            if (dst[i] >= 0) {
                kk[i] = src_k[i][u];
                vv[i] = src_v[i][u];
            }
#pragma unroll
        for (int i = 0; i < M; ++i)
            if (dst[i] >= 0) {
                k[dst[i] + u] = kk[i];
                v[dst[i] + u] = vv[i];
            }
    }
}

int most_moves(const SpinnHipKvEvictDesc *d) {
    return d->max_len > d->budget ? std::min(d->budget, d->max_len - d->budget) : 0;
}

} // namespace

size_t kv_evict_workspace_bytes(const SpinnHipKvEvictDesc *d) {
    const size_t rows = (size_t)d->kv.seqs * d->kv.kv_heads;
    return round16(4 * (size_t)d->kv.seqs) + round16(4 * rows) + 2 * round16(4 * rows * most_moves(d));
}

int kv_evict(const SpinnHipKvEvictDesc *d, const int32_t *table, const int32_t *lengths, const int32_t *next_pos,
             const float *acc, const int32_t *pos, float *acc_out, int32_t *pos_out, int32_t *lengths_out, void *k,
             void *v, void *ws, hipStream_t st) {
    const SpinnHipKvDesc &kv = d->kv;
    const size_t rows = (size_t)kv.seqs * kv.kv_heads;
    EvictArgs a{};
    a.table = table;
    a.lengths = lengths;
    a.next_pos = next_pos;
    a.pos = pos;
    a.acc = acc;
    a.acc_out = acc_out;
    a.pos_out = pos_out;
    a.lengths_out = lengths_out;
    a.most = most_moves(d);
    char *w = (char *)ws;
    a.left = (int32_t *)w;
    w += round16(4 * (size_t)kv.seqs);
    a.n_moves = (int32_t *)w;
    w += round16(4 * rows);
    a.from = (int32_t *)w;
    w += round16(4 * rows * a.most);
    a.to = (int32_t *)w;
    a.acc_stride = d->acc_stride;
    a.kv_heads = kv.kv_heads;
    a.page_size = kv.page_size;
    a.n_pages = kv.n_pages;
    a.max_pages = kv.max_pages;
    a.budget = d->budget;
    a.recent = d->recent;
    a.sinks = d->sinks;
    a.max_len = d->max_len;
    if (!launch_fits((int64_t)rows, kPick)) return SPINN_HIP_EUNSUPPORTED;
    a.runs = d->acc_stride % 4 == 0 && aligned16(acc) && aligned16(pos) && aligned16(acc_out) && aligned16(pos_out);
    if (d->max_len <= 256 * kHeld) evict_pick_kernel<256, true><<<(unsigned)rows, 256, 0, st>>>(a);
    else if (d->max_len <= kPick * kHeld) evict_pick_kernel<kPick, true><<<(unsigned)rows, kPick, 0, st>>>(a);
    else evict_pick_kernel<kPick, false><<<(unsigned)rows, kPick, 0, st>>>(a);
    int rc = check_launch();
    if (rc) return rc;
    // units of 16 bytes where rows are whole runs of them
    const int e = dtype_bytes(kv.dtype), per = 16 / e;
    const bool vec = kv.head_dim % per == 0 && kv.page_stride % per == 0 && kv.head_stride % per == 0 &&
                     kv.slot_stride % per == 0 && aligned16(k) && aligned16(v);
    const int div = vec ? per : 1;
    a.page_stride = kv.page_stride / div;
    a.head_stride = kv.head_stride / div;
    a.slot_stride = kv.slot_stride / div;
    const int units = kv.head_dim / div;
    // all shares of moves in one launch, unless that has too many workgroups
    const int chunks = std::max(1, (a.most + kMovesPer - 1) / kMovesPer);
    const int at_once = (int)std::max<int64_t>(1, std::min<int64_t>(chunks, kMoveGroups / (int64_t)rows));
    for (int first = 0; first < chunks && !rc; first += at_once) {
        const unsigned grid = (unsigned)(rows * at_once);
        if (vec) evict_move_kernel<<<grid, 256, 0, st>>>(a, (u32x4 *)k, (u32x4 *)v, units, at_once, first);
        else if (e == 4) evict_move_kernel<<<grid, 256, 0, st>>>(a, (uint32_t *)k, (uint32_t *)v, units, at_once, first);
        else evict_move_kernel<<<grid, 256, 0, st>>>(a, (uint16_t *)k, (uint16_t *)v, units, at_once, first);
        rc = check_launch();
    }
    return rc;
}

} // namespace spinn
