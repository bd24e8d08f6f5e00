// kv_evict.hip - eviction from a paged key-value cache by accumulated attention weight.
//
// Per (sequence, kv head): of n slots the `budget` of the highest (key, lowest slot) stay, key
// ordering safe tokens before all others and those by weight. Two launches:
//  * one workgroup per row finds the budget-th key by radix selection (four passes over 8 bits, counts in
//    LDS), then walks the slots once, numbering the places below the budget that fall free and
//    the kept slots behind it; the n-th of these goes to the n-th of those. A source is
//    never below the budget and a destination always is, so nothing is read after it was
//    overwritten, and no more rows move than have to;
//  * the rows are moved, a quarter wave per row of K and V.
#include "decode.h"

namespace spinn {
namespace {

constexpr int kPick = 1024;      // threads of a selecting workgroup
constexpr int kCached = 8192;    // keys that it holds in LDS
constexpr int kMovesPer = 64;    // moves per workgroup of the second launch

struct EvictArgs {
    const int32_t *table, *lengths, *next_pos, *pos;
    const float *acc;
    float *acc_out;
    int32_t *pos_out, *lengths_out;
    int32_t *left;      // [seqs] slots left
    int32_t *n_moves;   // [rows]
    int32_t *from, *to; // [rows][most]
    int64_t acc_stride, page_stride, head_stride, slot_stride;
    int32_t seqs, kv_heads, dim, page_size, n_pages, max_pages, budget, recent, sinks, max_len, most;
};

// Order of slots as unsigned numbers: NaN 0, then -inf .. +inf, safe tokens last.
__device__ __forceinline__ uint32_t key_of(const EvictArgs &a, float w, int pos, int64_t first_recent) {
    if (pos < a.sinks || (int64_t)pos >= first_recent) return 0xffffffffu;
    if (w != w) return 0u;
    const uint32_t b = __builtin_bit_cast(uint32_t, w == 0.f ? 0.f : w); // both zeros are equal
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Exclusive prefix sum of v over the workgroup, in thread order; total in `all`. Two barriers.
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
    for (int w = 0; w < kPick / 64; ++w) {
        const int c = waves[w];
        if (w < wave) before += c;
        all += c;
    }
    return before + s - v;
}

__global__ __launch_bounds__(kPick) void evict_pick_kernel(EvictArgs a) {
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
        for (int i = tid; i < left; i += kPick) {
            acc_out[i] = acc[i];
            pos_out[i] = pos[i];
        }
        return;
    }
    const int64_t first_recent = (int64_t)a.next_pos[seq] - a.recent;
    __shared__ uint32_t cached[kCached];
    __shared__ int hist[256];
    __shared__ int waves[kPick / 64];
    __shared__ uint32_t s_prefix;
    __shared__ int s_want;
    const bool in_lds = n <= kCached;
    auto key = [&](int i) { return in_lds ? cached[i] : key_of(a, acc[i], pos[i], first_recent); };
    if (in_lds)
        for (int i = tid; i < n; i += kPick) cached[i] = key_of(a, acc[i], pos[i], first_recent);

    // the left-th largest key: `prefix` holds its upper bits, `want` its rank among the keys that share them
    uint32_t found = 0;
    int want = left;
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t high = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
        for (int i = tid; i < n; i += kPick) {
            const uint32_t k = key(i);
            if ((k & high) == found) atomicAdd(&hist[k >> shift & 255u], 1);
        }
        __syncthreads();
        if (tid < 64) { // lane l: bins 255-4l .. 252-4l, from the top
            int c[4], sum = 0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                c[j] = hist[255 - 4 * tid - j];
                sum += c[j];
            }
            int incl = sum;
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int o = __shfl_up(incl, off);
                if (tid >= off) incl += o;
            }
            int above = incl - sum;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (above < want && want <= above + c[j]) {
                    s_prefix = found | (uint32_t)(255 - 4 * tid - j) << shift;
                    s_want = want - above;
                }
                above += c[j];
            }
        }
        __syncthreads();
        found = s_prefix;
        want = s_want;
    }

    // places that fall free and kept slots behind the budget, each numbered in slot order
    int32_t *from = a.from + (int64_t)row * a.most, *to = a.to + (int64_t)row * a.most;
    int equal_before = 0, free_before = 0, moved_before = 0;
    for (int base = 0; base < n; base += kPick) {
        const int i = base + tid;
        const uint32_t k = i < n ? key(i) : 0u;
        const bool eq = i < n && k == found;
        int all;
        const int eq_rank = equal_before + prefix(eq, waves, all);
        equal_before += all;
        const bool kept = i < n && (k > found || (eq && eq_rank < want));
        const bool hole = i < left && !kept, mover = i >= left && kept;
        // one sum for both: at most kPick of each per step
        const int both = prefix((int)hole | (int)mover << 16, waves, all);
        if (hole) to[free_before + (both & 0xffff)] = i;
        if (mover) from[moved_before + (both >> 16)] = i;
        free_before += all & 0xffff;
        moved_before += all >> 16;
    }
    __syncthreads();
    // as many of the one as of the other: both are `left` less the kept slots below the budget
    if (tid == 0) a.n_moves[row] = moved_before;
    if (acc_out != acc || pos_out != pos)
        for (int i = tid; i < left; i += kPick) {
            if (acc_out != acc) acc_out[i] = acc[i];
            if (pos_out != pos) pos_out[i] = pos[i];
        }
    __syncthreads();
    for (int i = tid; i < moved_before; i += kPick) {
        acc_out[to[i]] = acc[from[i]];
        pos_out[to[i]] = pos[from[i]];
    }
}

// 16 lanes per move, `U` the unit of copying.
template <class U>
__global__ __launch_bounds__(256) void evict_move_kernel(EvictArgs a, U *k, U *v, int units, int chunks) {
    const int row = blockIdx.x / chunks, chunk = blockIdx.x - row * chunks;
    const int seq = row / a.kv_heads, head = row - seq * a.kv_heads;
    if (chunk == 0 && head == 0 && threadIdx.x == 0) a.lengths_out[seq] = a.left[seq];
    const int n = a.n_moves[row];
    const int32_t *table = a.table + (int64_t)seq * a.max_pages;
    const int l = threadIdx.x & 15;
    for (int i = chunk * kMovesPer + (threadIdx.x >> 4); i < min(n, (chunk + 1) * kMovesPer); i += 16) {
        const int from = a.from[(int64_t)row * a.most + i], to = a.to[(int64_t)row * a.most + i];
        const int fp = from / a.page_size, tp = to / a.page_size;
        const int from_page = table[fp], to_page = table[tp];
        if ((unsigned)from_page >= (unsigned)a.n_pages || (unsigned)to_page >= (unsigned)a.n_pages) continue;
        const int64_t s = (int64_t)from_page * a.page_stride + (int64_t)head * a.head_stride +
                          (int64_t)(from - fp * a.page_size) * a.slot_stride;
        const int64_t d = (int64_t)to_page * a.page_stride + (int64_t)head * a.head_stride +
                          (int64_t)(to - tp * a.page_size) * a.slot_stride;
        for (int u = l; u < units; u += 16) {
            const U kk = k[s + u], vv = v[s + u];
            k[d + u] = kk;
            v[d + u] = vv;
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
    a.seqs = kv.seqs;
    a.kv_heads = kv.kv_heads;
    a.dim = kv.head_dim;
    a.page_size = kv.page_size;
    a.n_pages = kv.n_pages;
    a.max_pages = kv.max_pages;
    a.budget = d->budget;
    a.recent = d->recent;
    a.sinks = d->sinks;
    a.max_len = d->max_len;
    const int chunks = std::max(1, (a.most + kMovesPer - 1) / kMovesPer);
    if ((int64_t)rows * chunks > INT32_MAX) return SPINN_HIP_EUNSUPPORTED;
    evict_pick_kernel<<<(unsigned)rows, kPick, 0, st>>>(a);
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
    const unsigned grid = (unsigned)(rows * chunks);
    const int units = kv.head_dim / div;
    if (vec) evict_move_kernel<<<grid, 256, 0, st>>>(a, (u32x4 *)k, (u32x4 *)v, units, chunks);
    else if (e == 4) evict_move_kernel<<<grid, 256, 0, st>>>(a, (uint32_t *)k, (uint32_t *)v, units, chunks);
    else evict_move_kernel<<<grid, 256, 0, st>>>(a, (uint16_t *)k, (uint16_t *)v, units, chunks);
    return check_launch();
}

} // namespace spinn
