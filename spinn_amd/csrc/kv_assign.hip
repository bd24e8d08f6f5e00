// kv_assign.hip - pages for the next tokens of every sequence, and where each token goes.
//
// Three prefix sums over the sequences: of the pages that ended ones give back, of the tokens, and of the pages that are
// needed; then the pages' numbers are copied between the stack of free ones and the rows of the table, and each token
// finds its sequence by a search among the starts. Nothing here has work to speak of: dependent steps bound it. The
// sums are one workgroup's, 1024 sequences at a time; few tokens are placed by it, too, in the same launch, many by a
// second one, which needs all the starts. 64 sequences of one token: a launch (7.2 us a call); 500, of which 50 bring prompts of
// up to 8000 tokens and 25 end: 22.8 us, 5 of them the second launch's.
#include "decode.h"

namespace spinn {
namespace {

constexpr int kThreads = 1024;
constexpr uint32_t kMany = 1u << 30; // sums stop here: no valid one reaches it

struct AssignArgs {
    const int32_t *new_tokens, *lengths, *next, *held, *free_count;
    int32_t *free_pages, *table, *lengths_out, *next_out, *held_out, *free_count_out, *starts, *served, *seq, *slot, *position;
    int32_t seqs, page_size, n_pages, max_pages, max_tokens;
};

__device__ __forceinline__ uint32_t sum(uint32_t a, uint32_t b) { return min(a + b, kMany); }

// Sum of v over the threads before this one, and over all; `parts` is not used again before the next barrier but one.
__device__ __forceinline__ uint32_t scan(uint32_t v, uint32_t *parts, uint32_t &total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t upto = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t o = __shfl_up(upto, d);
        if (lane >= d) upto = sum(upto, o);
    }
    if (lane == 63) parts[wave] = upto;
    uint32_t before = __shfl_up(upto, 1);
    if (lane == 0) before = 0;
    __syncthreads();
    uint32_t p = lane < kThreads / 64 ? parts[lane] : 0;
#pragma unroll
    for (int d = 1; d < kThreads / 64; d *= 2) {
        const uint32_t o = __shfl_up(p, d);
        if (lane >= d) p = sum(p, o);
    }
    total = __shfl(p, kThreads / 64 - 1);
    return wave ? sum(before, __shfl(p, wave - 1)) : before;
}

// Largest i in [lo, hi) with v(i) <= t, v ascending, v(lo) <= t.
template <class V>
__device__ __forceinline__ int last_upto(V v, int lo, int hi, int t) {
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if (v(mid) <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}
// The same for a t that all lanes share: 64 places a step.
template <class V>
__device__ __forceinline__ int wave_last_upto(V v, int lo, int hi, int t) {
    const int lane = threadIdx.x & 63;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64, at = lo + lane * step;
        const int n = __popcll(__ballot(at < hi && v(at) <= t));
        lo += (n - 1) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}
// The same for t = first.. +63, one a lane, up to `last` (the lanes behind it get its place): one search where they all share a place,
// as a long prompt's tokens do.
template <class V>
__device__ __forceinline__ int lanes_last_upto(V v, int hi, int first, int last) {
    const int lo = wave_last_upto(v, 0, hi, first), end = min(first + 63, last);
    if (lo + 1 >= hi || v(lo + 1) > end) return lo;
    return last_upto(v, lo, wave_last_upto(v, lo, hi, end) + 1, min(first + (int)(threadIdx.x & 63), last));
}

// Page numbers 0 .. n - 1, each of the sequence (of 1024) that `offset` places it in, from one list to another. A wave has a stretch
// of them and goes on from the sequence that it is in; those of four rounds are asked for before the first is written (12600 pages
// there and back, one round after the other with a search each: 17 us, so 10).
template <class V, class From, class To>
__device__ __forceinline__ void move_pages(V offset, int n, From from, To to) {
    constexpr int R = 4, kWaves = kThreads / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int each = ((n + kWaves - 1) / kWaves + 63) & ~63, end = min(n, (wave + 1) * each);
    int first = wave * each;
    if (first >= end) return;
    int at = wave_last_upto(offset, 0, kThreads, first);
    for (; first < end; first += 64 * R) {
        int32_t page[R];
        int owner[R];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = first + 64 * r, last = min(i + 63, end - 1);
            owner[r] = at;
            if (i < end && at + 1 < kThreads && __builtin_amdgcn_readfirstlane(offset(at + 1)) <= last) {
                const int to_at = wave_last_upto(offset, at, kThreads, last);
                owner[r] = last_upto(offset, at, to_at + 1, min(i + lane, last));
                at = to_at;
            }
            page[r] = from(min(i + lane, n - 1), owner[r]);
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = first + 64 * r + lane;
            if (i < end) to(i, owner[r], page[r]);
        }
    }
}

// Tokens first.. +63, one a lane: all lanes of a wave together.
__device__ __forceinline__ void place_tokens(const AssignArgs &a, int first, int total) {
    const int t = first + (int)(threadIdx.x & 63);
    int seq = -1, slot = -1, position = 0;
    if (first < total) {
        const int s = lanes_last_upto([&](int i) { return a.starts[i]; }, a.seqs, first, total - 1);
        if (t < total) {
            if (a.served[s]) {
                const int left = a.starts[s + 1] - t; // tokens to its end
                seq = s;
                slot = a.lengths_out[s] - left;
                position = a.next ? (int32_t)((uint32_t)a.next_out[s] - (uint32_t)left) : slot;
            }
        }
    }
    if (t < a.max_tokens) {
        a.seq[t] = seq;
        a.slot[t] = slot;
        if (a.position) a.position[t] = position;
    }
}

__global__ __launch_bounds__(kThreads) void kv_assign_kernel(AssignArgs a, int place) {
    __shared__ uint32_t before[kThreads + 1], parts[2][kThreads / 64], s_taken;
    __shared__ int32_t s_held[kThreads];
    const int tid = threadIdx.x;
    auto offset = [&](int i) { return (int)before[i]; };
    uint32_t count = (uint32_t)min(max(*a.free_count, 0), a.n_pages);
    if (tid == 0) s_taken = 0;

    bool any = false;
    for (int s = tid; s < a.seqs; s += kThreads) any |= a.new_tokens[s] == -1;
    if (__syncthreads_or(any)) {
        for (int base = 0; base < a.seqs; base += kThreads) {
            const int s = base + tid;
            const uint32_t back = s < a.seqs && a.new_tokens[s] == -1 ? (uint32_t)min(max(a.held[s], 0), a.max_pages) : 0u;
            uint32_t total;
            before[tid] = scan(back, parts[0], total);
            if (tid == 0) before[kThreads] = total;
            __syncthreads();
            total = min(total, (uint32_t)a.n_pages - count);
            move_pages(offset, (int)total, [&](int i, int j) { return a.table[(int64_t)(base + j) * a.max_pages + (i - before[j])]; },
                       [&](int i, int, int32_t page) { a.free_pages[count + i] = page; });
            count += total;
            __syncthreads();
        }
    }

    uint32_t tokens = 0, needed = 0;
    const int64_t capacity = (int64_t)a.page_size * a.max_pages;
    for (int base = 0; base < a.seqs; base += kThreads) {
        const int s = base + tid;
        const bool in = s < a.seqs;
        const int n = in ? a.new_tokens[s] : 0, len = in ? max(a.lengths[s], 0) : 0;
        const int held = in ? min(max(a.held[s], 0), a.max_pages) : 0;
        const uint32_t add = min((uint32_t)max(n, 0), kMany);
        uint32_t total, total_need;
        const uint32_t start = sum(tokens, scan(add, parts[0], total));
        const uint32_t end = sum(start, add);
        const bool fits = n >= -1 && (add == 0 || ((int64_t)len + add <= capacity && end <= (uint32_t)a.max_tokens));
        uint32_t need = 0;
        if (fits && add) need = (uint32_t)max((int)(((uint32_t)len + add - 1u) / (uint32_t)a.page_size) + 1 - held, 0);
        const uint32_t need0 = scan(need, parts[1], total_need);
        const uint32_t upto = sum(needed, sum(need0, need));
        const bool served = fits && (need == 0 || upto <= count);
        before[tid] = need0;
        if (tid == 0) before[kThreads] = total_need;
        s_held[tid] = held;
        if (served && need) atomicMax(&s_taken, upto); // the served ones' needs are the first ones
        if (in) {
            const bool ended = n == -1;
            const uint32_t got = served ? need : 0u, more = served ? add : 0u;
            a.starts[s] = (int32_t)min(start, (uint32_t)a.max_tokens);
            a.served[s] = served;
            if (a.next) a.next_out[s] = ended ? 0 : (int32_t)((uint32_t)max(a.next[s], 0) + more);
            a.lengths_out[s] = ended ? 0 : (int32_t)((uint32_t)len + more);
            a.held_out[s] = ended ? 0 : (int32_t)((uint32_t)held + got);
        }
        __syncthreads();
        const uint32_t most = needed < count ? min(total_need, count - needed) : 0u;
        move_pages(offset, (int)most, [&](int i, int) { return a.free_pages[count - 1 - (needed + i)]; },
                   [&](int i, int j, int32_t page) {
                       if (sum(needed, before[j + 1]) <= count) a.table[(int64_t)(base + j) * a.max_pages + s_held[j] + (i - before[j])] = page;
                   });
        tokens = sum(tokens, total);
        needed = sum(needed, total_need);
        __syncthreads();
    }
    if (tid == 0) {
        *a.free_count_out = (int32_t)(count - s_taken);
        a.starts[a.seqs] = (int32_t)min(tokens, (uint32_t)a.max_tokens);
    }
    if (!place) return;
    __syncthreads();
    for (int t = tid & ~63; t < a.max_tokens; t += kThreads) place_tokens(a, t, (int)min(tokens, (uint32_t)a.max_tokens));
}

__global__ __launch_bounds__(256) void kv_place_kernel(AssignArgs a) {
    const int total = a.starts[a.seqs];
    for (int t = (int)(blockIdx.x * 256 + (threadIdx.x & ~63u)); t < a.max_tokens; t += (int)gridDim.x * 256) place_tokens(a, t, total);
}

} // namespace

int kv_assign(const SpinnHipKvAssignDesc *d, const int32_t *new_tokens, const int32_t *lengths, const int32_t *next,
              const int32_t *held, const int32_t *free_count, int32_t *free_pages, int32_t *table, int32_t *lengths_out,
              int32_t *next_out, int32_t *held_out, int32_t *free_count_out, int32_t *starts, int32_t *served, int32_t *seq,
              int32_t *slot, int32_t *position, hipStream_t st) {
    AssignArgs a{};
    a.new_tokens = new_tokens;
    a.lengths = lengths;
    a.next = next;
    a.held = held;
    a.free_count = free_count;
    a.free_pages = free_pages;
    a.table = table;
    a.lengths_out = lengths_out;
    a.next_out = next_out;
    a.held_out = held_out;
    a.free_count_out = free_count_out;
    a.starts = starts;
    a.served = served;
    a.seq = seq;
    a.slot = slot;
    a.position = position;
    a.seqs = d->seqs;
    a.page_size = d->page_size;
    a.n_pages = d->n_pages;
    a.max_pages = d->max_pages;
    a.max_tokens = d->max_tokens;
    const bool one = d->max_tokens <= 4096;
    kv_assign_kernel<<<1, kThreads, 0, st>>>(a, one);
    if (!one) kv_place_kernel<<<(unsigned)std::min((d->max_tokens + 255) / 256, 4096), 256, 0, st>>>(a);
    return check_launch();
}

} // namespace spinn
