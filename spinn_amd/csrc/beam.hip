// beam.hip - beam search: the k best continuations over all beams and the vocabulary, and
// the reordering of the beams' states after their parents.
//
// key(b,t) = score_b + x_bt - lse_b. Within a beam the keys order as the logits do, so one pass over a
// chunk of a row finds the chunk's share of lse (its maximum and its sum of exponentials) and its k
// first candidates together, from registers. The second launch joins a batch item's chunks.
// Both pick k of n unique 64-bit ranks the same way: of the threads' own maxima the k-th largest
// bounds the k-th largest of all from below, few elements pass it (at most k threads hold any),
// and those few are ranked by counting. Bound: memory, each logit read once.
#include "decode.h"

namespace spinn {
namespace {

constexpr int kBeamThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

// fp32 to an unsigned number of the same order, both zeros equal; NaN as -inf, +inf as the largest finite.
__device__ __forceinline__ float clean(float v) {
    if (v != v) return -INFINITY;
    v = v == 0.f ? 0.f : v;
    return fminf(v, 3.402823466e38f);
}
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
    return __builtin_bit_cast(float, o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t ordered64(double v) {
    const uint64_t b = __builtin_bit_cast(uint64_t, v == 0.0 ? 0.0 : v);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

struct BeamArgs {
    const void *logits;
    const float *scores;
    const uint8_t *finished;
    float *out_scores;
    int32_t *out_parents, *out_tokens;
    float *chunk_max;    // [rows][chunks]
    double *chunk_sum;   // [rows][chunks]: sum of exp(x - chunk_max)
    uint64_t *candidate; // [rows][chunks][k]: ordered logit << 32 | ~token, 0 = none
    int64_t stride;
    int32_t batch, beams, vocab, k, end, chunks;
};

// Elements per thread of a chunk of kBeamThreads * EPT.
template <class T, int EPT, bool VEC>
__global__ __launch_bounds__(kBeamThreads) void beam_chunk_kernel(BeamArgs a) {
    constexpr int E = 16 / (int)sizeof(T);
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *x = (const T *)a.logits + (int64_t)row * a.stride;
    const int base = chunk * kBeamThreads * EPT;
    const float score = clean(a.scores[row]);
    const bool ended = a.finished && a.finished[row], empty = score == -INFINITY;

    // runs of E elements, a workgroup's runs side by side: equal logits then spread over the threads
    float v[EPT];
    int first[EPT / E]; // token of each run's first element
#pragma unroll
    for (int r = 0; r < EPT / E; ++r) first[r] = base + (r * kBeamThreads + tid) * E;
    if (ended || empty) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) v[i] = ended && !empty && first[i / E] + i % E == a.end ? 0.f : -INFINITY;
    } else if constexpr (VEC) {
#pragma unroll
        for (int r = 0; r < EPT / E; ++r) { // a row is whole runs
            u32x4 w = {0, 0, 0, 0};
            if (first[r] < a.vocab) w = *reinterpret_cast<const u32x4 *>(x + first[r]);
            const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int i = 0; i < E; ++i) v[r * E + i] = (float)e[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const int t = first[i / E] + i % E;
            v[i] = t < a.vocab ? (float)x[t] : 0.f;
        }
    }
    // the thread's maximum, by value and then by the lower token
    float best = -INFINITY;
    uint64_t mine = 0;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        const int t = first[i / E] + i % E;
        v[i] = clean(v[i]);
        const uint64_t u = t < a.vocab ? (uint64_t)ordered(v[i]) << 32 | (uint32_t)~t : 0ull;
        mine = u > mine ? u : mine;
        if (t < a.vocab) best = fmaxf(best, v[i]);
    }

    __shared__ uint64_t top[kBeamThreads];
    __shared__ float wmax[kBeamThreads / 64];
    __shared__ double wsum[kBeamThreads / 64];
    __shared__ uint64_t bound;
    __shared__ int count;
    extern __shared__ uint64_t list[]; // [k * EPT]
    top[tid] = mine;
#pragma unroll
    for (int off = 32; off; off >>= 1) best = fmaxf(best, __shfl_xor(best, off));
    if (lane == 0) wmax[wave] = best;
    if (tid == 0) {
        bound = 0;
        count = 0;
    }
    __syncthreads();
    float m = wmax[0];
#pragma unroll
    for (int w = 1; w < kBeamThreads / 64; ++w) m = fmaxf(m, wmax[w]);

    // share of the sum: exponentials in fp32, added in fp64, so that beams compare to about 1e-8
    if (!ended && !empty) {
        double sum = 0.0;
        if (m != -INFINITY) {
#pragma unroll
            for (int i = 0; i < EPT; i += 4) {
                float part = 0.f;
#pragma unroll
                for (int j = i; j < i + 4; ++j)
                    part += first[j / E] + j % E < a.vocab ? __builtin_amdgcn_exp2f((v[j] - m) * kLog2e) : 0.f;
                sum += (double)part;
            }
        }
#pragma unroll
        for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off);
        if (lane == 0) wsum[wave] = sum;
    }

    // the k-th largest of the threads' maxima (unique but for the 0 of threads without elements)
    if (a.k < kBeamThreads && mine != 0) {
        int above = 0;
        for (int i = 0; i < kBeamThreads; ++i) above += top[i] > mine;
        if (above == a.k - 1) bound = mine;
    }
    __syncthreads();
    if (tid == 0) {
        a.chunk_max[blockIdx.x] = ended ? 0.f : m;
        double sum = 1.0;
        if (!ended && !empty) {
            sum = wsum[0];
#pragma unroll
            for (int w = 1; w < kBeamThreads / 64; ++w) sum += wsum[w];
        }
        a.chunk_sum[blockIdx.x] = sum;
    }
    const uint64_t least = bound;
    if (mine != 0 && mine >= least) {
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const int t = first[i / E] + i % E;
            const uint64_t u = t < a.vocab ? (uint64_t)ordered(v[i]) << 32 | (uint32_t)~t : 0ull;
            if (u != 0 && u >= least) list[atomicAdd(&count, 1)] = u;
        }
    }
    __syncthreads();
    // ranks by counting: which slot of the list an element got does not matter
    const int n = count;
    uint64_t *out = a.candidate + (int64_t)blockIdx.x * a.k;
    for (int i = tid; i < n; i += kBeamThreads) {
        const uint64_t u = list[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += list[j] > u;
        if (rank < a.k) out[rank] = u;
    }
    for (int i = n + tid; i < a.k; i += kBeamThreads) out[i] = 0;
}

// One workgroup per batch item: lse per beam, then the k first of the chunks' candidates in the order
// of (key, lower beam, logit, lower token).
constexpr int kJoinThreads = 512;
constexpr int kJoinList = 1024; // candidates that pass the bound and are ranked by counting

struct Rank {
    uint64_t key; // of the double, ordered; 0 = none
    uint32_t tie; // beams - beam
    uint64_t cand;
};
__device__ __forceinline__ bool above(const Rank &p, const Rank &q) {
    return p.key != q.key ? p.key > q.key : (p.tie != q.tie ? p.tie > q.tie : p.cand > q.cand);
}

__global__ __launch_bounds__(kJoinThreads) void beam_join_kernel(BeamArgs a) {
    constexpr int kWaves = kJoinThreads / 64;
    const int item = blockIdx.x, tid = threadIdx.x;
    const int lane = tid & 63, wave = tid >> 6;
    __shared__ double lse[SPINN_HIP_BEAM_MAX], score[SPINN_HIP_BEAM_MAX];
    __shared__ Rank list[kJoinList]; // first the threads' maxima, then what passes the bound
    __shared__ Rank bound, best[kWaves];
    __shared__ int count;
    if (tid == 0) {
        bound = Rank{0, 0, 0};
        count = 0;
    }
    for (int b = wave; b < a.beams; b += kWaves) {
        const int row = item * a.beams + b;
        const float *cm = a.chunk_max + (int64_t)row * a.chunks;
        const double *cs = a.chunk_sum + (int64_t)row * a.chunks;
        float m = -INFINITY;
        for (int i = lane; i < a.chunks; i += 64) m = fmaxf(m, cm[i]);
#pragma unroll
        for (int off = 32; off; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
        double s = 0.0;
        if (m != -INFINITY)
            for (int i = lane; i < a.chunks; i += 64) s += cs[i] * exp((double)cm[i] - (double)m);
#pragma unroll
        for (int off = 32; off; off >>= 1) s += __shfl_xor(s, off);
        if (lane == 0) {
            const bool ended = a.finished && a.finished[row];
            score[b] = (double)clean(a.scores[row]);
            lse[b] = ended || m == -INFINITY ? 0.0 : (double)m + log(s);
        }
    }
    __syncthreads();
    // lists of k, each in order: thread t takes every kJoinThreads-th candidate counted by
    // place first, so that the lists' heads lie with different threads
    const int lists = a.beams * a.chunks, total = lists * a.k;
    const uint64_t *cand = a.candidate + (int64_t)item * total;
    auto rank_of = [&](int i) {
        const int place = i / lists, which = i - place * lists, b = which / a.chunks;
        Rank r;
        r.cand = cand[(int64_t)which * a.k + place];
        r.tie = (uint32_t)(a.beams - b);
        const float x = unordered((uint32_t)(r.cand >> 32));
        r.key = r.cand == 0 ? 0ull : ordered64(x == -INFINITY ? -INFINITY : score[b] + ((double)x - lse[b]));
        return r;
    };
    auto put = [&](const Rank &r, int rank) {
        const int64_t at = (int64_t)item * a.k + rank;
        const uint64_t kb = r.key >> 63 ? r.key & 0x7fffffffffffffffull : ~r.key;
        a.out_scores[at] = (float)__builtin_bit_cast(double, kb);
        a.out_parents[at] = a.beams - (int)r.tie;
        a.out_tokens[at] = (int32_t) ~(uint32_t)r.cand;
    };
    Rank mine{0, 0, 0};
    for (int i = tid; i < total; i += kJoinThreads) {
        const Rank r = rank_of(i);
        if (r.key != 0 && above(r, mine)) mine = r;
    }
    list[tid] = mine;
    __syncthreads();
    if (mine.key != 0) {
        int n = 0;
        for (int i = 0; i < kJoinThreads; ++i) n += above(list[i], mine);
        if (n == a.k - 1) bound = mine;
    }
    __syncthreads();
    const Rank least = bound;
    if (mine.key != 0 && !above(least, mine))
        for (int i = tid; i < total; i += kJoinThreads) {
            const Rank r = rank_of(i);
            if (r.key != 0 && !above(least, r)) {
                const int at = atomicAdd(&count, 1);
                if (at < kJoinList) list[at] = r;
            }
        }
    __syncthreads();
    const int n = count;
    if (n <= kJoinList) {
        for (int i = tid; i < n; i += kJoinThreads) {
            const Rank r = list[i];
            int rank = 0;
            for (int j = 0; j < n; ++j) rank += above(list[j], r);
            if (rank < a.k) put(r, rank);
        }
        return;
    }
    // more pass than the list holds (one thread's candidates far above the others'): one place at a time
    Rank last{~0ull, ~0u, ~0ull};
    for (int place = 0; place < a.k; ++place) {
        Rank r{0, 0, 0};
        for (int i = tid; i < total; i += kJoinThreads) {
            const Rank c = rank_of(i);
            if (c.key != 0 && above(last, c) && above(c, r)) r = c;
        }
#pragma unroll
        for (int off = 32; off; off >>= 1) {
            const Rank o{__shfl_xor(r.key, off), __shfl_xor(r.tie, off), __shfl_xor(r.cand, off)};
            if (above(o, r)) r = o;
        }
        __syncthreads(); // the last place's readers are done
        if (lane == 0) best[wave] = r;
        __syncthreads();
        r = best[0];
        for (int w = 1; w < kWaves; ++w)
            if (above(best[w], r)) r = best[w];
        if (tid == 0) put(r, place);
        last = r;
    }
}

struct ReorderArgs {
    SpinnHipBeamState s[SPINN_HIP_MAX_BLOCKS];
};
// Units of U per row and state: a grid row of workgroups per destination row, the states side by side.
template <class U>
__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a, const int32_t *__restrict__ parents, int beams,
                                                           int k, int parts, int rows) {
    const int64_t blk = blockIdx.x;
    const int part = (int)(blk % parts);
    const int row = (int)(blk / parts % rows);
    const SpinnHipBeamState &s = a.s[blk / parts / rows];
    const int parent = parents[row];
    if ((unsigned)parent >= (unsigned)beams) return;
    const U *src = (const U *)((const char *)s.src + ((int64_t)(row / k) * beams + parent) * s.src_stride);
    U *dst = (U *)((char *)s.dst + (int64_t)row * s.dst_stride);
    const int64_t units = s.row_bytes / (int64_t)sizeof(U);
    for (int64_t u = (int64_t)part * 256 + threadIdx.x; u < units; u += (int64_t)parts * 256) dst[u] = src[u];
}

struct Plan {
    int ept, chunks;
    size_t max_bytes, sum_bytes, cand_bytes;
};
Plan plan(const SpinnHipBeamDesc *d) {
    Plan p;
    const int64_t rows = (int64_t)d->batch * d->beams;
    auto chunks = [&](int ept) { return ((int64_t)d->vocab + kBeamThreads * ept - 1) / (kBeamThreads * ept); };
    // long chunks leave less to join, short ones fill the device
    p.ept = 32;
    while (p.ept > 8 && rows * chunks(p.ept) < 2 * (int64_t)device_cu_count()) p.ept /= 2;
    p.chunks = (int)chunks(p.ept);
    p.max_bytes = round16((size_t)rows * p.chunks * 4);
    p.sum_bytes = round16((size_t)rows * p.chunks * 8);
    p.cand_bytes = (size_t)rows * p.chunks * d->k * 8;
    return p;
}

template <class T, int EPT>
void launch_chunks(const BeamArgs &a, bool vec, hipStream_t st) {
    const unsigned grid = (unsigned)((int64_t)a.batch * a.beams * a.chunks);
    const size_t lds = (size_t)a.k * EPT * 8;
    if (vec) beam_chunk_kernel<T, EPT, true><<<grid, kBeamThreads, lds, st>>>(a);
    else beam_chunk_kernel<T, EPT, false><<<grid, kBeamThreads, lds, st>>>(a);
}

} // namespace

size_t beam_select_workspace_bytes(const SpinnHipBeamDesc *d) {
    const Plan p = plan(d);
    return p.max_bytes + p.sum_bytes + p.cand_bytes;
}

int beam_select(const SpinnHipBeamDesc *d, const void *logits, const float *scores, const uint8_t *finished,
                float *out_scores, int32_t *out_parents, int32_t *out_tokens, void *ws, hipStream_t st) {
    const Plan p = plan(d);
    BeamArgs a{};
    a.logits = logits;
    a.scores = scores;
    a.finished = finished;
    a.out_scores = out_scores;
    a.out_parents = out_parents;
    a.out_tokens = out_tokens;
    char *w = (char *)ws;
    a.chunk_max = (float *)w;
    a.chunk_sum = (double *)(w + p.max_bytes);
    a.candidate = (uint64_t *)(w + p.max_bytes + p.sum_bytes);
    a.stride = d->logits_stride;
    a.batch = d->batch;
    a.beams = d->beams;
    a.vocab = d->vocab;
    a.k = d->k;
    a.end = d->end_token;
    a.chunks = p.chunks;
    if ((int64_t)a.batch * a.beams * a.chunks > INT32_MAX) return SPINN_HIP_EUNSUPPORTED;
    const int rc = with_dtype(d->dtype, [&](auto t) {
        typedef decltype(t) T;
        const int e = 16 / (int)sizeof(T);
        const bool vec = d->vocab % e == 0 && d->logits_stride % e == 0 && aligned16(logits);
        if (p.ept == 32) launch_chunks<T, 32>(a, vec, st);
        else if (p.ept == 16) launch_chunks<T, 16>(a, vec, st);
        else launch_chunks<T, 8>(a, vec, st);
        return check_launch();
    });
    if (rc) return rc;
    beam_join_kernel<<<(unsigned)a.batch, kJoinThreads, 0, st>>>(a);
    return check_launch();
}

int beam_reorder(const SpinnHipBeamState *states, int n, int batch, int beams, int k, const int32_t *parents,
                 hipStream_t st) {
    ReorderArgs a{};
    int used = 0;
    int64_t longest = 0;
    uint64_t bits = 0; // of every address and length: what they are all multiples of
    for (int i = 0; i < n; ++i) {
        const SpinnHipBeamState &s = states[i];
        if (s.row_bytes == 0) continue;
        a.s[used++] = s;
        longest = std::max(longest, s.row_bytes);
        bits |= (uint64_t)(uintptr_t)s.src | (uint64_t)(uintptr_t)s.dst | (uint64_t)s.row_bytes | (uint64_t)s.src_stride |
                (uint64_t)s.dst_stride;
    }
    if (!used) return SPINN_HIP_OK;
    const int unit = (bits & 15) == 0 ? 16 : ((bits & 3) == 0 ? 4 : 1);
    const int rows = batch * k;
    // about 16 KB a workgroup, at most 64 workgroups a row
    const int parts = (int)std::min<int64_t>(64, (longest + 16383) / 16384);
    if ((int64_t)rows * used * parts > INT32_MAX) return SPINN_HIP_EUNSUPPORTED;
    const unsigned grid = (unsigned)((int64_t)rows * used * parts);
    if (unit == 16) beam_reorder_kernel<u32x4><<<grid, 256, 0, st>>>(a, parents, beams, k, parts, rows);
    else if (unit == 4) beam_reorder_kernel<uint32_t><<<grid, 256, 0, st>>>(a, parents, beams, k, parts, rows);
    else beam_reorder_kernel<uint8_t><<<grid, 256, 0, st>>>(a, parents, beams, k, parts, rows);
    return check_launch();
}

} // namespace spinn
