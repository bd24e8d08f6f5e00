// beam.hip - beam search: the k best continuations over all beams and the vocabulary, and
// the reordering of the beams' states after their parents.
//
// key(b,t) = score_b + x_bt - lse_b. Within a beam the keys order as the logits do, so one pass over a
// chunk of a row finds the chunk's share of lse (its maximum and its sum of exponentials) and its k
// first candidates together, from registers: a lower bound for the k-th comes from the lanes' own
// maxima, and the few elements that pass it are ranked by counting. The second launch joins a
// batch item's chunks, merging their ordered lists by their heads.
// Bound: memory, each logit read once, and as much again the vector units' work on it (a conversion, a maximum
// and an exponential each), which overlaps with other workgroups' reading only as far as registers let them be there.
// 32 x 8 beams of 128000 bf16, k = 16: chunks 23 us (2.8 TB/s), join 10.3; 4 beams of
// 32000 fp32, k = 8: 5.1 and 6.2, two launches' latency.
#include "decode.h"
#include <type_traits>

namespace spinn {
namespace {

constexpr int kBeamThreads = 256;
constexpr float kLog2e = 1.4426950408889634f;

// fp32 to an unsigned number of the same order, both zeros equal; NaN as -inf, +inf as the largest finite.
// (By the bits: the maximum of a signalling NaN and a number is a NaN, and a bf16 one becomes an fp32 one.)
__device__ __forceinline__ float clean(float v) {
    return (__builtin_bit_cast(uint32_t, v) & 0x7fffffffu) > 0x7f800000u ? -INFINITY : fminf(v, 3.402823466e38f);
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

// Maximum over a wave of unsigned numbers, in every lane.
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_max(uint64_t v) {
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, 0xf, 0xf, false);
    const uint64_t o = (uint64_t)hi << 32 | lo;
    return o > v ? o : v;
}
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_umax(uint32_t v) {
    const uint32_t o = __builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, false);
    return o > v ? o : v;
}
__device__ __forceinline__ uint32_t wave_umax(uint32_t v) {
    v = dpp_umax<0x111>(v);
    v = dpp_umax<0x112>(v);
    v = dpp_umax<0x114>(v);
    v = dpp_umax<0x118>(v);
    v = dpp_umax<0x142>(v);
    v = dpp_umax<0x143>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ uint64_t wave_max(uint64_t v) {
    v = dpp_max<0x111>(v); // row_shr 1, 2, 4, 8: lane 15 of each row of 16 has the row's
    v = dpp_max<0x112>(v);
    v = dpp_max<0x114>(v);
    v = dpp_max<0x118>(v);
    v = dpp_max<0x142>(v); // row_bcast 15 and 31: lane 63 has all
    v = dpp_max<0x143>(v);
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), 63) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, 63);
}

// Order by logit, then by the lower token; never 0.
__device__ __forceinline__ uint64_t rank32(float v, int token) {
    return (uint64_t)ordered(v == 0.f ? 0.f : v) << 32 | (uint32_t)~token;
}
// -inf in every element of a word.
__device__ __forceinline__ uint32_t no_logits(float) { return 0xff800000u; }
__device__ __forceinline__ uint32_t no_logits(_Float16) { return 0xfc00fc00u; }
__device__ __forceinline__ uint32_t no_logits(__bf16) { return 0xff80ff80u; }
// Maximum over a wave, in every lane.
template <int CTRL>
__device__ __forceinline__ float dpp_fmax(float v) {
    return fmaxf(v, __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, v), __builtin_bit_cast(int, v),
                                                                         CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ float wave_fmax(float v) {
    v = dpp_fmax<0x111>(v);
    v = dpp_fmax<0x112>(v);
    v = dpp_fmax<0x114>(v);
    v = dpp_fmax<0x118>(v);
    v = dpp_fmax<0x142>(v);
    v = dpp_fmax<0x143>(v);
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
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

// Lanes whose elements the list of a chunk has room for: k and more.
__host__ __device__ constexpr int beam_lanes(int k) { return 2 * k + 16 < kBeamThreads ? 2 * k + 16 : kBeamThreads; }

// Elements per thread of a chunk of kBeamThreads * EPT.
template <class T, int EPT, bool VEC>
__global__ __launch_bounds__(kBeamThreads) void beam_chunk_kernel(BeamArgs a) {
    typedef typename Bits<T>::type B;
    constexpr int E = 16 / (int)sizeof(T), P = 4 / (int)sizeof(T); // elements of a run and of a word
    const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const T *x = (const T *)a.logits + (int64_t)row * a.stride;
    const int base = chunk * kBeamThreads * EPT;
    const float score = clean(a.scores[row]);
    const bool ended = a.finished && a.finished[row], empty = score == -INFINITY;

    if (ended || empty) { // the end token, where it is this chunk's, and the lowest others at -inf
        const int in_chunk = min(a.vocab - base, kBeamThreads * EPT);
        const int lead = ended && !empty && a.end >= base && a.end < base + in_chunk ? a.end : -1;
        uint64_t *out = a.candidate + (int64_t)blockIdx.x * a.k;
        for (int i = tid; i < a.k; i += kBeamThreads) {
            int t = base + i;
            if (lead >= 0) t = i == 0 ? lead : (t - 1 < lead ? t - 1 : t);
            out[i] = i < in_chunk ? rank32(i == 0 && lead >= 0 ? 0.f : -INFINITY, t) : 0ull;
        }
        if (tid == 0) {
            a.chunk_max[blockIdx.x] = -INFINITY;
            a.chunk_sum[blockIdx.x] = 0.0;
        }
        return;
    }
    // runs of E elements, a workgroup's runs side by side: equal logits then spread over the threads.
    // What lies behind the row is -inf like a hidden token, and comes after all tokens.
    // They stay as they are in memory and each pass converts them again: 85 registers and five workgroups on a CU
    // instead of 180 and two (25 -> 23 us over 32 x 8 beams of 128000, bf16).
    uint32_t w[EPT / P];
    const int first = base + tid * E; // token of the first run
    auto token = [&](int i) { return first + (i / E) * kBeamThreads * E + i % E; };
    if constexpr (VEC) {
#pragma unroll
        for (int r = 0; r < EPT / E; ++r) { // a row is whole runs
            u32x4 run = (u32x4)(no_logits(T()));
            if (token(r * E) < a.vocab) run = *reinterpret_cast<const u32x4 *>(x + token(r * E));
#pragma unroll
            for (int i = 0; i < 4; ++i) w[4 * r + i] = run[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < EPT; i += P) {
            w[i / P] = no_logits(T());
#pragma unroll
            for (int j = 0; j < P; ++j)
                if (token(i + j) < a.vocab) {
                    const uint32_t one = (uint32_t) reinterpret_cast<const B *>(x)[token(i + j)];
                    if constexpr (P == 1) w[i] = one;
                    else w[i / P] = j ? (w[i / P] & 0xffffu) | one << 16 : (w[i / P] & 0xffff0000u) | one;
                }
        }
    }
    auto logit = [&](int i) {
        if constexpr (P == 1) return __builtin_bit_cast(float, w[i]);
        else return (float)__builtin_bit_cast(T, (uint16_t)(w[i / P] >> (16 * (i % P))));
    };
    // (keeps the compiler from holding what it converted for the next pass)
    auto again = [&]() {
#pragma unroll
        for (int i = 0; i < EPT / P; ++i) asm volatile("" : "+v"(w[i]));
    };
    constexpr int kWaves = kBeamThreads / 64;
    __shared__ float wmax[kWaves], wfloor[kWaves];
    __shared__ double wsum[kWaves];
    __shared__ uint64_t bound;
    __shared__ int count, passing;
    extern __shared__ uint64_t list[]; // [beam_lanes(k) * EPT]
    constexpr int R = EPT / 8; // groups of 8 elements, with their maxima
    float top[R];
    const int q = (a.k + kWaves - 1) / kWaves;
    float best, floor, m;
    double sum;
    auto scan = [&](auto cleaned) {
        auto value = [&](int i) { return decltype(cleaned)::value ? clean(logit(i)) : logit(i); };
        best = -INFINITY; // a NaN leaves it as it is
#pragma unroll
        for (int r = 0; r < R; ++r) {
            top[r] = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i) top[r] = fmaxf(top[r], value(8 * r + i));
            best = fmaxf(best, top[r]);
        }
        // Of each wave the q-th largest lane maximum, 4 q >= k: at least q of its elements reach it, so k
        // of the chunk reach the least of the four (-inf, which all reach, where a chunk has fewer).
        float nth = -INFINITY, left = best;
        m = -INFINITY;
        for (int i = 0; i < q; ++i) {
            nth = wave_fmax(left);
            if (i == 0) m = nth;
            if (nth == -INFINITY) break;
            if (lane == __ffsll((unsigned long long)__ballot(left == nth)) - 1) left = -INFINITY;
        }
        if (lane == 0) {
            wmax[wave] = m;
            wfloor[wave] = nth;
        }
        if (tid == 0) {
            count = 0;
            passing = 0;
            bound = 0;
        }
        __syncthreads();
        floor = wfloor[0];
        m = wmax[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) {
            m = fmaxf(m, wmax[w]);
            floor = fminf(floor, wfloor[w]);
        }
        const uint64_t pass = __ballot(best >= floor);
        if (lane == 0 && pass) atomicAdd(&passing, __popcll(pass));
        again();

        // share of the sum: exponentials in fp32 (their arguments rounded once, 2^-24 of themselves, and one step of
        // the exponential; four added in fp32), then fp64. Within 2^-20; over many alike terms the errors average to 1e-8
        sum = 0.0;
        if (m != -INFINITY) {
            // exp(v - m) = 2^(v L - m L), in one rounding; what m L lost is a factor of the whole sum. Half a step of m L is
            // at most 1/16 below 2^20; from 128 on, one of the two would be infinite and the other zero. Beyond, v - m first:
            // exact for the v that are anywhere near m.
            const float shift = m * kLog2e, lost = fmaf(m, kLog2e, -shift);
            if (fabsf(m) < 1e6f) {
#pragma unroll
                for (int i = 0; i < EPT; i += 4) {
                    float part = 0.f;
#pragma unroll
                    for (int j = i; j < i + 4; ++j) part += __builtin_amdgcn_exp2f(fmaf(value(j), kLog2e, -shift));
                    sum += (double)part;
                }
                sum *= (double)__builtin_amdgcn_exp2f(-lost);
            } else {
#pragma unroll
                for (int i = 0; i < EPT; ++i) sum += (double)__builtin_amdgcn_exp2f((value(i) - m) * kLog2e);
            }
        }
#pragma unroll
        for (int off = 32; off; off >>= 1) sum += __shfl_xor(sum, off);
        if (lane == 0) wsum[wave] = sum;
        __syncthreads();
        sum = wsum[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) sum += wsum[w];
        again();
    };
    scan(std::false_type());
    if (!(m > -INFINITY && m < INFINITY && sum == sum)) { // a NaN or +inf among the logits, or hardly any: once more without them
        __syncthreads();
        scan(std::true_type());
    }
    if (floor > -INFINITY && passing <= beam_lanes(a.k)) {
        // (few groups have one)
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (top[r] >= floor) {
#pragma unroll
                for (int i = 8 * r; i < 8 * r + 8; ++i)
                    if (logit(i) >= floor) list[atomicAdd(&count, 1)] = rank32(clean(logit(i)), token(i));
            }
    } else {
        // One wave's part of the row is far above another's, or many logits are equal: the k-th of all lane
        // maxima instead, ties told apart by their tokens, from the waves' sorted ones (kept where the list
        // comes later). At most k lanes reach it.
        int at = 0;
#pragma unroll
        for (int i = EPT - 1; i >= 0; --i) at = clean(logit(i)) == best ? i : at;
        const uint64_t mine = token(at) < a.vocab ? rank32(best, token(at)) : 0ull;
        const int most = a.k < 64 ? a.k : 64;
        uint64_t left = mine;
        for (int i = 0; i < most; ++i) {
            const uint64_t top = wave_max(left);
            if (lane == 0) list[wave * most + i] = top;
            if (left == top) left = 0;
        }
        __syncthreads();
        int over = 0;
        if (mine != 0)
            for (int i = 0; i < kWaves * most; ++i) over += list[i] > mine;
        if (mine != 0 && over == a.k - 1) bound = mine;
        __syncthreads();
        again();
        const uint64_t least = bound;
        if (mine != 0 && mine >= least) {
#pragma unroll
            for (int i = 0; i < EPT; ++i)
                if (token(i) < a.vocab) {
                    const uint64_t u = rank32(clean(logit(i)), token(i));
                    if (u >= least) list[atomicAdd(&count, 1)] = u;
                }
        }
    }
    __syncthreads();
    if (tid == 0) {
        a.chunk_max[blockIdx.x] = m;
        a.chunk_sum[blockIdx.x] = sum;
    }
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
struct Rank {
    uint64_t key; // of the double, ordered; 0 = none
    uint32_t tie; // beams - beam
    uint64_t cand;
};
__device__ __forceinline__ bool above(const Rank &p, const Rank &q) {
    return p.key != q.key ? p.key > q.key : (p.tie != q.tie ? p.tie > q.tie : p.cand > q.cand);
}
// The lane whose rank is above all others' in the wave (any lane where there is none).
__device__ __forceinline__ int first_lane(const Rank &r) {
    const uint32_t high = (uint32_t)(r.key >> 32);
    uint64_t tied = __ballot(high == wave_umax(high));
    if (__popcll(tied) > 1) {
        const uint64_t top = wave_max(r.key);
        const uint64_t t = wave_max(r.key == top ? r.tie : 0u);
        const bool in = r.key == top && r.tie == t;
        const uint64_t c = wave_max(in ? r.cand : 0ull);
        tied = __ballot(in && r.cand == c);
    }
    return __ffsll((unsigned long long)tied) - 1;
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int lane) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane) << 32 |
           (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
}
__device__ __forceinline__ Rank lane_rank(const Rank &r, int lane) {
    return Rank{lane_u64(r.key, lane), (uint32_t)__builtin_amdgcn_readlane((int)r.tie, lane), lane_u64(r.cand, lane)};
}

constexpr int kJoinWaves = 16;    // at most
constexpr int kJoinCached = 2048; // candidates held in LDS with their keys

// Every lane has the heads of its lists (one, until there are more lists than lanes), and a
// wave takes the first of them k times without a barrier; then one wave does the same with the waves' lists.
template <bool CACHED>
__global__ __launch_bounds__(64 * kJoinWaves) void beam_join_kernel(BeamArgs a, int merging) {
    const int item = blockIdx.x, tid = threadIdx.x, waves = blockDim.x >> 6;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // lse in two parts: beside a large maximum the sum's logarithm would be lost
    __shared__ double most[SPINN_HIP_BEAM_MAX], log_sum[SPINN_HIP_BEAM_MAX], score[SPINN_HIP_BEAM_MAX];
    __shared__ uint64_t key_at[CACHED ? kJoinCached : 1], cand_at[CACHED ? kJoinCached : 1];
    extern __shared__ Rank merged[]; // [merging][k], where several waves merge
    const int lists = a.beams * a.chunks, total = lists * a.k, per_beam = a.chunks * a.k;
    const uint64_t *cand = a.candidate + (int64_t)item * total;
    if constexpr (CACHED)
        for (int i = tid; i < total; i += blockDim.x) cand_at[i] = cand[i];
    for (int b = wave; b < a.beams; b += waves) {
        const int row = item * a.beams + b;
        const float *cm = a.chunk_max + (int64_t)row * a.chunks;
        const double *cs = a.chunk_sum + (int64_t)row * a.chunks;
        const float sc = a.scores[row];
        // (a lane's first chunk at once, both its numbers)
        const float m0 = lane < a.chunks ? cm[lane] : -INFINITY;
        const double s0 = lane < a.chunks ? cs[lane] : 0.0;
        float m = m0;
        for (int i = lane + 64; i < a.chunks; i += 64) m = fmaxf(m, cm[i]);
        m = wave_fmax(m);
        double s = 0.0;
        if (m != -INFINITY) {
            s = s0 * exp((double)m0 - (double)m);
            for (int i = lane + 64; i < a.chunks; i += 64) s += cs[i] * exp((double)cm[i] - (double)m);
        }
#pragma unroll
        for (int off = 32; off; off >>= 1) s += __shfl_xor(s, off);
        if (lane == 0) {
            score[b] = (double)clean(sc);
            most[b] = m == -INFINITY ? 0.0 : (double)m;
            log_sum[b] = m == -INFINITY ? 0.0 : log(s);
        }
    }
    __syncthreads();
    auto key_of = [&](uint64_t c, int b) {
        const float x = unordered((uint32_t)(c >> 32));
        return c == 0 ? 0ull : ordered64(x == -INFINITY ? -INFINITY : score[b] + (((double)x - most[b]) - log_sum[b]));
    };
    if constexpr (CACHED) {
        for (int i = tid; i < total; i += blockDim.x) key_at[i] = key_of(cand_at[i], i / per_beam);
        __syncthreads();
    }
    auto rank_of = [&](int list, int place) {
        const int i = list * a.k + place, b = list / a.chunks;
        if constexpr (CACHED) return Rank{key_at[i], (uint32_t)(a.beams - b), cand_at[i]};
        else return Rank{key_of(cand[i], b), (uint32_t)(a.beams - b), cand[i]};
    };
    auto put = [&](const Rank &r, int rank) {
        const int64_t at = (int64_t)item * a.k + rank;
        const uint64_t kb = r.key >> 63 ? r.key & 0x7fffffffffffffffull : ~r.key;
        a.out_scores[at] = (float)__builtin_bit_cast(double, kb);
        a.out_parents[at] = a.beams - (int)r.tie;
        a.out_tokens[at] = (int32_t) ~(uint32_t)r.cand;
    };
    if (wave < merging) {
        const int first = wave * 64 + lane, step = merging * 64;
        const bool one = lists <= step; // list per lane
        int pos = 0;
        auto at = [&](int place) { return first < lists && place < a.k ? rank_of(first, place) : Rank{0, 0, 0}; };
        // the lane's first candidate after `last` over several lists, each in order
        auto after = [&](const Rank &last) {
            Rank r{0, 0, 0};
            for (int l = first; l < lists; l += step)
                for (int p = 0; p < a.k; ++p) {
                    const Rank c = rank_of(l, p);
                    if (c.key == 0) break;
                    if (above(last, c)) {
                        if (above(c, r)) r = c;
                        break;
                    }
                }
            return r;
        };
        Rank mine, follow{0, 0, 0}, taken{0, 0, 0};
        if (one) {
            mine = at(0);
            follow = at(1);
            pos = 2;
        } else {
            mine = after(Rank{~0ull, ~0u, ~0ull});
        }
        for (int i = 0; i < a.k; ++i) {
            const int w = first_lane(mine);
            const Rank r = lane_rank(mine, w);
            if (lane == (i & 63)) taken = r;
            if ((i & 63) == 63 || i == a.k - 1) {
                const int to = (i & ~63) + lane;
                if (to <= i) {
                    if (merging == 1) put(taken, to);
                    else merged[wave * a.k + to] = taken;
                }
            }
            if (lane == w) {
                if (one) {
                    mine = follow;
                    follow = at(pos++);
                } else if (r.key != 0) {
                    mine = after(r);
                }
            }
        }
    }
    if (merging == 1) return;
    __syncthreads();
    if (wave) return;
    int pos = 0;
    auto head = [&]() { return lane < merging && pos < a.k ? merged[lane * a.k + pos] : Rank{0, 0, 0}; };
    Rank mine = head(), taken{0, 0, 0};
    for (int i = 0; i < a.k; ++i) {
        const int w = first_lane(mine);
        const Rank r = lane_rank(mine, w);
        if (lane == (i & 63)) taken = r;
        if ((i & 63) == 63 || i == a.k - 1) {
            const int to = (i & ~63) + lane;
            if (to <= i) put(taken, to);
        }
        if (lane == w) {
            ++pos;
            mine = head();
        }
    }
}

struct ReorderArgs {
    SpinnHipBeamState s[SPINN_HIP_MAX_BLOCKS];
};
// Units of U per row and state: `parts` shares of a destination row each, the states side by side; a workgroup takes
// every gridDim.x-th share.
template <class U>
__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a, const int32_t *__restrict__ parents, int beams,
                                                           int k, int parts, int rows, int64_t shares) {
    for (int64_t blk = blockIdx.x; blk < shares; blk += gridDim.x) {
        const int part = (int)(blk % parts);
        const int row = (int)(blk / parts % rows);
        const SpinnHipBeamState &s = a.s[blk / parts / rows];
        const int parent = parents[row];
        if ((unsigned)parent >= (unsigned)beams) continue;
        const U *src = (const U *)((const char *)s.src + ((int64_t)(row / k) * beams + parent) * s.src_stride);
        U *dst = (U *)((char *)s.dst + (int64_t)row * s.dst_stride);
        const int64_t units = s.row_bytes / (int64_t)sizeof(U);
        for (int64_t u = (int64_t)part * 256 + threadIdx.x; u < units; u += (int64_t)parts * 256) dst[u] = src[u];
    }
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
    p.ept = beam_lanes(d->k) <= 64 ? 64 : 32; // (the list of a chunk: 32 KB of LDS for 64 lanes)
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
    const size_t lds = (size_t)std::max(beam_lanes(a.k) * EPT, 4 * std::min(a.k, 64)) * 8;
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
    if (!launch_fits((int64_t)a.batch * a.beams * a.chunks, kBeamThreads)) return SPINN_HIP_EUNSUPPORTED;
    const int rc = with_dtype(d->dtype, [&](auto t) {
        typedef decltype(t) T;
        const int e = 16 / (int)sizeof(T);
        const bool vec = d->vocab % e == 0 && d->logits_stride % e == 0 && aligned16(logits);
        if (p.ept == 64) launch_chunks<T, 64>(a, vec, st);
        else if (p.ept == 32) launch_chunks<T, 32>(a, vec, st);
        else if (p.ept == 16) launch_chunks<T, 16>(a, vec, st);
        else launch_chunks<T, 8>(a, vec, st);
        return check_launch();
    });
    if (rc) return rc;
    const int64_t lists = (int64_t)a.beams * a.chunks;
    const int merging = (int)std::min<int64_t>(kJoinWaves, (lists + 63) / 64);
    const int waves = std::max(merging, std::min(kJoinWaves, std::max(4, a.beams))); // a wave per beam's lse
    const size_t lds = merging > 1 ? (size_t)merging * a.k * sizeof(Rank) : 0;
    if (lists * a.k <= kJoinCached) beam_join_kernel<true><<<(unsigned)a.batch, 64 * waves, lds, st>>>(a, merging);
    else beam_join_kernel<false><<<(unsigned)a.batch, 64 * waves, lds, st>>>(a, merging);
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
    const int64_t shares = (int64_t)rows * used * parts;
    const unsigned grid = (unsigned)std::min<int64_t>(shares, 1 << 20); // (a launch has at most 2^32 threads)
    if (unit == 16) beam_reorder_kernel<u32x4><<<grid, 256, 0, st>>>(a, parents, beams, k, parts, rows, shares);
    else if (unit == 4) beam_reorder_kernel<uint32_t><<<grid, 256, 0, st>>>(a, parents, beams, k, parts, rows, shares);
    else beam_reorder_kernel<uint8_t><<<grid, 256, 0, st>>>(a, parents, beams, k, parts, rows, shares);
    return check_launch();
}

} // namespace spinn
