// kv_attention.hip - a paged key-value cache: rows appended to it, and the attention of one new
// token per sequence over it.
//
// Per query head: s_i = scale q.k_i, p_i = exp(s_i - m) / sum_j exp(s_j - m), o = sum_i p_i v_i,
// in one pass with the running maximum m and sum: a tile of slots raises m to m', and what
// was summed so far is scaled by exp(m - m'). Every row of the cache is read once, for all the
// query heads of its kv head, so the bound is memory: 2 rows a slot against 4 * heads * head_dim flops.
// 8 kv heads of 128, bf16: one sequence of 131001 slots 101 us (5.3 TB/s), 32 of 37 to 8000 122 us (4.3 TB/s: the
// last parts run alone, since the split goes by max_len). 16 x 1500..2000, 16 heads of 80 fp32, with
// weights: 75 us, 7 of them the second launch.
//
// The matrix cores then have time to spare (one new token fills few of a tile's 16 columns, and
// at 5 TB/s they are still under 8 % busy), which decides the layout: nothing goes through LDS in the
// loop. S^T = K Q^T has slots as rows, and lane (g = l/16, n = l%16) ends up with
// head n, slots 4g..4g+3 of each half tile: exactly the elements that the second product wants
// from it as its operand (contraction over slots may run in any order, so V's rows
// are fetched in that order). O^T = V^T P^T: a lane fetches the same 16-byte columns of
// eight slots, a full row per 16 lanes, and transposes them in registers (one
// v_perm per two elements).
#include "decode.h"

namespace spinn {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kStep = 128;    // slots of a split are a multiple of this: a 32-slot step of four waves
constexpr int kHeadTile = 16; // query heads of one kv head per workgroup

__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }

struct AttendArgs {
    const void *q, *k, *v;
    const int32_t *table, *lengths;
    const uint8_t *mask;
    void *o;
    float *lse;
    float *part_o, *part_ml; // [seqs][heads][splits][part_row], [..][2] (maximum and sum, base 2)
    float *scores;           // [seqs][heads][score_row], base 2; null when no weights are wanted
    int64_t q_stride, o_stride, mask_stride, page_stride, head_stride, slot_stride, score_row;
    float scale2; // scale * log2 e
    int32_t seqs, heads, kv_heads, group, dim, page_size, n_pages, max_pages, max_len;
    uint32_t page_mul, page_shift; // slot / page_size = slot * page_mul >> 32 + page_shift (page_mul 0: slot)
    int32_t q_runs;        // query rows are whole 16-byte runs
    int32_t part_row;      // dim rounded up to a multiple of 4
    int32_t splits, chunk; // chunk: slots per split, a multiple of kStep
    int32_t head_tiles, parts; // parts: seqs * kv_heads * splits
};

// A number that no kernel writes meanwhile, at an index that is the same in every lane: through the scalar cache.
__device__ __forceinline__ int32_t scalar_at(const int32_t *p, int i) {
    return ((const __attribute__((address_space(4))) int32_t *)p)[i];
}

__device__ __forceinline__ int page_of(const AttendArgs &a, int slot) {
    return a.page_mul ? (int)(__umulhi((uint32_t)slot, a.page_mul) >> a.page_shift) : slot;
}

// T: element; DP: head_dim padded to 64, 128 or 256; ROWS: how rows are read;
// UNI: pages are multiples of 16 slots, so that each half tile lies in one page.
// kWaves: 4, or 8 for a short sequence in one workgroup.
template <class T, int DP, Rows ROWS, bool UNI, int kWaves>
__global__ __launch_bounds__(64 * kWaves) void kv_attend_kernel(AttendArgs a) {
    constexpr int E = 16 / (int)sizeof(T);    // elements per 16 bytes
    constexpr int KC = DP / kFrag<T>;         // fragments of a row of K or Q
    constexpr int DPL = DP / 16;              // a lane's elements of a V row: DPL n .. +DPL-1
    constexpr int VB = DPL * (int)sizeof(T);  // their bytes
    constexpr int VW = VB / 4;                // and words
    constexpr int H = sizeof(T) == 2 ? 2 : 1; // halves of 16 slots in a wave's step: a 16-bit product takes 32
    constexpr int kTile = 16 * H;
    constexpr float kPScale = sizeof(T) == 2 && !__is_same(T, __bf16) ? 16384.f : 1.f;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n = lane & 15;

    // the head tiles of a part, which read the same rows, are workgroups of one XCD (b % 8) one after the other
    const int per = 8 * a.head_tiles, ht = (int)(blockIdx.x % per) >> 3;
    int b = (int)(blockIdx.x / per) * 8 + (int)(blockIdx.x & 7);
    if (b >= a.parts) return;
    // Lengths differ, so a row's last parts are short or empty. Up to four parts: all rows' first ones, then the second
    // ones, ..., so that what starts late is short (24 sequences of 100 to 8000 slots, 8 x 128 bf16: 88 us,
    // row by row 110; 48 of 100 to 3000: 72, 86). More: row by row, turned so that no XCD has only last ones
    // (8 of 100 to 60000: 198 us, unturned 200, first parts first 208; 16 of 100 to 16000: 123, 130, 125).
    int sp;
    if (a.splits <= 4) {
        const int rows = a.seqs * a.kv_heads;
        sp = b / rows;
        b -= sp * rows;
    } else {
        sp = b % a.splits;
        b /= a.splits;
        sp = (sp + b / 2) % a.splits;
    }
    const int kvh = b % a.kv_heads, seq = b / a.kv_heads;
    const int h0 = kvh * a.group + ht * kHeadTile;              // first query head of the tile
    const int nh = min(kHeadTile, a.group - ht * kHeadTile);    // query heads in it
    const int begin = sp * a.chunk;
    const int len_read = scalar_at(a.lengths, seq);
    const int32_t *table = a.table + (int64_t)seq * a.max_pages;
    // UNI: where each half of a tile starts. The page number comes through the scalar cache (a vector load would
    // wait for all rows in flight before it) a step ahead of its use.
    // The first tile's are asked for with the length, not after it: among max_len slots, whatever they name behind the
    // length (one sequence of 8000 slots, 8 x 128 bf16: 17.6 -> 17.2 us).
    // Otherwise every lane looks up its rows' pages, a step ahead, too.
    constexpr int L = UNI ? H : 5 * H; // page numbers of a tile: of the halves, or of the lane's K rows and V rows
    auto slot_of = [&](int t0, int i, int n_slots) {
        if constexpr (UNI) return min(t0 + 16 * i, max(n_slots - 1, 0) & ~15);
        else return min(t0 + (i < H ? 16 * i + n : 16 * ((i - H) >> 2) + 4 * g + ((i - H) & 3)), max(n_slots - 1, 0));
    };
    int coming[L];  // page numbers of the next tile
    int64_t at[L];  // where the current tile's rows are
    uint32_t there; // bit i: they are in a page
    auto look_up = [&](int t0, int n_slots) {
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int pi = page_of(a, slot_of(t0, i, n_slots));
            if constexpr (UNI) coming[i] = scalar_at(table, pi);
            else coming[i] = table[pi];
        }
    };
    auto place = [&](int t0, int n_slots) {
        there = 0;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int slot = slot_of(t0, i, n_slots);
            const bool ok = (unsigned)coming[i] < (unsigned)a.n_pages;
            there |= (uint32_t)ok << i;
            at[i] = (int64_t)(ok ? coming[i] : 0) * a.page_stride + (int64_t)(slot - page_of(a, slot) * a.page_size) * a.slot_stride;
        }
    };
    int t0 = begin + wave * kTile;
    if constexpr (UNI) look_up(t0, a.max_len);
    const int len = min(max(len_read, 0), a.max_len), end = begin + min(len - begin, a.chunk);
    if (begin >= len && sp > 0) { // nothing here (a sequence's first part writes o and lse where it is the only one)
        if ((int)threadIdx.x < nh) {
            float *ml = a.part_ml + (((int64_t)seq * a.heads + h0 + threadIdx.x) * a.splits + sp) * 2;
            ml[0] = -INFINITY;
            ml[1] = 0.f;
        }
        return;
    }
    const uint8_t *mask = a.mask ? a.mask + (int64_t)seq * a.mask_stride : nullptr;

    // Q: lane (g, n) holds head n, the same k as the K fragments
    u32x4 q[KC];
    {
        const T *qp = (const T *)a.q + (int64_t)seq * a.q_stride + (int64_t)(h0 + min(n, nh - 1)) * a.dim;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            const int d0 = c * kFrag<T> + g * E;
            if (a.q_runs) q[c] = n < nh && d0 < a.dim ? *reinterpret_cast<const u32x4 *>(qp + d0) : (u32x4){0, 0, 0, 0};
            else q[c] = load_edge<T>(qp + d0, n < nh ? a.dim - d0 : 0);
        }
    }

    f32x4 acc[DPL] = {};
    float m = -INFINITY, l = 0.f;
    const T *kb = (const T *)a.k + (int64_t)kvh * a.head_stride;
    const T *vb = (const T *)a.v + (int64_t)kvh * a.head_stride;

    // K's rows of a tile: lane (g, n) takes row n of each half
    u32x4 kr[H][KC];
    auto load_k = [&](int t0) {
#pragma unroll
        for (int h = 0; h < H; ++h) {
            const T *kp = kb + at[h];
            if constexpr (UNI) kp += (int64_t)n * a.slot_stride;
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const int d0 = c * kFrag<T> + g * E;
                if constexpr (ROWS == kRuns) kr[h][c] = d0 < a.dim ? *reinterpret_cast<const u32x4 *>(kp + d0) : (u32x4){0, 0, 0, 0};
                else if constexpr (ROWS == kShort) kr[h][c] = load_edge<T>(kp + d0, a.dim - d0);
                else {
                    uint32_t w[4];
                    load_loose<T, E>(kp, d0, a.dim, w);
                    kr[h][c] = (u32x4){w[0], w[1], w[2], w[3]};
                }
            }
        }
    };
    // V's: lane (g, n) takes its columns of rows 4g..4g+3 of each half; which of them are visible
    uint32_t vr[4 * H][VW];
    uint32_t seen; // bit j: the lane's j-th slot, t0 + 16 (j/4) + 4g + j%4, is one of the part's
    uint8_t shown[4 * H];
    auto load_v = [&](int t0) {
        seen = 0;
#pragma unroll
        for (int h = 0; h < H; ++h) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const T *vp = vb + n * DPL;
                if constexpr (UNI) vp += at[h] + (int64_t)(4 * g + j) * a.slot_stride;
                else vp += at[H + 4 * h + j];
                const int slot = t0 + 16 * h + 4 * g + j;
                if ((there >> (UNI ? h : H + 4 * h + j) & 1u) && slot < end) {
                    seen |= 1u << (4 * h + j);
                    if (mask) shown[4 * h + j] = mask[slot]; // read where it is needed
                }
                uint32_t(&to)[VW] = vr[4 * h + j];
                if constexpr (ROWS == kRuns) {
                    // in 16-byte runs (8 where a lane's share is 8); a row ends between runs
                    constexpr int R = VB >= 16 ? 16 : VB;
#pragma unroll
                    for (int r = 0; r < VB / R; ++r) {
                        const bool in = n * DPL + r * (R / (int)sizeof(T)) < a.dim;
                        if constexpr (R == 16) {
                            const u32x4 w = in ? *reinterpret_cast<const u32x4 *>(vp + r * E) : (u32x4){0, 0, 0, 0};
#pragma unroll
                            for (int i = 0; i < 4; ++i) to[4 * r + i] = w[i];
                        } else {
                            const u32x2 w = in ? *reinterpret_cast<const u32x2 *>(vp) : (u32x2){0, 0};
                            to[0] = w[0];
                            to[1] = w[1];
                        }
                    }
                } else {
                    constexpr int N = DPL < E ? DPL : E; // elements per load
#pragma unroll
                    for (int r = 0; r < DPL / N; ++r) {
                        uint32_t w[N * sizeof(T) / 4];
                        if constexpr (ROWS == kLoose) load_loose<T, N>(vp - n * DPL, n * DPL + r * N, a.dim, w);
                        else {
                            const u32x4 e = load_edge<T>(vp + r * N, min(a.dim - n * DPL - r * N, N));
#pragma unroll
                            for (int i = 0; i < N * (int)sizeof(T) / 4; ++i) w[i] = e[i];
                        }
#pragma unroll
                        for (int i = 0; i < N * (int)sizeof(T) / 4; ++i) to[r * (N * (int)sizeof(T) / 4) + i] = w[i];
                    }
                }
            }
        }
    };

    // The registers of K are free once the scores are there and those of V at the end of a step: each takes
    // the next tile's rows at once, which then travel during the other's products.
    if (t0 < end) {
        if constexpr (!UNI) look_up(t0, len);
        place(t0, UNI ? a.max_len : len);
        load_k(t0);
        load_v(t0);
        look_up(t0 + kTile * kWaves, len);
    }
    for (; t0 < end; t0 += kTile * kWaves) {
        const int t1 = t0 + kTile * kWaves;
        uint32_t vis = seen;
        if (mask) {
#pragma unroll
            for (int j = 0; j < 4 * H; ++j)
                if (shown[j] == 0) vis &= ~(1u << j);
        }

        // scores, base 2
        float s[4 * H];
#pragma unroll
        for (int h = 0; h < H; ++h) {
            f32x4 c = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < KC; ++i) mfma_frag(c, kr[h][i], q[i], T());
#pragma unroll
            for (int i = 0; i < 4; ++i) s[4 * h + i] = (vis >> (4 * h + i) & 1u) ? c[i] * a.scale2 : -INFINITY;
        }
        if (t1 < end) {
            place(t1, len);
            look_up(t1 + kTile * kWaves, len);
            load_k(t1);
        }
        if (a.scores && n < nh) {
            float *row = a.scores + ((int64_t)seq * a.heads + h0 + n) * a.score_row + t0 + 4 * g;
#pragma unroll
            for (int h = 0; h < H; ++h)
                *reinterpret_cast<f32x4 *>(row + 16 * h) = (f32x4){s[4 * h], s[4 * h + 1], s[4 * h + 2], s[4 * h + 3]};
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < 4 * H; ++j) top = fmaxf(top, s[j]);
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float base = top == -INFINITY ? 0.f : top;
        if (__any(top > m)) {
            const float alpha = exp2_hw(m - base);
            l *= alpha;
#pragma unroll
            for (int c = 0; c < DPL; ++c) acc[c] *= alpha;
            m = top;
        }
        float p[4 * H];
#pragma unroll
        for (int j = 0; j < 4 * H; ++j) {
            p[j] = exp2_hw(s[j] - base);
            l += p[j];
        }
        // rows that are not visible may hold anything, and 0 * NaN is NaN
        if (__any(vis != (1u << 4 * H) - 1)) {
#pragma unroll
            for (int j = 0; j < 4 * H; ++j)
                if (!(vis >> j & 1u))
#pragma unroll
                    for (int i = 0; i < VW; ++i) vr[j][i] = 0u;
        }

        if constexpr (sizeof(T) == 2) {
            // p as 16-bit parts, each the rounding of what those before it left, for more passes of a unit that is idle: three
            // of bf16 hold all 24 bits, two of fp16 carry p to 2^-22. fp16 takes p times 2^14: its least number is 2^-24,
            // which weights of a long sequence fall under.
            constexpr int kParts = __is_same(T, __bf16) ? 3 : 2;
            uint32_t part[kParts][2 * H];
#pragma unroll
            for (int i = 0; i < 2 * H; ++i) {
                float v[2] = {p[2 * i] * kPScale, p[2 * i + 1] * kPScale};
#pragma unroll
                for (int w = 0; w < kParts; ++w) {
                    part[w][i] = 0;
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const T r = (T)v[e];
                        v[e] -= (float)r;
                        part[w][i] |= (uint32_t) __builtin_bit_cast(uint16_t, r) << (16 * e);
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < DPL; ++c) {
                uint32_t f[2 * H]; // V^T: row c of the lane's columns, its slots
#pragma unroll
                for (int i = 0; i < 2 * H; ++i)
                    f[i] = __builtin_amdgcn_perm(vr[2 * i + 1][c / 2], vr[2 * i][c / 2], c % 2 ? 0x07060302u : 0x05040100u);
                const u32x4 fv = {f[0], f[1], f[2], f[3]};
#pragma unroll
                for (int w = 0; w < kParts; ++w) mfma_frag(acc[c], fv, (u32x4){part[w][0], part[w][1], part[w][2], part[w][3]}, T());
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4 * H; ++j)
#pragma unroll
                for (int c = 0; c < DPL; ++c)
                    acc[c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vr[j][c]), p[j], acc[c], 0, 0, 0);
        }
        if (t1 < end) load_v(t1);
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);

    // The waves' parts, joined in wave order: acc[c][r] of lane (g, n) is head n, element DPL (4g + r) + c.
    __shared__ float sm[kWaves][16], sl[kWaves][16];
    extern __shared__ float so[]; // [kWaves][nh][DP + 1]
    constexpr int kRow = DP + 1;
    if (g == 0) {
        sm[wave][n] = m;
        sl[wave][n] = l;
    }
    __syncthreads();
    float M = sm[0][n];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) M = fmaxf(M, sm[w][n]);
    const float mbase = M == -INFINITY ? 0.f : M;
    const float mine = exp2_hw(m - mbase) * (1.f / kPScale);
    if (n < nh) {
        float *row = so + (wave * nh + n) * kRow;
#pragma unroll
        for (int c = 0; c < DPL; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) row[DPL * (4 * g + r) + c] = acc[c][r] * mine;
    }
    __syncthreads();
    const bool whole = a.splits == 1;
    for (int h = wave; h < nh; h += kWaves) {
        float Mh = sm[0][h];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) Mh = fmaxf(Mh, sm[w][h]);
        const float bh = Mh == -INFINITY ? 0.f : Mh;
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) L += sl[w][h] * exp2_hw(sm[w][h] - bh);
        const int64_t sh = (int64_t)seq * a.heads + h0 + h;
        const float inv = whole && L > 0.f ? 1.f / L : (whole && L == 0.f ? 0.f : (whole ? L : 1.f));
        if (whole || Mh != -INFINITY)
            for (int d = lane; d < a.dim; d += 64) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) v += so[(w * nh + h) * kRow + d];
                if (whole) ((T *)a.o)[(int64_t)seq * a.o_stride + (int64_t)(h0 + h) * a.dim + d] = (T)(v * inv);
                else a.part_o[(sh * a.splits + sp) * a.part_row + d] = v;
            }
        if (lane == 0) {
            if (whole && a.lse) a.lse[sh] = L == 0.f ? -INFINITY : (Mh + __log2f(L)) * kLn2;
            if (a.part_ml) {
                a.part_ml[(sh * a.splits + sp) * 2] = Mh;
                a.part_ml[(sh * a.splits + sp) * 2 + 1] = L;
            }
        }
    }
}

// Maximum and sum of one head over its splits, by the lanes of a wave; the same in every lane.
__device__ __forceinline__ void join_ml(const float *ml, int splits, int lane, float &M, float &L) {
    M = -INFINITY;
    for (int i = lane; i < splits; i += 64) M = fmaxf(M, ml[2 * i]);
#pragma unroll
    for (int off = 32; off; off >>= 1) M = fmaxf(M, __shfl_xor(M, off));
    const float base = M == -INFINITY ? 0.f : M;
    L = 0.f;
    for (int i = lane; i < splits; i += 64) L += ml[2 * i + 1] * exp2_hw(ml[2 * i] - base);
#pragma unroll
    for (int off = 32; off; off >>= 1) L += __shfl_xor(L, off);
}

// Blocks below join_blocks: one (sequence, head) each, the splits' sums joined in split order
// by strands of threads and the strands in order. The others: 1024 slots of one (sequence, kv head),
// the heads' weights added up.
constexpr int kAccSlots = 1024;
template <class T>
__global__ __launch_bounds__(256) void kv_join_kernel(AttendArgs a, int join_blocks, const float *__restrict__ acc_in,
                                                      float *acc_out, int64_t acc_stride, int acc_chunks) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if ((int)blockIdx.x < join_blocks) {
        const int sh = blockIdx.x, seq = sh / a.heads, h = sh - seq * a.heads;
        const float *ml = a.part_ml + (int64_t)sh * a.splits * 2;
        float M, L;
        join_ml(ml, a.splits, lane, M, L);
        const float base = M == -INFINITY ? 0.f : M;
        // strands of threads, each over the row's runs of 4, take every strands-th split
        __shared__ float sum[256 * 4];
        const int runs = (a.dim + 3) / 4;
        int cols = 1;
        while (cols < runs) cols *= 2;
        const int strands = 256 / cols, strand = threadIdx.x / cols, d = threadIdx.x % cols * 4;
        const float *po = a.part_o + (int64_t)sh * a.splits * a.part_row + d;
        f32x4 v = {0.f, 0.f, 0.f, 0.f};
        if (d < a.dim) {
#pragma unroll 4
            for (int i = strand; i < a.splits; i += strands) {
                const float mi = ml[2 * i];
                // (a split with nothing visible wrote no row)
                if (mi != -INFINITY) v += *reinterpret_cast<const f32x4 *>(po + (int64_t)i * a.part_row) * exp2_hw(mi - base);
            }
        }
        *reinterpret_cast<f32x4 *>(sum + threadIdx.x * 4) = v;
        __syncthreads();
        if ((int)threadIdx.x < a.dim) {
            float r = 0.f;
            for (int i = 0; i < strands; ++i) r += sum[i * cols * 4 + threadIdx.x];
            ((T *)a.o)[(int64_t)seq * a.o_stride + (int64_t)h * a.dim + threadIdx.x] = (T)(L == 0.f ? 0.f : r / L);
        }
        if (threadIdx.x == 0 && a.lse) a.lse[sh] = L == 0.f ? -INFINITY : (M + __log2f(L)) * kLn2;
        return;
    }
    const int b = blockIdx.x - join_blocks;
    const int chunk = b % acc_chunks, sg = b / acc_chunks, seq = sg / a.kv_heads, kvh = sg - seq * a.kv_heads;
    const int len = min(max(a.lengths[seq], 0), a.max_len);
    const int s0 = chunk * kAccSlots;
    if (s0 >= len) return;
    extern __shared__ float hml[]; // [group][2]: base and 1 / sum
    const int64_t first = (int64_t)seq * a.heads + (int64_t)kvh * a.group;
    for (int h = wave; h < a.group; h += 4) {
        float M, L;
        join_ml(a.part_ml + (first + h) * a.splits * 2, a.splits, lane, M, L);
        if (lane == 0) {
            hml[2 * h] = M == -INFINITY ? 0.f : M;
            hml[2 * h + 1] = L == 0.f ? 0.f : 1.f / L;
        }
    }
    __syncthreads();
    const int64_t row = (int64_t)sg * acc_stride;
    const int stop = min(len, s0 + kAccSlots);
    for (int i = s0 + threadIdx.x; i < stop; i += 256) {
        float v = 0.f;
        for (int h = 0; h < a.group; ++h)
            v += exp2_hw(a.scores[(first + h) * a.score_row + i] - hml[2 * h]) * hml[2 * h + 1];
        acc_out[row + i] = acc_in[row + i] + v;
    }
}

// Rows of `units` units of U, strides in units. One workgroup per token, threads over its rows of all heads.
template <class U>
__global__ __launch_bounds__(256) void kv_append_kernel(SpinnHipKvDesc d, int units, int64_t tokens, const int32_t *seq,
                                                        const int32_t *slot, const int32_t *position, const U *k,
                                                        int64_t k_stride, const U *v, int64_t v_stride,
                                                        const int32_t *table, U *k_pages, U *v_pages, float *acc,
                                                        int32_t *pos, int64_t acc_stride) {
    const int row = d.kv_heads * units;
    for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
        const int s = seq ? seq[t] : (int)t;
        const int at = slot[t];
        if ((unsigned)s >= (unsigned)d.seqs || at < 0) continue;
        const int pi = at / d.page_size;
        if (pi >= d.max_pages) continue;
        const int page = table[(int64_t)s * d.max_pages + pi];
        if ((unsigned)page >= (unsigned)d.n_pages) continue;
        const int64_t base = (int64_t)page * d.page_stride + (int64_t)(at - pi * d.page_size) * d.slot_stride;
        for (int i = threadIdx.x; i < row; i += blockDim.x) {
            const int h = i / units;
            const int64_t to = base + (int64_t)h * d.head_stride + (i - h * units);
            k_pages[to] = k[t * k_stride + i];
            v_pages[to] = v[t * v_stride + i];
        }
        if (at < acc_stride)
            for (int h = threadIdx.x; h < d.kv_heads; h += blockDim.x) {
                const int64_t e = ((int64_t)s * d.kv_heads + h) * acc_stride + at;
                if (acc) acc[e] = 0.f;
                if (pos) pos[e] = position ? position[t] : at;
            }
    }
}

struct Plan {
    int head_tiles, splits, chunk, waves;
    int64_t score_row;
    size_t o_bytes, ml_bytes, score_bytes;
};

Plan plan(const SpinnHipKvAttentionDesc *d) {
    Plan p;
    const int group = d->heads / d->kv.kv_heads;
    p.head_tiles = (group + kHeadTile - 1) / kHeadTile;
    const int64_t units = (int64_t)d->kv.seqs * d->kv.kv_heads * p.head_tiles;
    const int64_t steps = std::max<int64_t>(1, (d->max_len + kStep - 1) / kStep);
    // Parts of about 1 MB at most: a workgroup's start and end cost as much as 100 KB of reading (32 sequences of 37 to 8000
    // slots, 8 x 128 bf16: 159 us at 128 KB, 141 at 256, 132 at 512, 122 at 1 MB, 137 unsplit).
    // Shorter ones, down to a step per wave, where longer ones would leave CUs idle.
    const int64_t fill = (steps * units + 2 * device_cu_count() - 1) / (2 * device_cu_count());
    const int64_t bytes = (int64_t)2 * kStep * d->kv.head_dim * dtype_bytes(d->kv.dtype);
    const int64_t most = std::max<int64_t>(1, std::min(fill, (1048576 + bytes - 1) / bytes)); // steps per split
    p.splits = (int)((steps + most - 1) / most);
    // Short sequences in one workgroup of eight waves, two steps each, where a workgroup per CU is enough: no second
    // launch (1 sequence of 500 slots, fp16: 10.0 -> 7.9 us; 32 of 250, bf16: 14.2 -> 10.4; 64 of 200: 13.3 -> 17.0,
    // so not there).
    p.waves = 4;
    const int eight = 8 * (dtype_bytes(d->kv.dtype) == 2 ? 32 : 16); // slots per step
    if (p.splits > 1 && d->max_len <= 2 * eight && d->kv.head_dim <= 128 && units <= device_cu_count()) {
        p.splits = 1;
        p.waves = 8;
    }
    const int64_t per = (steps + p.splits - 1) / p.splits; // alike
    p.splits = (int)((steps + per - 1) / per);               // none begins behind max_len, however they round
    p.chunk = (int)(per * kStep);
    const int64_t rows = (int64_t)d->kv.seqs * d->heads;
    p.score_row = ((int64_t)d->max_len + 31) / 32 * 32;
    p.o_bytes = p.splits > 1 ? (size_t)rows * p.splits * ((d->kv.head_dim + 3) & ~3) * 4 : 0;
    p.ml_bytes = p.splits > 1 || d->accumulate ? round16((size_t)rows * p.splits * 8) : 0;
    p.score_bytes = d->accumulate ? (size_t)rows * p.score_row * 4 : 0;
    return p;
}

template <class T, int DP, int W>
void launch_attend(const AttendArgs &a, Rows rows, bool uni, dim3 grid, hipStream_t st) {
    const size_t lds = (size_t)W * std::min(a.group, kHeadTile) * (DP + 1) * sizeof(float);
    if (rows == kRuns && uni) kv_attend_kernel<T, DP, kRuns, true, W><<<grid, 64 * W, lds, st>>>(a);
    else if (rows == kRuns) kv_attend_kernel<T, DP, kRuns, false, W><<<grid, 64 * W, lds, st>>>(a);
    else if (rows == kLoose && uni) kv_attend_kernel<T, DP, kLoose, true, W><<<grid, 64 * W, lds, st>>>(a);
    else if (rows == kLoose) kv_attend_kernel<T, DP, kLoose, false, W><<<grid, 64 * W, lds, st>>>(a);
    else if constexpr (DP == 64) kv_attend_kernel<T, DP, kShort, false, W><<<grid, 64 * W, lds, st>>>(a);
}

} // namespace

size_t kv_attention_workspace_bytes(const SpinnHipKvAttentionDesc *d) {
    const Plan p = plan(d);
    return p.o_bytes + p.ml_bytes + p.score_bytes;
}

int kv_attention(const SpinnHipKvAttentionDesc *d, const void *q, const void *k, const void *v, const int32_t *table,
                 const int32_t *lengths, const uint8_t *mask, const float *acc, float *acc_out, void *o, float *lse,
                 void *ws, hipStream_t st) {
    const Plan p = plan(d);
    const SpinnHipKvDesc &kv = d->kv;
    AttendArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.table = table;
    a.lengths = lengths;
    a.mask = mask;
    a.o = o;
    a.lse = lse;
    char *w = (char *)ws;
    a.part_o = p.o_bytes ? (float *)w : nullptr;
    a.part_ml = p.ml_bytes ? (float *)(w + p.o_bytes) : nullptr;
    a.scores = p.score_bytes ? (float *)(w + p.o_bytes + p.ml_bytes) : nullptr;
    a.q_stride = d->q_stride;
    a.o_stride = d->o_stride;
    a.mask_stride = d->mask_stride;
    a.page_stride = kv.page_stride;
    a.head_stride = kv.head_stride;
    a.slot_stride = kv.slot_stride;
    a.score_row = p.score_row;
    a.scale2 = d->scale * kLog2e;
    a.seqs = kv.seqs;
    a.heads = d->heads;
    a.kv_heads = kv.kv_heads;
    a.group = d->heads / kv.kv_heads;
    a.dim = kv.head_dim;
    a.page_size = kv.page_size;
    // Rounded up, page_mul is off by less than 1, so the product for a slot below 2^31 by less than 2^31: under
    // one part in page_size of 2^(32 + shift) as long as page_size <= 2^(shift + 1).
    if (kv.page_size > 1) {
        a.page_shift = 31 - __builtin_clz((unsigned)kv.page_size - 1);
        a.page_mul = (uint32_t)((((uint64_t)1 << (32 + a.page_shift)) + kv.page_size - 1) / kv.page_size);
    }
    a.n_pages = kv.n_pages;
    a.max_pages = kv.max_pages;
    a.max_len = d->max_len;
    a.part_row = (kv.head_dim + 3) & ~3;
    a.splits = p.splits;
    a.chunk = p.chunk;
    a.head_tiles = p.head_tiles;
    const int64_t parts = (int64_t)kv.seqs * kv.kv_heads * p.splits;
    const int64_t blocks = (parts + 7) / 8 * 8 * p.head_tiles;
    a.parts = (int32_t)parts;
    const int acc_chunks = (d->max_len + kAccSlots - 1) / kAccSlots;
    const int64_t join_blocks = p.splits > 1 ? (int64_t)kv.seqs * d->heads : 0;
    const int64_t acc_blocks = d->accumulate ? (int64_t)kv.seqs * kv.kv_heads * acc_chunks : 0;
    if (!launch_fits(blocks, 64 * p.waves) || !launch_fits(join_blocks + acc_blocks, 256)) return SPINN_HIP_EUNSUPPORTED;
    const size_t hml = (size_t)a.group * 8;
    if (hml > 32768) return SPINN_HIP_EUNSUPPORTED;
    const int rc = with_dtype(kv.dtype, [&](auto t) {
        typedef decltype(t) T;
        const int e = 16 / (int)sizeof(T);
        const bool vec = kv.head_dim % e == 0 && kv.page_stride % e == 0 && kv.head_stride % e == 0 &&
                         kv.slot_stride % e == 0 && aligned16(k) && aligned16(v);
        const Rows rows = vec ? kRuns : (kv.head_dim >= e ? kLoose : kShort);
        const bool uni = kv.page_size % 16 == 0;
        a.q_runs = kv.head_dim % e == 0 && d->q_stride % e == 0 && aligned16(q);
        const dim3 grid((unsigned)blocks);
        if (kv.head_dim <= 64) p.waves == 8 ? launch_attend<T, 64, 8>(a, rows, uni, grid, st) : launch_attend<T, 64, 4>(a, rows, uni, grid, st);
        else if (kv.head_dim <= 128) p.waves == 8 ? launch_attend<T, 128, 8>(a, rows, uni, grid, st) : launch_attend<T, 128, 4>(a, rows, uni, grid, st);
        else launch_attend<T, 256, 4>(a, rows, uni, grid, st);
        return check_launch();
    });
    if (rc || join_blocks + acc_blocks == 0) return rc;
    return with_dtype(kv.dtype, [&](auto t) {
        typedef decltype(t) T;
        kv_join_kernel<T><<<(unsigned)(join_blocks + acc_blocks), 256, hml, st>>>(a, (int)join_blocks, acc, acc_out,
                                                                                  d->acc_stride, acc_chunks);
        return check_launch();
    });
}

int kv_append(const SpinnHipKvDesc *d, int64_t tokens, const int32_t *seq, const int32_t *slot, const int32_t *position,
              const void *k, int64_t k_stride, const void *v, int64_t v_stride, const int32_t *table, void *k_pages,
              void *v_pages, float *acc, int32_t *pos, int64_t acc_stride, hipStream_t st) {
    // in units of 16 bytes where rows are whole, aligned runs of them (16384 tokens of 8 x 128, bf16: 24 us, 5.7 TB/s;
    // by elements 42)
    const int e = dtype_bytes(d->dtype), per = 16 / e;
    const bool vec = d->head_dim % per == 0 && d->page_stride % per == 0 && d->head_stride % per == 0 &&
                     d->slot_stride % per == 0 && k_stride % per == 0 && v_stride % per == 0 && aligned16(k) && aligned16(v) &&
                     aligned16(k_pages) && aligned16(v_pages);
    const int unit = vec ? per : 1;
    SpinnHipKvDesc u = *d;
    u.page_stride /= unit;
    u.head_stride /= unit;
    u.slot_stride /= unit;
    auto launch = [&](auto one) {
        typedef decltype(one) U;
        kv_append_kernel<U><<<(unsigned)std::min<int64_t>(tokens, 65536), 256, 0, st>>>(
            u, d->head_dim / unit, tokens, seq, slot, position, (const U *)k, k_stride / unit, (const U *)v, v_stride / unit,
            table, (U *)k_pages, (U *)v_pages, acc, pos, acc_stride);
        return check_launch();
    };
    if (vec) return launch(u32x4());
    return e == 4 ? launch(uint32_t()) : launch(uint16_t());
}

} // namespace spinn
