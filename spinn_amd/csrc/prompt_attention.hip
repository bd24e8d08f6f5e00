// prompt_attention.hip - attention within packed sequences: every row of a prompt over the rows that it sees.
//
// o_i = sum_j p_ij v_j, p = softmax over the visible j of scale q_i.k_j, in one pass over the keys with the running maximum and sum.
// 4 head_dim flops a visible pair: the matrix cores bound it, and beside them the exponentials, one a pair.
//
// The rows of a tile are (token, query head of the group) pairs, so that all heads that share a kv head share its
// tiles in LDS. S^T = K Q^T: an accumulator's column, so a lane and one (fp32: three) more, is one row of queries; its maximum and sum
// need an exchange among those, and a mask is one number a lane. The products' elements that a lane
// holds are exactly the operand that O^T = V^T P^T wants from it (contraction over keys may run in any order); V^T comes
// out of LDS transposed by the read itself (16-bit types) or by whole runs of a row (fp32).
//
// 16-bit types: 128 rows a workgroup, tiles of 64 keys, 32 x 32 instructions, two workgroups a CU (heads of 128). 16000 rows, 32 heads on 8
// of 128, bf16, causal: 1830 to 2040 us by the card, up to 1150 TFLOP/s, bound by power (1400 us on zeros); 24 sequences of 37 to 2000 rows: 326 to 342 us.
// fp32: 64 rows, tiles of 16 keys, 16 x 16 instructions at the same rate: less padding (80 columns are five blocks) and small
// enough for five workgroups a CU. 8 x 577 rows, 16 heads of 80: 127 us, 107 TFLOP/s (32 x 32 instructions, 128 rows: 179); 4 x 2000 of 128
// 618 (670); 2 x 1000, 8 heads on 2 of 256: 141 (277).
#include "decode.h"
#include <cmath>
#include <limits>
#include <type_traits>

namespace spinn {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// The maximum that a row's weights are relative to may lag behind by 2^kLag, so that sums are rescaled seldom.
constexpr float kLag = 8.f;
// Rows of a wave and of a workgroup: the matrix instructions' size, 32 x 32 for 16-bit types, 16 x 16 for fp32.
template <class T> constexpr int kWaveRows = sizeof(T) == 2 ? 32 : 16;
template <class T> constexpr int kRows = 4 * kWaveRows<T>;

struct PromptArgs {
    const void *q, *k, *v;
    void *o;
    float *lse;
    const int32_t *starts, *kv_starts;
    int64_t q_stride, k_stride, v_stride, o_stride;
    float scale2;      // |scale| log2 e
    uint32_t flip;     // sign bits of two 16-bit elements or one fp32 where the scale is negative
    float *part_o, *part_ml; // [item][kv head][split][kRows][head_dim padded], [..][2] (maximum and sum, base 2)
    int32_t seqs, heads, kv_heads, group, dim, causal, q_rows, kv_rows, splits;
    uint32_t group_mul, group_shift; // row / group = row * group_mul >> 32 + group_shift (group_mul 0: row)
    int32_t o_runs;    // rows of o are whole, aligned 16-byte runs
    int32_t at_once;   // all workgroups are on the device together
};

__device__ __forceinline__ int token_of(const PromptArgs &a, int row) {
    return a.group_mul ? (int)(__umulhi((uint32_t)row, a.group_mul) >> a.group_shift) : row;
}

// Which tile of which sequence is `item`, and the sequence's rows.
struct Place {
    int tile; // < 0: none
    int q0, nq, k0, nk;
};
__device__ __forceinline__ int clamped(const int32_t *starts, int i, int rows) { return min(max(starts[i], 0), rows); }
// Sequence by sequence, so that what runs at a time shares keys in the L2 (24 sequences of 37 to 2000 rows, in an earlier form: 406 us; all their
// last tiles first, then the ones before them, 421), each from its end, where a causal mask leaves the most keys. Up to 64, one a
// lane, the longest first, so that what starts last is short.
__device__ __forceinline__ Place find_place(const PromptArgs &a, int item, int rows) {
    const int lane = threadIdx.x & 63;
    const int32_t *ks = a.kv_starts ? a.kv_starts : a.starts;
    if (a.seqs <= 64) {
        const int s = min(lane, a.seqs - 1);
        const int q0 = clamped(a.starts, s, a.q_rows), q1 = clamped(a.starts, s + 1, a.q_rows);
        const int k0 = clamped(ks, s, a.kv_rows), k1 = clamped(ks, s + 1, a.kv_rows);
        const int n = lane < a.seqs ? (max(q1 - q0, 0) * a.group + rows - 1) / rows : 0;
        // tiles of the sequences that come first: those of more tiles (up to 2^25), or as many and an earlier lane
        const uint32_t key = (uint32_t)n << 6 | (uint32_t)(63 - lane);
        int before = 0;
        if (a.seqs > 1) {
#pragma unroll 8
            for (int i = 0; i < ((a.seqs + 7) & ~7); ++i) { // lanes behind the last sequence have no tiles
                const uint32_t o = (uint32_t)__builtin_amdgcn_readlane((int)key, i);
                before += o > key ? (int)(o >> 6) : 0;
            }
        }
        const unsigned long long mine = __ballot(item >= before && item - before < n);
        const int seq = __ffsll(mine) - 1;
        if (seq < 0) return {-1, 0, 0, 0, 0};
        const int tile = __builtin_amdgcn_readlane(n - 1 - (item - before), seq);
        const int first = __builtin_amdgcn_readlane(q0, seq), kfirst = __builtin_amdgcn_readlane(k0, seq);
        return {tile, first, __builtin_amdgcn_readlane(q1, seq) - first, kfirst,
                max(__builtin_amdgcn_readlane(k1, seq) - kfirst, 0)};
    }
    // More: a sequence's tiles stand from `place` on, which no sum is needed for: sequence s + 1's is at least s's tiles behind it (the whole
    // part of a sum grows by the rounded-up length less one at least; the second term by one where there are rows). 64 shares of the
    // sequences left a step: two steps up to 4096 sequences, four up to 2^24 (5000 sequences of 1 to 8 rows, 32 heads on 8 of 128: 529 us, with
    // every workgroup adding up all sequences' tiles 1630; 300 of 1 to 400: 361 and 389).
    auto place = [&](int s) {
        const int row = clamped(a.starts, s, a.q_rows);
        return row * a.group / rows + min(s, row);
    };
    int first = 0, left = a.seqs;
    while (left > 1) {
        const int each = (left + 63) / 64, at = lane * each;
        const int upto = __popcll(__ballot(at < left && place(first + at) <= item));
        if (upto == 0) return {-1, 0, 0, 0, 0};
        first += (upto - 1) * each;
        left = min(each, left - (upto - 1) * each);
    }
    const int q0 = clamped(a.starts, first, a.q_rows), k0 = clamped(ks, first, a.kv_rows);
    const int nq = max(clamped(a.starts, first + 1, a.q_rows) - q0, 0);
    const int n = (nq * a.group + rows - 1) / rows, tile = item - place(first);
    if (tile < 0 || tile >= n) return {-1, 0, 0, 0, 0};
    return {n - 1 - tile, q0, nq, k0, max(clamped(ks, first + 1, a.kv_rows) - k0, 0)};
}

// How 16-byte runs of a row lie in LDS, so that lanes that read a column of them (K), and lanes that read pieces of four rows (V in 16-bit
// types), meet all banks. V in fp32 is read by whole 256 bytes of a row.
template <class T, int DP>
struct Tile {
    static constexpr int E = 16 / (int)sizeof(T);
    static constexpr int kRow = DP * (int)sizeof(T);  // bytes
    static constexpr int kRuns = kRow / 16;
    static constexpr int kPow2 = (kRuns & -kRuns) < 16 ? (kRuns & -kRuns) : 16; // runs that may change places among each other
    static constexpr int kBlocks = kRow / 64, kBlockPow2 = (kBlocks & -kBlocks) < 4 ? (kBlocks & -kBlocks) : 4;
    static constexpr int log2of(int n) { return n > 1 ? 1 + log2of(n / 2) : 0; }
    __device__ __forceinline__ static int k_run(int row, int run) { return run_of(false, row, run); }
    __device__ __forceinline__ static int v_run(int row, int run) { return run_of(true, row, run); }
    __device__ __forceinline__ static int run_of(bool v, int row, int run) { // without a branch on v, which a wave knows
        const int down = v ? log2of(4 / kBlockPow2) : log2of(16 / kPow2), up = v ? 2 : 0;
        const int mask = v ? (sizeof(T) == 2 ? kBlockPow2 - 1 : 0) : kPow2 - 1;
        return run ^ ((row >> down & mask) << up);
    }
};

__device__ __forceinline__ f32x16 mfma_piece(u32x4 a, u32x4 b, f32x16 c, _Float16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma_piece(u32x4 a, u32x4 b, f32x16 c, __bf16) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_piece(u32x4 a, u32x4 b, f32x4 c, float) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
        c = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, (uint32_t)a[e]), __builtin_bit_cast(float, (uint32_t)b[e]), c, 0, 0, 0);
    return c;
}

template <class T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    typedef T T2 __attribute__((ext_vector_type(2)));
    T2 v;
    v[0] = (T)a;
    v[1] = (T)b;
    return __builtin_bit_cast(uint32_t, v);
}

// A row's value out of those of its lanes, lane % 32 (or 16).
template <int R, class F>
__device__ __forceinline__ float across(float v, F f) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto far = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    v = f(__builtin_bit_cast(float, (uint32_t)far[0]), __builtin_bit_cast(float, (uint32_t)far[1]));
    if constexpr (R == 16) {
        const uint32_t c = __builtin_bit_cast(uint32_t, v);
        const auto near = __builtin_amdgcn_permlane16_swap(c, c, false, false);
        v = f(__builtin_bit_cast(float, (uint32_t)near[0]), __builtin_bit_cast(float, (uint32_t)near[1]));
    }
    return v;
}

// 16 bytes a lane from base + off to byte `to` + 16 lane of LDS; all_ready() waits for it. In assembly, since the compiler would wait for all
// of these before every transposing read of LDS that follows, whatever it reads (16000 rows, before other steps: 2020 -> 1916 us).
// lanes: -1 all of those that are here, 0 none, without a branch.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm" // m0 among what the statement changes is meant
__device__ __forceinline__ void async_run(const char *base, uint32_t off, uint32_t to, int lanes = -1) {
    uint64_t here;
    asm volatile("s_mov_b32 m0, %1\n\ts_and_saveexec_b64 %0, %4\n\tglobal_load_lds_dwordx4 %2, %3\n\ts_mov_b64 exec, %0"
                 : "=&s"(here)
                 : "s"(__builtin_amdgcn_readfirstlane(to)), "v"(off), "s"(base), "s"((int64_t)__builtin_amdgcn_readfirstlane(lanes))
                 : "memory", "m0", "scc");
}
#pragma clang diagnostic pop

// This wave's copies have landed and its LDS reads are done, and so are every other wave's.
__device__ __forceinline__ void all_ready() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// Workgroups on a CU, as registers and LDS allow.
template <class T, int DP, bool RUNS>
constexpr int kAtOnce = sizeof(T) == 4 ? (DP <= 96 ? 4 + RUNS : DP == 128 ? 3 + RUNS : 2) : DP <= 128 ? (DP == 96 && RUNS ? 3 : 2) : 1;

// What a matrix product has just left in s may be read. The compiler counts the wait that is due along one way into a block only
// (16 x 16 x 4 fp32: 10 instructions by the masked way, 1 by the other, where it put none), so it is written out here.
template <class T, int B, class Acc>
__device__ __forceinline__ void settle(Acc (&s)[B]) {
    if constexpr (sizeof(T) == 2) asm volatile("s_nop 7\n\ts_nop 3" : "+v"(s[B - 1]));
    else asm volatile("s_nop 7\n\ts_nop 1" : "+v"(s[B - 1]));
#pragma unroll
    for (int b = 0; b < B - 1; ++b) asm volatile("" : "+v"(s[b]));
}

// T: element; DP: head_dim padded to whole matrix operands; KB: keys of a tile;
// RUNS: rows of q, k and v are whole, aligned 16-byte runs.
template <class T, int DP, int KB, bool RUNS>
__global__ __launch_bounds__(256, (kAtOnce<T, DP, RUNS>)) void prompt_kernel(PromptArgs a) {
    typedef Tile<T, DP> Lay;
    constexpr int R = kWaveRows<T>, G = 64 / R, kRows = ::spinn::kRows<T>; // G: lanes of a row
    typedef float Acc __attribute__((ext_vector_type(R * R / 64)));
    constexpr int A4 = R * R / 256; // fours of an accumulator: rows 4 G i + 4 h ..
    constexpr int E = Lay::E, kRow = Lay::kRow, NC = kRow / (16 * G); // NC: operand pieces of a row
    constexpr int B = KB / R, DB = DP / R;
    // fp32: the columns of O that four (two, one) accumulators in a row hold go round among them, so that a lane's pieces of V's row lie
    // next to each other, and so do four elements of O's.
    constexpr int kFull = DB / 4 * 4, kRest = DB % 4;
    static_assert(sizeof(T) == 2 || kRest != 3, "");
    constexpr int kTile = KB * kRow;        // bytes of a tile of K or V
    constexpr int kCopies = kTile / 1024;   // of 1 KB: two waves copy K, two V
    constexpr int P = (kCopies + 1) / 2;    // a wave's
    static_assert(kTile % 1024 == 0 && NC * 16 * G == kRow && P <= B * NC, "");
    // fp16's weights are kept 2^7 higher: its least number is 2^-24, which many small ones together fall under
    constexpr float kUp = __is_same(T, _Float16) ? 7.f : 0.f;
    __shared__ __attribute__((aligned(16))) char lds[4 * kTile]; // K, V of the even tiles, then of the odd ones
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane % R, h = lane / R;
    const int kvh = (int)blockIdx.x % a.kv_heads, sp = (int)blockIdx.x / a.kv_heads % a.splits, item = (int)blockIdx.x / a.kv_heads / a.splits;
    const Place at = find_place(a, item, kRows);
    if (at.tile < 0) return;
    const int q0 = at.q0, nq = at.nq;
    const int rows = nq * a.group, row0 = at.tile * kRows;
    // rows beyond the last take part as copies of it
    auto keys_of = [&](int row) { // how many a row sees
        return a.causal ? min(max(token_of(a, min(row, rows - 1)) + at.nk - nq + 1, 0), at.nk) : at.nk;
    };
    // This split's tiles of those that the last row sees; from here on keys are counted from their first.
    const int all = (keys_of(row0 + kRows - 1) + KB - 1) / KB;
    const int t_first = (int)((int64_t)all * sp / a.splits), tiles = (int)((int64_t)all * (sp + 1) / a.splits) - t_first;
    const int k0 = at.k0 + t_first * KB, nk = min(at.nk - t_first * KB, tiles * KB);
    auto limit_of = [&](int row) { return min(max(keys_of(row) - t_first * KB, 0), nk); };
    const int wrow = row0 + wave * R, limit = limit_of(wrow + n);
    const int wave_min = limit_of(wrow), wave_max = limit_of(wrow + R - 1);
    const bool is_v = wave >= 2; // what this wave copies
    const int64_t stride = is_v ? a.v_stride : a.k_stride;
    const char *const from_first = (const char *)((const T *)(is_v ? a.v : a.k) + (int64_t)k0 * stride + (int64_t)kvh * a.dim);
    const uint32_t row_bytes = (uint32_t)(stride * (int)sizeof(T));
    const int copy0 = (wave & 1) * P; // its first copy of the tile's
    // Bytes from a tile's first row to a lane's runs. Runs behind dim are copies of the last one: Q's are zeros there.
    uint32_t from[P];
    auto from_rows = [&](int left) { // of a tile whose row `left` is the last that there is: rows behind it are copies of it
        int here = lane;
        asm volatile("" : "+v"(here)); // so that nothing of this is kept in registers throughout
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int at = (copy0 + p) * 1024 + here * 16, run = min(Lay::run_of(is_v, at / kRow, at % kRow / 16), a.dim / E - 1);
            from[p] = (uint32_t)min(at / kRow, left) * row_bytes + (uint32_t)run * 16u;
        }
    };
    if constexpr (RUNS) from_rows(min(nk, KB) - 1);
    const char *from_at = from_first; // the tile to fetch next
    const uint32_t lds_at = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char *)lds;
    uint32_t fetch_to = is_v * kTile + copy0 * 1024; // its bytes of LDS, from lds on
    int lanes = -1;
    auto fetch_piece = [&](int p) { // of P; the second wave's may be one less
        async_run(from_at, from[p], lds_at + fetch_to + p * 1024, kCopies % 2 && p == P - 1 && copy0 ? 0 : lanes);
    };
    auto next_fetch = [&](int t) { // what is fetched next is tile t
        from_at = from_first + (int64_t)t * KB * row_bytes;
        fetch_to = (t & 1) * 2 * kTile + is_v * kTile + copy0 * 1024;
        if (RUNS && nk - t * KB < KB) from_rows(nk - t * KB - 1); // the last one
    };
    // The same through registers. 16-bit types: they go to LDS when the tile before is done (24 x 500 rows, 32 heads on 8 of 99, bf16: 237 us, at
    // once 287; 2 x 1000, 8 heads of 255: 119 and 176); fp32, with more waves to wait for: at once (2 x 1000, 8 heads of 255: 222, late 298;
    // smaller ones within 4 %).
    constexpr bool kLate = sizeof(T) == 2;
    typedef LooseRun<T, E> Run;
    u32x4 kept[RUNS ? 1 : P];
    auto load_loose_tile = [&](int t) {
        const int left = nk - t * KB - 1;
        int here = lane;
        if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(here)); // as in from_rows; fp32 has the registers
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int at = (copy0 + p) * 1024 + here * 16, d0 = Lay::run_of(is_v, at / kRow, at % kRow / 16) * E;
            if (kCopies % 2 && p == P - 1 && copy0) break;
            const T *rp = (const T *)(from_at + (int64_t)min(at / kRow, left) * row_bytes);
            kept[p] = a.dim >= E ? Run::load(rp, d0, a.dim) : load_edge<T>(rp + d0, a.dim - d0);
        }
    };
    auto store_loose_tile = [&]() {
        int here = lane;
        if constexpr (sizeof(T) == 2) asm volatile("" : "+v"(here));
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int at = (copy0 + p) * 1024 + here * 16, d0 = Lay::run_of(is_v, at / kRow, at % kRow / 16) * E;
            if (kCopies % 2 && p == P - 1 && copy0) break;
            uint32_t w[4] = {kept[p][0], kept[p][1], kept[p][2], kept[p][3]};
            if (a.dim >= E) Run::shift(kept[p], d0, a.dim, w);
            *reinterpret_cast<u32x4 *>(lds + fetch_to + p * 1024 + lane * 16) = (u32x4){w[0], w[1], w[2], w[3]};
        }
    };
    if (tiles > 0) {
        if constexpr (RUNS) {
#pragma unroll
            for (int p = 0; p < P; ++p) fetch_piece(p);
        } else {
            load_loose_tile(0);
            store_loose_tile();
        }
    }
    // where a row of the tile lies in q and o, in elements from the first one's token and the kv head's first query head
    const int tok0 = token_of(a, row0);
    auto row_at = [&](int row, int64_t stride) {
        const int tok = token_of(a, row);
        return (uint32_t)(tok - tok0) * (uint32_t)stride + (uint32_t)((row - tok * a.group) * a.dim);
    };
    const T *const q_first = (const T *)a.q + (int64_t)(q0 + tok0) * a.q_stride + (int64_t)kvh * a.group * a.dim;
    // Q's rows come through the odd tiles' place where they fit, whole lines at a time, a wave's own ones (24 sequences of 500 rows,
    // 32 heads on 8 of 128: 89.6 us, straight to registers 91.1; heads of 64 gain nothing, 155 and 151 at 1000 rows; fp32's do not fit)
    constexpr bool kStageQ = RUNS && DP > 64 && kRows * kRow <= 2 * kTile;
    if constexpr (kStageQ) {
        constexpr int PQ = R * kRow / 1024;
        const uint32_t to = lds_at + 2 * kTile + wave * PQ * 1024;
#pragma unroll
        for (int p = 0; p < PQ; ++p) {
            const int off = p * 1024 + lane * 16, r = wave * R + off / kRow, run = min(Lay::k_run(r, off % kRow / 16), a.dim / E - 1);
            async_run((const char *)q_first, row_at(min(row0 + r, rows - 1), a.q_stride) * (uint32_t)sizeof(T) + (uint32_t)run * 16u, to + p * 1024);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    const int my_row = min(wrow + n, rows - 1), token = token_of(a, my_row), head = kvh * a.group + (my_row - token * a.group);
    u32x4 q[NC];
    {
        const T *qp = q_first + row_at(my_row, a.q_stride);
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int d0 = (G * c + h) * E;
            if constexpr (kStageQ)
                q[c] = d0 >= a.dim ? (u32x4){0, 0, 0, 0}
                                   : *reinterpret_cast<const u32x4 *>(lds + 2 * kTile + (wave * R + n) * kRow + Lay::k_run(n, G * c + h) * 16);
            else if constexpr (RUNS) q[c] = d0 < a.dim ? *reinterpret_cast<const u32x4 *>(qp + d0) : (u32x4){0, 0, 0, 0};
            else q[c] = load_edge<T>(qp + d0, a.dim - d0);
#pragma unroll
            for (int w = 0; w < 4; ++w) q[c][w] ^= a.flip;
        }
    }

    // where a lane reads: K's row n (+ R a block), piece c; V's rows 4h + (lane % 16) / 4 (+ 8, + 16 cc, + 32 b), columns of block db
    // (the swap of runs is among the first ones; the others follow at the same distances), or in fp32 rows 4h + r (+ 16 b)
    constexpr int NK = Lay::kPow2 / G, NV = sizeof(T) == 2 ? Lay::kBlockPow2 : 1;
    int k_off[NK], v_off[NV];
#pragma unroll
    for (int c = 0; c < NK; ++c) k_off[c] = n * kRow + Lay::k_run(n, G * c + h) * 16;
#pragma unroll
    for (int d = 0; d < NV; ++d) {
        const int row = 4 * h + (lane & 15) / 4, run = 4 * d + 2 * ((lane >> 4) & 1) + (lane & 3) / 2;
        v_off[d] = sizeof(T) == 2 ? row * kRow + Lay::v_run(row, run) * 16 + (lane & 1) * 8 : 4 * h * kRow;
    }

    Acc o[DB] = {};
    float m = -INFINITY, l = 0.f; // base 2; l: this lane's share of the keys
    for (int t = 0; t < tiles; ++t) {
        // fp32: workgroups that are all on the device at once end together if those behind go first; the oldest ones would (8 x 577 rows, 16
        // heads of 80: 127.5 us, 133 without). Where others follow, they fill that gap themselves (8 x 2000 of 64: 672 with this, 628 without).
        if (sizeof(T) == 4 && a.at_once) {
            if (t == 0) __builtin_amdgcn_s_setprio(3);
            else if (t == tiles / 4) __builtin_amdgcn_s_setprio(2);
            else if (t == tiles / 2) __builtin_amdgcn_s_setprio(1);
            else if (t == tiles * 3 / 4) __builtin_amdgcn_s_setprio(0);
        }
        all_ready(); // tile t is there, and every wave is done with tile t - 1
        if (t + 1 < tiles) {
            next_fetch(t + 1);
            if constexpr (!RUNS) {
                load_loose_tile(t + 1);
                if constexpr (!kLate) store_loose_tile();
            }
        } else {
            lanes = 0;
        }
        const int first = t * KB;
        if (first >= wave_max) {
            if constexpr (RUNS) {
#pragma unroll
                for (int p = 0; p < P; ++p) fetch_piece(p);
            } else if constexpr (kLate) {
                if (lanes) store_loose_tile();
            }
            continue;
        }
        const char *kt = lds + (t & 1) * 2 * kTile, *vt = kt + kTile;

        Acc s[B] = {};
        // pieces of K's rows are read kAhead products before they are needed
        constexpr int kMostAhead = sizeof(T) == 2 ? 8 : 4, kAhead = NC < kMostAhead ? NC : kMostAhead;
        auto read_k = [&](int j) { return *reinterpret_cast<const u32x4 *>(kt + k_off[j % NC % NK] + j % NC / NK * NK * 16 * G + j / NC * R * kRow); };
        // The next tile's copies go out one by one between the products: a copy waits at its issue for those of the other waves to
        // pass (64 bytes a cycle for all of the CU), 600 cycles for the eight of a wave in a row.
        u32x4 kf[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) kf[j] = read_k(j);
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int j = 0; j < B * NC; ++j) {
            s[j / NC] = mfma_piece(kf[j % kAhead], q[j % NC], s[j / NC], T());
            if constexpr (RUNS) {
                const int p = ((j + 1) * P - 1) / (B * NC); // the copy whose turn comes within product j's
                if (j == (p + 1) * B * NC / P - 1) fetch_piece(p);
            }
            __builtin_amdgcn_sched_group_barrier(0x8, sizeof(T) == 2 ? 1 : 4, 0);
            if (j + kAhead < B * NC) {
                kf[j % kAhead] = read_k(j + kAhead);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
        }
        settle<T>(s);
        if (first + KB > wave_min) {
#pragma unroll
            for (int b = 0; b < B; ++b)
#pragma unroll
                for (int r = 0; r < 4 * A4; ++r)
                    if (first + R * b + 4 * G * (r / 4) + 4 * h + r % 4 >= limit) s[b][r] = -INFINITY;
        }
        float vf[2][DB]; // fp32: V's row r of each four, read while the row before the last one is multiplied
        auto read_v = [&](int b, int r) {
            const char *row = vt + v_off[0] + (R * b + r) * kRow;
#pragma unroll
            for (int d = 0; d < kFull; ++d) vf[r % 2][d] = (*reinterpret_cast<const f32x4 *>(row + d / 4 * 256 + n * 16))[d % 4];
#pragma unroll
            for (int d = kFull; kRest == 2 && d < DB; ++d) vf[r % 2][d] = (*reinterpret_cast<const f32x2 *>(row + kFull * 64 + n * 8))[d % 2];
            if constexpr (kRest == 1) vf[r % 2][kFull] = *reinterpret_cast<const float *>(row + kFull * 64 + n * 4);
        };
        if constexpr (sizeof(T) == 4) {
            read_v(0, 0);
            read_v(0, 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        float tops[4]; // shorter chains
#pragma unroll
        for (int r = 0; r < 4; ++r) tops[r] = s[0][r];
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int r = b ? 0 : 4; r < 4 * A4; ++r) tops[r % 4] = fmaxf(tops[r % 4], s[b][r]);
        float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
        top = across<R>(top, [](float x, float y) { return fmaxf(x, y); }) * a.scale2;
        if (__any(top > m + kLag)) {
            const float to = fmaxf(m, top), alpha = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= alpha;
        }
        const float base = m == -INFINITY ? 0.f : m - kUp;
#pragma unroll
        for (int b = 0; b < B; ++b)
#pragma unroll
            for (int r = 0; r < 4 * A4; ++r) {
                s[b][r] = __builtin_amdgcn_exp2f(fmaf(s[b][r], a.scale2, -base));
                l += s[b][r];
            }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            if constexpr (sizeof(T) == 2) {
                // weights enter the second product rounded once to T, as its operands have to be: off by half a step of T each, where
                // the result is rounded by as much (their sum is taken of the unrounded ones). In all 1.3 to 1.4 times the error of
                // the result's rounding alone; a second part of each weight would cost half as much again of the products.
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                    u32x4 p;
#pragma unroll
                    for (int w = 0; w < 4; ++w) p[w] = pack2<T>(s[b][8 * cc + 2 * w], s[b][8 * cc + 2 * w + 1]);
#pragma unroll
                    for (int d = 0; d < DB; ++d) {
                        typedef __attribute__((address_space(3))) s16x4 *Piece;
                        const char *vp = vt + v_off[d % NV] + d / NV * NV * 64 + (32 * b + 16 * cc) * kRow;
                        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Piece)vp);
                        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Piece)(vp + 8 * kRow));
                        const u32x2 wl = __builtin_bit_cast(u32x2, lo), wh = __builtin_bit_cast(u32x2, hi);
                        o[d] = mfma_piece((u32x4){wl[0], wl[1], wh[0], wh[1]}, p, o[d], T());
                    }
                }
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
#pragma unroll
                    for (int d = 0; d < DB; ++d) o[d] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[r % 2][d], s[b][r], o[d], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                    if (r < 2) read_v(b, r + 2);
                    else if (b + 1 < B) read_v(b + 1, r - 2);
                }
            }
        }
        if constexpr (!RUNS && kLate) {
            if (lanes) store_loose_tile();
        }
    }

    // four elements of o next to each other, and where: k of DB A4
    auto four = [&](int k) {
        if constexpr (sizeof(T) == 2) {
            return (f32x4){o[k / A4][k % A4 * 4], o[k / A4][k % A4 * 4 + 1], o[k / A4][k % A4 * 4 + 2], o[k / A4][k % A4 * 4 + 3]};
        } else {
            const int W = k < kFull ? 4 : kRest, d = k < kFull ? k / 4 * 4 : kFull, t = (k - d) * 4;
            return (f32x4){o[d + t % W][t / W], o[d + (t + 1) % W][(t + 1) / W], o[d + (t + 2) % W][(t + 2) / W], o[d + (t + 3) % W][(t + 3) / W]};
        }
    };
    auto four_at = [&](int k) {
        if constexpr (sizeof(T) == 2) return R * (k / A4) + 4 * G * (k % A4) + 4 * h;
        else return k < kFull ? k / 4 * 64 + 16 * h + k % 4 * 4 : kFull * 16 + 4 * kRest * h + (k - kFull) * 4;
    };
    const float sum = across<R>(l, [](float x, float y) { return x + y; });
    const bool mine = wrow + n < rows;
    if (a.splits > 1) { // as they are, for prompt_join_kernel
        const int64_t part = ((int64_t)(item * a.kv_heads + kvh) * a.splits + sp) * kRows + wave * R + n;
        if (mine) {
#pragma unroll
            for (int k = 0; k < DB * A4; ++k) *reinterpret_cast<f32x4 *>(a.part_o + part * DP + four_at(k)) = four(k);
            if (h == 0) *reinterpret_cast<float2 *>(a.part_ml + part * 2) = make_float2(m - kUp, sum);
        }
        return;
    }
    __syncthreads(); // the tiles' place takes o's
    const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
#pragma unroll
    for (int k = 0; k < DB * A4; ++k) {
        const int at4 = four_at(k);
        const f32x4 w = four(k);
        typedef T T4 __attribute__((ext_vector_type(4)));
        T4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(w[e] * inv);
        *reinterpret_cast<T4 *>(lds + (wave * R + n) * kRow + Lay::k_run(n, at4 / E) * 16 + at4 % E * (int)sizeof(T)) = v;
    }
    if (a.lse && h == 0 && mine) a.lse[(int64_t)(q0 + token) * a.heads + head] = sum == 0.f ? -INFINITY : (m - kUp + __log2f(sum)) * kLn2;
    // a wave's rows, whole lines at a time
    T *const o_first = (T *)a.o + (int64_t)(q0 + tok0) * a.o_stride + (int64_t)kvh * a.group * a.dim;
    if (a.o_runs) {
        constexpr int PO = R * kRow / 1024;
#pragma unroll
        for (int p = 0; p < PO; ++p) {
            const int off = p * 1024 + lane * 16, r = wave * R + off / kRow, run = off % kRow / 16;
            const u32x4 v = *reinterpret_cast<const u32x4 *>(lds + r * kRow + Lay::k_run(r, run) * 16);
            if (row0 + r < rows && run * E < a.dim) *reinterpret_cast<u32x4 *>(o_first + (row_at(row0 + r, a.o_stride) + run * E)) = v;
        }
    } else {
        for (int r = wave * R; r < (wave + 1) * R && row0 + r < rows; ++r) {
            T *op = o_first + row_at(row0 + r, a.o_stride);
            for (int d = lane; d < a.dim; d += 64)
                op[d] = *reinterpret_cast<const T *>(lds + r * kRow + Lay::k_run(r, d / E) * 16 + d % E * (int)sizeof(T));
        }
    }
}

// The splits' sums of a row, added in split order: a wave a row, a lane a split's weight, then four elements.
template <class T>
__global__ __launch_bounds__(256) void prompt_join_kernel(PromptArgs a, int part_row) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    constexpr int kRows = ::spinn::kRows<T>, kFours = kRows / 4; // of an (item, kv head)
    const int block = (int)blockIdx.x / kFours, r = (int)blockIdx.x % kFours * 4 + wave, kvh = block % a.kv_heads;
    const Place at = find_place(a, block / a.kv_heads, kRows);
    const int row = at.tile * kRows + r;
    if (at.tile < 0 || row >= at.nq * a.group) return;
    const int tok = token_of(a, row), head = kvh * a.group + (row - tok * a.group);
    const int64_t part = (int64_t)block * a.splits * kRows + r; // its first split
    const float2 ml = lane < a.splits ? *reinterpret_cast<const float2 *>(a.part_ml + (part + (int64_t)lane * kRows) * 2) : make_float2(-INFINITY, 0.f);
    float M = ml.x;
#pragma unroll
    for (int d = 32; d; d >>= 1) M = fmaxf(M, __shfl_xor(M, d));
    const float w = __builtin_amdgcn_exp2f(ml.x - (M == -INFINITY ? 0.f : M));
    float L = ml.y * w;
#pragma unroll
    for (int d = 32; d; d >>= 1) L += __shfl_xor(L, d);
    const float inv = L > 0.f ? 1.f / L : (L == 0.f ? 0.f : L);
    if (a.lse && lane == 0) a.lse[(int64_t)(at.q0 + tok) * a.heads + head] = L == 0.f ? -INFINITY : (M + __log2f(L)) * kLn2;
    T *op = (T *)a.o + (int64_t)(at.q0 + tok) * a.o_stride + (int64_t)head * a.dim;
    const int d0 = lane * 4;
    if (d0 >= a.dim) return;
    const float *from = a.part_o + part * part_row + d0;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; ++s)
        v += *reinterpret_cast<const f32x4 *>(from + (int64_t)s * kRows * part_row) *
             __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), s));
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (d0 + e < a.dim) op[d0 + e] = (T)(v[e] * inv);
}

// How the rows and keys are cut.
struct Cut {
    int rows;      // of a tile
    int64_t items; // tiles at most
    int pad;       // head_dim padded
    int splits;
};
Cut cut(const SpinnHipPromptAttentionDesc *d) {
    Cut c;
    const int64_t group = d->heads / d->kv_heads;
    c.rows = dtype_bytes(d->dtype) == 4 ? kRows<float> : kRows<__bf16>;
    c.items = (int64_t)d->q_rows * group / c.rows + std::min(d->seqs, d->q_rows); // `place` of the sequence behind the last
    // Each of these has its kernel: 24 x 500 rows, 32 heads on 8 of 32, bf16: 43 us, with 64 columns 52; 8 x 1000, 16 heads of 32, fp32: 137 and 206.
    for (const int pad : {256, 128, 96, 80, 64, 32})
        if (d->head_dim <= pad && (pad != 80 || c.rows == kRows<float>)) c.pad = pad;
    // Keys are split where workgroups of whole rows leave most of the device idle: into as many parts as two workgroups a CU take, of
    // 8 tiles at least, up to the join's 64. The parts' sums and the second launch cost some 10 us, so that is for 16 tiles less at least
    // (32 heads on 8 of 128, bf16: 16 rows over 4000 keys 68 -> 19 us, over 64000 1014 -> 66, 100 over 4000 69 -> 27; 1000 over 1000,
    // which stays whole, 24, in two 36).
    const int64_t tiles = ((int64_t)d->kv_rows / std::max(d->seqs, 1) + 63) / 64; // of an ordinary sequence
    const int64_t most = std::min({2 * device_cu_count() / std::max<int64_t>(c.items * d->kv_heads, 1), tiles / 8, (int64_t)64});
    c.splits = most >= 2 && tiles * (most - 1) / most >= 16 ? (int)most : 1;
    return c;
}

template <class T, int DP, int KB>
int launch(PromptArgs &a, const Cut &c, bool runs, hipStream_t st) {
    const int64_t grid = c.items * a.kv_heads * c.splits;
    if (!launch_fits(grid, 256)) return SPINN_HIP_EUNSUPPORTED;
    a.at_once = grid <= (runs ? kAtOnce<T, DP, true> : kAtOnce<T, DP, false>) * device_cu_count();
    if (runs) prompt_kernel<T, DP, KB, true><<<(unsigned)grid, 256, 0, st>>>(a);
    else prompt_kernel<T, DP, KB, false><<<(unsigned)grid, 256, 0, st>>>(a);
    if (c.splits > 1) prompt_join_kernel<T><<<(unsigned)(c.items * a.kv_heads * (c.rows / 4)), 256, 0, st>>>(a, DP);
    return check_launch();
}

} // namespace

size_t prompt_attention_workspace_bytes(const SpinnHipPromptAttentionDesc *d) {
    const Cut c = cut(d);
    return c.splits > 1 ? (size_t)(c.items * d->kv_heads * c.splits) * c.rows * (c.pad + 2) * 4 : 0;
}

int prompt_attention(const SpinnHipPromptAttentionDesc *d, const void *q, const void *k, const void *v, const int32_t *starts,
                     const int32_t *kv_starts, void *o, float *lse, void *ws, hipStream_t st) {
    const Cut c = cut(d);
    PromptArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.o = o;
    a.lse = lse;
    a.starts = starts;
    a.kv_starts = kv_starts;
    a.q_stride = d->q_stride;
    a.k_stride = d->k_stride;
    a.v_stride = d->v_stride;
    a.o_stride = d->o_stride;
    // A scale of nothing still multiplies the -inf of hidden keys: the least number takes its place, with which no score passes 2^-21.
    a.scale2 = std::max(std::fabs(d->scale) * kLog2e, std::numeric_limits<float>::denorm_min());
    const int e = dtype_bytes(d->dtype);
    a.flip = d->scale < 0 ? (e == 2 ? 0x80008000u : 0x80000000u) : 0u;
    a.seqs = d->seqs;
    a.heads = d->heads;
    a.kv_heads = d->kv_heads;
    a.group = d->heads / d->kv_heads;
    a.dim = d->head_dim;
    a.causal = d->causal;
    a.splits = c.splits;
    a.part_o = (float *)ws;
    a.part_ml = (float *)ws + c.items * d->kv_heads * c.splits * c.rows * c.pad;
    if (a.group > 1) { // exact for rows under 2^31
        while ((2u << a.group_shift) < (uint32_t)a.group) ++a.group_shift;
        a.group_mul = (uint32_t)(((1ull << (32 + a.group_shift)) + a.group - 1) / a.group);
    }
    a.q_rows = d->q_rows;
    a.kv_rows = d->kv_rows;
    const int per = 16 / e;
    const bool runs = a.dim % per == 0 && d->q_stride * e <= (1 << 24) && (d->q_stride | d->k_stride | d->v_stride) % per == 0 && aligned16(q) && aligned16(k) && aligned16(v);
    a.o_runs = a.dim % per == 0 && d->o_stride % per == 0 && aligned16(o);
    return with_dtype(d->dtype, [&](auto t) {
        typedef decltype(t) T;
        constexpr int K = sizeof(T) == 2 ? 64 : 16;
        if (c.pad == 32) return launch<T, 32, K>(a, c, runs, st);
        if (c.pad == 64) return launch<T, 64, K>(a, c, runs, st);
        if constexpr (sizeof(T) == 4) {
            if (c.pad == 80) return launch<T, 80, K>(a, c, runs, st);
        }
        if (c.pad == 96) return launch<T, 96, K>(a, c, runs, st);
        if (c.pad == 128) return launch<T, 128, K>(a, c, runs, st);
        return launch<T, 256, sizeof(T) == 2 ? 32 : 16>(a, c, runs, st);
    });
}

} // namespace spinn
