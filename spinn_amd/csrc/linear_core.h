// linear_core.h - kernels of linear layers, for floating-point types (linear.hip) and 8-bit integers (linear_i8.hip).
// T: element of x and w, O: of bias, residual and y.
#pragma once
#include "decode.h"
#include <type_traits>

namespace spinn {
namespace {

constexpr int kFragBytes = 1024;

// A block's sums
template <class T>
struct SumsOf {
    typedef f32x4 type;
};
template <>
struct SumsOf<int8_t> {
    typedef i32x4 type;
};
template <class T>
using Sums = typename SumsOf<T>::type;

// v Phi(v), within 3 * 2^-24 |v| (a correctly rounded 1 + erf has 2) and, for v < 0, within (10 + v^2) 2^-24 of itself.
// Up to 1.25, Phi(v) = 1/2 + v S(v^2); beyond, Phi(-a) = exp(-a^2 / 2) R(a), R(a) = exp(a^2 / 2) Phi(-a) = t P(t) for
// t = 1 / (1 + a/2). S and P are polynomials fitted to them with the least relative error (1e-8 and 1.4e-8, up to
// a = 14.6, where exp has left fp32). 26 instructions; an epilogue unrolls them over up to 128 values, and the whole of
// 1568 x 2048 x 512 fp32 takes 41.1 us (40.2 with a seven-digit erfc of half the length).
__device__ __forceinline__ float gelu_erf(float v) {
    const float a = fabsf(v), w = v * v;
    const float s = fmaf(fmaf(fmaf(fmaf(fmaf(-6.80949188e-06f, w, 1.11041125e-04f), w, -1.18383719e-03f), w, 9.97228269e-03f), w,
                              -6.64902106e-02f), w, 3.98942262e-01f);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.5f, a, 1.f));
    const float p = fmaf(fmaf(fmaf(fmaf(fmaf(fmaf(fmaf(-1.39945731e-01f, t, 4.05194312e-01f), t, -3.73826802e-01f), t, 2.40476951e-02f), t,
                                        3.27784605e-02f), t, 1.51606306e-01f), t, 1.99343786e-01f), t, 1.99474499e-01f);
    const float below = t * p * __builtin_amdgcn_exp2f(w * -0.72134752044448170f); // Phi(-a)
    return v * (a < 1.25f ? fmaf(v, s, 0.5f) : (v < 0.f ? below : 1.f - below));
}
// v/2 (1 + tanh u) = v / (1 + exp(-2u))
__device__ __forceinline__ float gelu_tanh(float v) {
    const float u = 0.7978845608028654f * (v + 0.044715f * v * v * v);
    return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * (-2.f * 1.4426950408889634f)));
}
template <int ACT>
__device__ __forceinline__ float linear_act(float v) {
    if constexpr (ACT == SPINN_LINEAR_RELU) return v < 0.f ? 0.f : v;
    else if constexpr (ACT == SPINN_LINEAR_SILU) return silu(v);
    else if constexpr (ACT == SPINN_LINEAR_GELU) return gelu_erf(v);
    else if constexpr (ACT == SPINN_LINEAR_GELU_TANH) return gelu_tanh(v);
    else return v;
}
// f(integral_constant<activation>)
template <class F>
__device__ __forceinline__ void with_act(int act, F f) {
    switch (act) {
    case SPINN_LINEAR_RELU: f(std::integral_constant<int, SPINN_LINEAR_RELU>()); break;
    case SPINN_LINEAR_SILU: f(std::integral_constant<int, SPINN_LINEAR_SILU>()); break;
    case SPINN_LINEAR_GELU: f(std::integral_constant<int, SPINN_LINEAR_GELU>()); break;
    case SPINN_LINEAR_GELU_TANH: f(std::integral_constant<int, SPINN_LINEAR_GELU_TANH>()); break;
    default: f(std::integral_constant<int, SPINN_LINEAR_NONE>()); break;
    }
}

struct LinearArgs {
    const void *x, *bias, *res; // x: rows, or granules [M/16][frags/2]
    const float *sx, *sw;       // 8-bit integers: scales of x's rows and of the columns
    const char *w;              // packed
    void *y;
    int64_t ldx, ldres, ldy;
    int32_t m, n, k, act;
    int32_t kf;      // fragments along K
    int32_t ntiles;  // of 16 columns
    int32_t vec;     // rows of residual and y are whole runs of 16 bytes
};

// C neighbouring columns n.. of a row: bias and residual as they are in memory, the sum, the activation, the result.
// Loads and stores are 16-byte runs where all C columns exist and the rows allow it, else element by element.
template <class T, int C>
struct Columns {
    static_assert(C * sizeof(T) % 8 == 0, "");
    typedef T Run __attribute__((ext_vector_type(C)));
    typedef float Sum __attribute__((ext_vector_type(C)));
    static constexpr int kAlign = C * sizeof(T) < 16 ? C * sizeof(T) : 16;
    typedef Run AlignedRun __attribute__((aligned(kAlign)));
    __device__ __forceinline__ static Run load(const T *p, int left, bool runs) {
        Run r;
        if (runs && left >= C) {
            r = *reinterpret_cast<const AlignedRun *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i) r[i] = i < left ? p[i] : (T)0.f;
        }
        return r;
    }
    template <int ACT>
    __device__ __forceinline__ static void store(T *p, int left, bool runs, Sum v) {
        Run r;
#pragma unroll
        for (int i = 0; i < C; ++i) r[i] = (T)linear_act<ACT>(v[i]);
        if (runs && left >= C) {
            *reinterpret_cast<AlignedRun *>(p) = r;
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (i < left) p[i] = r[i];
        }
    }
};

// Columns that accumulator block `tile` of a lane with l/16 = g holds: four from here on. Of 64 columns the
// blocks tile % 4 together are 16-byte runs, run q of lane group g at q 4 C + g C (C columns a run), so that the
// four lanes of a row store 64 neighbouring bytes at a time.
// (8-bit weights are packed as for 16-bit results, whatever these are.)
template <class T>
constexpr int kRunCols = sizeof(T) == 1 ? 8 : 16 / (int)sizeof(T);
template <class T>
__device__ __forceinline__ int first_col(int tile, int g) {
    constexpr int C = kRunCols<T>, B = C / 4; // blocks per run
    const int t = tile & 3;
    return (tile >> 2) * 64 + (t / B) * 4 * C + g * C + 4 * (t % B);
}

// x goes to LDS in granules of 16 rows by two fragments, 128 bytes (a cache line) of every row: row r's eight
// 16-byte runs at 128 r, run c in place c ^ (r / 2), so that the 16 lanes that read run c of 16 rows at once
// meet all banks. (64-byte pieces of rows, a fragment at a time, ask the L2 for every line twice:
// 348 against 275 us for the whole 4096 x 8192 x 4096 product.)
constexpr int kGranule = 2 * kFragBytes;
// Byte of the run that operand lane `lane` reads for the granule's fragment `half`.
__device__ __forceinline__ int granule_at(int lane, int half) {
    const int r = lane & 15, c = half * 4 + (lane >> 4);
    return r * 128 + ((c ^ (r >> 1)) << 4);
}

// The waves' sums of a workgroup's MT x NT blocks (from block row m0 and tile t0 on), added in wave order, to y.
template <class T, class O, int MT, int NT, int NW>
__device__ __forceinline__ void join_waves(const LinearArgs &a, int m0, int t0, int wave, int lane, const Sums<T> (&acc)[MT][NT]) {
    __shared__ Sums<T> part[NW][MT * NT][64];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
    // a wave finishes every NW-th block; what it adds is on its way while the others' sums come together
    constexpr int B = (MT * NT + NW - 1) / NW;
    typedef Columns<O, 4> Col;
    typename Col::Run bias[B], res[B];
    int rows[B], cols[B], left[B];
#pragma unroll
    for (int k = 0; k < B; ++k) {
        const int b = wave + k * NW, tile = t0 + b % NT;
        rows[k] = (m0 + b / NT) * 16 + (lane & 15);
        cols[k] = first_col<T>(tile, lane >> 4);
        left[k] = b < MT * NT && tile < a.ntiles && rows[k] < a.m ? a.n - cols[k] : 0;
        if (left[k] > 0) {
            if (a.bias) bias[k] = Col::load((const O *)a.bias + cols[k], left[k], false);
            if (a.res) res[k] = Col::load((const O *)a.res + (int64_t)rows[k] * a.ldres + cols[k], left[k], a.vec);
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < B; ++k)
        if (left[k] > 0) {
            const int b = wave + k * NW;
            Sums<T> s = part[0][b][lane];
#pragma unroll
            for (int w = 1; w < NW; ++w) s += part[w][b][lane];
            f32x4 v;
            if constexpr (sizeof(T) == 1) {
                const float sx = a.sx[rows[k]];
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = (float)s[i] * (i < left[k] ? a.sw[cols[k] + i] : 0.f) * sx;
            } else {
                v = s;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (a.bias) v[i] += (float)bias[k][i];
                if (a.res) v[i] += (float)res[k][i];
            }
            O *y = (O *)a.y + (int64_t)rows[k] * a.ldy + cols[k];
            with_act(a.act, [&](auto act) { Col::template store<decltype(act)::value>(y, left[k], a.vec, v); });
        }
}

template <class T, class O, int MT, int NT, int NW, Rows ROWS>
__global__ __launch_bounds__(64 * NW) void linear_stream_kernel(LinearArgs a) {
    constexpr int E = 16 / (int)sizeof(T);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t0 = blockIdx.x * NT, m0 = blockIdx.y * MT;
    const char *wp[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
        wp[j] = a.w + (int64_t)min(t0 + j, a.ntiles - 1) * a.kf * kFragBytes + lane * 16;
    const T *xp[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        if constexpr (ROWS == kLaidOut) xp[i] = (const T *)((const char *)a.x + (int64_t)min(m0 + i, (a.m - 1) >> 4) * a.kf * kFragBytes);
        else xp[i] = (const T *)a.x + (int64_t)min((m0 + i) * 16 + (lane & 15), a.m - 1) * a.ldx + (ROWS == kRuns ? (lane >> 4) * E : 0);
    }
    Sums<T> acc[MT][NT] = {};
    constexpr int U = MT * NT >= 8 ? 2 : 4;
    for (int f0 = wave; f0 < a.kf; f0 += NW * U) {
        u32x4 w[U][NT], x[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int f = min(f0 + u * NW, a.kf - 1);
#pragma unroll
            for (int j = 0; j < NT; ++j) w[u][j] = *reinterpret_cast<const u32x4 *>(wp[j] + (int64_t)f * kFragBytes);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                const int k0 = f * kFrag<T> + (lane >> 4) * E;
                if constexpr (ROWS == kLaidOut)
                    x[u][i] = *reinterpret_cast<const u32x4 *>((const char *)xp[i] + (int64_t)(f >> 1) * kGranule + granule_at(lane, f & 1));
                else if constexpr (ROWS == kRuns) x[u][i] = k0 < a.k ? *reinterpret_cast<const u32x4 *>(xp[i] + (int64_t)f * kFrag<T>) : (u32x4){0, 0, 0, 0};
                else if constexpr (ROWS == kShort) x[u][i] = load_edge<T>(xp[i] + k0, a.k - k0);
                else {
                    uint32_t r[4];
                    load_loose<T, E>(xp[i], k0, a.k, r);
                    x[u][i] = (u32x4){r[0], r[1], r[2], r[3]};
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (f0 + u * NW < a.kf) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j) mfma_frag(acc[i][j], w[u][j], x[u][i], T());
            }
    }
    join_waves<T, O, MT, NT, NW>(a, m0, t0, wave, lane, acc);
}

__device__ __forceinline__ void copy_to_lds(const char *src, char *lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                     (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}
// All but this wave's last `LEFT` copies have landed, its LDS reads are done, and so are every other wave's.
// (Counted: between copies and this there is no other access of a wave to memory, a spilled register's included.)
template <int LEFT>
__device__ __forceinline__ void stage_ready() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// A lane's sums of TM rows of blocks, four 16-column blocks each (from a multiple of 64 on), to y.
template <class T, class O, int TM>
__device__ __forceinline__ void finish_rows(const LinearArgs &a, int row0, int tile, int g, const Sums<T> (&acc)[TM][4]) {
    constexpr int C = kRunCols<T>, Q = 16 / C; // Q runs of C columns
    typedef Columns<O, C> Col;
    constexpr int R = TM < 4 ? TM : 4; // rows whose residuals travel at a time
    static_assert(TM % R == 0, "");
    const int col = first_col<T>(tile, g); // run q: 4 C q behind it
    if (col >= a.n) return;
    typename Col::Run bias[Q];
    if (a.bias) {
#pragma unroll
        for (int q = 0; q < Q; ++q) bias[q] = Col::load((const O *)a.bias + col + q * 4 * C, a.n - col - q * 4 * C, false);
    }
    float sw[Q][C];
    if constexpr (sizeof(T) == 1) {
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
            for (int c = 0; c < C; ++c) sw[q][c] = col + q * 4 * C + c < a.n ? a.sw[col + q * 4 * C + c] : 0.f;
    }
    with_act(a.act, [&](auto act) {
#pragma unroll
        for (int i0 = 0; i0 < TM; i0 += R) {
            const int row = row0 + 16 * i0;
            typename Col::Run res[R][Q];
            if (a.res) {
#pragma unroll
                for (int i = 0; i < R; ++i)
                    if (row + 16 * i < a.m)
#pragma unroll
                        for (int q = 0; q < Q; ++q)
                            res[i][q] = Col::load((const O *)a.res + (int64_t)(row + 16 * i) * a.ldres + col + q * 4 * C,
                                                  a.n - col - q * 4 * C, a.vec);
            }
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (row + 16 * i >= a.m) continue;
                float sx = 0.f;
                if constexpr (sizeof(T) == 1) sx = a.sx[row + 16 * i];
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    typename Col::Sum v;
#pragma unroll
                    for (int c = 0; c < C; ++c) {
                        if constexpr (sizeof(T) == 1) v[c] = (float)acc[i0 + i][q * (C / 4) + c / 4][c % 4] * sw[q][c] * sx;
                        else v[c] = acc[i0 + i][q * (C / 4) + c / 4][c % 4];
                        if (a.bias) v[c] += (float)bias[q][c];
                        if (a.res) v[c] += (float)res[i][q][c];
                    }
                    Col::template store<decltype(act)::value>((O *)a.y + (int64_t)(row + 16 * i) * a.ldy + col + q * 4 * C,
                                                              a.n - col - q * 4 * C, a.vec, v);
                }
            }
        }
    });
}

// BM x BN of y per workgroup of WVM x WVN waves, wave tiles 64 columns wide. LDS holds WF fragments of w along K
// and WF / 2 + 1 granules of x: while fragment f is computed, the reads of f + 1 go to registers (x's
// as each is used up), and f + 2 .. f + WF are on their way from memory. One barrier per fragment.
// `splits` > 1: a workgroup takes its share of K and leaves its sums in part[split][tile][block][lane].
constexpr int tile_lds(int BM, int BN, int WF) { return (WF / 2 + 1) * (BM / 16) * kGranule + WF * (BN / 16) * kFragBytes; }
template <class T, class O, int BM, int BN, int WVM, int WVN, int WF, bool XP>
__global__ __launch_bounds__(64 * WVM * WVN, WVM * WVN == 8 || 2 * tile_lds(BM, BN, WF) <= 160 * 1024 ? 2 : 1) void linear_tile_kernel(LinearArgs a, int mblocks, int nblocks, int splits,
                                                                     Sums<T> *part) {
    constexpr int E = 16 / (int)sizeof(T);
    constexpr int NW = WVM * WVN;
    constexpr int TM = BM / WVM / 16, TN = BN / WVN / 16;   // a wave's blocks
    constexpr int PX = BM / 16 * 2 / NW, PW = BN / 16 / NW; // a wave's 1 KB copies of a granule and of a fragment
    static_assert(BM / 16 * 2 % NW == 0 && BN / 16 % NW == 0 && TN == 4 && (WF & (WF - 1)) == 0, "");
    constexpr int GX = WF / 2 + 1;
    constexpr int kX = BM / 16 * kGranule, kW = BN / 16 * kFragBytes;
    __shared__ __attribute__((aligned(16))) char lds[tile_lds(BM, BN, WF)];
    char *const ldw = lds + GX * kX;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // workgroup b runs on XCD b % 8: an XCD takes neighbouring tiles, columns of 4 tiles high, so that
    // its CUs share rows of x and of w in its L2
    int bm, bn, split, id;
    {
        const int tiles = mblocks * nblocks, total = tiles * splits, q = total / 8, r = total % 8, x = blockIdx.x % 8;
        id = x * q + min(x, r) + (int)blockIdx.x / 8;
        split = id / tiles;
        id -= split * tiles;
        constexpr int G = 4;
        const int group = id / (G * nblocks), high = min(G, mblocks - group * G);
        const int in = id - group * G * nblocks;
        bm = group * G + in % high;
        bn = in / high;
    }
    const int mt0 = bm * (BM / 16), nt0 = bn * (BN / 16);
    // this split's granules along K
    const int g0 = (int)((int64_t)(a.kf / 2) * split / splits), g1 = (int)((int64_t)(a.kf / 2) * (split + 1) / splits);
    const int kf = 2 * (g1 - g0); // at least 2

    // copy p of a granule: eight rows, lane l run l % 8 of row l / 8 as it lies in LDS
    const char *xs[PX];
    int run[PX]; // first k of the lane's run in granule 0
#pragma unroll
    for (int p = 0; p < PX; ++p) {
        const int c = wave * PX + p, r = (c & 1) * 8 + (lane >> 3);
        run[p] = g0 * 2 * kFrag<T> + ((lane & 7) ^ (r >> 1)) * E;
        if constexpr (XP) {
            const int mt = min(mt0 + (c >> 1), (a.m - 1) >> 4);
            xs[p] = (const char *)a.x + ((int64_t)mt * a.kf + 2 * g0) * kFragBytes + (c & 1) * kFragBytes + lane * 16;
        } else {
            const int row = min((mt0 + (c >> 1)) * 16 + r, a.m - 1);
            xs[p] = (const char *)((const T *)a.x + (int64_t)row * a.ldx + run[p]);
        }
    }
    const char *ws[PW];
#pragma unroll
    for (int p = 0; p < PW; ++p) {
        const int nt = min(nt0 + wave * PW + p, a.ntiles - 1);
        ws[p] = a.w + ((int64_t)nt * a.kf + 2 * g0) * kFragBytes + lane * 16;
    }
    const char *zeros = a.w + (int64_t)a.ntiles * a.kf * kFragBytes;
    auto fetch_x = [&](int g, int place, bool whole) { // granule g of the split's; whole: it does not pass the rows' end
        char *to = lds + place * kX + wave * PX * kFragBytes;
        if (XP || whole || (g0 + g + 1) * 2 * kFrag<T> <= a.k) {
#pragma unroll
            for (int p = 0; p < PX; ++p) copy_to_lds(xs[p] + (int64_t)g * (XP ? kGranule : 128), to + p * kFragBytes);
        } else { // the runs behind a row's end come from the packed weights' zeros
#pragma unroll
            for (int p = 0; p < PX; ++p)
                copy_to_lds(g * 2 * kFrag<T> + run[p] < a.k ? xs[p] + (int64_t)g * 128 : zeros, to + p * kFragBytes);
        }
    };
    auto fetch_w = [&](int f) {
        char *to = ldw + (f & (WF - 1)) * kW + wave * PW * kFragBytes;
#pragma unroll
        for (int p = 0; p < PW; ++p) copy_to_lds(ws[p] + (int64_t)f * kFragBytes, to + p * kFragBytes);
    };

    const int wm = wave % WVM, wn = wave / WVM;
    const char *const lx[2] = {lds + wm * TM * kGranule + granule_at(lane, 0), lds + wm * TM * kGranule + granule_at(lane, 1)};
    const char *const lw = ldw + wn * TN * kFragBytes + lane * 16;
    auto read = [&](const char *p) { return *reinterpret_cast<const u32x4 *>(p); };
    Sums<T> acc[TM][TN] = {};
    u32x4 x[TM], w[2][TN];

    // In the order of the steps before the first: x of a granule, then w, every odd step a granule.
    fetch_x(0, 0, false);
#pragma unroll
    for (int s = 0; s < WF; ++s) {
        if (s % 2 && s + 1 < kf) fetch_x((s + 1) / 2, (s + 1) / 2, false);
        if (s < kf) fetch_w(s);
    }
    if (kf > WF) stage_ready<WF / 2 * PX + (WF - 1) * PW>();
    else stage_ready<0>();
#pragma unroll
    for (int j = 0; j < TN; ++j) w[0][j] = read(lw + j * kFragBytes);
#pragma unroll
    for (int i = 0; i < TM; ++i) x[i] = read(lx[0] + i * kGranule);
    // One fragment f, half = f % 2. x's granule is in place `here`, the one after it in `next`; every wave has read fragment
    // f, so its place takes f + WF, and an odd one's granule the GX-th after it.
    // steady: all that a step asks for is there, and not the last granule (no branches in the loop)
    auto step = [&](int f, auto half_, auto steady_, int here, int next) {
        constexpr int half = decltype(half_)::value;
        constexpr bool steady = decltype(steady_)::value;
        const bool more = steady || f + 1 < kf;
        // copies since fragment f + 1 was asked for: w of f + 2 .. f + WF - 1, and a granule for every two
        if (steady || f + WF < kf) stage_ready<(WF - 2) / 2 * PX + (WF - 2) * PW>();
        else if (more) stage_ready<0>();
        if (half && (steady || f + WF + 1 < kf)) fetch_x(f / 2 + GX, here, steady);
        if (steady || f + WF < kf) fetch_w(f + WF);
        const char *px = half ? lx[0] + next * kX : lx[1] + here * kX;
        if (more) {
            const char *pw = lw + ((f + 1) & (WF - 1)) * kW;
#pragma unroll
            for (int j = 0; j < TN; ++j) w[!half][j] = read(pw + j * kFragBytes);
        }
        if constexpr (sizeof(T) == 4) { // neighbouring instructions on different accumulators
            constexpr int I = 2;
#pragma unroll
            for (int i0 = 0; i0 < TM; i0 += I) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = i0; i < i0 + I; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j)
                            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                                __builtin_bit_cast(float, (uint32_t)w[half][j][e]),
                                __builtin_bit_cast(float, (uint32_t)x[i][e]), acc[i][j], 0, 0, 0);
                if (more) {
#pragma unroll
                    for (int i = i0; i < i0 + I; ++i) x[i] = read(px + i * kGranule);
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < TM; ++i) {
#pragma unroll
                for (int j = 0; j < TN; ++j) mfma_frag(acc[i][j], w[half][j], x[i], T());
                if (more) x[i] = read(px + i * kGranule);
            }
        }
    };
    int f = 0, here = 0;
    auto pair = [&](auto steady) {
        const int next = here == GX - 1 ? 0 : here + 1;
        step(f, std::integral_constant<int, 0>(), steady, here, next);
        step(f + 1, std::integral_constant<int, 1>(), steady, here, next);
        here = next;
        f += 2;
    };
    while (f + WF + 4 < kf) pair(std::true_type());
    while (f < kf) pair(std::false_type());
    if (splits > 1) {
        Sums<T> *to = part + (((int64_t)split * mblocks * nblocks + id) * NW + wave) * (TM * TN) * 64 + lane;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j) to[(i * TN + j) * 64] = acc[i][j];
        return;
    }
    finish_rows<T, O, TM>(a, (mt0 + wm * TM) * 16 + (lane & 15), nt0 + wn * TN, lane >> 4, acc);
}

// The splits' sums of one row of blocks of a wave's tile, added in split order. One wave each.
template <class T, class O, int BM, int BN, int WVM, int WVN>
__global__ __launch_bounds__(256) void linear_join_kernel(LinearArgs a, int mblocks, int nblocks, int splits,
                                                          const Sums<T> *part) {
    constexpr int NW = WVM * WVN, TM = BM / WVM / 16;
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); // (tile, wave, block row)
    const int64_t tiles = (int64_t)mblocks * nblocks;
    if (unit >= tiles * NW * TM) return;
    const int id = (int)(unit / (NW * TM)), wave = (int)(unit / TM % NW), i = (int)(unit % TM);
    constexpr int G = 4;
    const int group = id / (G * nblocks), high = min(G, mblocks - group * G), in = id - group * G * nblocks;
    const int bm = group * G + in % high, bn = in / high;
    Sums<T> acc[1][4] = {};
    const Sums<T> *from = part + unit * 4 * 64 + lane;
#pragma unroll 4
    for (int s = 0; s < splits; ++s)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[0][j] += from[(s * tiles * NW * TM * 4 + j) * 64];
    finish_rows<T, O, 1>(a, (bm * (BM / 16) + wave % WVM * TM + i) * 16 + (lane & 15),
                      bn * (BN / 16) + wave / WVM * 4, lane >> 4, acc);
}

// One thread per 16 bytes of the packed weights, and of a fragment of zeros behind them.
template <class T>
__global__ __launch_bounds__(256) void linear_pack_kernel(const T *__restrict__ w, u32x4 *__restrict__ out, int n, int k,
                                                          int trans_w, int64_t kf, int64_t total) {
    constexpr int E = 16 / (int)sizeof(T);
    typedef typename Bits<T>::type B;
    const B *wb = reinterpret_cast<const B *>(w);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total + 64; i += (int64_t)gridDim.x * 256) {
        const int lane = (int)(i & 63);
        const int64_t frag = i >> 6;
        const int64_t tile = frag / kf, f = frag - tile * kf;
        const int r = lane & 15;
        const int64_t col = (tile >> 2) * 64 + first_col<T>((int)(tile & 3), r >> 2) + (r & 3);
        const int64_t k0 = f * kFrag<T> + (lane >> 4) * E;
        u32x4 v = {0, 0, 0, 0};
        if (i < total && col < n) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (k0 + e < k) {
                    const uint32_t b = trans_w ? wb[col * k + k0 + e] : wb[(k0 + e) * n + col];
                    if constexpr (E == 4) v[e] = b;
                    else if constexpr (E == 8) v[e / 2] |= b << (16 * (e % 2));
                    else v[e / 4] |= b << (8 * (e % 4));
                }
        }
        out[i] = v;
    }
}

template <class T, class O, int MT, int NT, int NW>
int launch_stream(const LinearArgs &a, Rows rows, hipStream_t st) {
    const dim3 grid((a.ntiles + NT - 1) / NT, (a.m + 16 * MT - 1) / (16 * MT));
    if (!launch_fits(grid.x, 64 * NW) || grid.y > 65535) return SPINN_HIP_EUNSUPPORTED;
    if (rows == kRuns) linear_stream_kernel<T, O, MT, NT, NW, kRuns><<<grid, 64 * NW, 0, st>>>(a);
    else if (rows == kLaidOut) linear_stream_kernel<T, O, MT, NT, NW, kLaidOut><<<grid, 64 * NW, 0, st>>>(a);
    else if (rows == kLoose) linear_stream_kernel<T, O, MT, NT, NW, kLoose><<<grid, 64 * NW, 0, st>>>(a);
    else linear_stream_kernel<T, O, MT, NT, NW, kShort><<<grid, 64 * NW, 0, st>>>(a);
    return check_launch();
}

template <class T, class O, int BM, int BN, int WVM, int WVN, int WF>
int launch_tile(const LinearArgs &a, bool xp, int splits, void *part, hipStream_t st) {
    const int mb = (a.m + BM - 1) / BM, nb = (a.ntiles * 16 + BN - 1) / BN;
    if (!launch_fits((int64_t)mb * nb * splits, 64 * WVM * WVN)) return SPINN_HIP_EUNSUPPORTED;
    const unsigned grid = (unsigned)(mb * nb * splits);
    bool laid_out = false;
    if constexpr (sizeof(T) > 1) { // rows of 8-bit integers are whole runs
        laid_out = xp;
        if (xp) linear_tile_kernel<T, O, BM, BN, WVM, WVN, WF, true><<<grid, 64 * WVM * WVN, 0, st>>>(a, mb, nb, splits, (Sums<T> *)part);
    }
    if (!laid_out) linear_tile_kernel<T, O, BM, BN, WVM, WVN, WF, false><<<grid, 64 * WVM * WVN, 0, st>>>(a, mb, nb, splits, (Sums<T> *)part);
    if (splits > 1)
        linear_join_kernel<T, O, BM, BN, WVM, WVN><<<(unsigned)(((int64_t)mb * nb * (BM * BN / 1024) + 3) / 4), 256, 0, st>>>(
            a, mb, nb, splits, (const Sums<T> *)part);
    return check_launch();
}

// Which kernel a layer runs on.
struct Choice {
    enum { kStream, kTile64, kTile128, kTile256 } kind;
    int mt, nt;  // kStream: blocks of 16 rows and columns per workgroup
    int splits;  // kTile64: along K
};
// From measurements over m = 1..4096, n, k = 64..16384 (fp32 and bf16; us at k = 4096 unless stated):
//  * up to 64 rows, and grids too short to fill the device at a short K: the stream kernel, on the largest blocks that
//    still leave a workgroup per CU (64 x 4096: 2 x 2 blocks 11.7, 4 x 2 18.8, 1 x 2 14.0; 64 x 16384: 4 x 4
//    36, 2 x 2 53; 512 x 1024 at k = 1024: 7.1 against 11.1 and more on tiles); up to 16 rows 1 x 1 with 16 waves
//    (1 x 4096 7.1, 1 x 2 blocks 8.7);
//  * 256 x 256 tiles from one per CU (4096 x 4096: 124; 2048 x 4096, half as many: 92 against 75 on 128 x 128);
//  * 128 x 128 from more than one per CU (2048 x 4096: 75 against 97 on 64 x 128; 1024 x 4096, exactly one: 51 against 46);
//  * 64 x 128 otherwise, K split where that leaves CUs idle (256 x 4096: 29 whole, 22 in two; 128 x 4096: 28, 16 in
//    four; 200 x 1024 at k = 16384: 92, 23 in eight), parts of at least 16 fragments.
inline Choice choose(int64_t mt, int64_t nt, int64_t kf) { // tiles of 16 rows and columns, fragments
    const int64_t cus = device_cu_count();
    auto grid = [&](int64_t rows, int64_t cols) { return ((mt + rows - 1) / rows) * ((nt + cols - 1) / cols); };
    Choice c{Choice::kStream, 1, 1, 1};
    if (mt <= 1) return c;
    const int64_t tiles = grid(4, 8);
    if (mt <= 4 || (tiles < cus && kf < 64)) {
        static const int blocks[][2] = {{4, 4}, {4, 2}, {2, 4}, {2, 2}, {1, 2}};
        for (auto &b : blocks)
            if ((b[0] <= mt || b[0] < 2 * mt) && grid(b[0], b[1]) >= cus) {
                c.mt = b[0];
                c.nt = b[1];
                return c;
            }
        return c;
    }
    if (grid(16, 16) >= cus) c.kind = Choice::kTile256;
    else if (grid(8, 8) > cus) c.kind = Choice::kTile128;
    else {
        c.kind = Choice::kTile64;
        c.splits = (int)std::max<int64_t>(1, std::min(cus / tiles, kf / 16));
    }
    return c;
}

// A layer on tiles. part: the splits' sums.
template <class T, class O>
int launch_tiles(const LinearArgs &a, const Choice &c, bool xp, void *part, hipStream_t st) {
    const int64_t tiles = (((int64_t)(a.m + 15) / 16 + 3) / 4) * ((a.ntiles + 7) / 8);
    const bool deep = tiles * c.splits <= device_cu_count();
    if (c.kind == Choice::kTile256) return launch_tile<T, O, 256, 256, 2, 4, 4>(a, xp, 1, nullptr, st);
    if (c.kind == Choice::kTile128) return launch_tile<T, O, 128, 128, 2, 2, 4>(a, xp, 1, nullptr, st);
    // one workgroup per CU can have all of its LDS
    if (deep) return launch_tile<T, O, 64, 128, 2, 2, 8>(a, xp, c.splits, part, st);
    return launch_tile<T, O, 64, 128, 2, 2, 4>(a, xp, c.splits, part, st);
}

// The kernel of `c` for a layer.
template <class T, class O>
int launch_linear(const LinearArgs &a, const Choice &c, Rows rows, void *part, hipStream_t st) {
    if (c.kind != Choice::kStream) return launch_tiles<T, O>(a, c, rows == kLaidOut, part, st);
    if (c.mt == 4 && c.nt == 4) return launch_stream<T, O, 4, 4, 4>(a, rows, st);
    if (c.mt == 4) return launch_stream<T, O, 4, 2, 8>(a, rows, st);
    if (c.mt == 2 && c.nt == 4) return launch_stream<T, O, 2, 4, 4>(a, rows, st);
    if (c.mt == 2) return launch_stream<T, O, 2, 2, 8>(a, rows, st);
    if (c.nt == 2) return launch_stream<T, O, 1, 2, 8>(a, rows, st);
    return launch_stream<T, O, 1, 1, 16>(a, rows, st);
}

} // namespace
} // namespace spinn
