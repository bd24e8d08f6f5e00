// linear.hip - linear layers: y = act(x w^T + bias + residual) in fp32, fp16 and bf16.
//
// Weights are packed once into MFMA operand fragments, [N/16][K/kFrag][64 lanes][16 bytes] with
// zeros around, so that a wave reads 1 KB of them with one load and feeds a matrix instruction
// as they come. The weights are the A operand (its rows are the accumulators' rows), x is the
// B operand; tile t of four holds columns 64 G + 16 g + 4 t + i, g = l/16, so that a lane's
// accumulators over the four tiles are 16 neighbouring columns of one row of y.
//
//  * few rows (single tokens): the weights are read once and bound it. linear_stream_kernel: tiles of
//    16 MT x 16 NT, K spread over a workgroup's waves, operands straight from memory into
//    registers, the waves' sums joined in LDS in wave order.
//  * many rows: the matrix cores bound it. linear_tile_kernel: both operands through LDS, whole
//    fragments copied there without passing registers, two stages.
#include "decode.h"

namespace spinn {
namespace {

constexpr int kFragBytes = 1024;

inline int64_t frags(const SpinnHipLinearDesc *d) { // along K, an even number
    const int f = 64 / dtype_bytes(d->dtype);
    return ((int64_t)d->k + 2 * f - 1) / (2 * f) * 2;
}
inline int64_t n_tiles(const SpinnHipLinearDesc *d) { return ((int64_t)d->n + 63) / 64 * 4; }
inline int64_t m_tiles(const SpinnHipLinearDesc *d) { return ((int64_t)d->m + 15) / 16; }
// x's rows are not whole 16-byte runs: they are laid out as fragments first
inline bool x_loose(const SpinnHipLinearDesc *d) {
    const int e = 16 / dtype_bytes(d->dtype);
    return d->x_unaligned || d->ldx % e || d->k % e;
}

__device__ __forceinline__ float gelu_erf(float v) { return 0.5f * v * (1.f + erff(v * 0.70710678118654752f)); }
// v/2 (1 + tanh u) = v / (1 + exp(-2u))
__device__ __forceinline__ float gelu_tanh(float v) {
    const float u = 0.7978845608028654f * (v + 0.044715f * v * v * v);
    return v * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(u * (-2.f * 1.4426950408889634f)));
}
__device__ __forceinline__ float linear_act(float v, int act) {
    switch (act) {
    case SPINN_LINEAR_RELU: return v < 0.f ? 0.f : v;
    case SPINN_LINEAR_SILU: return silu(v);
    case SPINN_LINEAR_GELU: return gelu_erf(v);
    case SPINN_LINEAR_GELU_TANH: return gelu_tanh(v);
    default: return v;
    }
}

struct LinearArgs {
    const void *x, *bias, *res; // x: rows, or fragments [M/16][frags]
    const char *w;              // packed
    void *y;
    int64_t ldx, ldres, ldy;
    int32_t m, n, k, act;
    int32_t kf;      // fragments along K
    int32_t ntiles;  // of 16 columns
    int32_t vec;     // residual and y are read and written in runs of 4
};

// Four neighbouring columns n.. of a row.
template <class T>
__device__ __forceinline__ void finish4(const LinearArgs &a, int row, int n, f32x4 v) {
    if (row >= a.m || n >= a.n) return;
    typedef T T4 __attribute__((ext_vector_type(4)));
    const int64_t ry = (int64_t)row * a.ldy + n, rr = (int64_t)row * a.ldres + n;
    if (a.vec && n + 3 < a.n) {
        if (a.bias) {
            const T *b = (const T *)a.bias + n;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += (float)b[i];
        }
        if (a.res) {
            const T4 r = *reinterpret_cast<const T4 *>((const T *)a.res + rr);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] += (float)r[i];
        }
        T4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = (T)linear_act(v[i], a.act);
        *reinterpret_cast<T4 *>((T *)a.y + ry) = o;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < a.n) {
                float s = v[i];
                if (a.bias) s += (float)((const T *)a.bias)[n + i];
                if (a.res) s += (float)((const T *)a.res)[rr + i];
                ((T *)a.y)[ry + i] = (T)linear_act(s, a.act);
            }
    }
}

// First column of the four that accumulator block `tile` of a lane with l/16 = g holds.
__device__ __forceinline__ int first_col(int tile, int g) { return (tile >> 2) * 64 + 16 * g + 4 * (tile & 3); }

// XP: x is laid out as fragments.
template <class T, int MT, int NT, int NW, bool XP>
__global__ __launch_bounds__(64 * NW) void linear_stream_kernel(LinearArgs a) {
    constexpr int E = 16 / (int)sizeof(T);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t0 = blockIdx.x * NT, m0 = blockIdx.y * MT;
    const char *wp[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
        wp[j] = a.w + (int64_t)min(t0 + j, a.ntiles - 1) * a.kf * kFragBytes + lane * 16;
    const char *xp[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        if constexpr (XP) {
            const int mt = min(m0 + i, (a.m - 1) >> 4);
            xp[i] = (const char *)a.x + (int64_t)mt * a.kf * kFragBytes + lane * 16;
        } else {
            const int row = min((m0 + i) * 16 + (lane & 15), a.m - 1);
            xp[i] = (const char *)((const T *)a.x + (int64_t)row * a.ldx + (lane >> 4) * E);
        }
    }
    f32x4 acc[MT][NT] = {};
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
                if constexpr (XP) x[u][i] = *reinterpret_cast<const u32x4 *>(xp[i] + (int64_t)f * kFragBytes);
                else {
                    const bool in = f * kFrag<T> + (lane >> 4) * E < a.k;
                    x[u][i] = in ? *reinterpret_cast<const u32x4 *>(xp[i] + (int64_t)f * 64) : (u32x4){0, 0, 0, 0};
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
    __shared__ f32x4 part[NW][MT * NT][64];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) part[wave][i * NT + j][lane] = acc[i][j];
    __syncthreads();
    for (int b = wave; b < MT * NT; b += NW) {
        f32x4 v = part[0][b][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += part[w][b][lane];
        const int i = b / NT, j = b % NT;
        if (t0 + j < a.ntiles) finish4<T>(a, (m0 + i) * 16 + (lane & 15), first_col(t0 + j, lane >> 4), v);
    }
}

__device__ __forceinline__ void copy_to_lds(const char *src, char *lds) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)src,
                                     (__attribute__((address_space(3))) void *)lds, 16, 0, 0);
}

// BM x BN of y per workgroup of WVM x WVN waves.
template <class T, int BM, int BN, int WVM, int WVN, bool XP>
__global__ __launch_bounds__(64 * WVM * WVN) void linear_tile_kernel(LinearArgs a, int mblocks) {
    constexpr int E = 16 / (int)sizeof(T);
    constexpr int NW = WVM * WVN;
    constexpr int TM = BM / WVM / 16, TN = BN / WVN / 16; // a wave's blocks
    constexpr int S = 2;                                  // fragments along K per stage
    constexpr int FX = BM / 16 * S, FW = BN / 16 * S;     // fragments of a stage
    constexpr int PW = (FX + FW) / NW;                    // a wave's share of the copies
    static_assert((FX + FW) % NW == 0 && FX % PW == 0, "a wave copies fragments of one operand");
    __shared__ __attribute__((aligned(16))) char lds[2][(FX + FW) * kFragBytes];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int bm = blockIdx.x % mblocks, bn = blockIdx.x / mblocks;
    const int mt0 = bm * (BM / 16), nt0 = bn * (BN / 16);

    // fragment c of a stage: x's first, [tile][s]
    const char *src[PW];
    const bool wx = wave * PW < FX;
#pragma unroll
    for (int p = 0; p < PW; ++p) {
        const int c = wave * PW + p;
        if (wx) {
            if constexpr (XP) {
                const int mt = min(mt0 + c / S, (a.m - 1) >> 4);
                src[p] = (const char *)a.x + ((int64_t)mt * a.kf + c % S) * kFragBytes + lane * 16;
            } else {
                const int row = min((mt0 + c / S) * 16 + (lane & 15), a.m - 1);
                src[p] = (const char *)((const T *)a.x + (int64_t)row * a.ldx + (c % S) * kFrag<T> + (lane >> 4) * E);
            }
        } else {
            const int nt = min(nt0 + (c - FX) / S, a.ntiles - 1);
            src[p] = a.w + ((int64_t)nt * a.kf + (c - FX) % S) * kFragBytes + lane * 16;
        }
    }
    const char *zeros = a.w + (int64_t)a.ntiles * a.kf * kFragBytes;
    auto fetch = [&](int f, int buf) {
#pragma unroll
        for (int p = 0; p < PW; ++p) {
            const int c = wave * PW + p;
            const char *s;
            if (wx && !XP) {
                // runs behind a row's end come from the packed weights' zeros
                const bool in = (f + c % S) * kFrag<T> + (lane >> 4) * E < a.k;
                s = in ? src[p] + (int64_t)f * 64 : zeros;
            } else {
                s = src[p] + (int64_t)f * kFragBytes;
            }
            copy_to_lds(s, lds[buf] + c * kFragBytes);
        }
    };

    const int wm = wave % WVM, wn = wave / WVM;
    f32x4 acc[TM][TN] = {};
    fetch(0, 0);
    for (int f = 0, buf = 0; f < a.kf; f += S, buf ^= 1) {
        __builtin_amdgcn_s_waitcnt(0x0f70); // vmcnt(0): this wave's copies have landed
        __syncthreads();                    // everyone's have, and the other buffer has been read
        if (f + S < a.kf) fetch(f + S, buf ^ 1);
        const char *lx = lds[buf] + (wm * TM * S) * kFragBytes + lane * 16;
        const char *lw = lds[buf] + (FX + wn * TN * S) * kFragBytes + lane * 16;
#pragma unroll
        for (int s = 0; s < S; ++s) {
            u32x4 x[TM], w[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) w[j] = *reinterpret_cast<const u32x4 *>(lw + (j * S + s) * kFragBytes);
#pragma unroll
            for (int i = 0; i < TM; ++i) x[i] = *reinterpret_cast<const u32x4 *>(lx + (i * S + s) * kFragBytes);
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) mfma_frag(acc[i][j], w[j], x[i], T());
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int tile = nt0 + wn * TN + j;
            if (tile < a.ntiles)
                finish4<T>(a, (mt0 + wm * TM + i) * 16 + (lane & 15), first_col(tile, lane >> 4), acc[i][j]);
        }
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
        const int64_t col = (tile >> 2) * 64 + 16 * (r >> 2) + 4 * (tile & 3) + (r & 3);
        const int64_t k0 = f * kFrag<T> + (lane >> 4) * E;
        u32x4 v = {0, 0, 0, 0};
        if (i < total && col < n) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (k0 + e < k) {
                    const uint32_t b = trans_w ? wb[col * k + k0 + e] : wb[(k0 + e) * n + col];
                    if constexpr (E == 4) v[e] = b;
                    else v[e / 2] |= b << (16 * (e % 2));
                }
        }
        out[i] = v;
    }
}

// x as fragments [M/16][kf][64][16 bytes], zeros behind its rows and columns.
template <class T>
__global__ __launch_bounds__(256) void linear_pack_x_kernel(const T *__restrict__ x, u32x4 *__restrict__ out, int m, int k,
                                                            int64_t ldx, int64_t kf, int64_t total) {
    constexpr int E = 16 / (int)sizeof(T);
    typedef typename Bits<T>::type B;
    const B *xb = reinterpret_cast<const B *>(x);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int lane = (int)(i & 63);
        const int64_t frag = i >> 6;
        const int64_t tile = frag / kf, f = frag - tile * kf;
        const int64_t row = tile * 16 + (lane & 15), k0 = f * kFrag<T> + (lane >> 4) * E;
        u32x4 v = {0, 0, 0, 0};
        if (row < m) {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (k0 + e < k) {
                    const uint32_t b = xb[row * ldx + k0 + e];
                    if constexpr (E == 4) v[e] = b;
                    else v[e / 2] |= b << (16 * (e % 2));
                }
        }
        out[i] = v;
    }
}

template <class T, int MT, int NT, int NW>
void launch_stream(const LinearArgs &a, bool xp, hipStream_t st) {
    const dim3 grid((a.ntiles + NT - 1) / NT, (a.m + 16 * MT - 1) / (16 * MT));
    if (xp) linear_stream_kernel<T, MT, NT, NW, true><<<grid, 64 * NW, 0, st>>>(a);
    else linear_stream_kernel<T, MT, NT, NW, false><<<grid, 64 * NW, 0, st>>>(a);
}

template <class T, int BM, int BN, int WVM, int WVN>
void launch_tile(const LinearArgs &a, bool xp, hipStream_t st) {
    const int mb = (a.m + BM - 1) / BM, nb = (a.ntiles * 16 + BN - 1) / BN;
    if (xp) linear_tile_kernel<T, BM, BN, WVM, WVN, true><<<mb * nb, 64 * WVM * WVN, 0, st>>>(a, mb);
    else linear_tile_kernel<T, BM, BN, WVM, WVN, false><<<mb * nb, 64 * WVM * WVN, 0, st>>>(a, mb);
}

} // namespace

size_t linear_packed_bytes(const SpinnHipLinearDesc *d) {
    return (size_t)(n_tiles(d) * frags(d) + 1) * kFragBytes;
}

size_t linear_workspace_bytes(const SpinnHipLinearDesc *d) {
    return x_loose(d) ? (size_t)(m_tiles(d) * frags(d)) * kFragBytes : 0;
}

int linear_pack(const SpinnHipLinearDesc *d, const void *w, void *packed, hipStream_t st) {
    const int64_t total = n_tiles(d) * frags(d) * 64;
    const unsigned grid = (unsigned)std::min<int64_t>((total + 64 + 255) / 256, 65536);
    return with_dtype(d->dtype, [&](auto t) {
        typedef decltype(t) T;
        linear_pack_kernel<T><<<grid, 256, 0, st>>>((const T *)w, (u32x4 *)packed, d->n, d->k, d->trans_w, frags(d), total);
        return check_launch();
    });
}

int linear_run(const SpinnHipLinearDesc *d, const void *x, const void *packed, const void *bias, const void *res,
               void *y, void *ws, hipStream_t st) {
    LinearArgs a{};
    a.x = x;
    a.bias = bias;
    a.res = res;
    a.w = (const char *)packed;
    a.y = y;
    a.ldx = d->ldx;
    a.ldres = d->ldres;
    a.ldy = d->ldy;
    a.m = d->m;
    a.n = d->n;
    a.k = d->k;
    a.act = d->act;
    a.kf = (int32_t)frags(d);
    a.ntiles = (int32_t)n_tiles(d);
    const size_t run = 4 * (size_t)dtype_bytes(d->dtype);
    a.vec = (uintptr_t)y % run == 0 && d->ldy % 4 == 0 && (!res || ((uintptr_t)res % run == 0 && d->ldres % 4 == 0));
    const bool xp = x_loose(d);
    const int64_t wgs = (int64_t)((d->m + 63) / 64) * (a.ntiles / 4);
    if (wgs > INT32_MAX / 4 || (d->m + 15) / 16 > 65535 * 4) return SPINN_HIP_EUNSUPPORTED;
    return with_dtype(d->dtype, [&](auto t) {
        typedef decltype(t) T;
        if (xp) {
            const int64_t total = m_tiles(d) * a.kf * 64;
            linear_pack_x_kernel<T><<<(unsigned)std::min<int64_t>((total + 255) / 256, 65536), 256, 0, st>>>(
                (const T *)x, (u32x4 *)ws, d->m, d->k, d->ldx, a.kf, total);
            const int rc = check_launch();
            if (rc) return rc;
            a.x = ws;
        }
        const int cus = device_cu_count();
        const int64_t big = (int64_t)((d->m + 255) / 256) * ((a.ntiles + 15) / 16);
        const int64_t mid = (int64_t)((d->m + 127) / 128) * ((a.ntiles + 7) / 8);
        if (d->m <= 16) launch_stream<T, 1, 1, 8>(a, xp, st);
        else if (d->m <= 32) launch_stream<T, 2, 1, 8>(a, xp, st);
        else if (d->m <= 64) launch_stream<T, 4, 1, 8>(a, xp, st);
        else if (big >= cus) launch_tile<T, 256, 256, 2, 4>(a, xp, st);
        else if (mid >= cus / 2) launch_tile<T, 128, 128, 2, 2>(a, xp, st);
        else launch_stream<T, 4, 4, 4>(a, xp, st);
        return check_launch();
    });
}

} // namespace spinn
