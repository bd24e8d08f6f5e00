// linear_i8.hip - linear layers in 8-bit integers, and rows quantised for them.
//
// The layers run on the kernels of linear_core.h: a fragment of 64 k of 8-bit integers has the bytes of one of 32 k of a
// 16-bit type and its matrix instruction the same time, so that tiles, copies and waits are the same, with twice the
// products. Sums are exact 32-bit integers; the scales come in with the epilogue, in fp32.
//
// Many rows: the matrix cores bound it (4000 x 8192 x 4096: 131 to 144 us by the clock, up to 2050 TOP/s). Few rows have a stream kernel
// here, bound by what a CU takes in (1 x 8192 x 4096: 4.9 us, 6.8 TB/s, with the weights in caches; 45 x 5120 x 8192: 12.2).
#include "linear_core.h"

namespace spinn {
namespace {

constexpr int kUnit = 16; // elements that a lane quantises at a time

// Elements u kUnit.. of a row of k, in fp32, zeros behind its end.
template <class T>
__device__ __forceinline__ void load_unit(const T *row, int u, int k, float (&v)[kUnit]) {
    constexpr int E = 16 / (int)sizeof(T);
    typedef T Vec __attribute__((ext_vector_type(E)));
    typedef Vec Loose __attribute__((aligned(sizeof(T))));
    const int64_t at = (int64_t)u * kUnit;
    if (at + kUnit <= k) {
        Vec w[kUnit / E];
#pragma unroll
        for (int i = 0; i < kUnit / E; ++i) w[i] = *reinterpret_cast<const Loose *>(row + at + i * E);
#pragma unroll
        for (int i = 0; i < kUnit; ++i) v[i] = (float)w[i / E][i % E];
    } else {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) v[i] = at + i < k ? (float)row[at + i] : 0.f;
    }
}

// v / s to the nearest integer, ties to even, decided by the remainder of a first guess: the remainder is exact
// where it is near s / 2.
__device__ __forceinline__ int quantized(float v, float s, float inv) {
    float r = fminf(fmaxf(rintf(v * inv), -127.f), 127.f);
    const float d = fmaf(-r, s, v), far = fabsf(d), half = 0.5f * s;
    const int i = (int)r;
    return far > half || (far == half && (i & 1)) ? min(max(i + (d > 0.f ? 1 : -1), -127), 127) : i;
}

// The same where s has few bits or none above fp32's least number and a reciprocal would overflow.
__device__ __forceinline__ int quantized_tiny(float v, float s) {
    return s > 0.f ? (int)fmin(fmax(rint((double)v / (double)s), -127.0), 127.0) : 0;
}

// A row per NW waves, 4 / NW (at least one) rows a workgroup; a lane's first unit stays in registers between the two passes. Only rows of 16 waves have more.
// 1 x 4096 bf16 is one workgroup's latency (4 us); many rows are bound by memory (4000 x 4096: 9.4 us behind the launch before it, 5.2 TB/s).
// From 4097 elements on k / 16 of a row's 1024 lanes work, up to 16384 (launches in a row: 4000 x 4096 14.2 us, 3.5 TB/s; x 5120 27.8, 2.2; x 8192
// 29.9, 3.3; x 14336 44.0, 3.9).
template <class T, int NW>
__global__ __launch_bounds__(64 * (NW < 4 ? 4 : NW)) void quantize_rows_kernel(const T *__restrict__ x, int64_t ldx, int8_t *__restrict__ xq,
                                                                           int64_t ldq, float *__restrict__ scale, int64_t rows, int k) {
    constexpr int R = NW < 4 ? 4 / NW : 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * R + wave / NW;
    const int first = (wave % NW) * 64 + lane, units = (int)(((int64_t)k + kUnit - 1) / kUnit);
    const bool in = row < rows;
    const T *xr = x + (in ? row : 0) * ldx;
    float v[kUnit];
    uint32_t top = 0; // bits of the largest magnitude; infinities and NaN are above all numbers
    auto look = [&](const float (&w)[kUnit]) {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) top = max(top, __builtin_bit_cast(uint32_t, w[i]) & 0x7fffffffu);
    };
    if (in && first < units) {
        load_unit<T>(xr, first, k, v);
        look(v);
    }
    if (NW == 16 && in)
        for (int u = first + 64 * NW; u < units; u += 64 * NW) {
            float w[kUnit];
            load_unit<T>(xr, u, k, w);
            look(w);
        }
#pragma unroll
    for (int d = 32; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if constexpr (NW > 1) {
        __shared__ uint32_t tops[NW];
        if (lane == 0) tops[wave] = top;
        __syncthreads();
        top = tops[lane % NW];
#pragma unroll
        for (int d = NW / 2; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    }
    if (!in) return;
    const bool bad = top >= 0x7f800000u;
    const float most = __builtin_bit_cast(float, top);
    const float s = bad ? __builtin_bit_cast(float, 0x7fc00000u) : most / 127.f;
    const float inv = 1.f / s;
    if (first == 0) scale[row] = s;
    int8_t *out = xq + row * ldq;
    auto store = [&](int u, const float (&w)[kUnit]) {
        u32x4 b = {0, 0, 0, 0};
        if (top < 0x0d800000u) { // 2^-100
#pragma unroll
            for (int i = 0; i < kUnit; ++i) b[i / 4] |= (uint32_t)(uint8_t)quantized_tiny(w[i], s) << (8 * (i % 4));
        } else if (!bad) {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) b[i / 4] |= (uint32_t)(uint8_t)quantized(w[i], s, inv) << (8 * (i % 4));
        }
        *reinterpret_cast<u32x4 *>(out + (int64_t)u * kUnit) = b;
    };
    if (first < units) store(first, v);
    if (NW == 16)
        for (int u = first + 64 * NW; u < units; u += 64 * NW) {
            float w[kUnit];
            load_unit<T>(xr, u, k, w);
            store(u, w);
        }
}

template <class T, int NW>
int launch_quantize(int64_t rows, int k, const void *x, int64_t ldx, int8_t *xq, int64_t ldq, float *scale, hipStream_t st) {
    constexpr int R = NW < 4 ? 4 / NW : 1, threads = 64 * (NW < 4 ? 4 : NW);
    const int64_t grid = (rows + R - 1) / R;
    if (!launch_fits(grid, threads)) return SPINN_HIP_EUNSUPPORTED;
    quantize_rows_kernel<T, NW><<<(unsigned)grid, threads, 0, st>>>((const T *)x, ldx, xq, ldq, scale, rows, k);
    return check_launch();
}

// Few rows: as linear_stream_kernel, with the next U fragments of a wave on their way while U are multiplied. What bounds it is what a CU takes in,
// some 50 GB/s of weights and of rows (12.8 TB/s over all), whichever level of memory they come from: see choose().
template <class O, int MT, int NT, int NW, int U>
__global__ __launch_bounds__(64 * NW) void linear_i8_stream_kernel(LinearArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t0 = blockIdx.x * NT, m0 = blockIdx.y * MT;
    const char *wp[NT], *xp[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) wp[j] = a.w + (int64_t)min(t0 + j, a.ntiles - 1) * a.kf * kFragBytes + lane * 16;
#pragma unroll
    for (int i = 0; i < MT; ++i) xp[i] = (const char *)a.x + (int64_t)min((m0 + i) * 16 + (lane & 15), a.m - 1) * a.ldx;
    const int last = ((a.k + 15) & ~15) - 16; // what is behind a row meets zeros of w: any 16 bytes of it do
    Sums<int8_t> acc[MT][NT] = {};
    u32x4 w[2][U][NT], x[2][U][MT];
    // a wave takes fragments in pairs: 128 bytes, a cache line, of every row of x
    auto fragment = [](int u) { return u / 2 * 2 * NW + u % 2; };
    auto fetch = [&](int f0, u32x4 (&wb)[U][NT], u32x4 (&xb)[U][MT]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int f = f0 + fragment(u);
            if (f >= a.kf) break;
#pragma unroll
            for (int j = 0; j < NT; ++j) wb[u][j] = *reinterpret_cast<const u32x4 *>(wp[j] + (int64_t)f * kFragBytes);
            const int k0 = min(f * kFrag<int8_t> + (lane >> 4) * 16, last);
#pragma unroll
            for (int i = 0; i < MT; ++i) xb[u][i] = *reinterpret_cast<const u32x4 *>(xp[i] + k0);
        }
    };
    auto multiply = [&](int f0, const u32x4 (&wb)[U][NT], const u32x4 (&xb)[U][MT]) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (f0 + fragment(u) >= a.kf) break;
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) mfma_frag(acc[i][j], wb[u][j], xb[u][i], int8_t());
        }
    };
    constexpr int S = NW * U;
    fetch(2 * wave, w[0], x[0]);
    for (int f = 2 * wave; f < a.kf; f += 2 * S) {
        fetch(f + S, w[1], x[1]);
        multiply(f, w[0], x[0]);
        fetch(f + 2 * S, w[0], x[0]);
        multiply(f + S, w[1], x[1]);
    }
    join_waves<int8_t, O, MT, NT, NW>(a, m0, t0, wave, lane, acc);
}

template <class O, int MT, int NT, int NW, int U>
int launch_stream_i8(const LinearArgs &a, hipStream_t st) {
    const dim3 grid((a.ntiles + NT - 1) / NT, (a.m + 16 * MT - 1) / (16 * MT));
    if (!launch_fits(grid.x, 64 * NW) || grid.y > 65535) return SPINN_HIP_EUNSUPPORTED;
    linear_i8_stream_kernel<O, MT, NT, NW, U><<<grid, 64 * NW, 0, st>>>(a);
    return check_launch();
}

inline int64_t frags(const SpinnHipLinearI8Desc *d) { return ((int64_t)d->k + 127) / 128 * 2; }
inline int64_t n_tiles(const SpinnHipLinearI8Desc *d) { return ((int64_t)d->n + 63) / 64 * 4; }
inline int64_t m_tiles(const SpinnHipLinearI8Desc *d) { return ((int64_t)d->m + 15) / 16; }

// Which kernel a layer runs on, by its time as measured over m = 1..2000, n = 1024..14336, k = 1024..16384 (us; f fragments of 64 along K,
// 256 CUs, one workgroup of the stream kernel at a time on each):
//  * stream kernel on MT x NT blocks: 2 + 0.02 f (MT + NT) a round of its grid (45 x 5120 x 8192: 1 x 4 blocks 16.2, 2 x 2
//    18.4, 2 x 4 17.5, 4 x 4 25.0; 64 x 14336 x 4096: 18.8 on 4 x 4, 23.0 on 2 x 4, 36.6 on 1 x 4; 100 x 4096 x 4096: 8.7 on 2 x 4, 11.4 on
//    1 x 4, 12.9 on 4 x 4; 8 x 14336 x 4096: 12.5 on 1 x 2, 14.9 on 1 x 1);
//  * 64 x 128 tiles: 5.5 + 0.2 f / splits, 6 more where K is split, 5.5 + 0.18 f a round from more than one per CU (200 x 1024 x 16384:
//    54.6 whole, 34.1 in two, 22.6 in four, the stream kernel 24.8; 500 x 1024 x 1024: 8.2, stream 5.0);
//  * 128 x 128 tiles: 5.5 + 0.23 f up to one per CU (150 x 14336 x 4096: 24.0, 64 x 128 27.5, stream 38.1); beyond, and for
//    256 x 256 from one per CU, as the other types;
//  * up to 128 rows of so many columns that there are more 128 x 128 tiles than CUs (a vocabulary), where rounds of a grid tell nothing any more: up to
//    16 rows the stream kernel on 1 x 2 blocks (1 x 128000 x 4096: 81, 1 x 1 87, 1 x 4 88, 64 x 128 tiles 87; 8 rows 84, 108, 93, 89), up to 64
//    tiles of 64 x 128 (64 rows: 98, 128 x 128 101, 256 x 256 130, stream 137 at best; 17 rows 90, 92, 124, 99), then 128 x 128 (65 rows: 101, 64 x 128
//    117, 256 x 256 129; 128 x 40000 x 8192: 88, 94, 98).
Choice choose(const SpinnHipLinearI8Desc *d) {
    const int64_t cus = device_cu_count(), mt = m_tiles(d), nt = n_tiles(d), f = frags(d);
    auto grid = [&](int64_t rows, int64_t cols) { return ((mt + rows - 1) / rows) * ((nt + cols - 1) / cols); };
    auto rounds = [&](int64_t blocks) { return (blocks + cus - 1) / cus; };
    if (grid(8, 8) > cus) {
        if (mt > 8) return choose(mt, nt, f);
        if (mt == 1) return {Choice::kStream, 1, 2, 1};
        return {mt <= 4 ? Choice::kTile64 : Choice::kTile128, 1, 1, 1};
    }
    Choice c{Choice::kStream, 1, 1, 1};
    double least = 1e30;
    static const int blocks[][2] = {{1, 1}, {1, 2}, {1, 4}, {2, 2}, {2, 4}, {3, 2}, {3, 4}, {4, 2}, {4, 4}};
    for (auto &b : blocks) {
        const double t = (2 + 0.02 * f * (b[0] + b[1])) * rounds(grid(b[0], b[1]));
        if (b[0] <= mt && t < least) {
            least = t;
            c.mt = b[0];
            c.nt = b[1];
        }
    }
    const int64_t tiles = grid(4, 8);
    const int64_t splits = std::max<int64_t>(1, std::min(cus / tiles, f / 16));
    const double whole = tiles <= cus ? 5.5 + 0.2 * f : 5.5 + 0.18 * f * rounds(tiles), parts = 11.5 + 0.2 * f / splits;
    if (std::min(whole, parts) < least) {
        least = std::min(whole, parts);
        c.kind = Choice::kTile64;
        c.splits = splits > 1 && parts < whole ? (int)splits : 1;
    }
    if (5.5 + 0.23 * f < least) c.kind = Choice::kTile128;
    return c;
}

} // namespace

int quantize_rows(int dtype, int64_t rows, int k, const void *x, int64_t ldx, int8_t *xq, int64_t ldq, float *scale, hipStream_t st) {
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        if (k <= 1024) return launch_quantize<T, 1>(rows, k, x, ldx, xq, ldq, scale, st);
        if (k <= 4096) return launch_quantize<T, 4>(rows, k, x, ldx, xq, ldq, scale, st);
        return launch_quantize<T, 16>(rows, k, x, ldx, xq, ldq, scale, st);
    });
}

size_t linear_i8_packed_bytes(const SpinnHipLinearI8Desc *d) { return (size_t)(n_tiles(d) * frags(d) + 1) * kFragBytes; }

size_t linear_i8_workspace_bytes(const SpinnHipLinearI8Desc *d) {
    const Choice c = choose(d);
    const size_t tiles = (size_t)((m_tiles(d) + 3) / 4) * ((n_tiles(d) + 7) / 8);
    return c.kind == Choice::kTile64 && c.splits > 1 ? tiles * c.splits * 64 * 128 * 4 : 0;
}

int linear_i8_pack(const SpinnHipLinearI8Desc *d, const int8_t *w, void *packed, hipStream_t st) {
    const int64_t total = n_tiles(d) * frags(d) * 64;
    const unsigned grid = (unsigned)std::min<int64_t>((total + 64 + 255) / 256, 65536);
    linear_pack_kernel<int8_t><<<grid, 256, 0, st>>>(w, (u32x4 *)packed, d->n, d->k, d->trans_w, frags(d), total);
    return check_launch();
}

int linear_i8_run(const SpinnHipLinearI8Desc *d, const int8_t *x, const float *x_scale, const void *packed, const float *w_scale,
                  const void *bias, const void *res, void *y, void *ws, hipStream_t st) {
    LinearArgs a{};
    a.x = x;
    a.bias = bias;
    a.res = res;
    a.sx = x_scale;
    a.sw = w_scale;
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
    const int per = 16 / dtype_bytes(d->dtype);
    a.vec = aligned16(y) && d->ldy % per == 0 && (!res || (aligned16(res) && d->ldres % per == 0));
    const Choice c = choose(d);
    return with_dtype(d->dtype, [&](auto o) {
        typedef decltype(o) O;
        if (c.kind != Choice::kStream) return launch_tiles<int8_t, O>(a, c, false, ws, st);
        switch (c.mt * 10 + c.nt) {
        case 44: return launch_stream_i8<O, 4, 4, 8, 2>(a, st);
        case 34: return launch_stream_i8<O, 3, 4, 8, 2>(a, st);
        case 24: return launch_stream_i8<O, 2, 4, 8, 2>(a, st);
        case 42: return launch_stream_i8<O, 4, 2, 8, 2>(a, st);
        case 32: return launch_stream_i8<O, 3, 2, 8, 4>(a, st);
        case 22: return launch_stream_i8<O, 2, 2, 8, 4>(a, st);
        case 14: return launch_stream_i8<O, 1, 4, 8, 4>(a, st);
        case 12: return launch_stream_i8<O, 1, 2, 8, 4>(a, st);
        default: return launch_stream_i8<O, 1, 1, 16, 4>(a, st);
        }
    });
}

} // namespace spinn
