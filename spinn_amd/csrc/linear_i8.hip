// linear_i8.hip - linear layers in 8-bit integers, and rows quantised for them.
//
// The layers run on the kernels of linear_core.h: a fragment of 64 k of 8-bit integers has the bytes of one of 32 k of a
// 16-bit type and its matrix instruction the same time, so that tiles, copies and waits are the same, with twice the
// products. Sums are exact 32-bit integers; the scales come in with the epilogue, in fp32.
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
// where it is near s / 2. tiny: s has few bits or none above fp32's least number, where a reciprocal would overflow.
__device__ __forceinline__ int quantized(float v, float s, float inv, bool tiny) {
    if (tiny) return s > 0.f ? (int)fmin(fmax(rint((double)v / (double)s), -127.0), 127.0) : 0;
    float r = fminf(fmaxf(rintf(v * inv), -127.f), 127.f);
    const float d = fmaf(-r, s, v), far = fabsf(d), half = 0.5f * s;
    const int i = (int)r;
    return far > half || (far == half && (i & 1)) ? min(max(i + (d > 0.f ? 1 : -1), -127), 127) : i;
}

// A row per NW waves, 4 / NW (at least one) rows a workgroup; up to HOLD units of a lane stay in registers between the two passes.
// 1 x 4096 bf16 is one workgroup's latency; many rows are bound by memory.
template <class T, int NW, int HOLD>
__global__ __launch_bounds__(64 * (NW < 4 ? 4 : NW)) void quantize_rows_kernel(const T *__restrict__ x, int64_t ldx, int8_t *__restrict__ xq,
                                                                           int64_t ldq, float *__restrict__ scale, int64_t rows, int k) {
    constexpr int R = NW < 4 ? 4 / NW : 1;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t row = (int64_t)blockIdx.x * R + wave / NW;
    const int first = (wave % NW) * 64 + lane, units = (int)(((int64_t)k + kUnit - 1) / kUnit);
    const bool in = row < rows;
    const T *xr = x + (in ? row : 0) * ldx;
    float v[HOLD][kUnit];
    uint32_t top = 0; // bits of the largest magnitude; infinities and NaN are above all numbers
    auto look = [&](const float (&w)[kUnit]) {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) top = max(top, __builtin_bit_cast(uint32_t, w[i]) & 0x7fffffffu);
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        const int u = first + h * 64 * NW;
        if (in && u < units) {
            load_unit<T>(xr, u, k, v[h]);
            look(v[h]);
        }
    }
    if (in)
        for (int u = first + HOLD * 64 * NW; u < units; u += 64 * NW) {
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
    const bool tiny = top < 0x0d800000u; // 2^-100
    const float inv = 1.f / s;
    if (first == 0) scale[row] = s;
    int8_t *out = xq + row * ldq;
    auto store = [&](int u, const float (&w)[kUnit]) {
        u32x4 b = {0, 0, 0, 0};
        if (!bad) {
#pragma unroll
            for (int i = 0; i < kUnit; ++i) b[i / 4] |= (uint32_t)(uint8_t)quantized(w[i], s, inv, tiny) << (8 * (i % 4));
        }
        *reinterpret_cast<u32x4 *>(out + (int64_t)u * kUnit) = b;
    };
#pragma unroll
    for (int h = 0; h < HOLD; ++h) {
        const int u = first + h * 64 * NW;
        if (u < units) store(u, v[h]);
    }
    for (int u = first + HOLD * 64 * NW; u < units; u += 64 * NW) {
        float w[kUnit];
        load_unit<T>(xr, u, k, w);
        store(u, w);
    }
}

template <class T, int NW, int HOLD>
int launch_quantize(int64_t rows, int k, const void *x, int64_t ldx, int8_t *xq, int64_t ldq, float *scale, hipStream_t st) {
    constexpr int R = NW < 4 ? 4 / NW : 1, threads = 64 * (NW < 4 ? 4 : NW);
    const int64_t grid = (rows + R - 1) / R;
    if (!launch_fits(grid, threads)) return SPINN_HIP_EUNSUPPORTED;
    quantize_rows_kernel<T, NW, HOLD><<<(unsigned)grid, threads, 0, st>>>((const T *)x, ldx, xq, ldq, scale, rows, k);
    return check_launch();
}

inline int64_t frags(const SpinnHipLinearI8Desc *d) { return ((int64_t)d->k + 127) / 128 * 2; }
inline int64_t n_tiles(const SpinnHipLinearI8Desc *d) { return ((int64_t)d->n + 63) / 64 * 4; }
inline int64_t m_tiles(const SpinnHipLinearI8Desc *d) { return ((int64_t)d->m + 15) / 16; }
Choice choose(const SpinnHipLinearI8Desc *d) { return choose(m_tiles(d), n_tiles(d), frags(d)); }

} // namespace

int quantize_rows(int dtype, int64_t rows, int k, const void *x, int64_t ldx, int8_t *xq, int64_t ldq, float *scale, hipStream_t st) {
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        if (k <= 1024) return launch_quantize<T, 1, 1>(rows, k, x, ldx, xq, ldq, scale, st);
        if (k <= 4096) return launch_quantize<T, 4, 1>(rows, k, x, ldx, xq, ldq, scale, st);
        return launch_quantize<T, 16, 1>(rows, k, x, ldx, xq, ldq, scale, st);
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
    return with_dtype(d->dtype, [&](auto o) { return launch_linear<int8_t, decltype(o)>(a, c, kRuns, ws, st); });
}

} // namespace spinn
