// linear.hip - linear layers: y = act(x w^T + bias + residual) in fp32, fp16 and bf16.
//
// Weights are packed once into MFMA operand fragments, [N/16][K/kFrag][64 lanes][16 bytes] with
// zeros around, so that a wave reads 1 KB of them with one load and feeds a matrix instruction
// as they come. The weights are the A operand (its rows are the accumulators' rows), x is the
// B operand; which columns of 64 a tile holds is chosen for the stores of y (first_col).
//
//  * few rows (single tokens): the weights are read once and bound it. linear_stream_kernel: tiles of
//    16 MT x 16 NT, K spread over a workgroup's waves, operands straight from memory into
//    registers, the waves' sums joined in LDS in wave order. 1 x 4096 x 4096 bf16: 7.2 us, 4.7 TB/s;
//    33 x 8192 x 2048 fp16: 8.5 us, 4.0 TB/s.
//  * many rows: the matrix cores bound it. linear_tile_kernel: both operands through LDS, whole
//    fragments copied there without passing registers, four of them along K. 4096 x 8192 x 4096 bf16:
//    218 us, 1260 TFLOP/s; 1568 x 2048 x 512 fp32: 41 us, 80 TFLOP/s (400 tiles for 256 CUs).
#include "linear_core.h"

namespace spinn {
namespace {

inline int64_t frags(const SpinnHipLinearDesc *d) { // along K, an even number
    const int f = 64 / dtype_bytes(d->dtype);
    return ((int64_t)d->k + 2 * f - 1) / (2 * f) * 2;
}
inline int64_t n_tiles(const SpinnHipLinearDesc *d) { return ((int64_t)d->n + 63) / 64 * 4; }
inline int64_t m_tiles(const SpinnHipLinearDesc *d) { return ((int64_t)d->m + 15) / 16; }
// x's rows are not whole, aligned 16-byte runs
inline bool x_loose(const SpinnHipLinearDesc *d) {
    const int e = 16 / dtype_bytes(d->dtype);
    return d->x_unaligned || d->ldx % e || d->k % e;
}

Choice choose(const SpinnHipLinearDesc *d) { return choose(m_tiles(d), n_tiles(d), frags(d)); }

// x as granules [M/16][kf/2][2 KB], zeros behind its rows and columns; one thread per 16 bytes.
template <class T>
__global__ __launch_bounds__(256) void linear_pack_x_kernel(const T *__restrict__ x, u32x4 *__restrict__ out, int m, int k,
                                                            int64_t ldx, int64_t kf, int64_t total) {
    constexpr int E = 16 / (int)sizeof(T);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int in = (int)(i & 127), r = in >> 3;
        const int64_t granule = i >> 7, tile = granule / (kf / 2), g = granule - tile * (kf / 2);
        const int64_t row = tile * 16 + r;
        const int k0 = (int)(g * 2 * kFrag<T>) + ((in & 7) ^ (r >> 1)) * E;
        uint32_t w[4] = {0, 0, 0, 0};
        if (row < m && k0 < k) {
            if (k >= E) {
                load_loose<T, E>(x + row * ldx, k0, k, w);
            } else {
                const u32x4 v = load_edge<T>(x + row * ldx + k0, k - k0);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = v[j];
            }
        }
        out[i] = (u32x4){w[0], w[1], w[2], w[3]};
    }
}

// How a layer reads x. Rows that are no whole, aligned runs are laid out in the workspace by a launch of their own,
// but the stream kernel reads them where they are while a workgroup's rows stay under 32 KB: its unaligned loads then
// cost less than the launch (1 x 4096 x 4097 bf16: 10.8 -> 7.8 us, 427 x 131 x 275: 10.3 -> 7.6; 40 KB, 202 x 1758 x 632:
// 9.9 -> 13.0; 131 KB, 16 x 4096 x 4097: 10.0 -> 16.8).
Rows x_rows(const SpinnHipLinearDesc *d, const Choice &c) {
    if (!x_loose(d)) return kRuns;
    const int64_t bytes = (int64_t)d->k * dtype_bytes(d->dtype);
    if (c.kind != Choice::kStream || std::min(d->m, 16 * c.mt) * bytes > 32768) return kLaidOut;
    return bytes >= 16 ? kLoose : kShort;
}

size_t x_bytes(const SpinnHipLinearDesc *d, const Choice &c) {
    return x_rows(d, c) == kLaidOut ? (size_t)(m_tiles(d) * frags(d)) * kFragBytes : 0;
}

} // namespace

size_t linear_packed_bytes(const SpinnHipLinearDesc *d) {
    return (size_t)(n_tiles(d) * frags(d) + 1) * kFragBytes;
}

size_t linear_workspace_bytes(const SpinnHipLinearDesc *d) {
    const Choice c = choose(d);
    const size_t tiles = (size_t)((m_tiles(d) + 3) / 4) * ((n_tiles(d) + 7) / 8);
    return x_bytes(d, c) + (c.kind == Choice::kTile64 && c.splits > 1 ? tiles * c.splits * 64 * 128 * 4 : 0);
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
    const int per = 16 / dtype_bytes(d->dtype);
    a.vec = aligned16(y) && d->ldy % per == 0 && (!res || (aligned16(res) && d->ldres % per == 0));
    const Choice c = choose(d);
    const Rows rows = x_rows(d, c);
    return with_dtype(d->dtype, [&](auto t) {
        typedef decltype(t) T;
        if (rows == kLaidOut) {
            const int64_t total = m_tiles(d) * a.kf * 64;
            linear_pack_x_kernel<T><<<(unsigned)std::min<int64_t>((total + 255) / 256, 65536), 256, 0, st>>>(
                (const T *)x, (u32x4 *)ws, d->m, d->k, d->ldx, a.kf, total);
            const int rc = check_launch();
            if (rc) return rc;
            a.x = ws;
        }
        return launch_linear<T, T>(a, c, rows, (char *)ws + x_bytes(d, c), st);
    });
}

} // namespace spinn
