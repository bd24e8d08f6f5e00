// rope.hip - rotary positions: pairs of a head's elements turned by an angle that grows with the position.
//
// Memory bounds it: every element is read and written once. The sines and cosines of a token are the same in all of its heads,
// so a workgroup computes those of its tokens once into LDS and then walks over the heads in 16-byte
// runs. Angles: a frequency is kept as a fraction of a turn in 64-bit fixed point, right to its last two units, whose product with the position,
// modulo 2^64, is the angle without its whole turns, to 2^-32: positions in the thousands of millions are as good as the first.
// 16384 x 40 heads of 128, bf16: 62 to 67 us, 5.0 to 5.4 TB/s; 5001 x 17 heads, 32 of 80, interleaved, fp32: 10.5 us, 5.2 TB/s; 32 x 20 heads of
// 128: 6.8 us a call, a launch.
#include "decode.h"

namespace spinn {
namespace {

struct RopeArgs {
    const int32_t *position;
    const uint64_t *table;
    const void *x;
    void *y;
    int64_t tokens, x_stride, x_head_stride, y_stride, y_head_stride;
    float magnitude;
    int32_t heads, dim, rot, interleaved;
    int32_t per_block;         // tokens of a workgroup
    int32_t turned, units;     // of a head: runs (or pairs of runs) that turn, and those and the ones to copy
    int32_t rest_runs;         // what is to copy are whole runs, else single elements
    uint32_t unit_mul, unit_shift, head_mul, head_shift; // i / units and i / heads by a product
};

// (sin, cos) of 2 pi p / 2^64: the nearest quarter turn and what is left of it, within 1/8 of a turn.
// sin x = x + x^3 S(x^2) and cos x = 1 - x^2/2 + x^4 C(x^2), S and C fitted on [-pi/4, pi/4] with the least error of the
// results (5e-9 relative and 1e-10).
__device__ __forceinline__ void sin_cos_turns(uint64_t p, float &s, float &c) {
    const uint32_t q = (uint32_t)((p + (1ull << 61)) >> 62);
    const int64_t r = (int64_t)(p - ((uint64_t)q << 62));
    const float x = (float)r * 3.4061215800304e-19f; // 2 pi / 2^64
    const float z = x * x;
    const float sn = fmaf(x * z, fmaf(fmaf(-1.9517e-4f, z, 8.33218e-3f), z, -1.6666655e-1f), x);
    const float cs = fmaf(z * z, fmaf(fmaf(2.44383793e-5f, z, -1.38873669e-3f), z, 4.16666469e-2f), fmaf(-0.5f, z, 1.f));
    const bool swap = q & 1;
    s = swap ? cs : sn;
    c = swap ? sn : cs;
    if (q & 2) s = -s;          // sin: + + - -
    if ((q + 1) & 2) c = -c;    // cos: + - - +
}

__device__ __forceinline__ uint32_t quotient(uint32_t i, uint32_t mul, uint32_t shift) {
    return mul ? __umulhi(i, mul) >> shift : i;
}

// One unit: run u of V elements of a head. Half layout: those at u V and rot/2 + u V; interleaved: those at u V.
// LOOSE: runs start at any element.
template <class T, int V, bool INTER, bool LOOSE>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    extern __shared__ float2 turn[]; // [per_block][rot / 2]: (sin, cos)
    const int half = a.rot / 2;
    const int64_t t0 = (int64_t)blockIdx.x * a.per_block;
    const int n = (int)min((int64_t)a.per_block, a.tokens - t0);
    for (int i = threadIdx.x; i < n * half; i += 256) {
        const int t = i / half, k = i - t * half;
        float s, c;
        sin_cos_turns((uint64_t)(int64_t)a.position[t0 + t] * a.table[k], s, c);
        turn[i] = make_float2(s * a.magnitude, c * a.magnitude);
    }
    __syncthreads();
    typedef T Vec __attribute__((ext_vector_type(V)));
    typedef Vec InMemory __attribute__((aligned(LOOSE ? sizeof(T) : V * sizeof(T))));
    auto load = [](const T *p) { return (Vec) * reinterpret_cast<const InMemory *>(p); };
    auto store = [](T *p, Vec v) { *reinterpret_cast<InMemory *>(p) = v; };
    const uint32_t total = (uint32_t)n * a.heads * a.units;
    for (uint32_t i = threadIdx.x; i < total; i += 256) {
        const uint32_t th = quotient(i, a.unit_mul, a.unit_shift), u = i - th * a.units;
        const uint32_t t = quotient(th, a.head_mul, a.head_shift), h = th - t * a.heads;
        const T *x = (const T *)a.x + (t0 + t) * a.x_stride + h * a.x_head_stride;
        T *y = (T *)a.y + (t0 + t) * a.y_stride + h * a.y_head_stride;
        const float2 *sc = turn + t * half;
        if (u >= (uint32_t)a.turned) { // behind the turned part, its bits
            typedef typename Bits<T>::type B;
            typedef B Word __attribute__((ext_vector_type(V)));
            typedef Word LooseWord __attribute__((aligned(LOOSE ? sizeof(T) : V * sizeof(T))));
            const int k = (int)(u - a.turned);
            if (a.rest_runs) *reinterpret_cast<LooseWord *>(y + a.rot + k * V) = *reinterpret_cast<const LooseWord *>(x + a.rot + k * V);
            else reinterpret_cast<B *>(y)[a.rot + k] = reinterpret_cast<const B *>(x)[a.rot + k];
        } else if constexpr (INTER) {
            const int at = (int)u * V;
            const Vec v = load(x + at);
            Vec r;
#pragma unroll
            for (int k = 0; k < V; k += 2) {
                const float2 w = sc[(at + k) >> 1];
                const float p = (float)v[k], q = (float)v[k + 1];
                r[k] = (T)fmaf(w.y, p, -(w.x * q));
                r[k + 1] = (T)fmaf(w.x, p, w.y * q);
            }
            store(y + at, r);
        } else {
            const int at = (int)u * V;
            const Vec va = load(x + at), vb = load(x + half + at);
            Vec ra, rb;
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float2 w = sc[at + k];
                const float p = (float)va[k], q = (float)vb[k];
                ra[k] = (T)fmaf(w.y, p, -(w.x * q));
                rb[k] = (T)fmaf(w.x, p, w.y * q);
            }
            store(y + at, ra);
            store(y + half + at, rb);
        }
    }
}

// Numbers of 106 bits, hi + lo: a position of up to 2^31 multiplies what an angle's frequency is off by.
struct Wide {
    double hi, lo;
};
__device__ Wide normal(double a, double b) { // a + b, |a| >= |b|
#pragma clang fp contract(off)
    const double s = a + b;
    return {s, b - (s - a)};
}
__device__ Wide sum(double a, double b) {
#pragma clang fp contract(off)
    const double s = a + b, t = s - a;
    return {s, (a - (s - t)) + (b - t)};
}
__device__ Wide operator+(Wide a, Wide b) {
#pragma clang fp contract(off)
    const Wide s = sum(a.hi, b.hi), t = sum(a.lo, b.lo), u = normal(s.hi, s.lo + t.hi);
    return normal(u.hi, u.lo + t.lo);
}
__device__ Wide operator-(Wide a) { return {-a.hi, -a.lo}; }
__device__ Wide operator*(Wide a, Wide b) {
#pragma clang fp contract(off)
    const double p = a.hi * b.hi, e = fma(a.hi, b.hi, -p);
    return normal(p, e + (a.hi * b.lo + a.lo * b.hi));
}
__device__ Wide operator/(Wide a, Wide b) { // three quotients of what is left
#pragma clang fp contract(off)
    const double q1 = a.hi / b.hi;
    const Wide r1 = a + -(b * Wide{q1, 0.0});
    const double q2 = r1.hi / b.hi;
    const Wide r2 = r1 + -(b * Wide{q2, 0.0});
    return normal(q1, q2) + Wide{r2.hi / b.hi, 0.0};
}
__device__ Wide power(Wide a, int n) {
    Wide r = {1.0, 0.0};
    for (; n; n >>= 1) {
        if (n & 1) r = r * a;
        a = a * a;
    }
    return r;
}

// One entry a lane: its frequency in turns a position, without the whole ones, in units of 2^-64. Within 2 of them for frequencies up to 2^30.
__global__ __launch_bounds__(256) void rope_table_kernel(uint64_t *out, int half, int scaling, double base, double factor,
                                                         double low, double high, double trained) {
    const int i = threadIdx.x;
    if (i >= half) return;
    // f = base^(-i / half): two steps of Newton's method for f^half base^i = 1 from the library's power, which is off by up to 2^-46. Each
    // squares the distance (times half); the powers' own roundings are 2^-95 of the equation's, 2^-95 / half of f. Exponents apart, so that
    // nothing leaves the range.
    int exp_b, exp_f;
    const double mant_b = frexp(base, &exp_b);
    Wide f = {pow(base, -(double)i / half), 0.0};
    frexp(f.hi, &exp_f);
    const Wide base_i = power({mant_b, 0.0}, i);
    for (int step = 0; step < 2; ++step) {
        const Wide p = power({ldexp(f.hi, -exp_f), ldexp(f.lo, -exp_f)}, half) * base_i;
        const int e = exp_f * half + exp_b * i;
        const Wide off = Wide{1.0, 0.0} + Wide{-ldexp(p.hi, e), -ldexp(p.lo, e)};
        f = f + f * (off / Wide{(double)half, 0.0});
    }
    const Wide per_radian = {0x1.45f306dc9c883p-3, -0x1.6b01ec5417056p-57};
    Wide turns = f * per_radian;
    if (scaling == SPINN_ROPE_LINEAR) {
        turns = turns / Wide{factor, 0.0};
    } else if (scaling == SPINN_ROPE_BY_PARTS) {
        const Wide t = (turns * Wide{trained, 0.0} + Wide{-low, 0.0}) / sum(high, -low);
        const Wide stretched = turns / Wide{factor, 0.0};
        if (t.hi <= 0.0) turns = stretched;
        else if (t.hi < 1.0) turns = t * turns + (Wide{1.0, 0.0} + -t) * stretched;
    }
    constexpr double kUnits = 18446744073709551616.0; // 2^64
    const double part = (turns.hi - floor(turns.hi)) * kUnits, rest = (turns.lo - rint(turns.lo)) * kUnits;
    const double whole = floor(part);
    out[i] = (uint64_t)whole + (uint64_t)(int64_t)rint(rest + (part - whole));
}

// mul and shift so that i / n = mulhi(i, mul) >> shift for all i < 2^31 (mul 0: i itself).
void reciprocal(uint32_t n, uint32_t &mul, uint32_t &shift) {
    mul = shift = 0;
    if (n == 1) return;
    while ((2u << shift) < n) ++shift; // 2^shift < n <= 2^(shift + 1)
    mul = (uint32_t)(((1ull << (32 + shift)) + n - 1) / n);
}

template <class T, int V>
int launch(const RopeArgs &a, bool loose, unsigned grid, size_t lds, hipStream_t st) {
    if (a.interleaved) {
        if constexpr (V >= 2) {
            if (loose) rope_kernel<T, V, true, true><<<grid, 256, lds, st>>>(a);
            else rope_kernel<T, V, true, false><<<grid, 256, lds, st>>>(a);
        }
    } else if (loose) {
        rope_kernel<T, V, false, true><<<grid, 256, lds, st>>>(a);
    } else {
        rope_kernel<T, V, false, false><<<grid, 256, lds, st>>>(a);
    }
    return check_launch();
}

} // namespace

int rope_table(const SpinnHipRopeDesc *d, void *table, hipStream_t st) {
    rope_table_kernel<<<1, 256, 0, st>>>((uint64_t *)table, d->rot_dim / 2, d->scaling, d->base, d->factor, d->low, d->high, d->trained);
    return check_launch();
}

int rope_run(const SpinnHipRopeDesc *d, int64_t tokens, const int32_t *position, const void *table, const void *x, void *y,
             hipStream_t st) {
    RopeArgs a{};
    a.position = position;
    a.table = (const uint64_t *)table;
    a.x = x;
    a.y = y;
    a.tokens = tokens;
    a.x_stride = d->x_stride;
    a.x_head_stride = d->x_head_stride;
    a.y_stride = d->y_stride;
    a.y_head_stride = d->y_head_stride;
    a.magnitude = d->magnitude;
    a.heads = d->heads;
    a.dim = d->head_dim;
    a.rot = d->rot_dim;
    a.interleaved = d->interleaved;
    const int e = dtype_bytes(d->dtype), half = a.rot / 2, rest = y == x ? 0 : a.dim - a.rot;
    const int turns = a.interleaved ? a.rot : half;
    int v = 16 / e; // elements of a run
    while (turns % v) v /= 2;
    const bool loose = (d->x_stride | d->y_stride | d->x_head_stride | d->y_head_stride | a.rot) % v != 0 ||
                       ((uintptr_t)x | (uintptr_t)y) % (uintptr_t)(v * e) != 0;
    a.rest_runs = rest % v == 0;
    a.turned = turns / v;
    a.units = a.turned + (a.rest_runs ? rest / v : rest);
    reciprocal((uint32_t)a.units, a.unit_mul, a.unit_shift);
    reciprocal((uint32_t)a.heads, a.head_mul, a.head_shift);
    const int64_t per_token = (int64_t)a.heads * a.units;
    // 1024 units or more a workgroup (sines and cosines shared by what there is), but two workgroups a CU first
    int64_t n = 1;
    while (2 * n * half * 8 <= 32768 && ((n * per_token < 1024 && tokens / (2 * n) >= 2 * device_cu_count()) || !launch_fits((tokens + n - 1) / n, 256)) &&
           2 * n * per_token < (int64_t)1 << 31)
        n *= 2;
    a.per_block = (int32_t)n;
    const int64_t grid = (tokens + n - 1) / n;
    if (!launch_fits(grid, 256)) return SPINN_HIP_EUNSUPPORTED;
    const size_t lds = (size_t)n * half * sizeof(float2);
    return with_dtype(d->dtype, [&](auto t) {
        typedef decltype(t) T;
        switch (v) {
        case 8:
            if constexpr (sizeof(T) == 2) return launch<T, 8>(a, loose, (unsigned)grid, lds, st);
            return (int)SPINN_HIP_EINVAL;
        case 4: return launch<T, 4>(a, loose, (unsigned)grid, lds, st);
        case 2: return launch<T, 2>(a, loose, (unsigned)grid, lds, st);
        default: return launch<T, 1>(a, loose, (unsigned)grid, lds, st);
        }
    });
}

} // namespace spinn
