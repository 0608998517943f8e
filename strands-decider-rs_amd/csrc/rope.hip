// Rotary positions apart from the engine's own rotation: the angles of any positions, as a table or applied to rows, and a
// step's positions of requests that have dropped cached rows (no counterpart in the reference, whose positions are the
// cache's rows and whose pairs are half the rotated dims apart).
//
// Pair j of a row at position p turns by x = p f_j: (a, b) -> m (a cos x - b sin x, b cos x + a sin x).  f comes in f64,
// radians per position, and so does everything up to the cosine and the sine: at position 3 000 000 the fastest pair's
// angle has 22 bits before the point, and f32 would leave it 2 behind.
#include "paged.h"

namespace sd {
namespace {

struct Turn {
    float c, s;
};

// m (cos, sin) of p f radians: p f in turns, less whole turns, less the nearest quarter; what is left, at most 1/8 turn,
// goes through the first terms of the two series, up to x^11 and x^12 (the next ones are below 2^-37), in f64.  Each result
// is rounded to f32 once.  About 30 f64 instructions: a table of 16396 rows of 64 pairs takes 5.4 us where its bytes, 8.4 MB, would
// take 1.8.
__device__ __forceinline__ Turn turn_of(int p, double f, double m) {
    double t = (double)p * (f * 0.15915494309189533577);
    t -= __builtin_rint(t);
    const double q = __builtin_rint(t * 4.0);
    const double x = (t - q * 0.25) * 6.28318530717958647693, z = x * x;
    double s = -1.0 / 39916800, c = 1.0 / 479001600;
    s = s * z + 1.0 / 362880, c = c * z - 1.0 / 3628800;
    s = s * z - 1.0 / 5040, c = c * z + 1.0 / 40320;
    s = s * z + 1.0 / 120, c = c * z - 1.0 / 720;
    s = s * z - 1.0 / 6, c = c * z + 1.0 / 24;
    c = c * z - 0.5;
    s = m * (x * z * s + x), c = m * (c * z + 1.0);
    const int k = (int)q;
    const double a = k & 1 ? s : c, b = k & 1 ? c : s;
    return {(float)((k + 1) & 2 ? -a : a), (float)(k & 2 ? -b : b)};
}

// One (cosine, sine) per thread.
__global__ __launch_bounds__(256) void k_rope_table(const double* __restrict__ freqs, uint32_t pairs, double m,
                                                    const int* __restrict__ pos, uint32_t total, float2* __restrict__ table) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const uint32_t r = i / pairs, j = i - r * pairs;
    const Turn t = turn_of(pos ? pos[r] : (int)r, freqs[j], m);
    table[i] = make_float2(t.c, t.s);
}

constexpr int MAX_R = 8;  // rows of a workgroup at most

// Rows r0 .. r0 + R - 1 of a workgroup, or a slice of one row's units.  A unit is 8 dims of a head with the 8 that turn
// with them (HALF), or 4 neighbouring pairs (PAIRS), or 8 dims that are only copied.  The workgroup's angles come once,
// into LDS, for all heads, while its rows are on their way.  Bound by bytes: 8192 rows of 8 and 2 heads of 256 dims,
// 64 of them rotated, written elsewhere: 18 to 20 us for 84 MB, 4.3 TB/s (four units a thread; one: 24); 64 rows 3.0 us, a launch
// and two loads in series.
enum { HALF, PAIRS, ODD };  // ODD: pairs half the rotated dims apart where that is no multiple of 8: element by element (those rows with
                            // 40 dims rotated 68 us, in f32 126; f32 with 64 dims 40)
template <class T>
struct RopeSide {  // q's or k's heads
    const T* in;
    T* out;
    uint32_t stride, step, ostride, ostep;
};
// Division by a number that is the same for all, as one upper half of a product: exact where the dividend times it is below 2^32.
struct Div {
    uint32_t d, magic;
    explicit Div(uint32_t n) : d(n), magic((uint32_t)((1ull << 32) / n + 1)) {}
    __device__ __forceinline__ uint32_t of(uint32_t x) const { return d == 1 ? x : __umulhi(x, magic); }
};
template <class T, int MODE, int N>
__global__ __launch_bounds__(256) void k_rope(const double* __restrict__ freqs, int RD, double m, float sign,
                                              const int* __restrict__ pos, int rows, int HD, RopeSide<T> q, int HQ,
                                              RopeSide<T> k, Div per, uint32_t turning, Div units, int R, uint32_t slices) {
    typedef T T8 __attribute__((ext_vector_type(8), aligned(16)));
    __shared__ Turn turns[MAX_R * 128];
    const int tid = threadIdx.x, rd2 = RD / 2;
    const uint32_t slice = slices == 1 ? 0 : blockIdx.x % slices;
    const int r0 = (slices == 1 ? blockIdx.x : blockIdx.x / slices) * R, nr = min(R, rows - r0);
    const uint32_t first = slice * (256 * N), last = min((uint32_t)nr * per.d, first + 256 * N);  // (R is 1 where a row has several slices)
    const T* const q0 = q.in + (size_t)r0 * q.stride;
    const T* const k0 = k.in + (size_t)r0 * k.stride;
    T* const q1 = q.out + (size_t)r0 * q.ostride;
    T* const k1 = k.out + (size_t)r0 * k.ostride;
    T8 a[N], b[N];
    const T* src[N];
    T* dst[N];
    uint32_t at[N], row[N];
#pragma unroll
    for (int n = 0; n < N; n++) {
        const uint32_t i = first + n * 256 + tid;
        if (i >= last) continue;
        row[n] = slices == 1 ? per.of(i) : 0;
        const uint32_t x = i - row[n] * per.d, h = units.of(x);
        at[n] = x - h * units.d;
        const bool isq = h < (uint32_t)HQ;
        const uint32_t hh = isq ? h : h - HQ;
        src[n] = (isq ? q0 : k0) + (uint64_t)row[n] * (isq ? q.stride : k.stride) + (uint64_t)hh * (isq ? q.step : k.step);
        dst[n] = (isq ? q1 : k1) + (uint64_t)row[n] * (isq ? q.ostride : k.ostride) + (uint64_t)hh * (isq ? q.ostep : k.ostep);
        if (MODE == ODD) continue;
        if (at[n] < turning) {
            a[n] = *reinterpret_cast<const T8*>(src[n] + 8 * at[n]);
            if (MODE == HALF) b[n] = *reinterpret_cast<const T8*>(src[n] + 8 * at[n] + rd2);
        } else {
            a[n] = *reinterpret_cast<const T8*>(src[n] + 8 * at[n] + (MODE == HALF ? rd2 : 0));
        }
    }
    for (int i = tid; i < nr * rd2; i += 256) {
        const int r = i / rd2;
        Turn t = turn_of(pos ? pos[r0 + r] : r0 + r, freqs[i - r * rd2], m);
        t.s *= sign;
        turns[i] = t;
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; n++) {
        if (first + n * 256 + tid >= last) continue;
        const Turn* const w = turns + row[n] * rd2;
        if (MODE == ODD) {
            const int u = 8 * at[n];
            if (at[n] < turning) {
                for (int j = u; j < min(u + 8, rd2); j++) {
                    const float x = (float)src[n][j], y = (float)src[n][j + rd2];
                    dst[n][j] = (T)(x * w[j].c - y * w[j].s);
                    dst[n][j + rd2] = (T)(y * w[j].c + x * w[j].s);
                }
            } else {
                const int d0 = RD + 8 * (at[n] - turning);
                for (int d = d0; d < min(d0 + 8, HD); d++) dst[n][d] = src[n][d];
            }
            continue;
        }
        if (at[n] >= turning) {
            *reinterpret_cast<T8*>(dst[n] + 8 * at[n] + (MODE == HALF ? rd2 : 0)) = a[n];
            continue;
        }
        if (MODE == HALF) {
            T8 x, y;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const Turn t = w[8 * at[n] + e];
                x[e] = (T)((float)a[n][e] * t.c - (float)b[n][e] * t.s);
                y[e] = (T)((float)b[n][e] * t.c + (float)a[n][e] * t.s);
            }
            *reinterpret_cast<T8*>(dst[n] + 8 * at[n]) = x;
            *reinterpret_cast<T8*>(dst[n] + 8 * at[n] + rd2) = y;
        } else {
            T8 x = a[n];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = 4 * at[n] + e;
                if (j < rd2) {  // (dims past the rotated ones in the last of the turning units stay)
                    const Turn t = w[j];
                    x[2 * e] = (T)((float)a[n][2 * e] * t.c - (float)a[n][2 * e + 1] * t.s);
                    x[2 * e + 1] = (T)((float)a[n][2 * e + 1] * t.c + (float)a[n][2 * e] * t.s);
                }
            }
            *reinterpret_cast<T8*>(dst[n] + 8 * at[n]) = x;
        }
    }
}

// Each row's request by a search of cu in LDS.  (64 requests 1.6 us, 16396 rows 2.3)
__global__ __launch_bounds__(1024) void k_page_positions(const int* __restrict__ cu, const int* __restrict__ dropped, int B,
                                                         int T, const int* pos, int* out) {
    __shared__ int to[PAGE_PLAN_MAX_B + 1];
    for (int b = threadIdx.x; b <= B; b += 1024) to[b] = cu[b];
    __syncthreads();
    for (int t = blockIdx.x * 1024 + threadIdx.x; t < T; t += gridDim.x * 1024) {
        const int b = find_range(to, B, t);
        const bool there = to[b] <= t && t < to[b + 1];
        out[t] = (int)((uint32_t)pos[t] + (there ? (uint32_t)dropped[b] : 0u));
    }
}

template <class T>
void rope_as(const RopeRows& a, hipStream_t st) {
    const int rd2 = a.RD / 2;
    const int mode = a.pairs ? PAIRS : rd2 % 8 == 0 ? HALF : ODD;
    // a head's units: those that turn, and those that are copied (none in place)
    uint32_t turning, copied;
    if (mode == HALF) turning = rd2 / 8, copied = (a.HD - a.RD) / 8;
    else if (mode == PAIRS) turning = (a.RD + 7) / 8, copied = a.HD / 8 - turning;
    else turning = (rd2 + 7) / 8, copied = (a.HD - a.RD + 7) / 8;
    const bool moved = a.q.out != a.q.in || (a.HK && a.k.out != a.k.in);
    const uint32_t units = turning + (moved ? copied : 0), heads = a.HQ + a.HK;
    const size_t per = (size_t)heads * units, total = per * a.rows;
    auto side = [](const RopeHeads& h) {
        return RopeSide<T>{static_cast<const T*>(h.in), static_cast<T*>(h.out), (uint32_t)h.stride, (uint32_t)h.step,
                           (uint32_t)h.ostride, (uint32_t)h.ostep};
    };
    auto launch = [&](auto kernel, int N) {
        const size_t wg = 256 * (size_t)N, slices = (per + wg - 1) / wg;
        const int R = slices > 1 ? 1 : (int)std::min<size_t>(MAX_R, wg / per);
        const size_t groups = (a.rows + R - 1) / R * slices;
        if (groups >= size_t(1) << 24) throw Error("sd_op_rope: too many rows for one launch");
        hipLaunchKernelGGL(kernel, dim3((unsigned)groups), dim3(256), 0, st, a.freqs, a.RD, a.magnitude,
                           a.inverse ? -1.f : 1.f, a.pos, a.rows, a.HD, side(a.q), a.HQ, side(a.k), Div((uint32_t)per), turning, Div(units), R, (uint32_t)slices);
        launched("rope");
    };
    auto sized = [&](auto mode_c) {
        constexpr int M = decltype(mode_c)::value;
        if (total >= 1024 * 512) launch(k_rope<T, M, 4>, 4);
        else launch(k_rope<T, M, 1>, 1);
    };
    if (mode == HALF) sized(std::integral_constant<int, HALF>());
    else if (mode == PAIRS) sized(std::integral_constant<int, PAIRS>());
    else sized(std::integral_constant<int, ODD>());
}

}  // namespace

void rope_table(const double* freqs, int pairs, double magnitude, const int* pos, int n, float* table, hipStream_t st) {
    const uint32_t total = (uint32_t)n * (uint32_t)pairs;
    hipLaunchKernelGGL(k_rope_table, dim3((total + 255) / 256), dim3(256), 0, st, freqs, (uint32_t)pairs, magnitude, pos, total,
                       reinterpret_cast<float2*>(table));
    launched("rope_table");
}

void rope(const RopeRows& a, hipStream_t st) {
    if (a.type == 0) rope_as<f16>(a, st);
    else if (a.type == 1) rope_as<bf16>(a, st);
    else rope_as<float>(a, st);
}

void page_positions(const int* cu, const int* dropped, int B, int T, const int* pos, int* out, hipStream_t st) {
    hipLaunchKernelGGL(k_page_positions, dim3(std::min((T + 1023) / 1024, 128)), dim3(1024), 0, st, cu, dropped, B, T, pos, out);
    launched("page_positions");
}

}  // namespace sd
