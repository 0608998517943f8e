// What the kernels of the paged cache share: the rows' types and their products, a request's part in a launch, blocks of
// 32 rows, and the numerics of the base-2 softmax.
//
// A page holds PS rows (a power of two from 32) of every kv head: K [HK][PS / 32][HD / 32][32 rows][32 dims], V transposed
// [HK][PS / 32][HD][32 rows].  Page p starts `pstride` elements after page p - 1.  Row j of a request lies in page
// table[j / PS] at row j % PS; a table entry outside [0, n_pages) is a hole, whose rows nothing reads or writes.
#pragma once

#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "common.h"
#include "device.h"

namespace sd {
namespace {

constexpr float LOG2E = 1.4426950408889634f;

typedef __bf16 bf16;
template <class T>
struct Vec8;
template <>
struct Vec8<f16> {
    typedef f16x8 type;
};
template <>
struct Vec8<bf16> {
    typedef __bf16 type __attribute__((ext_vector_type(8)));
};

// The last index b of [0, B) with to[b] <= x, for to[0] = 0 <= x < to[B] ascending (empty ranges are passed over).
__device__ __forceinline__ int find_range(const int* to, int B, int x) {
    int lo = 0, hi = B;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (to[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Element offset of (slot, kv head) in a cache whose rows' 32-row blocks hold HD x 32 elements.
template <int HD>
__device__ __forceinline__ size_t block_at(int slot, int kh, int lps, size_t pstride) {
    return (size_t)(slot >> lps) * pstride + ((size_t)kh * (1 << (lps - 5)) + ((slot & ((1 << lps) - 1)) >> 5)) * (HD * 32);
}

// (left to itself the compiler keeps the larger lambdas as calls, and with them their captures in memory)
#define INL __attribute__((always_inline))
// (and it moves work that the products are to cover out from between them: a volatile asm keeps its place)
#if defined(__HIP_DEVICE_COMPILE__)
#define PIN_V(x) asm volatile("" : "+v"(x))
#else
#define PIN_V(x) (void)(x)
#endif

// From here on f32 has no fractions.
constexpr float FAR = 8388608.f;

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// A score as it is before c turns it into c s - m, c s rounded.
__device__ __forceinline__ float less_max(float s, float c, float m) {
#pragma clang fp contract(off)
    const float x = s * c;
    return (x - m) * __builtin_amdgcn_rcpf(c);
}

// The largest of a value and the one 32 lanes away, and of the four 16 lanes apart.  (The swap of a register with itself
// leaves one half's values in both halves of each result.)
__device__ __forceinline__ float max_halves(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t lo = sw[0], hi = sw[1];
    return fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi));
#else
    return x;
#endif
}
__device__ __forceinline__ float max_quarters(float x) {
#if defined(__HIP_DEVICE_COMPILE__)
    const auto sw = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    const uint32_t lo = sw[0], hi = sw[1];
    return max_halves(fmaxf(__builtin_bit_cast(float, lo), __builtin_bit_cast(float, hi)));
#else
    return x;
#endif
}

template <class T>
struct Num;
template <>
struct Num<f16> {
    static constexpr uint32_t EXP = 0x7C00;
    static constexpr float UP = 8.0f;
    static __device__ __forceinline__ f32x4 mfma16(f16x8 a, f16x8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(f16x8 a, f16x8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Num<bf16> {
    static constexpr uint32_t EXP = 0x7F80;
    static constexpr float UP = -16.0f;
    typedef Vec8<bf16>::type B8;
    static __device__ __forceinline__ f32x4 mfma16(B8 a, B8 b, f32x4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ f32x16 mfma32(B8 a, B8 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

// One request's part in a launch, cut to the bounds that the launch is made for.
struct Req {
    int q0;        // its first row
    int n;         // rows to do
    int p0;        // position of its first row
    int kcap;      // keys that may be read
};
__device__ __forceinline__ Req request(const int* __restrict__ cu, const int* __restrict__ kv_lens, int b, int rows,
                                       int max_new, int kcap) {
    const int a = cu[b], e = cu[b + 1], kv = max(kv_lens[b], -(1 << 30));
    Req r;
    r.q0 = min(max(a, 0), rows);
    const int n = min(max(e, r.q0), rows) - r.q0;
    r.n = min(n, max_new);
    r.p0 = kv - n;
    r.kcap = min(kcap, max(kv, 0));
    return r;
}

// The sum over lanes 0 to the own, by moves between lanes: within rows of 16, then from each row's last lane on.
__device__ __forceinline__ int lanes_upto(int x) {
    auto add = [&](auto ctrl, auto rows) {
        x += __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
    };
    using std::integral_constant;
    add(integral_constant<int, 0x111>(), integral_constant<int, 0xF>());  // 1 lane up in each row
    add(integral_constant<int, 0x112>(), integral_constant<int, 0xF>());  // 2
    add(integral_constant<int, 0x114>(), integral_constant<int, 0xF>());  // 4
    add(integral_constant<int, 0x118>(), integral_constant<int, 0xF>());  // 8
    add(integral_constant<int, 0x142>(), integral_constant<int, 0xA>());  // rows 0 and 2 into 1 and 3
    add(integral_constant<int, 0x143>(), integral_constant<int, 0xC>());  // the lower half into the upper
    return x;
}

struct Tile {
    int b, i;  // request and tile in it; b < 0: none
    int x;     // its number
};
// Tile x of the requests' tiles numbered through (tiles(b) of request b, at most 2^24), the last one first.
template <class F>
__device__ __forceinline__ Tile find_tile(int B, int x, F&& of) {
    const int lane = threadIdx.x & 63, per = (B + 63) >> 6;
    if (B == 1) {
        const int total = of(0);
        return {x < total ? 0 : -1, total - 1 - x, total - 1 - x};
    }
    auto tiles = [&](int b) {
        const int n = of(min(b, B - 1));
        return b < B ? n : 0;  // (no branch: several loads in flight)
    };
    // lane l counts requests l, l + 64, ..., the tiles are numbered lane by lane
    // (cut at 2^24 per lane, which row starts that do not ascend could pass: the sums stay in range)
    int own = 0;
#pragma unroll 8
    for (int i = 0; i < per; i++) own = min(own + tiles(64 * i + lane), 1 << 24);
    const int to = lanes_upto(own), total = __builtin_amdgcn_readlane(to, 63);
    if (x >= total) return {-1, 0, 0};
    const int number = x = total - 1 - x;
    const int at = __ffsll((long long)__ballot(to > x)) - 1;
    x -= __builtin_amdgcn_readlane(to, at) - __builtin_amdgcn_readlane(own, at);
    if (per == 1) return {at, x, number};
    for (int i = 0; i < per; i += 64) {  // lane l: request 64 (i + l) + at
        const int n = i + lane < per ? tiles(64 * (i + lane) + at) : 0, t = lanes_upto(n), sum = __builtin_amdgcn_readlane(t, 63);
        if (x < sum) {
            const int l = __ffsll((long long)__ballot(t > x)) - 1;
            return {64 * (i + l) + at, x - (__builtin_amdgcn_readlane(t, l) - __builtin_amdgcn_readlane(n, l)), number};
        }
        x -= sum;
    }
    return {-1, 0, 0};
}

// Weight of a part of a row's keys (a wave's, a split's) whose running maximum is m, where the largest is mx.  A part that
// saw no score above -inf has 0, and its zeros, or its NaN (0 times a value that is not finite), are multiplied like any
// other's: what is seen stays seen, whatever the split.
__device__ __forceinline__ float part_weight(float m, float mx) { return m == -INFINITY ? 0.f : exp2_fast(m - mx); }

// 16 bytes per lane; ONCE: of data that nothing reads again before it has left the caches (the non-temporal hint).
template <bool ONCE>
__device__ __forceinline__ u32x4 load16(Rsrc r, uint32_t voff, uint32_t soff) {
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (ONCE) return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, voff, soff, 2));
#endif
    return buf_b128(r, voff, soff);
}

inline int log2i(int x) { return 31 - __builtin_clz((unsigned)x); }

// f(type tag, head_dim constant)
template <class F>
void by_type(const PagedShape& s, F&& f) {
    auto dims = [&](auto t) {
        if (s.HD == 64) f(t, std::integral_constant<int, 64>());
        else if (s.HD == 128) f(t, std::integral_constant<int, 128>());
        else f(t, std::integral_constant<int, 256>());
    };
    if (s.bf16) dims(bf16());
    else dims(f16());
}

}  // namespace
}  // namespace sd
