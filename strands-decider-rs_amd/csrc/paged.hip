// A K/V cache in pages, shared by many requests: the step's page plan, the norm + rotation + cache write of its new
// rows, and their attention (no counterpart in the reference, whose cache holds one sequence).
//
// A page holds PS rows (a power of two from 32) of every kv head, in the blocks of 32 rows that the engine's own cache
// has: K [HK][PS / 32][HD / 32][32 rows][32 dims], V transposed [HK][PS / 32][HD][32 rows].  Page p starts `pstride`
// elements after page p - 1.  Row j of a request lies in page table[j / PS] at row j % PS; a table entry outside
// [0, n_pages) is a hole, whose rows nothing reads or writes.
#include "paged.h"

namespace sd {
namespace {

// ---- the page plan --------------------------------------------------------------------------------------------------

constexpr int PLAN_T = 1024;  // threads of a plan workgroup

// Two sums side by side over the workgroup: exclusive prefixes of (a, b) in thread order.
__device__ __forceinline__ void scan2(long long& a, long long& b, long long (*ws)[2]) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const long long a0 = a, b0 = b;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long x = __shfl_up(a, o), y = __shfl_up(b, o);
        if (lane >= o) a += x, b += y;
    }
    if (lane == 63) ws[wv][0] = a, ws[wv][1] = b;
    __syncthreads();
    long long pa = 0, pb = 0;
    for (int w = 0; w < wv; w++) pa += ws[w][0], pb += ws[w][1];
    a += pa - a0;
    b += pb - b0;
}

// Every workgroup scans all requests by itself (B counts from L2: cheaper than a second launch or a hand-off between
// workgroups), then takes its share of the rows and of the new table entries.  Nothing that a workgroup reads is
// written by another one: the outputs do not overlap the inputs, and of the table only entries of pages that a request
// had are read and only entries behind them written.
// First come, first admitted: requests 0 .. bad - 1 get their rows and pages, where `bad` is the first one that does
// not fit (rows, free pages, table width) or whose counts are negative.
// Bound by its launch and four barriers: 4.3 us for 8 requests, 5.4 for 384 with 13000 rows.
__global__ __launch_bounds__(PLAN_T) void k_page_plan(const int* __restrict__ lens, const int* __restrict__ news, int B,
                                                      int T, int lps, int n_pages, const int* __restrict__ free_pages,
                                                      const int* __restrict__ n_free, int* table, int max_blocks,
                                                      int* __restrict__ cu, int* __restrict__ kv_lens,
                                                      int* __restrict__ slots, int* __restrict__ pos,
                                                      int* __restrict__ status) {
    __shared__ int rows_to[PAGE_PLAN_MAX_B + 1], pages_to[PAGE_PLAN_MAX_B + 1];
    __shared__ long long ws[PLAN_T / 64][2];
    __shared__ int bad, total[2];
    const int tid = threadIdx.x, per = (B + PLAN_T - 1) / PLAN_T, b0 = tid * per, b1 = min(B, b0 + per);
    const long long nf = min(max(n_free[0], 0), n_pages);
    const long long ps1 = (1ll << lps) - 1;
    if (tid == 0) bad = B, total[0] = total[1] = 0;
    long long r = 0, p = 0;
    auto need = [&](int b, long long& len, long long& n) {
        len = lens[b], n = news[b];
        const bool ok = len >= 0 && n >= 0;
        if (!ok) len = n = 0;
        return ok;
    };
    for (int b = b0; b < b1; b++) {
        long long len, n;
        need(b, len, n);
        r += n;
        p += ((len + n + ps1) >> lps) - ((len + ps1) >> lps);
    }
    scan2(r, p, ws);  // (its barrier is also behind the shared variables' first values)
    const long long r0 = r, p0 = p;
    for (int b = b0; b < b1; b++) {
        long long len, n;
        const bool ok = need(b, len, n);
        const long long want = (len + n + ps1) >> lps;
        r += n;
        p += want - ((len + ps1) >> lps);
        if (!ok || r > T || p > nf || want > max_blocks) {
            atomicMin(&bad, b);
            break;
        }
    }
    __syncthreads();
    const int adm = bad;
    r = r0, p = p0;
    for (int b = b0; b < b1 && b < adm; b++) {
        long long len, n;
        need(b, len, n);
        rows_to[b] = (int)r;
        pages_to[b] = (int)p;
        r += n;
        p += ((len + n + ps1) >> lps) - ((len + ps1) >> lps);
        if (b == adm - 1) total[0] = (int)r, total[1] = (int)p;
    }
    __syncthreads();
    const int R = total[0], N = total[1];
    for (int b = max(b0, adm); b < b1; b++) rows_to[b] = R, pages_to[b] = N;
    if (tid == 0) rows_to[B] = R, pages_to[B] = N;
    __syncthreads();
    if (blockIdx.x == 0) {
        for (int b = tid; b <= B; b += PLAN_T) cu[b] = rows_to[b];
        for (int b = tid; b < B; b += PLAN_T) kv_lens[b] = lens[b] + (rows_to[b + 1] - rows_to[b]);
        if (tid == 0) status[0] = adm, status[1] = R, status[2] = N, status[3] = (int)nf - N;
    }
    const int step = gridDim.x * PLAN_T;
    for (int k = blockIdx.x * PLAN_T + tid; k < N; k += step) {
        const int b = find_range(pages_to, B, k);
        const int have = (int)((lens[b] + ps1) >> lps);
        table[(size_t)b * max_blocks + have + (k - pages_to[b])] = free_pages[nf - 1 - k];
    }
    for (int t = blockIdx.x * PLAN_T + tid; t < T; t += step) {
        int slot = -1, at = 0;
        if (t < R) {
            const int b = find_range(rows_to, B, t);
            const int len = lens[b], have = (int)((len + ps1) >> lps);
            at = len + (t - rows_to[b]);
            const int blk = at >> lps;
            const int page = blk < have ? table[(size_t)b * max_blocks + blk]
                                        : free_pages[nf - 1 - (pages_to[b] + (blk - have))];
            if (page >= 0 && page < n_pages) slot = (int)(((long long)page << lps) + (at & ps1));
        }
        slots[t] = slot;
        pos[t] = at;
    }
}

// ---- norm, rotation and cache write ---------------------------------------------------------------------------------

// The sum over each N adjacent lanes, in all of them.
template <int N>
__device__ __forceinline__ float head_sum(float x) {
    auto dpp = [&](auto ctrl) {
        x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xF, 0xF, false));
    };
    dpp(std::integral_constant<int, 0xB1>());   // lane i and i ^ 1
    dpp(std::integral_constant<int, 0x4E>());   // i ^ 2
    dpp(std::integral_constant<int, 0x141>());  // 7 - i of each 8
    if (N >= 16) dpp(std::integral_constant<int, 0x140>());  // 15 - i of each 16
    if (N >= 32) x += __shfl_xor(x, 16);
    return x;
}

constexpr int VT = 64, VD = 64;  // rows and dims of a V workgroup

// Workgroups [0, nv) transpose V, 64 rows of 64 dims of a kv head each, through LDS, so that 8 consecutive slots go out as
// 16 bytes.  Each of the others does 512 / HD rows of `hpt` q (or k) heads per thread: HD / 8 threads share a row and a
// head, 8 dims each, 4 heads side by side.  The rows' cosines and sines (f32 and gathered by axis: more work than a head)
// come once, through LDS, while each thread's first head is on its way; the next one always is.
// Bound by bytes: 4099 rows of 32 and 8 heads of 128 dims on three axes, 103 MB, 22.4 us, 4.6 TB/s, where a copy makes
// 4.8; 19.6 again and again on the same buffers, which the last-level cache holds in part.  (33.5 us with scalar loads of
// the weights and the angles gathered by every thread.  Two and four heads of a thread in flight at a time cost more
// registers than they hid: 20.2 and 21.9 where one takes 19.8.)
template <class T, int HD>
__global__ __launch_bounds__(256) void k_paged_prep(const T* __restrict__ big, int stride, int q_step,
                                                    const float* __restrict__ qw, const float* __restrict__ kw,
                                                    const float* __restrict__ rope, int rope_len,
                                                    const int* __restrict__ pos, int axes,
                                                    const uint8_t* __restrict__ axis, const int* __restrict__ slots,
                                                    int rows, int HQ, int HK, int RD, int lps, int n_pages,
                                                    size_t pstride, int hpt, int nv, T* __restrict__ Q,
                                                    T* __restrict__ Kp, T* __restrict__ Vp) {
    typedef typename Vec8<T>::type T8;
    constexpr int LPH = HD / 8, R = 512 / HD;
    const int tid = threadIdx.x;
    const int k_off = HQ * q_step, v_off = k_off + HK * HD;
    const long long n_slots = (long long)n_pages << lps;
    if ((int)blockIdx.x >= nv) {
        __shared__ __align__(16) float2 turns[R][HD / 2];
        const int tiles = (rows + R - 1) / R, u = (blockIdx.x - nv) / tiles, t0 = (blockIdx.x - nv) % tiles * R;
        const int gq = (HQ + 4 * hpt - 1) / (4 * hpt);
        const bool isq = u < gq;
        const int c = tid % LPH, r = tid / (4 * LPH), t = min(t0 + r, rows - 1);
        const int heads = isq ? HQ : HK, first = (isq ? u : u - gq) * 4 * hpt, end = min(heads, first + 4 * hpt);
        const int h0 = first + tid / LPH % 4;  // the thread's heads: h0, h0 + 4, ...
        const T* const src = big + (size_t)t * stride + (isq ? 0 : k_off);
        const int step = isq ? q_step : HD;
        auto load = [&](int h) { return *reinterpret_cast<const T8*>(src + (size_t)min(h, heads - 1) * step + 8 * c); };
        T8 next = load(h0);
        const int slot = slots[t];
        const float* const nw = isq ? qw : kw;
        // the pair of dim d: j = d % (RD / 2); its other dim is RD / 2 away
        const int rd2 = RD / 2;
        const bool whole = rd2 % 8 == 0;  // a chunk's others are one chunk
        auto other = [&](int e) { const int d = 8 * c + e; return d < rd2 ? d + rd2 : d < RD ? d - rd2 : d; };
        float w[8], w2[8];  // the weights of the thread's dims and of their others
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = w2[e] = 1.f;
        if (nw && whole) {
            typedef float F4 __attribute__((ext_vector_type(4), aligned(4)));
            const F4* const a = reinterpret_cast<const F4*>(nw + 8 * c);
            const F4* const b = reinterpret_cast<const F4*>(nw + other(0));
            const F4 v[4] = {a[0], a[1], b[0], b[1]};
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = v[e >> 2][e & 3], w2[e] = v[2 + (e >> 2)][e & 3];
        } else if (nw) {
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = nw[8 * c + e], w2[e] = nw[other(e)];
        }
        for (int i = tid; i < R * rd2; i += 256) {
            const int y = i / rd2, j = i % rd2, ty = min(t0 + y, rows - 1);
            int at[4];
#pragma unroll
            for (int a = 0; a < 4; a++) at[a] = a < axes ? pos[(size_t)a * rows + ty] : 0;
            const int b = axes > 1 ? axis[j] : 0;
            const int p = axes == 1 || b == 0 ? at[0] : min(b, axes - 1) == 1 ? at[1] : min(b, axes - 1) == 2 ? at[2] : at[3];
            turns[y][j] = *reinterpret_cast<const float2*>(rope + ((size_t)min(max(p, 0), rope_len - 1) * rd2 + j) * 2);
        }
        __syncthreads();
        // a result is (x cs + x' sn) / rms, x' its other dim, cs and sn with the weights in them
        float cs[8], sn[8];
#pragma unroll
        for (int e = 0; e < 8; e++) cs[e] = 1.f, sn[e] = 0.f;
        if (whole && 8 * c < RD) {
            const f32x4* const p = reinterpret_cast<const f32x4*>(&turns[r][8 * c < rd2 ? 8 * c : 8 * c - rd2]);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const f32x4 v = p[e];
                cs[2 * e] = v[0], sn[2 * e] = v[1], cs[2 * e + 1] = v[2], sn[2 * e + 1] = v[3];
            }
        } else if (!whole) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int d = 8 * c + e;
                if (d < RD) cs[e] = turns[r][d < rd2 ? d : d - rd2].x, sn[e] = turns[r][d < rd2 ? d : d - rd2].y;
            }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
            cs[e] *= w[e];
            sn[e] *= 8 * c + e < rd2 ? -w2[e] : w2[e];
        }
        if (t0 + r >= rows || slot < 0 || slot >= n_slots) return;
        for (int h = h0; h < end; h += 4) {
            const T8 x8 = next;
            if (h + 4 < end) next = load(h + 4);
            T8 o8;
            if (whole) {
                const int s = rd2 / 8, from = c < s ? c + s : c - s;
                const u32x4 v = __builtin_bit_cast(u32x4, x8);
                u32x4 o;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const uint32_t y = __shfl(v[e], from, LPH);
                    o[e] = 8 * c < RD ? y : 0;
                }
                o8 = __builtin_bit_cast(T8, o);
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) o8[e] = 8 * c + e < RD ? src[(size_t)h * step + other(e)] : (T)0.f;
            }
            float inv = 1.f;
            if (nw) {
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) ss += (float)x8[e] * (float)x8[e];
                inv = __builtin_amdgcn_rsqf(head_sum<LPH>(ss) * (1.0f / HD) + 1e-6f);
            }
            T8 y8;
#pragma unroll
            for (int e = 0; e < 8; e++) y8[e] = (T)(((float)x8[e] * cs[e] + (float)o8[e] * sn[e]) * inv);
            if (isq) *reinterpret_cast<T8*>(Q + ((size_t)t * HQ + h) * HD + 8 * c) = y8;
            else
                *reinterpret_cast<T8*>(Kp + block_at<HD>(slot, h, lps, pstride) + (c / 4) * 1024 + (slot & 31) * 32 + 8 * (c % 4)) = y8;
        }
        return;
    }
    __shared__ __align__(16) T tile[VT][VD + 8];
    __shared__ int sl[VT];
    __shared__ int cut, whole8[VT / 8 + 1];
    const int v = blockIdx.x, d0 = v % (HD / VD) * VD, kh = v / (HD / VD) % HK, t0 = v / (HD / VD) / HK * VT, nt = min(VT, rows - t0);
    T8 y8[VT * VD / 8 / 256];
#pragma unroll
    for (int i = 0; i < VT * VD / 8 / 256; i++) {
        const int x = tid + 256 * i;
        y8[i] = *reinterpret_cast<const T8*>(big + (size_t)(t0 + min(x / (VD / 8), nt - 1)) * stride + v_off + kh * HD + d0 + 8 * (x % (VD / 8)));
    }
    if (tid < VT) {  // (the first wave)
        const int s = tid < nt ? slots[t0 + tid] : -1, mine = s >= 0 && s < n_slots ? s : -1;
        sl[tid] = mine;
        // octets of rows cut where the slots of the first request here are multiples of 8: which of them are 8 slots on end
        const unsigned long long any = __ballot(mine >= 0);
        const int first = any ? __ffsll((long long)any) - 1 : 0, s0 = __shfl(mine, first);
        const int c = s0 < 0 ? 0 : ((first - s0) & 7) - 8, before = __shfl_up(mine, 1);
        const unsigned long long next = __ballot(tid > 0 && mine == before + 1);
        const int r0 = c + 8 * tid, at = __shfl(mine, min(max(r0, 0), VT - 1));
        if (tid < VT / 8 + 1)
            whole8[tid] = r0 >= 0 && r0 + 7 < VT && at >= 0 && at % 8 == 0 && (next >> (r0 + 1) & 127) == 127;
        if (tid == 0) cut = c;
    }
#pragma unroll
    for (int i = 0; i < VT * VD / 8 / 256; i++) {
        const int x = tid + 256 * i;
        *reinterpret_cast<T8*>(&tile[x / (VD / 8)][8 * (x % (VD / 8))]) = y8[i];
    }
    __syncthreads();
    for (int i = tid; i < VD * (VT / 8 + 1); i += 256) {
        const int d = i / (VT / 8 + 1), o = i % (VT / 8 + 1), r0 = cut + 8 * o;
        if (whole8[o]) {
            T8 y;
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = tile[r0 + e][d];
            *reinterpret_cast<T8*>(Vp + block_at<HD>(sl[r0], kh, lps, pstride) + (d0 + d) * 32 + (sl[r0] & 31)) = y;
        } else {
            for (int r = max(r0, 0); r < min(r0 + 8, nt); r++)
                if (sl[r] >= 0) Vp[block_at<HD>(sl[r], kh, lps, pstride) + (d0 + d) * 32 + (sl[r] & 31)] = tile[r][d];
        }
    }
}

// ---- attention ------------------------------------------------------------------------------------------------------
//
// A kv head's rows are its request's (token, query head) pairs, token-major: row r is token r / G and head kh G + r % G,
// G = HQ / HK, so that all query heads of a kv head share each key that is fetched.  Scores are S^T = K Q^T (keys x
// rows) on MFMA with the keys of a 32-row block ordered so that S^T's accumulator layout is the B operand's of O^T +=
// V^T P^T: probabilities never move between lanes, and both operands come out of the cache's blocks 16 bytes at a time.
//
// The online softmax is in base 2 and f32: p = 2^(c s - m + UP), c = scale log2(e), m the running maximum of c s.  P is
// rounded to the rows' type before the second product (f32 sums; the row sum takes the unrounded values): half a step
// of the type relative to each weight, as the result's own rounding.  m is raised, and O and the sum rescaled, only
// when a block's maximum exceeds it by more than 6, so p stays below 2^(UP + 7) and most blocks rescale nothing.  f16's
// UP is 8: its normal range then is at weights down to 2^-22 of the largest (30000 keys of 2^-22 each are 0.7 % of a
// result), and p within it.  bf16, whose range is f32's, has -16: sums of a thousand of the type's largest values stay in
// range, and weights down to 2^-110.  From FAR on, where f32 has no fractions left, m and c s in the exponent's one rounding
// would be apart by more than p's range: there c s is rounded as m was, and the difference taken first (a wave whose m
// are all nearer, as good as ever, skips it).
//
// A masked product is 0 times the value, which is NaN where that is not finite.  Blocks that some row does not see
// whole (the diagonal, a window's edge, the last block) look at their values first; where one is not finite, the
// products take it as 0, and where some row sees it, the rows that do add it at the end, element by element, in those
// blocks alone (add_seen).  (Cache rows behind a request's last that were never written may be NaN: 64 requests of 1000
// to 8191 keys take 144 us with them and without; with a look at every block at the end 697.)

constexpr float RAISE = 6.0f;

// Nonzero where one of 8 values is not finite (its exponent's bits all set: one more carries into the sign's place).
template <class T>
__device__ __forceinline__ uint32_t not_finite(u32x4 v) {
    constexpr uint32_t M = Num<T>::EXP * 0x10001u, A = (0x8000u - Num<T>::EXP) * 0x10001u;
    uint32_t r = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) r |= (v[i] & M) + A;
    return r & 0x80008000u;
}
// 8 values with 0 in the place of those that are not finite.
template <class T>
__device__ __forceinline__ u32x4 finite8(u32x4 v) {
    constexpr uint32_t M = Num<T>::EXP * 0x10001u, A = (0x8000u - Num<T>::EXP) * 0x10001u;
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = v[i] & ~(((((v[i] & M) + A) & 0x80008000u) >> 15) * 0xFFFFu);
    return r;
}

// All bits of the values of keys j to j + 7 that are in [lo, hi).
__device__ __forceinline__ u32x4 keys_within(int j, int lo, int hi) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; i++)
        r[i] = (j + 2 * i >= lo && j + 2 * i < hi ? 0xFFFFu : 0u) | (j + 2 * i + 1 >= lo && j + 2 * i + 1 < hi ? 0xFFFF0000u : 0u);
    return r;
}

// The launch's arguments that all attention kernels share.
struct AttnArgs {
    const int *table, *cu, *kv_lens;
    int max_blocks, B, rows, HQ, HK, G, lps, n_pages, max_new, kcap, window, stride;
    int few, few_ks, few_span;       // rows of a request that k_paged_few does, its splits and the blocks in each
    int tiles, rows_ks, rows_span;   // of k_paged_rows
    float c;  // scale log2(e)
    size_t pstride;
    // the first key that a row at position p sees (one before position 0 sees none, whatever this says)
    __device__ __forceinline__ int from(int p) const { return window ? max(p, -1) - window + 1 : 0; }
};

// Output of 4 dims of a row: unnormalised o over the sum l, times the sigmoid of its gates where it has some, rounded once.
template <class T>
__device__ __forceinline__ void finish4(f32x4 o, float l, bool gated, u32x2 gate, T* out) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    const T4 v = __builtin_bit_cast(T4, gate);
    T4 r;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float sg = gated ? __builtin_amdgcn_rcpf(1.0f + exp2_fast((float)v[e] * -LOG2E)) : 1.f;
        r[e] = (T)((l == 0.f ? 0.f : o[e] * inv) * sg);
    }
    *reinterpret_cast<T4*>(out) = r;
}
template <class T>
__device__ __forceinline__ u32x2 gate4(const T* big, size_t at) {
    return big ? *reinterpret_cast<const u32x2*>(big + at) : u32x2{0, 0};
}

// ---- few rows: up to 16 NR rows per (request, kv head), one new token's heads or a short draft's ----
//
// Bound by the cache's bytes: each is read once and used for a handful of rows.  The keys are split over workgroups
// (span blocks of 32 each) and inside one over its NW waves, block by block; a wave loads K and V straight into registers
// in MFMA operand order, 16 rows on v_mfma_f32_16x16x32, the next block while it works on one (LDS would be a second trip
// for bytes that one wave alone uses).  64 requests of 1000 to 8191 keys, 32 and 8 heads of 128 dims, 776 MB: 143 us, 5.4
// TB/s; two of 90 and 131 thousand, 8 and 2 heads of 256 dims: 79 us, 6.2 TB/s.  A CU alone draws 60 GB/s, so short
// caches are split as far as a join lets them: 700 keys of those heads 9.0 us, launches and two trips to memory.
template <int HD, int NR>
constexpr int few_waves() { return HD * NR <= 128 ? 8 : 4; }  // 8 where two fit a SIMD's registers (157 -> 143)
// Workgroup x of request b, of NW waves: om(w) gives LDS of R x HD floats for each wave, Ms and Ls are R of them per wave.
template <class T, int HD, int NR, bool ONCE, int NW, class Om>
__device__ __forceinline__ void few_part(const int x, const int b, const T* __restrict__ Q, const T* __restrict__ Kp,
                                         const T* __restrict__ Vp, const AttnArgs& a, const T* __restrict__ big,
                                         T* __restrict__ out, float* __restrict__ pacc, float* __restrict__ pml, Om om,
                                         float* Ms, float* Ls) {
    typedef typename Vec8<T>::type T8;
    constexpr int NS = HD / 32, ND = HD / 16, R = 16 * NR, D = 2;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int fq = lane & 15, fg = lane >> 4;
    const int kh = x % a.HK, z = x / a.HK;
    const Req rq = request(a.cu, a.kv_lens, b, a.rows, a.max_new, a.kcap);
    const int nrows = rq.n * a.G;
    if (nrows == 0 || nrows > a.few) return;
    // keys [lo, hi) are seen by some row; this workgroup's blocks of them
    const int hi = min(rq.p0 + rq.n, rq.kcap), lo = max(0, a.from(rq.p0));
    const int blk0 = (lo >> 5) + z * a.few_span;
    const int blk1 = z + 1 < a.few_ks ? min((hi + 31) >> 5, blk0 + a.few_span) : (hi + 31) >> 5;
    const int first = blk0 + wv, cnt = first < blk1 ? (blk1 - first + NW - 1) / NW : 0;
    int jlo[NR], jhi[NR];  // keys [jlo, jhi) are seen by this lane's row
    T8 qf[NR][NS];
#pragma unroll
    for (int u = 0; u < NR; u++) {
        const int r = min(16 * u + fq, nrows - 1), t = r / a.G, h = kh * a.G + r % a.G;
        const int p = rq.p0 + t;
        jlo[u] = a.from(p);
        jhi[u] = min(p + 1, hi);
        const T* q = Q + ((size_t)(rq.q0 + t) * a.HQ + h) * HD + 8 * fg;
#pragma unroll
        for (int s = 0; s < NS; s++) qf[u][s] = *reinterpret_cast<const T8*>(q + 32 * s);
    }
    // blocks in [open0, open1) are seen whole by every row
    const int open0 = a.from(rq.p0 + rq.n - 1), open1 = min(rq.p0 + 1, hi);

    const int lbpp = a.lps - 5;
    const int* const tb = a.table + (size_t)b * a.max_blocks;
    auto entries = [&](int i) {  // lane l: the table entry of the wave's block i + l
        return tb[min((first + NW * (i + lane)) >> lbpp, a.max_blocks - 1)];
    };
    int ids = cnt ? entries(0) : 0, ids2 = cnt > 64 ? entries(64) : 0;
    const uint32_t kofs = ((8 * (fq >> 2) + (fq & 3)) * 32 + fg * 8) * 2, vofs = (fq * 32 + fg * 8) * 2;
    f32x4 acc[NR][ND];
    float m[NR], l[NR];
#pragma unroll
    for (int u = 0; u < NR; u++) {
        m[u] = -INFINITY, l[u] = 0.f;
#pragma unroll
        for (int d = 0; d < ND; d++) acc[u][d] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    bool rare = false;  // some value that is seen was taken as 0
    struct Blk {
        u32x4 k[2][NS], v[ND];
        bool there;
    };
    auto load = [&](int i, Blk& x) INL {
        const int page = __builtin_amdgcn_readlane(ids, i & 63), blk = first + NW * i;
        x.there = i < cnt && (unsigned)page < (unsigned)a.n_pages;
        const size_t at = x.there ? (size_t)page * a.pstride + ((size_t)(kh << lbpp) + (blk & ((1 << lbpp) - 1))) * (HD * 32) : 0;
        const Rsrc rk = make_rsrc(Kp + at, x.there ? HD * 64u : 0u), rv = make_rsrc(Vp + at, x.there ? HD * 64u : 0u);
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int tt = 0; tt < 2; tt++) x.k[tt][s] = load16<ONCE>(rk, kofs + tt * 256, s * 2048);
#pragma unroll
        for (int d = 0; d < ND; d++) x.v[d] = load16<ONCE>(rv, vofs, d * 1024);
    };
    auto work = [&](int i, Blk& x) INL {
        const int j0 = (first + NW * i) * 32;
        const bool open = x.there && j0 >= open0 && j0 + 32 <= open1;
        f32x4 s2[NR][2];
#pragma unroll
        for (int u = 0; u < NR; u++) s2[u][0] = s2[u][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int tt = 0; tt < 2; tt++)
#pragma unroll
                for (int u = 0; u < NR; u++)
                    s2[u][tt] = Num<T>::mfma16(__builtin_bit_cast(T8, x.k[tt][s]), qf[u][s], s2[u][tt]);
        if (!open) {
#pragma unroll
            for (int u = 0; u < NR; u++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int j = j0 + 8 * fg + e;
                    const bool keep = x.there & (j >= jlo[u]) & (j < jhi[u]);
                    s2[u][e >> 2][e & 3] = keep ? s2[u][e >> 2][e & 3] : -INFINITY;
                }
        }
        float tmax[NR];
        bool up = false;
#pragma unroll
        for (int u = 0; u < NR; u++) {
            tmax[u] = s2[u][0][0];
#pragma unroll
            for (int e = 1; e < 8; e++) tmax[u] = fmaxf(tmax[u], s2[u][e >> 2][e & 3]);
            tmax[u] = max_quarters(tmax[u]) * a.c;
            up |= tmax[u] - m[u] > RAISE;
        }
        if (__any(up)) {
#pragma unroll
            for (int u = 0; u < NR; u++) {
                const float mn = fmaxf(m[u], tmax[u]), f = m[u] == -INFINITY ? 0.f : exp2_fast(m[u] - mn);
                m[u] = mn;
                l[u] *= f;
#pragma unroll
                for (int d = 0; d < ND; d++)
#pragma unroll
                    for (int e = 0; e < 4; e++) acc[u][d][e] *= f;
            }
        }
        float nm[NR];
        bool far = false;
#pragma unroll
        for (int u = 0; u < NR; u++) nm[u] = m[u] == -INFINITY ? 0.f : Num<T>::UP - m[u], far |= fabsf(nm[u]) >= FAR;
        if (__builtin_expect(__any(far), 0)) {
#pragma unroll
            for (int u = 0; u < NR; u++)
                if (fabsf(nm[u]) >= FAR) {
                    nm[u] = Num<T>::UP;
#pragma unroll
                    for (int e = 0; e < 8; e++) s2[u][e >> 2][e & 3] = less_max(s2[u][e >> 2][e & 3], a.c, m[u]);
                }
        }
        T8 pf[NR];
#pragma unroll
        for (int u = 0; u < NR; u++) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float p = exp2_fast(__builtin_fmaf(s2[u][e >> 2][e & 3], a.c, nm[u]));
                l[u] += p;
                pf[u][e] = (T)p;
            }
        }
        if (!open) {
            uint32_t odd = 0;
#pragma unroll
            for (int d = 0; d < ND; d++) odd |= not_finite<T>(x.v[d]);
            if (__builtin_expect(__any(odd != 0), 0)) {
                const u32x4 some = keys_within(j0 + 8 * fg, lo, hi);  // (seen by some row)
                odd = 0;
#pragma unroll
                for (int d = 0; d < ND; d++) x.v[d] &= some, odd |= not_finite<T>(x.v[d]);
                if (__any(odd != 0)) {
                    rare = true;
#pragma unroll
                    for (int d = 0; d < ND; d++) x.v[d] = finite8<T>(x.v[d]);
                }
            }
        }
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int u = 0; u < NR; u++) acc[u][d] = Num<T>::mfma16(__builtin_bit_cast(T8, x.v[d]), pf[u], acc[u][d]);
    };
    // D blocks' registers: block i is in set i % D, and while it is worked on the D - 1 after it are on their way
    Blk set[D];
    auto ahead = [&](int i) INL {  // before block i's load: its window of table entries
        if ((i & 63) == 0 && i) {
            ids = ids2;
            if (i + 64 < cnt) ids2 = entries(i + 64);
        }
    };
#pragma unroll
    for (int u = 0; u < D - 1; u++) load(u, set[u]);
    for (int i = 0; i < cnt; i += D) {
#pragma unroll
        for (int u = 0; u < D; u++) {
            if (u && i + u >= cnt) break;
            ahead(i + u + D - 1);
            load(i + u + D - 1, set[(u + D - 1) % D]);
            __builtin_amdgcn_sched_barrier(0);
            work(i + u, set[u]);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    if (__builtin_expect(rare, 0)) {  // add_seen: see above
#pragma unroll 1
        for (int i = 0; i < cnt; i++) {
            const int blk = first + NW * i, page = tb[blk >> lbpp], j0 = 32 * blk;
            if ((unsigned)page >= (unsigned)a.n_pages || (j0 >= open0 && j0 + 32 <= open1)) continue;
            const T* const v = Vp + (size_t)page * a.pstride + ((size_t)(kh << lbpp) + (blk & ((1 << lbpp) - 1))) * (HD * 32);
#pragma unroll 1
            for (int j = j0; j < j0 + 32; j++)
#pragma unroll
                for (int u = 0; u < NR; u++)
                    if (j >= jlo[u] && j < jhi[u]) {
#pragma unroll
                        for (int d = 0; d < ND; d++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                const float x = (float)v[(16 * d + 4 * fg + e) * 32 + (j & 31)];
                                if (!__builtin_isfinite(x)) acc[u][d][e] += x;
                            }
                    }
        }
    }
    // the waves' states side by side: acc[u][d][e] is O[row 16 u + fq][dim 16 d + 4 fg + e].  (4 dims
    // at their place ^ row % 16, so that neither side meets a bank twice)
    float* const mine = om(wv);
#pragma unroll
    for (int u = 0; u < NR; u++) {
        l[u] += __shfl_xor(l[u], 16);
        l[u] += __shfl_xor(l[u], 32);
#pragma unroll
        for (int d = 0; d < ND; d++) *reinterpret_cast<f32x4*>(mine + (16 * u + fq) * HD + 4 * ((4 * d + fg) ^ fq)) = acc[u][d];
        if (fg == 0) Ms[wv * R + 16 * u + fq] = m[u], Ls[wv * R + 16 * u + fq] = l[u];
    }
    __syncthreads();
    for (int i = tid; i < nrows * (HD / 4); i += 64 * NW) {
        const int r = i / (HD / 4), d = 4 * (i % (HD / 4));
        float mx = -INFINITY, ls = 0.f;
#pragma unroll
        for (int w = 0; w < NW; w++) mx = fmaxf(mx, Ms[w * R + r]);
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; w++) {
            const float f = part_weight(Ms[w * R + r], mx);
            ls += Ls[w * R + r] * f;
            const f32x4 x = *reinterpret_cast<const f32x4*>(om(w) + r * HD + (d ^ 4 * (r & 15)));
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] += x[e] * f;
        }
        const int t = rq.q0 + r / a.G, h = kh * a.G + r % a.G;
        const size_t row = (size_t)t * a.HQ + h;
        if (a.few_ks == 1) {
            finish4<T>(o, ls, big, gate4(big, (size_t)t * a.stride + h * 2 * HD + HD + d), out + row * HD + d);
        } else {
            const size_t pr = (size_t)z * a.rows * a.HQ + row;
            *reinterpret_cast<f32x4*>(pacc + pr * HD + d) = o;
            if (d == 0) pml[2 * pr] = mx, pml[2 * pr + 1] = ls;
        }
    }
}

template <class T, int HD, int NR, bool ONCE>
__global__ __launch_bounds__((64 * few_waves<HD, NR>())) void k_paged_few(const T* __restrict__ Q, const T* __restrict__ Kp,
                                                                          const T* __restrict__ Vp, AttnArgs a,
                                                                          const T* __restrict__ big, T* __restrict__ out,
                                                                          float* __restrict__ pacc,
                                                                          float* __restrict__ pml) {
    constexpr int NW = few_waves<HD, NR>(), R = 16 * NR;
    __shared__ __align__(16) float Om[NW][R * HD];
    __shared__ float Ms[NW * R], Ls[NW * R];
    few_part<T, HD, NR, ONCE, NW>(blockIdx.x, blockIdx.y, Q, Kp, Vp, a, big, out, pacc, pml, [&](int w) { return Om[w]; }, Ms,
                                  Ls);
}

// Joins up to 64 splits of one row and writes it: 256 threads, HD / 4 of them side by side (4 dims each), their groups
// each every so many splits.  Every split of a row has written its maximum, sum and output, zeros where it saw no key.
constexpr int MAX_KS = 64;
template <class T, int HD>
__global__ __launch_bounds__(256) void k_paged_join_few(AttnArgs a, const float* __restrict__ pacc,
                                                        const float* __restrict__ pml, const T* __restrict__ big,
                                                        T* __restrict__ out, int rows_max) {
    constexpr int W = HD / 4, NG = 256 / W;
    __shared__ float wt[MAX_KS];
    __shared__ f32x4 part[NG][W];
    const int tid = threadIdx.x, lane = tid & 63;
    const int kh = blockIdx.x / rows_max, r = blockIdx.x % rows_max;
    const Req rq = request(a.cu, a.kv_lens, blockIdx.y, a.rows, a.max_new, a.kcap);
    const int nrows = rq.n * a.G;
    if (r >= nrows || nrows > a.few) return;
    const int t = rq.q0 + r / a.G, h = kh * a.G + r % a.G, d = 4 * (tid % W);
    const size_t row = (size_t)t * a.HQ + h, zs = (size_t)a.rows * a.HQ;
    const u32x2 gate = gate4(big, (size_t)t * a.stride + h * 2 * HD + HD + d);
    // (every wave for itself, the same)
    const float2 ml = lane < a.few_ks ? *reinterpret_cast<const float2*>(pml + 2 * (lane * zs + row)) : float2{-INFINITY, 0.f};
    float mx = ml.x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
    const float f = part_weight(ml.x, mx);
    float ls = ml.y * f;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) ls += __shfl_xor(ls, o);
    if (tid < 64) wt[lane] = f;
    __syncthreads();
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int z = tid / W; z < a.few_ks; z += NG) {
        const f32x4 x = *reinterpret_cast<const f32x4*>(pacc + (z * zs + row) * HD + d);
        const float w = wt[z];
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] += x[e] * w;
    }
    part[tid / W][tid % W] = o;
    __syncthreads();
    if (tid >= W) return;
#pragma unroll
    for (int g = 1; g < NG; g++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] += part[g][tid][e];
    finish4<T>(o, ls, big, gate, out + row * HD + d);
}

// ---- many rows: 128 rows of a kv head per workgroup ----
//
// Bound by MFMA and the softmax beside it: each wave has 32 rows on v_mfma_f32_32x32x16, its queries and outputs in
// registers, and all 4 share blocks of 32 keys that arrive by LDS DMA, three ahead.  A block's probabilities run between
// the products of the next one's scores and of its own output.  A prompt of 8192 tokens, 8 and 2 heads of 256 dims: 291
// to 303 us, up to 945 TFLOP/s; four chunks of 2048 on 2048 to 8192 old keys, 32 and 8 heads of 128 dims: 508 to 530 us,
// up to 1040 TFLOP/s, where
// a library product of 8192^3 makes 1200.  MFMA is busy half of the cycles, the softmax's vector instructions (half of
// them 16 exponentials of 16 cycles per block) the other half, and the power limit sets the clock: 2.0 GHz on random data,
// while zeros take 252 and 408 us.  Fragments read a step ahead, which probabilities run where, and wave priorities
// change 1 %.
// Workgroup x of the launch is kv head x % HK (with 8 heads, one per XCD's L2), split and tile; the tiles of all
// requests with more than `few` rows are numbered through, and taken from the last on: a causal chunk's late tiles are
// the long ones.  (Each workgroup finds its tile by itself, from all requests: 1086 us for 8192 requests of 20 new tokens
// on 300 keys, 8 and 2 heads of 128 dims, whose keys and values alone are 455.)
constexpr int TILE_ROWS = 128;
__device__ __forceinline__ Tile find_tile(const AttnArgs& a, int x) {
    return find_tile(a.B, x, [&](int b) {
        const int n = request(a.cu, a.kv_lens, b, a.rows, a.max_new, a.kcap).n * a.G;
        return n > a.few ? (n + TILE_ROWS - 1) / TILE_ROWS : 0;
    });
}

// FEW (2: with the non-temporal hint): the launch ends with the workgroups of the requests with few rows, which would
// otherwise wait for the last tile while most of the chip is idle.  us in a launch of their own and in this one: a chunk
// of 1501 tokens and 40 single ones, window 1024, 16 and 4 heads of 128 dims 42.8 and 31.1; 512 tokens among 64 single
// ones, 32 and 8 heads 186 and 174; 1024 among 32, 8 and 2 heads of 256 dims 85.6 and 61.6.
template <class T, int HD, int FEW>
__global__ __launch_bounds__(256, HD < 256 ? 2 : 1) void k_paged_rows(const T* __restrict__ Q, const T* __restrict__ Kp,
                                                       const T* __restrict__ Vp, AttnArgs a, const T* __restrict__ big,
                                                       T* __restrict__ out, float* __restrict__ pacc,
                                                       float* __restrict__ pml) {
    typedef typename Vec8<T>::type T8;
    constexpr int NS = HD / 16, ND = HD / 32, NB = 4;
    constexpr int BB = HD * 64;        // bytes of a block's K (or V)
    constexpr int PART = BB / 4;   // bytes of it that one wave fetches
    constexpr int IW = PART / 1024;  // in so many DMAs
    // (an array per buffer: the compiler then sees that the DMAs into one never alias the reads of another)
    __shared__ __align__(1024) uint8_t K0[BB], K1[BB], K2[BB], K3[BB], V0[BB], V1[BB], V2[BB], V3[BB];
    __shared__ int rare;  // some value that is seen was taken as 0
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, g = lane >> 5;
    if constexpr (FEW != 0) {
        const int x = (int)blockIdx.x - a.tiles * a.HK * a.rows_ks, per = a.HK * a.few_ks;
        if (x >= 0) {  // (a wave's states fit a block's buffer)
            few_part<T, HD, 1, FEW == 2, 4>(
                x % per, x / per, Q, Kp, Vp, a, big, out, pacc, pml,
                [&](int w) { return reinterpret_cast<float*>(w & 2 ? (w & 1 ? K3 : K2) : (w & 1 ? K1 : K0)); },
                reinterpret_cast<float*>(V0), reinterpret_cast<float*>(V1));
            return;
        }
    }
    const int kh = blockIdx.x % a.HK, z = blockIdx.x / a.HK % a.rows_ks;
    const Tile tl = find_tile(a, blockIdx.x / (a.HK * a.rows_ks));
    if (tl.b < 0) return;
    const Req rq = request(a.cu, a.kv_lens, tl.b, a.rows, a.max_new, a.kcap);
    const int nrows = rq.n * a.G, r0 = tl.i * TILE_ROWS, r1 = min(nrows, r0 + TILE_ROWS);
    const int w0 = r0 + 32 * wv, w1 = min(w0 + 32, r1);  // the wave's rows
    const bool live = w0 < r1;
    // keys seen by some row of the workgroup, and this split's blocks of them
    const int hi = min(rq.p0 + (r1 - 1) / a.G + 1, rq.kcap);
    const int lo = max(0, a.from(rq.p0 + r0 / a.G));
    const int blk0 = (lo >> 5) + z * a.rows_span, blk1 = z + 1 < a.rows_ks ? min((hi + 31) >> 5, blk0 + a.rows_span) : (hi + 31) >> 5;
    const int nb = max(blk1 - blk0, 0);
    // the lane's row (one past the last is the last again, also in the output) and the keys [jlo, jhi) that it sees
    const int r = min(w0 + c, r1 - 1), t = r / a.G, h = kh * a.G + r % a.G;
    const int jlo = a.from(rq.p0 + t), jhi = min(rq.p0 + t + 1, hi);
    // the keys that every row of the wave, and of the workgroup, sees
    const int all0 = a.from(rq.p0 + (w1 - 1) / a.G), all1 = min(rq.p0 + w0 / a.G + 1, hi);
    const int wg0 = a.from(rq.p0 + (r1 - 1) / a.G), wg1 = min(rq.p0 + r0 / a.G + 1, hi);
    if (tid == 0) rare = 0;

    const int lbpp = a.lps - 5;
    const int* const tb = a.table + (size_t)tl.b * a.max_blocks;
    // Lane l: where block `win` + l begins in a cache (bytes; the sign bit where it is not there: past the last block, in
    // a hole), and the same 32 blocks on.  The blocks in use at a time are less than 32 apart.
    int win = 0;
    struct Where {
        uint32_t lo, hi;
    };
    auto entries = [&](int j) INL {
        const int blk = blk0 + j + lane, page = tb[min(blk >> lbpp, a.max_blocks - 1)];
        const bool there = (unsigned)page < (unsigned)a.n_pages && blk < blk1;
        const size_t off = ((size_t)page * a.pstride + ((size_t)(kh << lbpp) + (blk & ((1 << lbpp) - 1))) * (HD * 32)) * 2;
        return Where{(uint32_t)off, there ? (uint32_t)(off >> 32) : 0x80000000u};
    };
    Where wh{0, 0x80000000u}, wh2{0, 0x80000000u};
    if (nb > 0) wh = entries(0), wh2 = entries(32);
    auto is_there = [&](int j) INL { return (int)__builtin_amdgcn_readlane(wh.hi, j - win) >= 0; };
    // block j of a cache: where it is not there nothing is read, and zeros come
    struct At {
        uint32_t lo, hi;
    };
    auto find = [&](int j) INL { return At{(uint32_t)__builtin_amdgcn_readlane(wh.lo, j - win), (uint32_t)__builtin_amdgcn_readlane(wh.hi, j - win)}; };
    auto block = [&](At w, const T* C) INL {
        const uint32_t lo = __builtin_amdgcn_readfirstlane(w.lo), hi = __builtin_amdgcn_readfirstlane(w.hi);
        return make_rsrc(reinterpret_cast<const uint8_t*>(C) + ((uint64_t)(hi & 0x7FFFFFFFu) << 32 | lo), (int)hi < 0 ? 0 : BB);
    };
    const uint32_t dlane = (uint32_t)((lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 4) & 3)) << 4));
    // A block of a cache into an LDS buffer: the wave's quarter, 16 bytes per lane, the 16-byte pieces
    // of each 64-byte row at p ^ (row / 4) % 4 (fragment reads then meet no bank twice).  Every call is the same DMAs.
    const int part = wv * PART;
    auto dma = [&](Rsrc rs, int u, uint8_t* buf) INL { buf_lds16(rs, dlane, part + u * 1024, buf + part + u * 1024); };
    auto fetch = [&](At w, const T* C, uint8_t* buf) INL {
        const Rsrc rs = block(w, C);
#pragma unroll
        for (int u = 0; u < IW; u++) dma(rs, u, buf);
    };
    T8 qf[NS];
    {
        const T* p = Q + ((size_t)(rq.q0 + t) * a.HQ + h) * HD + 8 * g;
#pragma unroll
        for (int s = 0; s < NS; s++) {
            qf[s] = *reinterpret_cast<const T8*>(p + 16 * s);
#if defined(__HIP_DEVICE_COMPILE__)
            if constexpr (HD == 256) asm("" : "+a"(qf[s]));  // (an MFMA reads AGPRs as it reads VGPRs)
#endif
        }
    }
    // row i of S^T is key 16 (i / 16) + 8 (i / 4 % 2) + 4 (i / 8 % 2) + i % 4 of its block: lane (row c, half g) then
    // has keys 16 k + 8 g + e in registers 8 k + e
    const int kperm = 16 * (c >> 4) + 8 * ((c >> 2) & 1) + 4 * ((c >> 3) & 1) + (c & 3);
    const int kfo = kperm * 64 + ((g ^ ((kperm >> 2) & 3)) << 4), vfo = c * 64 + ((g ^ ((c >> 2) & 3)) << 4);
    // K runs one block ahead of V: stage i is block i + 1's K and block i's V, in buffers i % NB; block 0's K begins in
    // the last stage's.
    auto stage = [&](int i, uint8_t* K, uint8_t* V) INL {
        fetch(find(i + 1), Kp, K);
        fetch(find(i), Vp, V);
    };
    constexpr int NK = NS / 4, NV = ND / 2, AHEAD = 2;
    if (nb > 0) {
        fetch(find(0), Kp, K3);
        stage(0, K0, V0);
        stage(1, K1, V1);
        stage(2, K2, V2);
    }
    f32x16 acc[ND];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[d][i] = 0.f;
    float m = -INFINITY, l = 0.f, nm = 0.f, tmax = -INFINITY;
    bool far = false;  // m is
    T8 pf[2];
    auto prob = [&](const f32x16& s, int e) INL {
        const float p = exp2_fast(__builtin_fmaf(s[e], a.c, nm));
        l += p;
        PIN_V(l);
        pf[e >> 3][e & 7] = (T)p;
    };
    // A step's fragments come in groups of 4: NK groups of K, then NV of V (ND dim tiles of the first 16 keys, then of
    // the others); group n is read while the groups up to AHEAD before it are in use.
    u32x4 fr[AHEAD + 1][4];
    auto read_k = [&](int n, int slot, const uint8_t* K) INL {
#pragma unroll
        for (int f = 0; f < 4; f++) {
            const int st = 4 * n + f;
            fr[slot][f] = *reinterpret_cast<const u32x4*>(K + (st >> 1) * 2048 + (kfo ^ ((st & 1) << 5)));
        }
    };
    auto read_v = [&](int n, int slot, const uint8_t* V) INL {
#pragma unroll
        for (int f = 0; f < 4; f++) {
            const int d = (4 * n + f) % ND, k = (4 * n + f) / ND;
            fr[slot][f] = *reinterpret_cast<const u32x4*>(V + d * 2048 + (vfo ^ (k << 5)));
        }
    };
    auto read = [&](int n, const uint8_t* K, const uint8_t* V) INL {
        if (n < NK) {
            read_k(n, n % (AHEAD + 1), K);
        } else if (n < NK + NV) read_v(n - NK, n % (AHEAD + 1), V);
    };
    // group n of S^T = K Q^T; mid(i) is work beside product i
    auto k_group = [&](int n, int slot, f32x16& s, auto mid) INL {
#pragma unroll
        for (int f = 0; f < 4; f++) {
            s = Num<T>::mfma32(__builtin_bit_cast(T8, fr[slot][f]), qf[4 * n + f], s);
            mid(4 * n + f);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // group n of O^T += V^T P^T
    auto v_group = [&](int n, int slot, auto mid) INL {
#pragma unroll
        for (int f = 0; f < 4; f++) {
            const int d = (4 * n + f) % ND, k = (4 * n + f) / ND;
            acc[d] = Num<T>::mfma32(__builtin_bit_cast(T8, fr[slot][f]), pf[k], acc[d]);
            mid(4 * n + f);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // The wave's part of the values of block i, which it has fetched itself: 0 in the place of what is not finite, where
    // some row of the workgroup does not see all of them.
    auto clean = [&](int i, uint8_t* V) INL {
        const int j0 = (blk0 + i) * 32;
        if (j0 >= wg0 && j0 + 32 <= wg1) return;
        uint8_t* const p = V + part + lane * 16;
        u32x4 v[IW];
        uint32_t x = 0;
#pragma unroll
        for (int u = 0; u < IW; u++) v[u] = *reinterpret_cast<const u32x4*>(p + u * 1024);
#pragma unroll
        for (int u = 0; u < IW; u++) x |= not_finite<T>(v[u]);
        if (__builtin_expect(__any(x != 0), 0)) {
            const u32x4 some = keys_within(j0 + 8 * ((lane & 3) ^ ((lane >> 4) & 3)), lo, hi);  // (seen by some row)
            x = 0;
#pragma unroll
            for (int u = 0; u < IW; u++) {
                v[u] &= some, x |= not_finite<T>(v[u]);
                *reinterpret_cast<u32x4*>(p + u * 1024) = finite8<T>(v[u]);
            }
            if (x != 0) rare = 1;
        }
    };
    // masks the scores of block j
    auto mask = [&](f32x16& s, int j) INL {
        const int j0 = (blk0 + j) * 32;
        const bool there = is_there(j);
        if (there && j0 >= all0 && j0 + 32 <= all1) return;
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int key = j0 + 16 * (e >> 3) + 8 * g + (e & 7);
            const bool keep = there & (key >= jlo) & (key < jhi);
            s[e] = keep ? s[e] : -INFINITY;
        }
    };
    auto raise = [&](f32x16& s) INL {  // (s: the scores whose maximum is tmax)
        if (__any(tmax - m > RAISE)) {
            const float mn = fmaxf(m, tmax), f = m == -INFINITY ? 0.f : exp2_fast(m - mn);
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < ND; d++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[d][e] *= f;
            nm = m == -INFINITY ? 0.f : Num<T>::UP - m;
            far = fabsf(nm) >= FAR;
            if (far) nm = Num<T>::UP;
        }
        if (__builtin_expect(__any(far), 0)) {
            if (far) {
#pragma unroll
                for (int e = 0; e < 16; e++) s[e] = less_max(s[e], a.c, m);
            }
        }
    };
    auto zero = [](f32x16& s) INL {
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = 0.f;
    };
    auto none = [](int) {};
    // Block i (scores s): its probabilities and output, beside the scores s2 of the next, whose keys are in K.  The first
    // EARLY keys' probabilities run beside the scores' products, the others beside the first half of the output's, the new
    // scores' maximum beside the second half.  The stage NB - 1 further on goes into (Kx, Vx).
    // (the pins keep the compiler from sinking work behind the products that it runs beside)
    constexpr int EARLY = 12;
    At nk{0, 0}, nv{0, 0};  // the blocks that the next step fetches: found in the shadow of this one's products
    auto find_next = [&](int i) INL { nk = find(i + NB), nv = find(i + NB - 1); };
    auto step = [&](int i, f32x16& s, f32x16& s2, const uint8_t* K, const uint8_t* V, uint8_t* Kx, uint8_t* Vx) INL {
#pragma unroll
        for (int n = 0; n < AHEAD; n++) read(n, K, V);
        __builtin_amdgcn_sched_barrier(0);
        raise(s);
        zero(s2);
        const Rsrc rk = block(nk, Kp), rv = block(nv, Vp);
#pragma unroll
        for (int n = 0; n < NK; n++) {
            read(n + AHEAD, K, V);
            __builtin_amdgcn_sched_barrier(0);
            k_group(n, n % (AHEAD + 1), s2, [&](int i) INL {
#pragma unroll
                for (int x = i * EARLY / NS; x < (i + 1) * EARLY / NS; x++) prob(s, x);
                // the DMAs one at a time: a burst of them holds up the wave
                if (i % (NS / IW) == NS / IW / 2) dma(rk, i / (NS / IW), Kx);
            });
        }
        OPAQUE_V(pf[0]);
        mask(s2, i + 1);
        constexpr int H = ND;  // products of each half
#pragma unroll
        for (int n = 0; n < NV; n++) {
            read(NK + n + AHEAD, K, V);
            __builtin_amdgcn_sched_barrier(0);
            v_group(n, (NK + n) % (AHEAD + 1), [&](int p) INL {
                if (p % (2 * H / IW) == H / IW) dma(rv, p / (2 * H / IW), Vx);
                if (p < H) {
                    constexpr int LATE = 16 - EARLY;
#pragma unroll
                    for (int x = p * LATE / H; x < (p + 1) * LATE / H; x++) prob(s, EARLY + x);
                    if (p == H - 1) OPAQUE_V(pf[1]);
                    if (p == H / 2) find_next(i + 1);
                } else {
                    constexpr int M = H - 1;  // the maximum beside all but the last
#pragma unroll
                    for (int x = (p - H) * 16 / M; x < (p - H + 1) * 16 / M && x < 16; x++)
                        tmax = x ? fmaxf(tmax, s2[x]) : s2[0];
                    if (p == 2 * H - 1) tmax = max_halves(tmax) * a.c;
                }
            });
        }
        OPAQUE_V(tmax);
    };
    // the wave's last block
    auto last = [&](f32x16& s, const uint8_t* V) INL {
        raise(s);
#pragma unroll
        for (int x = 0; x < 16; x++) prob(s, x);
#pragma unroll
        for (int n = 0; n < NV; n++) {
            read_v(n, 0, V);
            v_group(n, 0, none);
        }
    };
    // Stage i is there for every wave, the one before is done with.  (DMAs issued after it: NB - 2 stages.)
    auto arrive = [&](int i, uint8_t* V) INL {
        wait_loads<vmcnt_imm((NB - 2) * 2 * IW)>();
        clean(i, V);
        lds_barrier();
    };
    auto advance = [&](int i) INL {  // before blocks from i on are found
        if (i >= win + 32) win += 32, wh = wh2, wh2 = entries(win + 32);
    };
    if (nb > 0) {
        wait_loads<vmcnt_imm((NB - 1) * 2 * IW)>();
        lds_barrier();
    }
    if (live && nb > 0) {
        f32x16 sA, sB;
        zero(sA);
#pragma unroll
        for (int n = 0; n < NK; n++) {
            read_k(n, 0, K3);
            k_group(n, 0, sA, none);
        }
        mask(sA, 0);
        tmax = sA[0];
#pragma unroll
        for (int e = 1; e < 16; e++) tmax = fmaxf(tmax, sA[e]);
        tmax = max_halves(tmax) * a.c;
        find_next(0);
        // block i, its stage in (K, V), the stage NB - 1 further into (Kx, Vx)
        auto turn = [&](int i, f32x16& s, f32x16& s2, uint8_t* K, uint8_t* V, uint8_t* Kx, uint8_t* Vx) INL {
            arrive(i, V);
            advance(i);
            step(i, s, s2, K, V, Kx, Vx);
        };
        int i = 0;
        for (;;) {
            if (i + 1 >= nb) break;
            turn(i, sA, sB, K0, V0, K3, V3);
            if (++i + 1 >= nb) break;
            turn(i, sB, sA, K1, V1, K0, V0);
            if (++i + 1 >= nb) break;
            turn(i, sA, sB, K2, V2, K1, V1);
            if (++i + 1 >= nb) break;
            turn(i, sB, sA, K3, V3, K2, V2);
            ++i;
        }
        uint8_t* const V = i & 2 ? (i & 1 ? V3 : V2) : (i & 1 ? V1 : V0);
        arrive(i, V);
        if (i & 1) sA = sB;
        last(sA, V);
    } else {  // no rows: its part of the fetching
        auto buf = [&](int n, uint8_t* b0, uint8_t* b1, uint8_t* b2, uint8_t* b3) INL {
            return n & 2 ? (n & 1 ? b3 : b2) : (n & 1 ? b1 : b0);
        };
        for (int i = 0; i < nb; i++) {
            arrive(i, buf(i, V0, V1, V2, V3));
            advance(i);
            stage(i + NB - 1, buf(i + NB - 1, K0, K1, K2, K3), buf(i + NB - 1, V0, V1, V2, V3));
        }
    }
    wait_loads<vmcnt_imm(0)>();  // (no DMA outlives the workgroup whose LDS it writes)
    lds_barrier();
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(rare), 0)) {  // add_seen: see above
#pragma unroll 1
        for (int blk = blk0; blk < blk1; blk++) {
            const int j0 = 32 * blk, page = tb[blk >> lbpp];
            if ((unsigned)page >= (unsigned)a.n_pages || (j0 >= wg0 && j0 + 32 <= wg1)) continue;
            const T* const v = Vp + (size_t)page * a.pstride + ((size_t)(kh << lbpp) + (blk & ((1 << lbpp) - 1))) * (HD * 32);
#pragma unroll 1
            for (int j = j0; j < j0 + 32; j++)
                if (j >= jlo && j < jhi) {
#pragma unroll
                    for (int d = 0; d < ND; d++)
#pragma unroll
                        for (int e = 0; e < 16; e++) {
                            const float x = (float)v[(32 * d + 8 * (e >> 2) + 4 * g + (e & 3)) * 32 + (j & 31)];
                            if (!__builtin_isfinite(x)) acc[d][e] += x;
                        }
                }
        }
    }
    if (!live) return;
    // acc[d][e] is O[row c][dim 32 d + 8 (e / 4) + 4 g + e % 4]
    l += __shfl_xor(l, 32);
    const size_t row = (size_t)(rq.q0 + t) * a.HQ + h, pr = (size_t)z * a.rows * a.HQ + row;
    if (a.rows_ks > 1) {
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<f32x4*>(pacc + pr * HD + 32 * d + 8 * i + 4 * g) =
                    f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]};
        if (g == 0) pml[2 * pr] = m, pml[2 * pr + 1] = l;
        return;
    }
    // (all gates are loaded before the first is used: one after the other they were 17 us of a 256-dim call)
    u32x2 gate[ND][4];
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 4; i++) gate[d][i] = u32x2{0, 0};
    if (big) {
        const T* const p = big + (size_t)(rq.q0 + t) * a.stride + h * 2 * HD + HD + 4 * g;
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
            for (int i = 0; i < 4; i++) gate[d][i] = *reinterpret_cast<const u32x2*>(p + 32 * d + 8 * i);
    }
    T* const o = out + row * HD + 4 * g;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
        for (int i = 0; i < 4; i++)
            finish4<T>(f32x4{acc[d][4 * i], acc[d][4 * i + 1], acc[d][4 * i + 2], acc[d][4 * i + 3]}, l, big, gate[d][i],
                       o + 32 * d + 8 * i);
}

// Joins the splits of k_paged_rows: HD / 4 threads per row, 4 dims each, 8 splits at a time; the next 8 are on their way
// meanwhile (what goes past the last split is the last again).
template <class T, int HD>
__global__ __launch_bounds__(256) void k_paged_join_rows(AttnArgs a, const float* __restrict__ pacc,
                                                         const float* __restrict__ pml, const T* __restrict__ big,
                                                         T* __restrict__ out) {
    constexpr int W = HD / 4, PER = 256 / W, PARTS = TILE_ROWS / PER;
    const Tile tl = find_tile(a, blockIdx.x);
    if (tl.b < 0) return;
    const Req rq = request(a.cu, a.kv_lens, tl.b, a.rows, a.max_new, a.kcap);
    const int kh = blockIdx.y / PARTS, r = tl.i * TILE_ROWS + PER * (blockIdx.y % PARTS) + threadIdx.x / W;
    if (r >= rq.n * a.G) return;
    const int t = rq.q0 + r / a.G, h = kh * a.G + r % a.G, d = 4 * (threadIdx.x % W);
    const size_t row = (size_t)t * a.HQ + h, zs = (size_t)a.rows * a.HQ;
    constexpr int N = 8;
    struct Set {
        float2 ml[N];
        f32x4 x[N];
    };
    auto load = [&](int z0, Set& v) INL {
#pragma unroll
        for (int z = 0; z < N; z++) {
            const size_t at = min(z0 + z, a.rows_ks - 1) * zs + row;
            v.ml[z] = *reinterpret_cast<const float2*>(pml + 2 * at);
            v.x[z] = *reinterpret_cast<const f32x4*>(pacc + at * HD + d);
        }
    };
    Set v;
    load(0, v);
    const u32x2 gate = gate4(big, (size_t)t * a.stride + h * 2 * HD + HD + d);
    float mx = -INFINITY, ls = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int z0 = 0; z0 < a.rows_ks; z0 += N) {
        const Set now = v;
        if (z0 + N < a.rows_ks) load(z0 + N, v);
        float mn = mx;
#pragma unroll
        for (int z = 0; z < N; z++) mn = fmaxf(mn, now.ml[z].x);
        const float f0 = part_weight(mx, mn);
        mx = mn;
        ls *= f0;
#pragma unroll
        for (int e = 0; e < 4; e++) o[e] *= f0;
#pragma unroll
        for (int z = 0; z < N; z++) {
            if (z0 + z >= a.rows_ks) continue;
            const float f = part_weight(now.ml[z].x, mx);
            ls += now.ml[z].y * f;
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] += now.x[z][e] * f;
        }
    }
    finish4<T>(o, ls, big, gate, out + row * HD + d);
}

// How a call runs, from its sizes alone (the lengths themselves are on the device).
struct Plan {
    int nr = 0;                      // 16-row groups of k_paged_few, 0: not launched
    int few = 0;                     // requests with up to this many rows (new tokens times G) are its own
    int few_ks = 1, few_span = 1;    // splits, and blocks of 32 keys in each
    bool once = false;               // its cache is read past the last-level cache
    int tiles = 0;                   // of k_paged_rows (an upper bound), 0: not launched
    int rows_ks = 1, rows_span = 1;  // splits, and blocks in each
    size_t slots = 0;                // partial results of [rows][HQ] that they need at most, whatever the window
};

Plan plan_attn(const PagedShape& s, int B, int rows, int max_new, int max_kv, int window) {
    const int G = s.HQ / s.HK;
    const long long most = (long long)std::min(max_new, rows) * G;
    Plan p;
    const int fits = s.HD == 256 ? 16 : 32;  // (a second group's outputs and queries do not fit the registers at 256)
    // Among chunks, requests with few rows are k_paged_few's where most are such, and where some may have long caches,
    // which no tile of one row should walk: a prompt of 512 tokens and one token on 30000 keys, 32 and 8 heads of 128
    // dims, 260 us with both in tiles, 38 so.  Where all are chunks after all, the parts that exit and their join cost
    // 1 to 3 us.
    if (most <= fits) p.nr = most <= 16 ? 1 : 2, p.few = 16 * p.nr;
    else if (G <= fits && rows < (long long)max_new * B && (2ll * rows < (long long)max_new * B || max_kv >= 2048))
        p.nr = G <= 16 ? 1 : 2, p.few = 16 * p.nr;
    auto blocks = [&](long long n) {  // of 32 keys that n adjacent rows may see
        long long k = max_kv;
        if (window) k = std::min(k, (long long)window + n + 31);
        return (int)((k + 31) / 32);
    };
    if (p.nr) {
        const int nb = blocks(std::max(1, p.few / G));
        // One workgroup per CU wants keys to read, at least 2 blocks each (8 and 2 heads of 256 dims, 700 keys: 8.8 us, at
        // least 4 9.3, 8 10.6); but the parts cost a join: no split of few elements, and none where the unsplit workgroups
        // draw most of the bandwidth already.  us unsplit and split, at n keys of each request:
        // 8 workgroups, dims 64: 1000 6.9 7.8, 2000 10.5 7.5; 128: 700 9.1 7.8; 256: 200 7.8 7.9, 400 10.3 8.3
        // 128 workgroups, dims 64: 8000 39 44; 128: 4000 40 46, 8000 90 81; 256: 2000 41 46, 4000 93 82
        const int wgs = B * s.HK;
        const double elems = 32.0 * nb * s.HD;
        const int want = elems < (wgs < 128 ? 75e3 : 768e3) ? 1 : std::min(MAX_KS, std::max(1, 256 / wgs));
        p.few_span = ((nb + want - 1) / want + 1) / 2 * 2;
        p.few_ks = (nb + p.few_span - 1) / p.few_span;
        p.slots = std::min(want, (nb + 1) / 2);
        // beyond the 256 MB that stay in the last-level cache a layer's keys are gone before they are read again (64
        // requests of 1000 to 8191 rows 159 -> 142 us with the hint, two of 90 and 131 thousand 89 -> 78; 85 MB, read again
        // and again, 22 -> 24)
        p.once = (size_t)B * nb * s.HK * s.HD * 128 > (size_t(256) << 20);
    }
    if (most > p.few) {
        const long long all = (long long)rows * G;
        p.tiles = (int)(all / TILE_ROWS + std::min((long long)B, all / (p.few + 1)));
        const int nb = blocks(TILE_ROWS / G + 2);
        // One workgroup per CU: tiles as many as there will be, if every request has one (a request's 64 heads of 128 dims on
        // 8000 and 30000 keys 25 and 71 us in at most 8 splits, 15 and 23 in 64; 32 of them 33 and 101 us in 16, 31 and 93
        // in 8)
        const long long tiles = std::max({1ll, all / TILE_ROWS, p.nr ? 1ll : std::min(B, rows)});
        const int want = (int)std::min((long long)MAX_KS, std::max(1ll, 256 / (tiles * s.HK)));
        p.rows_span = std::max(8, ((nb + want - 1) / want + 1) / 2 * 2);
        p.rows_ks = (nb + p.rows_span - 1) / p.rows_span;
        p.slots = std::max(p.slots, (size_t)std::min(want, (nb + 7) / 8));
    }
    if (p.slots == 1) p.slots = 0;
    return p;
}

template <class T, int HD>
void prep_as(const PagedShape& s, const PagedPrep& a, hipStream_t st) {
    auto groups = [&](int hpt) {
        return ((size_t)a.rows * HD + 511) / 512 * ((s.HQ + 4 * hpt - 1) / (4 * hpt) + (s.HK + 4 * hpt - 1) / (4 * hpt));
    };
    // heads per thread: as many as leave nearly three workgroups per CU (us at 1, 2, 4, 8, on the same buffers again and
    // again: 32 and 8 heads of 128, three axes, 256 rows 6.4 7.5 7.1 7.5, 1024 rows 10.4 8.6 7.7 8.7, 4099 rows 30.9 22.4 20.7 20.1)
    int hpt = 8;
    while (hpt > 1 && groups(hpt) < 700) hpt /= 2;
    const size_t nv = (size_t)((a.rows + VT - 1) / VT) * s.HK * (HD / VD);
    if (nv + groups(hpt) >= size_t(1) << 24) throw Error("sd_op_paged_prep: too many rows for one launch");
    hipLaunchKernelGGL((k_paged_prep<T, HD>), dim3((unsigned)(nv + groups(hpt))), dim3(256), 0, st,
                       static_cast<const T*>(a.big), a.stride, a.gated ? 2 * HD : HD, a.qw, a.kw, a.rope, a.rope_len, a.pos,
                       a.axes, a.axis, a.slots, a.rows, s.HQ, s.HK, a.RD, log2i(s.PS), s.n_pages, s.pstride, hpt, (int)nv,
                       static_cast<T*>(a.Q), static_cast<T*>(a.Kp), static_cast<T*>(a.Vp));
    launched("paged_prep");
}

template <class T, int HD>
void attn_as(const PagedShape& s, const PagedAttn& a, hipStream_t st) {
    const Plan p = plan_attn(s, a.B, a.rows, a.max_new, a.max_kv, a.window);
    const AttnArgs g{a.table, a.cu, a.kv_lens, a.max_blocks, a.B, a.rows, s.HQ, s.HK, s.HQ / s.HK, log2i(s.PS), s.n_pages,
                     a.max_new, a.max_kv, a.window, a.stride, p.few, p.few_ks, p.few_span, p.tiles, p.rows_ks, p.rows_span,
                     a.scale * LOG2E, s.pstride};
    const T *Q = static_cast<const T*>(a.Q), *K = static_cast<const T*>(a.Kp), *V = static_cast<const T*>(a.Vp),
            *big = static_cast<const T*>(a.big);
    T* const out = static_cast<T*>(a.out);
    float* const pacc = static_cast<float*>(a.ws);
    float* const pml = pacc + p.slots * a.rows * s.HQ * HD;
    const size_t tiles = (size_t)p.tiles * s.HK * p.rows_ks, parts = (size_t)a.B * s.HK * p.few_ks;
    const bool both = p.tiles && p.nr == 1;
    if (tiles + parts >= size_t(1) << 24) throw Error("sd_op_paged_attention: too many rows and requests for one launch");
    auto launch = [&](auto kernel, dim3 grid, int threads) {
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, st, Q, K, V, g, big, out, pacc, pml);
        launched("paged_attention");
    };
    if (both) {
        if (p.once) launch(k_paged_rows<T, HD, 2>, dim3((unsigned)(tiles + parts)), 256);
        else launch(k_paged_rows<T, HD, 1>, dim3((unsigned)(tiles + parts)), 256);
    } else {
        if (p.tiles) launch(k_paged_rows<T, HD, 0>, dim3((unsigned)tiles), 256);
        const dim3 grid(s.HK * p.few_ks, a.B);
        if (p.nr == 1) {
            if (p.once) launch(k_paged_few<T, HD, 1, true>, grid, 64 * few_waves<HD, 1>());
            else launch(k_paged_few<T, HD, 1, false>, grid, 64 * few_waves<HD, 1>());
        }
        if constexpr (HD < 256)
            if (p.nr == 2) {
                if (p.once) launch(k_paged_few<T, HD, 2, true>, grid, 64 * few_waves<HD, 2>());
                else launch(k_paged_few<T, HD, 2, false>, grid, 64 * few_waves<HD, 2>());
            }
    }
    if (p.rows_ks > 1) {
        hipLaunchKernelGGL((k_paged_join_rows<T, HD>), dim3(p.tiles, TILE_ROWS / (1024 / HD) * s.HK), dim3(256), 0, st, g, pacc, pml,
                           big, out);
        launched("paged_attention");
    }
    if (p.few_ks > 1) {
        const int rows_max = (int)std::min((long long)p.few, (long long)std::min(a.max_new, a.rows) * g.G);
        hipLaunchKernelGGL((k_paged_join_few<T, HD>), dim3(s.HK * rows_max, a.B), dim3(256), 0, st, g, pacc, pml, big, out,
                           rows_max);
        launched("paged_attention");
    }
}

}  // namespace

void page_plan(const PagePlan& a, hipStream_t st) {
    const int groups = std::min((a.T + PLAN_T - 1) / PLAN_T, 128);
    hipLaunchKernelGGL(k_page_plan, dim3(groups), dim3(PLAN_T), 0, st, a.lens, a.news, a.B, a.T, log2i(a.PS), a.n_pages,
                       a.free_pages, a.n_free, a.table, a.max_blocks, a.cu, a.kv_lens, a.slots, a.pos, a.status);
    launched("page_plan");
}

void paged_prep(const PagedShape& s, const PagedPrep& a, hipStream_t st) {
    by_type(s, [&](auto t, auto hd) { prep_as<decltype(t), decltype(hd)::value>(s, a, st); });
}

size_t paged_attn_ws(const PagedShape& s, int B, int rows, int max_new, int max_kv) {
    // (a window only lowers the number of splits)
    return plan_attn(s, B, rows, max_new, max_kv, 0).slots * rows * s.HQ * (s.HD + 2) * 4;
}

void paged_attn(const PagedShape& s, const PagedAttn& a, hipStream_t st) {
    by_type(s, [&](auto t, auto hd) { attn_as<decltype(t), decltype(hd)::value>(s, a, st); });
}

}  // namespace sd
