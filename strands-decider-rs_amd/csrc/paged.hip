// A K/V cache in pages, shared by many requests: the step's page plan, the norm + rotation + cache write of its new
// rows, and their attention (no counterpart in the reference, whose cache holds one sequence).
//
// A page holds PS rows (a power of two from 32) of every kv head, in the blocks of 32 rows that the engine's own cache
// has: K [HK][PS / 32][HD / 32][32 rows][32 dims], V transposed [HK][PS / 32][HD][32 rows].  Page p starts `pstride`
// elements after page p - 1.  Row j of a request lies in page table[j / PS] at row j % PS; a table entry outside
// [0, n_pages) is a hole, whose rows nothing reads or writes.
#include <algorithm>
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

// ---- the page plan --------------------------------------------------------------------------------------------------

constexpr int PLAN_T = 1024;  // threads of a plan workgroup

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

// Element offset of (slot, kv head) in a cache whose rows' 32-row blocks hold HD x 32 elements.
template <int HD>
__device__ __forceinline__ size_t block_at(int slot, int kh, int lps, size_t pstride) {
    return (size_t)(slot >> lps) * pstride + ((size_t)kh * (1 << (lps - 5)) + ((slot & ((1 << lps) - 1)) >> 5)) * (HD * 32);
}

constexpr int VT = 64;  // rows of a V workgroup

// Workgroups [0, nqk): q and k heads.  HD / 8 threads share a (row, head), 8 dims each; a thread takes `nh` heads of its
// row one after the other with one set of cosines and sines (they are f32 and twice a row's bytes: fetched per head
// they, not the rows, were what a chunk's time went to).  Workgroups from nqk: 64 rows of one kv head's V, transposed
// through LDS so that 8 consecutive slots go out as 16 bytes.
template <class T, int HD>
__global__ __launch_bounds__(256) void k_paged_prep(const T* __restrict__ big, int stride, int q_step,
                                                    const float* __restrict__ qw, const float* __restrict__ kw,
                                                    const float* __restrict__ rope, int rope_len,
                                                    const int* __restrict__ pos, int axes,
                                                    const uint8_t* __restrict__ axis, const int* __restrict__ slots,
                                                    int rows, int HQ, int HK, int RD, int lps, int n_pages,
                                                    size_t pstride, int nh, int nqk, T* __restrict__ Q,
                                                    T* __restrict__ Kp, T* __restrict__ Vp) {
    typedef typename Vec8<T>::type T8;
    constexpr int LPH = HD / 8;
    const int tid = threadIdx.x;
    const int k_off = HQ * q_step, v_off = k_off + HK * HD;
    const long long n_slots = (long long)n_pages << lps;
    if ((int)blockIdx.x < nqk) {
        const int gq = (HQ + nh - 1) / nh, gk = (HK + nh - 1) / nh;
        const int unit = blockIdx.x * (256 / LPH) + tid / LPH, c = tid % LPH;
        const int t = unit / (gq + gk), u = unit % (gq + gk);
        if (t >= rows) return;
        const int slot = slots[t];
        if (slot < 0 || slot >= n_slots) return;
        const bool isq = u < gq;
        const int h0 = (isq ? u : u - gq) * nh, h1 = min(isq ? HQ : HK, h0 + nh);
        const T* const src = big + (size_t)t * stride + (isq ? 0 : k_off) + 8 * c;
        const int step = isq ? q_step : HD;
        const float* const nw = isq ? qw : kw;
        float w[8];
#pragma unroll
        for (int e = 0; e < 8; e++) w[e] = nw ? nw[8 * c + e] : 1.f;
        // the pair of dim d: j = d % (RD / 2); its other dim is RD / 2 away
        const int rd2 = RD / 2;
        const bool whole = rd2 % 8 == 0;  // a chunk's partners are one other chunk
        float cs[8], sn[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int d = 8 * c + e;
            cs[e] = 1.f, sn[e] = 0.f;
            if (d < RD) {
                const int j = d < rd2 ? d : d - rd2;
                const int a = axes > 1 ? min((int)axis[j], axes - 1) : 0;
                const int at = min(max(pos[(size_t)a * rows + t], 0), rope_len - 1);
                const float2 v = *reinterpret_cast<const float2*>(rope + ((size_t)at * rd2 + j) * 2);
                cs[e] = v.x;
                sn[e] = d < rd2 ? -v.y : v.y;
            }
        }
        for (int h = h0; h < h1; h++) {
            const T8 x8 = *reinterpret_cast<const T8*>(src + (size_t)h * step);
            float x[8], ss = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = (float)x8[e], ss += x[e] * x[e];
            float inv = 1.f;
            if (nw) {
#pragma unroll
                for (int o = 1; o < LPH; o <<= 1) ss += __shfl_xor(ss, o);
                inv = 1.0f / sqrtf(ss / (float)HD + 1e-6f);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = x[e] * inv * w[e];
            T8 y8;
            if (whole) {
                const int s = rd2 / 8;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float up = __shfl(x[e], c + s, LPH), dn = __shfl(x[e], c - s, LPH);
                    y8[e] = (T)(8 * c + e < RD ? x[e] * cs[e] + (c < s ? up : dn) * sn[e] : x[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int d = 8 * c + e, o = d < rd2 ? d + rd2 : d - rd2;
                    float r = x[e];
                    if (d < RD) r = x[e] * cs[e] + (float)src[(size_t)h * step - 8 * c + o] * inv * (nw ? nw[o] : 1.f) * sn[e];
                    y8[e] = (T)r;
                }
            }
            if (isq) *reinterpret_cast<T8*>(Q + ((size_t)t * HQ + h) * HD + 8 * c) = y8;
            else
                *reinterpret_cast<T8*>(Kp + block_at<HD>(slot, h, lps, pstride) + (c / 4) * 1024 + (slot & 31) * 32 +
                                       8 * (c % 4)) = y8;
        }
        return;
    }
    __shared__ __align__(16) T tile[VT][HD + 8];
    __shared__ int sl[VT];
    __shared__ int first, whole8[VT / 8 + 1];
    const int v = blockIdx.x - nqk, kh = v % HK, t0 = v / HK * VT, nt = min(VT, rows - t0);
    if (tid < VT) {
        const int s = tid < nt ? slots[t0 + tid] : -1;
        sl[tid] = s >= 0 && s < n_slots ? s : -1;
        const unsigned long long any = __ballot(sl[tid] >= 0);
        if (tid == 0) first = any ? __ffsll((long long)any) - 1 : 0;
    }
    for (int i = tid; i < nt * LPH; i += 256)
        *reinterpret_cast<T8*>(&tile[i / LPH][8 * (i % LPH)]) =
            *reinterpret_cast<const T8*>(big + (size_t)(t0 + i / LPH) * stride + v_off + kh * HD + 8 * (i % LPH));
    __syncthreads();
    // octets of rows cut where the slots of the first request here are multiples of 8
    const int s0 = sl[first], cut = s0 < 0 ? 0 : ((first - s0) & 7) - 8;
    if (tid < VT / 8 + 1) {
        const int r0 = cut + 8 * tid;
        bool ok = r0 >= 0 && r0 + 7 < VT && sl[max(r0, 0)] >= 0 && sl[max(r0, 0)] % 8 == 0;
        for (int i = 1; ok && i < 8; i++) ok = sl[r0 + i] == sl[r0] + i;
        whole8[tid] = ok;
    }
    __syncthreads();
    for (int i = tid; i < HD * (VT / 8 + 1); i += 256) {
        const int d = i / (VT / 8 + 1), o = i % (VT / 8 + 1), r0 = cut + 8 * o;
        if (whole8[o]) {
            T8 y;
#pragma unroll
            for (int e = 0; e < 8; e++) y[e] = tile[r0 + e][d];
            *reinterpret_cast<T8*>(Vp + block_at<HD>(sl[r0], kh, lps, pstride) + d * 32 + (sl[r0] & 31)) = y;
        } else {
            for (int r = max(r0, 0); r < min(r0 + 8, nt); r++)
                if (sl[r] >= 0) Vp[block_at<HD>(sl[r], kh, lps, pstride) + d * 32 + (sl[r] & 31)] = tile[r][d];
        }
    }
}

// ---- attention ------------------------------------------------------------------------------------------------------

// One wave per (row, q head), lanes over the dims, key after key.
template <class T, int HD>
__global__ __launch_bounds__(256) void k_paged_attn(const T* __restrict__ Q, const T* __restrict__ big, int stride,
                                                    const T* __restrict__ Kp, const T* __restrict__ Vp,
                                                    const int* __restrict__ table, int max_blocks,
                                                    const int* __restrict__ cu, const int* __restrict__ kv_lens, int B,
                                                    int rows, int HQ, int HK, int lps, int n_pages, size_t pstride,
                                                    int window, float scale, T* __restrict__ out) {
    constexpr int E = HD / 64;
    const int lane = threadIdx.x & 63, unit = blockIdx.x * 4 + (threadIdx.x >> 6);
    const int t = unit / HQ, h = unit % HQ, kh = h / (HQ / HK);
    if (t >= rows || t >= cu[B]) return;
    const int b = find_range(cu, B, t);
    const int p = kv_lens[b] - (cu[b + 1] - t);  // the row's own position
    const int last = min(p, (int)min((long long)max_blocks << lps, (long long)INT32_MAX) - 1);
    float q[E], acc[E], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < E; e++) q[e] = (float)Q[((size_t)t * HQ + h) * HD + lane + 64 * e], acc[e] = 0.f;
    for (int j = window > 0 ? max(0, p - window + 1) : 0; j <= last; j++) {
        const int page = table[(size_t)b * max_blocks + (j >> lps)];
        if (page < 0 || page >= n_pages) continue;
        const int row = j & ((1 << lps) - 1);
        const size_t at = (size_t)page * pstride + ((size_t)kh * (1 << (lps - 5)) + (row >> 5)) * (HD * 32);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int d = lane + 64 * e;
            s += q[e] * (float)Kp[at + (d / 32) * 1024 + (row & 31) * 32 + d % 32];
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
        s *= scale;
        const float mn = fmaxf(m, s), f = m == -INFINITY ? 0.f : exp2f((m - mn) * LOG2E);
        const float pr = exp2f((s - (mn == -INFINITY ? 0.f : mn)) * LOG2E);
        l = l * f + pr;
        m = mn;
#pragma unroll
        for (int e = 0; e < E; e++) acc[e] = acc[e] * f + pr * (float)Vp[at + (lane + 64 * e) * 32 + (row & 31)];
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
        const int d = lane + 64 * e;
        float o = l == 0.f ? 0.f : acc[e] / l;
        if (big) o *= 1.0f / (1.0f + exp2f(-LOG2E * (float)big[(size_t)t * stride + h * 2 * HD + HD + d]));
        out[((size_t)t * HQ + h) * HD + d] = (T)o;
    }
}

int log2i(int x) { return 31 - __builtin_clz((unsigned)x); }

template <class T, int HD>
void prep_as(const PagedShape& s, const PagedPrep& a, hipStream_t st) {
    constexpr int PER = 256 / (HD / 8);  // (row, head) units of a workgroup
    // heads per thread: as many as leave about four workgroups per CU
    int nh = 1;
    while (nh < 8 && (size_t)a.rows * (s.HQ + s.HK) / (2 * nh) / PER >= 1024) nh *= 2;
    const size_t units = (size_t)a.rows * ((s.HQ + nh - 1) / nh + (s.HK + nh - 1) / nh);
    const size_t nqk = (units + PER - 1) / PER, nv = (size_t)((a.rows + VT - 1) / VT) * s.HK;
    hipLaunchKernelGGL((k_paged_prep<T, HD>), dim3((unsigned)(nqk + nv)), dim3(256), 0, st, static_cast<const T*>(a.big),
                       a.stride, a.gated ? 2 * HD : HD, a.qw, a.kw, a.rope, a.rope_len, a.pos, a.axes, a.axis, a.slots,
                       a.rows, s.HQ, s.HK, a.RD, log2i(s.PS), s.n_pages, s.pstride, nh, (int)nqk, static_cast<T*>(a.Q),
                       static_cast<T*>(a.Kp), static_cast<T*>(a.Vp));
    launched("paged_prep");
}

template <class T, int HD>
void attn_as(const PagedShape& s, const PagedAttn& a, hipStream_t st) {
    hipLaunchKernelGGL((k_paged_attn<T, HD>), dim3((unsigned)(((size_t)a.rows * s.HQ + 3) / 4)), dim3(256), 0, st,
                       static_cast<const T*>(a.Q), static_cast<const T*>(a.big), a.stride, static_cast<const T*>(a.Kp),
                       static_cast<const T*>(a.Vp), a.table, a.max_blocks, a.cu, a.kv_lens, a.B, a.rows, s.HQ, s.HK,
                       log2i(s.PS), s.n_pages, s.pstride, a.window, a.scale, static_cast<T*>(a.out));
    launched("paged_attention");
}

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

void page_plan(const PagePlan& a, hipStream_t st) {
    const int groups = std::min((a.T + PLAN_T - 1) / PLAN_T, 128);
    hipLaunchKernelGGL(k_page_plan, dim3(groups), dim3(PLAN_T), 0, st, a.lens, a.news, a.B, a.T, log2i(a.PS), a.n_pages,
                       a.free_pages, a.n_free, a.table, a.max_blocks, a.cu, a.kv_lens, a.slots, a.pos, a.status);
    launched("page_plan");
}

void paged_prep(const PagedShape& s, const PagedPrep& a, hipStream_t st) {
    by_type(s, [&](auto t, auto hd) { prep_as<decltype(t), decltype(hd)::value>(s, a, st); });
}

size_t paged_attn_ws(const PagedShape&, int, int, int, int) { return 0; }

void paged_attn(const PagedShape& s, const PagedAttn& a, hipStream_t st) {
    by_type(s, [&](auto t, auto hd) { attn_as<decltype(t), decltype(hd)::value>(s, a, st); });
}

}  // namespace sd
