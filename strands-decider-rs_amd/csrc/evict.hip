// Rows that leave the paged cache: the attention weight that every cached key receives, the rows of each kv head that go
// when a request holds more than it may, the moves of those that stay into their places, and the pages behind them (no
// counterpart in the reference, whose cache holds one sequence and forgets nothing).
//
// Scores and positions of cached rows lie in arrays [n_pages][HK][PS], addressed by the same table as the caches.
#include "paged.h"

namespace sd {
namespace {

// Index of (page, kv head, row j) in an array [n_pages][HK][PS].
__device__ __forceinline__ size_t mark_at(int page, int HK, int h, int j, int lps) {
    return ((size_t)page * HK + h) * ((size_t)1 << lps) + (j & ((1 << lps) - 1));
}

// ---- the weight that every cached key receives ----------------------------------------------------------------------

struct WeightArgs {
    const int *table, *cu, *kv_lens, *pos;
    int max_blocks, B, rows, HQ, HK, G, lps, n_pages, max_new, kcap, window, observers;
    float c, decay;  // c: scale log2(e)
    size_t pstride;
    const float* scores;
    float* out;
    int* kpos;
    // the first key that a row at position p sees
    __device__ __forceinline__ int from(int p) const { return window ? max(p, -1) - window + 1 : 0; }
};

// The rows of a request that are counted: its last `observers`.
__device__ __forceinline__ int first_observer(const Req& r, int observers) { return observers ? max(0, r.n - observers) : 0; }

template <class T, int HD>
__device__ __forceinline__ const T* key_row(const T* Kp, const WeightArgs& a, int page, int h, int j) {
    return Kp + (size_t)page * a.pstride + ((size_t)(h << (a.lps - 5)) + ((j & ((1 << a.lps) - 1)) >> 5)) * (HD * 32) + (j & 31) * 32;
}
// c s, rounded: what a row's maximum is one of.  (In one fma with the maximum taken off, scores from 2^23 on, whose maximum
// has no fractions, would be off by more than an exponential's range.)
__device__ __forceinline__ float scaled(float s, float c) {
#pragma clang fp contract(off)
    return s * c;
}
template <class T, int HD>
__device__ __forceinline__ float dot(const T* q, const T* k) {
    float s = 0.f;
    for (int d = 0; d < HD; d++) s = __builtin_fmaf((float)q[d], (float)k[d / 32 * 1024 + d % 32], s);
    return s;
}

// A row's maximum and sum: one wave per (row, query head).
template <class T, int HD>
__global__ __launch_bounds__(64) void k_weights_stats(const T* __restrict__ Q, const T* __restrict__ Kp, WeightArgs a,
                                                      float2* __restrict__ ml) {
    const int b = blockIdx.y, lane = threadIdx.x, h = blockIdx.x % a.HQ;
    const Req rq = request(a.cu, a.kv_lens, b, a.rows, a.max_new, a.kcap);
    const int* const tb = a.table + (size_t)b * a.max_blocks;
    for (int i = first_observer(rq, a.observers) + blockIdx.x / a.HQ; i < rq.n; i += gridDim.x / a.HQ) {
        const int p = rq.p0 + i, lo = max(0, a.from(p)), hi = min(p + 1, rq.kcap);
        const T* const q = Q + ((size_t)(rq.q0 + i) * a.HQ + h) * HD;
        float m = -INFINITY, l = 0.f;
        for (int pass = 0; pass < 2; pass++)
            for (int j0 = lo; j0 < hi; j0 += 64) {
                const int j = j0 + lane, page = tb[min(j >> a.lps, a.max_blocks - 1)];
                if (j >= hi || (unsigned)page >= (unsigned)a.n_pages) continue;
                const float x = scaled(dot<T, HD>(q, key_row<T, HD>(Kp, a, page, h / a.G, j)), a.c);
                if (pass == 0) m = fmaxf(m, x);
                else l += m == -INFINITY && x == -INFINITY ? 0.f : exp2_fast(x - m);
            }
        float mx = m;  // (m is the lane's own)
        for (int o = 1; o < 64; o <<= 1) mx = fmaxf(mx, __shfl_xor(mx, o));
        l *= part_weight(m, mx);
        for (int o = 1; o < 64; o <<= 1) l += __shfl_xor(l, o);
        if (lane == 0) ml[(size_t)(rq.q0 + i) * a.HQ + h] = make_float2(mx, l);
    }
}

// A key's weight from all rows: one thread per (key, kv head).
template <class T, int HD>
__global__ __launch_bounds__(256) void k_weights_sum(const T* __restrict__ Q, const T* __restrict__ Kp, WeightArgs a,
                                                     const float2* __restrict__ ml) {
    const int b = blockIdx.z, kh = blockIdx.y, j = blockIdx.x * 256 + threadIdx.x;
    const Req rq = request(a.cu, a.kv_lens, b, a.rows, a.max_new, a.kcap);
    if (rq.n == 0 || j >= rq.kcap) return;
    const int page = a.table[(size_t)b * a.max_blocks + (j >> a.lps)];
    if ((unsigned)page >= (unsigned)a.n_pages) return;
    const T* const k = key_row<T, HD>(Kp, a, page, kh, j);
    float w = 0.f;
    for (int i = first_observer(rq, a.observers); i < rq.n; i++) {
        const int p = rq.p0 + i;
        if (j > p || j < a.from(p)) continue;
        for (int g = 0; g < a.G; g++) {
            const size_t row = (size_t)(rq.q0 + i) * a.HQ + kh * a.G + g;
            const float2 s = ml[row];
            if (s.y == 0.f) continue;
            w += exp2_fast(scaled(dot<T, HD>(Q + row * HD, k), a.c) - s.x) / s.y;
        }
    }
    const size_t at = mark_at(page, a.HK, kh, j, a.lps);
    const bool old = j < rq.p0;
    a.out[at] = old && a.decay != 0.f ? __builtin_fmaf(a.decay, a.scores[at], w) : w;
    if (!old && a.kpos) a.kpos[at] = a.pos[rq.q0 + j - rq.p0];
}

// ---- the rows that go -----------------------------------------------------------------------------------------------

// A score's place in the order, ascending: NaN, and a row in a hole, before all numbers; -0 is 0.
__device__ __forceinline__ uint32_t rank_of(float s) {
    if (s != s) return 0;
    const uint32_t u = __builtin_bit_cast(uint32_t, s + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int EVICT_T = 1024;

// The sum over the threads before this one, and over all; `ws` holds EVICT_T / 64 counts.
template <class I>
__device__ __forceinline__ I scan(I x, I* ws, I& total) {
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    I v = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const I y = __shfl_up(v, o);
        if (lane >= o) v += y;
    }
    __syncthreads();
    if (lane == 63) ws[wv] = v;
    __syncthreads();
    I before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < EVICT_T / 64; w++) before += w < wv ? ws[w] : 0, all += ws[w];
    total = all;
    return before + v - x;
}

// One workgroup per (request, kv head): the m-th largest rank by its 8-bit digits, from the highest down (a histogram of
// the rows whose digits above match), then one pass over the rows in order that numbers the holes below m and the rows
// that stay behind it.
__global__ __launch_bounds__(EVICT_T) void k_page_evict(const float* __restrict__ scores, const int* __restrict__ kpos,
                                                        const int* __restrict__ table, int max_blocks,
                                                        const int* __restrict__ kv_lens, const int* __restrict__ budgets,
                                                        int max_kv, int HK, int lps, int n_pages, int sink, int recent,
                                                        int* __restrict__ new_lens, int* __restrict__ moves,
                                                        int* __restrict__ counts) {
    __shared__ int hist[256], ws[EVICT_T / 64], newest, digit, above;
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, W = max(max_kv / 2, 1);
    const int n = kv_lens[b], budget = budgets[b];
    const bool over = n <= max_kv && budget >= 0 && n > budget;
    const int m = over ? budget : n;
    if (h == 0 && tid == 0) new_lens[b] = m;
    if (!over) {
        if (tid == 0) counts[(size_t)b * HK + h] = 0;
        return;
    }
    const int* const tb = table + (size_t)b * max_blocks;
    auto where = [&](int j, bool& there) {
        const int page = tb[j >> lps];
        there = (unsigned)page < (unsigned)n_pages;
        return mark_at(there ? page : 0, HK, h, j, lps);
    };
    if (tid == 0) newest = INT_MIN;
    __syncthreads();
    int most = INT_MIN;
    for (int j = tid; j < n; j += EVICT_T) {
        bool there;
        const size_t at = where(j, there);
        if (there) most = max(most, kpos ? kpos[at] : j);
    }
    atomicMax(&newest, most);
    __syncthreads();
    const long long keep_from = (long long)newest - recent;
    auto rank = [&](int j) {
        bool there;
        const size_t at = where(j, there);
        if (!there) return 0u;
        const int p = kpos ? kpos[at] : j;
        return p < sink || p > keep_from ? 0xFFFFFFFFu : min(rank_of(scores[at]), 0xFFFFFFFEu);
    };
    uint32_t prefix = 0;
    int left = m;  // of the largest ranks that begin with `prefix`, so many stay
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = tid; i < 256; i += EVICT_T) hist[i] = 0;
        __syncthreads();
        for (int j = tid; j < n; j += EVICT_T) {
            const uint32_t r = rank(j);
            if (shift == 24 || r >> (shift + 8) == prefix >> (shift + 8)) atomicAdd(&hist[r >> shift & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int d = 255, sum = 0;
            while (d > 0 && sum + hist[d] < left) sum += hist[d--];
            digit = d, above = sum;
        }
        __syncthreads();
        prefix |= (uint32_t)digit << shift;
        left -= above;
    }
    // ranks above `prefix` stay, and the first `left` rows that have it
    int ties = 0, holes = 0, rows = 0;
    int* const mv = moves + ((size_t)b * HK + h) * W * 2;
    for (int j0 = 0; j0 < n; j0 += EVICT_T) {
        const int j = j0 + tid;
        const uint32_t r = j < n ? rank(j) : 0;
        const bool tie = j < n && r == prefix;
        int total;
        const int nth = ties + scan((int)tie, ws, total);
        ties += total;
        const bool stays = j < n && (r > prefix || (tie && nth < left));
        const bool hole = j < m && !stays, row = j >= m && stays;
        const int x = holes + scan((int)hole, ws, total);
        holes += total;
        const int y = rows + scan((int)row, ws, total);
        rows += total;
        if (hole) mv[2 * x] = j;
        if (row) mv[2 * y + 1] = j;
    }
    if (tid == 0) counts[(size_t)b * HK + h] = rows;
}

// ---- their pages ----------------------------------------------------------------------------------------------------

constexpr int RELEASE_T = 1024;

// One workgroup: the requests' pages that go numbered through by a scan over the requests, then pushed in that order, a
// round of 1024 entries at a time, those out of range left out.
__global__ __launch_bounds__(RELEASE_T) void k_page_release(const int* __restrict__ kv_lens, const int* __restrict__ new_lens,
                                                            const int* __restrict__ dropped, const int* __restrict__ table,
                                                            int max_blocks, int B, int lps, int n_pages, int* free_pages,
                                                            const int* __restrict__ n_free, int* __restrict__ dropped_out,
                                                            int* __restrict__ n_free_out) {
    __shared__ int to[PAGE_PLAN_MAX_B + 1];
    __shared__ long long ws[RELEASE_T / 64];
    const int tid = threadIdx.x, per = (B + RELEASE_T - 1) / RELEASE_T, b0 = min(tid * per, B), b1 = min(B, b0 + per);
    const int ps1 = (1 << lps) - 1;
    auto pages = [&](int x) { return min((int)(((long long)x + ps1) >> lps), max_blocks); };
    auto gone = [&](int b) {  // pages of request b that go (max_blocks pages in all have fewer than 2^31 rows)
        const int n = kv_lens[b], m = new_lens[b];
        return m < 0 || n <= m ? 0 : pages(n) - pages(m);
    };
    long long own = 0;
    for (int b = b0; b < b1; b++) {
        const int n = kv_lens[b], m = new_lens[b];
        const bool cut = m >= 0 && m < n;
        dropped_out[b] = (int)((uint32_t)dropped[b] + (cut ? (uint32_t)(n - m) : 0u));
        own += gone(b);
    }
    long long all;
    long long at = scan(own, ws, all);
    const int total = (int)min(all, (long long)INT_MAX);  // (more than 2^26 pages there are not)
    for (int b = b0; b < b1; b++) {
        to[b] = (int)min(at, (long long)INT_MAX);
        at += gone(b);
    }
    if (tid == 0) to[B] = total;
    __syncthreads();
    int nf = min(max(n_free[0], 0), n_pages);
    for (int k0 = 0; k0 < total; k0 += RELEASE_T) {
        const int k = k0 + tid;
        int page = -1;
        if (k < total) {
            const int b = find_range(to, B, k), i = pages(new_lens[b]) + (k - to[b]);
            if (i < max_blocks) page = table[(size_t)b * max_blocks + i];
        }
        const bool there = (unsigned)page < (unsigned)n_pages;
        long long sum;
        const long long x = nf + scan((long long)there, ws, sum);
        if (there && x < n_pages) free_pages[x] = page;
        nf = (int)min(nf + sum, (long long)n_pages);
    }
    if (tid == 0) n_free_out[0] = nf;
}

// ---- their moves ----------------------------------------------------------------------------------------------------

// Sources lie behind all places that are written, so moves run in any order.  A workgroup takes every gridDim.x-th move of
// a (request, kv head): 256 threads, HD elements of K and of V.
template <int HD>
__global__ __launch_bounds__(256) void k_paged_move(const int* __restrict__ moves, const int* __restrict__ counts,
                                                    const int* __restrict__ table, int max_blocks, int W, int HK, int lps,
                                                    int n_pages, size_t pstride, uint16_t* Kp, uint16_t* Vp, float* scores,
                                                    int* kpos) {
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const size_t bh = (size_t)b * HK + h;
    const int n = min(counts[bh], W);
    const int* const mv = moves + bh * W * 2;
    const int* const tb = table + (size_t)b * max_blocks;
    const long long rows = (long long)max_blocks << lps;
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const int to = mv[2 * i], from = mv[2 * i + 1];
        if (to < 0 || from < 0 || to >= rows || from >= rows) continue;
        const int pt = tb[to >> lps], pf = tb[from >> lps];
        if ((unsigned)pt >= (unsigned)n_pages || (unsigned)pf >= (unsigned)n_pages) continue;
        auto block = [&](int page, int j) {
            return (size_t)page * pstride + ((size_t)(h << (lps - 5)) + ((j & ((1 << lps) - 1)) >> 5)) * (HD * 32);
        };
        const size_t x = block(pt, to), y = block(pf, from);
        for (int d = tid; d < HD; d += 256) {
            Kp[x + d / 32 * 1024 + (to & 31) * 32 + d % 32] = Kp[y + d / 32 * 1024 + (from & 31) * 32 + d % 32];
            Vp[x + d * 32 + (to & 31)] = Vp[y + d * 32 + (from & 31)];
        }
        if (tid == 0) {
            const size_t u = mark_at(pt, HK, h, to, lps), v = mark_at(pf, HK, h, from, lps);
            if (scores) scores[u] = scores[v];
            if (kpos) kpos[u] = kpos[v];
        }
    }
}

template <class T, int HD>
void weights_as(const PagedShape& s, const PagedWeights& a, hipStream_t st) {
    const WeightArgs g{a.table, a.cu, a.kv_lens, a.pos, a.max_blocks, a.B, a.rows, s.HQ, s.HK, s.HQ / s.HK, log2i(s.PS),
                       s.n_pages, a.max_new, a.max_kv, a.window, a.observers, a.scale * LOG2E, a.decay, s.pstride, a.scores,
                       a.out, a.kpos};
    const T *Q = static_cast<const T*>(a.Q), *K = static_cast<const T*>(a.Kp);
    float2* const ml = static_cast<float2*>(a.ws);
    const int most = std::min({a.max_new, a.rows, a.observers ? a.observers : INT_MAX});
    hipLaunchKernelGGL((k_weights_stats<T, HD>), dim3(s.HQ * std::min(most, 4096), a.B), dim3(64), 0, st, Q, K, g, ml);
    launched("paged_weights");
    hipLaunchKernelGGL((k_weights_sum<T, HD>), dim3((a.max_kv + 255) / 256, s.HK, a.B), dim3(256), 0, st, Q, K, g, ml);
    launched("paged_weights");
}

}  // namespace

size_t paged_weights_ws(const PagedShape& s, int, int rows, int, int, int) { return (size_t)rows * s.HQ * 8; }

void paged_weights(const PagedShape& s, const PagedWeights& a, hipStream_t st) {
    by_type(s, [&](auto t, auto hd) { weights_as<decltype(t), decltype(hd)::value>(s, a, st); });
}

size_t page_evict_ws(int, int, int) { return 0; }

void page_evict(const PageEvict& a, hipStream_t st) {
    hipLaunchKernelGGL(k_page_evict, dim3(a.HK, a.B), dim3(EVICT_T), 0, st, a.scores, a.kpos, a.table, a.max_blocks, a.kv_lens,
                       a.budgets, a.max_kv, a.HK, log2i(a.PS), a.n_pages, a.sink, a.recent, a.new_lens, a.moves, a.counts);
    launched("page_evict");
}

void page_release(const PageRelease& a, hipStream_t st) {
    hipLaunchKernelGGL(k_page_release, dim3(1), dim3(RELEASE_T), 0, st, a.kv_lens, a.new_lens, a.dropped, a.table, a.max_blocks,
                       a.B, log2i(a.PS), a.n_pages, a.free_pages, a.n_free, a.dropped_out, a.n_free_out);
    launched("page_release");
}

void paged_move(const PagedShape& s, const PagedMove& a, hipStream_t st) {
    const int W = std::max(a.max_kv / 2, 1);
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(std::min(W, std::max(1, 4096 / (s.HK * a.B))), s.HK, a.B), dim3(256), 0, st, a.moves,
                           a.counts, a.table, a.max_blocks, W, s.HK, log2i(s.PS), s.n_pages, s.pstride,
                           static_cast<uint16_t*>(a.Kp), static_cast<uint16_t*>(a.Vp), a.scores, a.kpos);
    };
    if (s.HD == 64) launch(k_paged_move<64>);
    else if (s.HD == 128) launch(k_paged_move<128>);
    else launch(k_paged_move<256>);
    launched("paged_move");
}

}  // namespace sd
