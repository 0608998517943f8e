// Rows that leave the paged cache: the attention weight that every cached key receives, the rows of each kv head that go
// when a request holds more than it may, the moves of those that stay into their places, and the pages behind them (no
// counterpart in the reference, whose cache holds one sequence and forgets nothing).
//
// Scores and positions of cached rows lie in arrays [n_pages][HK][PS], addressed by the same table as the caches.
#include "paged.h"

namespace sd {
namespace {

// 16 bytes of arrays that are aligned to 4.
typedef int i32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));

// Index of (page, kv head, row j) in an array [n_pages][HK][PS].
__device__ __forceinline__ size_t mark_at(int page, int HK, int h, int j, int lps) {
    return ((size_t)page * HK + h) * ((size_t)1 << lps) + (j & ((1 << lps) - 1));
}

// ---- the weight that every cached key receives ----------------------------------------------------------------------
//
// A key's weight is the sum over rows of exp(s - m) / l, and a row's maximum m and sum l are known only when all of its
// keys have been read: two passes over the scores.  A kv head's rows are its request's (token, query head) pairs as in the
// attention kernels.
//
// Few rows (one new token's heads, or up to 32): bound by the keys' bytes, so they are read once: the first pass leaves
// its scores, rows x 4 bytes a key where a key has 2 HD.  Many rows: bound by the products and the exponentials, and rows x
// 4 bytes a key would be the more: both passes compute the scores, with the roles swapped: the first keeps 32 rows of
// queries in a wave's registers and lets keys pass, the second keeps 32 keys and lets rows pass, so each sums in registers
// over what passes and neither needs another lane's values until its end.
//
// Scores are S^T = K Q^T (keys x rows) on MFMA, in f32, and so is all behind them; exponentials are in base 2, c = scale log2 e.
// Few rows keep c s, rounded, and its maximum m; exponents are the differences.  Many rows keep the maximum of s, and exponents
// are (s - m) c: a subtraction more than one fma of s, c and m, and with it sums and weights are the same function of s whatever
// the size of the scores, of other keys' or of other rows' (a fused c s - m, m rounded, leaves the rounding's 2^x in a row's sum,
// and has to be left from 2^23 on, where m has no fractions, at one key for the sum and at another for the weights).
// Sums have one order: over a lane's own keys or rows, then lanes, waves, and parts by their number.

struct WeightArgs {
    const int *table, *cu, *kv_lens, *pos;
    int max_blocks, B, rows, HQ, HK, G, lps, n_pages, max_new, kcap, window, observers;
    int few, few_ks, few_span, rw, kvp;        // rows of a request that the few rows' kernels do; their splits, blocks of 32
                                               // keys in each; rows and keys of a request's scores
    int first;                                 // request of a launch whose requests are some of all
    int tiles, ks, span;                       // many rows: tiles of rows, their splits, blocks in each;
    int part, parts, units;                    // tokens of a part, parts of a request at most, (key tile, part)s at most
    int slots;                                 // parts that `col` holds, of each key tile
    int ordered;                               // requests by length, the longest first
    int dt, dg;                                // 32 rows: tokens, and heads besides
    uint32_t magic;  // 2^32 / G and 1 more: x / G is the upper half of a product for x below 2^16
    float c, decay;  // c: scale log2(e)
    size_t pstride;
    const float* scores;
    float* out;
    int* kpos;
    float* S;         // [requests of a launch][HK][rw][kvp]: c s of the few rows
    float2* few_ml;   // [requests of a launch][HK][few_ks][rw]: their maxima and sums
    float2* ml;       // [ks][tiles][HK][ROW_TILE]: those of many rows
    float2* stat;     // [rows][HQ], a request's rows kv head by kv head: the maximum, and the whole sum's reciprocal
    float* col;       // [key tiles][slots][HK][KEY_TILE]: parts of the keys' weights
    int* index;       // [3][B + 1]: the first tile of every request, and how many there are: of rows, of (key tile, part)s, of
                      // keys of requests with several parts.  null: each workgroup finds its own
    // the first key that a row at position p sees
    __device__ __forceinline__ int from(int p) const { return window ? max(p, -1) - window + 1 : 0; }
};

// The rows of a request that are counted: its last `observers` tokens, from `t0` on, n of them.
struct Seen {
    int t0, n;
};
__device__ __forceinline__ Seen observed(const Req& r, int observers) {
    const int n = observers ? min(r.n, observers) : r.n;
    return {r.n - n, n};
}

// c s, rounded: what a few rows' maximum is one of.
__device__ __forceinline__ float scaled(float s, float c) {
#pragma clang fp contract(off)
    return s * c;
}

// A row's part: maximum and sum, and their turn to a row's whole.
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }  // (its sum is 0, or NaN)
__device__ __forceinline__ float inverse_of(float l) { return l == 0.f ? 0.f : 1.0f / l; }

// A row's sum over a split of its keys, block by block, and what its roundings have left out so far: the split may be the whole
// cache, and where one key's weight stands out over thousands of equal ones each addition would be off the same way (2.4e-4 of the
// sum after 32768 addends).  A block's exponentials are added in pairs.
struct LongSum {
    float sum = 0.f, rest = 0.f;
    __device__ __forceinline__ void add(float scale, float x) {  // the sum so far times `scale`, and x
#pragma clang fp contract(off)
        const float l = sum * scale, y = x + rest * scale;
        sum = l + y;
        rest = y - (sum - l);
    }
};
template <int N>
__device__ __forceinline__ float sum_pairs(float (&x)[N]) {
#pragma unroll
    for (int o = N / 2; o; o >>= 1)
#pragma unroll
        for (int e = 0; e < o; e++) x[e] += x[e + o];
    return x[0];
}

// Where the statistics of a request's rows of kv head kh begin.
__device__ __forceinline__ size_t stat_at(const WeightArgs& a, const Req& rq, const Seen& ob, int kh) {
    return (size_t)(rq.q0 + ob.t0) * a.HQ + (size_t)kh * ob.n * a.G;
}

// The weight of a part whose maximum of s is m, as part_weight.
__device__ __forceinline__ float part_of(float m, float mx, float c) { return m == -INFINITY ? 0.f : exp2_fast((m - mx) * c); }

// A row's whole, from its n parts, `step` apart: N lanes on end share it.  c: 1 where the maxima are c s.
template <int N>
__device__ __forceinline__ float2 join_parts(const float2* ml, size_t step, int n, float c) {
    float mx = -INFINITY, l = 0.f;
#pragma unroll 4
    for (int z = threadIdx.x % N; z < n; z += N) {
        const float2 v = ml[z * step];
        const float mn = fmaxf(mx, v.x);
        l = l * part_of(mx, mn, c) + v.y * part_of(v.x, mn, c);
        mx = mn;
    }
#pragma unroll
    for (int o = 1; o < N; o <<= 1) {
        const float m2 = __shfl_xor(mx, o), l2 = __shfl_xor(l, o), mn = fmaxf(mx, m2);
        l = l * part_of(mx, mn, c) + l2 * part_of(m2, mn, c);
        mx = mn;
    }
    return make_float2(base_of(mx), inverse_of(l));
}

// Key j's weight w of a request's rows, into the scores of kv head h.
__device__ __forceinline__ void put_weight(const WeightArgs& a, const Req& rq, size_t at, int j, float w) {
    const bool old = j < rq.p0;
    a.out[at] = old && a.decay != 0.f ? __builtin_fmaf(a.decay, a.scores[at], w) : w;
    if (!old && a.kpos) a.kpos[at] = a.pos[rq.q0 + j - rq.p0];
}

// ---- few rows ----

// What a few rows' kernel does with a request: its rows, the first one's position, and the keys [lo, hi) that some row sees.
struct Few {
    Req rq;
    Seen ob;
    int nrows, p0, lo, hi;
};
__device__ __forceinline__ Few few_of(const WeightArgs& a, int b) {
    Few f;
    f.rq = request(a.cu, a.kv_lens, b, a.rows, a.max_new, a.kcap);
    f.ob = observed(f.rq, a.observers);
    f.nrows = f.ob.n * a.G;
    f.p0 = f.rq.p0 + f.ob.t0;
    f.hi = min(f.p0 + f.ob.n, f.rq.kcap);
    f.lo = max(0, a.from(f.p0));
    return f;
}

// Scores of up to 16 NR rows of a (request, kv head) over blocks [blk0, blk1) of keys, by NW waves, into S (rows `stride`
// floats apart, key j at j), and each wave's maxima and sums of the rows over them.  A wave loads K straight into registers
// in MFMA operand order, D blocks of 32 keys in flight.
template <class T, int HD, int NR, bool ONCE, int NW, int D>
__device__ __forceinline__ void few_scores(const T* __restrict__ Q, const T* __restrict__ Kp, const WeightArgs& a, const Few& f, int b,
                                           int kh, int blk0, int blk1, float* S, int stride, float* Ms, float* Ls) {
    typedef typename Vec8<T>::type T8;
    constexpr int NS = HD / 32, R = 16 * NR;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int fq = lane & 15, fg = lane >> 4;
    const Req& rq = f.rq;
    const Seen& ob = f.ob;
    const int nrows = f.nrows, p0 = f.p0, hi = f.hi;
    const int first = blk0 + wv, cnt = first < blk1 ? (blk1 - first + NW - 1) / NW : 0;
    int jlo[NR], jhi[NR];  // keys [jlo, jhi) are seen by this lane's row
    T8 qf[NR][NS];
#pragma unroll
    for (int u = 0; u < NR; u++) {
        const int r = min(16 * u + fq, nrows - 1), t = ob.t0 + r / a.G, h = kh * a.G + r % a.G;
        jlo[u] = a.from(rq.p0 + t);
        jhi[u] = min(rq.p0 + t + 1, hi);
        const T* q = Q + ((size_t)(rq.q0 + t) * a.HQ + h) * HD + 8 * fg;
#pragma unroll
        for (int s = 0; s < NS; s++) qf[u][s] = *reinterpret_cast<const T8*>(q + 32 * s);
    }
    const int open0 = a.from(p0 + ob.n - 1), open1 = min(p0 + 1, hi);  // keys in [open0, open1) are seen by every row
    const int lbpp = a.lps - 5;
    const int* const tb = a.table + (size_t)b * a.max_blocks;
    auto entries = [&](int i) {  // lane l: the table entry of the wave's block i + l
        return tb[min((first + NW * (i + lane)) >> lbpp, a.max_blocks - 1)];
    };
    int ids = cnt ? entries(0) : 0, ids2 = cnt > 64 ? entries(64) : 0;
    // rows of K in the order in which a lane's 8 scores are 8 keys on end: j0 + 8 fg + e
    const uint32_t kofs = ((8 * (fq >> 2) + (fq & 3)) * 32 + fg * 8) * 2;
    float m[NR];
    LongSum l[NR];
#pragma unroll
    for (int u = 0; u < NR; u++) m[u] = -INFINITY;
    struct Blk {
        u32x4 k[2][NS];
        bool there;
    };
    auto load = [&](int i, Blk& x) INL {
        const int page = __builtin_amdgcn_readlane(ids, i & 63), blk = first + NW * i;
        x.there = i < cnt && (unsigned)page < (unsigned)a.n_pages;
        const size_t at = x.there ? (size_t)page * a.pstride + ((size_t)(kh << lbpp) + (blk & ((1 << lbpp) - 1))) * (HD * 32) : 0;
        const Rsrc rk = make_rsrc(Kp + at, x.there ? HD * 64u : 0u);
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int tt = 0; tt < 2; tt++) x.k[tt][s] = load16<ONCE>(rk, kofs + tt * 256, s * 2048);
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
#pragma unroll
        for (int u = 0; u < NR; u++) {
#pragma unroll
            for (int e = 0; e < 8; e++) s2[u][e >> 2][e & 3] = scaled(s2[u][e >> 2][e & 3], a.c);
            if (!open) {
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int j = j0 + 8 * fg + e;
                    const bool keep = x.there & (j >= jlo[u]) & (j < jhi[u]);
                    s2[u][e >> 2][e & 3] = keep ? s2[u][e >> 2][e & 3] : -INFINITY;
                }
            }
            if (16 * u + fq < nrows) {
                f32x4* const to = reinterpret_cast<f32x4*>(S + (size_t)(16 * u + fq) * stride + j0 + 8 * fg);
                to[0] = s2[u][0], to[1] = s2[u][1];
            }
            float mn = m[u];
#pragma unroll
            for (int e = 0; e < 8; e++) mn = fmaxf(mn, s2[u][e >> 2][e & 3]);
            const float base = base_of(mn);
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] = exp2_fast(s2[u][e >> 2][e & 3] - base);
            l[u].add(exp2_fast(m[u] - base), sum_pairs(x));
            m[u] = mn;
        }
    };
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
#pragma unroll
    for (int u = 0; u < NR; u++) {
        const float mx = max_quarters(m[u]);
        float sum = l[u].sum * part_weight(m[u], mx);
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (fg == 0) Ms[wv * R + 16 * u + fq] = mx, Ls[wv * R + 16 * u + fq] = sum;
    }
}

constexpr int FEW_W = 2;  // waves of a workgroup (1 and 4, with as many splits: level or slower)

// A split of the keys per workgroup.  One token of one request, 700 keys, 2 heads of 256 dims: 4.1 us, and 4.1 for the sums
// below: two launches whose loads (lengths, table, keys; parts, scores) come one after the other; the bytes would take 0.1.
template <class T, int HD, int NR, bool ONCE>
__global__ __launch_bounds__(64 * FEW_W) void k_weights_few(const T* __restrict__ Q, const T* __restrict__ Kp, WeightArgs a) {
    constexpr int R = 16 * NR;
    __shared__ float Ms[FEW_W * R], Ls[FEW_W * R];
    const int tid = threadIdx.x, kh = blockIdx.x % a.HK, z = blockIdx.x / a.HK, b = a.first + blockIdx.y;
    const size_t bh = (size_t)blockIdx.y * a.HK + kh;
    const Few f = few_of(a, b);
    if (f.nrows == 0 || f.nrows > a.few) return;
    const int blk0 = (f.lo >> 5) + z * a.few_span;
    const int blk1 = z + 1 < a.few_ks ? min((f.hi + 31) >> 5, blk0 + a.few_span) : (f.hi + 31) >> 5;
    few_scores<T, HD, NR, ONCE, FEW_W, HD == 64 ? 4 : HD == 128 ? 3 : 2>(Q, Kp, a, f, b, kh, blk0, blk1, a.S + bh * a.rw * a.kvp, a.kvp, Ms, Ls);
    __syncthreads();
    if (tid < f.nrows) {
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < FEW_W; w++) mx = fmaxf(mx, Ms[w * R + tid]);
#pragma unroll
        for (int w = 0; w < FEW_W; w++) sum += Ls[w * R + tid] * part_weight(Ms[w * R + tid], mx);
        a.few_ml[(bh * a.few_ks + z) * a.rw + tid] = make_float2(mx, sum);
    }
}

// 4 keys from j on: their place, and what they have.
struct Keys4 {
    int page;
    size_t at;
    f32x4u old;
};
__device__ __forceinline__ int page_of(const WeightArgs& a, int b, int j) {
    return a.table[(size_t)b * a.max_blocks + min(j >> a.lps, a.max_blocks - 1)];
}
__device__ __forceinline__ Keys4 keys4(const WeightArgs& a, const Few& f, int kh, int j, int page) {
    Keys4 k;
    k.page = page;
    const bool there = j < f.rq.kcap && (unsigned)k.page < (unsigned)a.n_pages;
    k.at = mark_at(there ? k.page : 0, a.HK, kh, there ? j : 0, a.lps);
    k.old = f32x4u{0.f, 0.f, 0.f, 0.f};
    if (there && a.decay != 0.f) k.old = *reinterpret_cast<const f32x4u*>(a.scores + k.at);
    return k;
}
__device__ __forceinline__ bool some_seen(const Few& f, int j) { return j > f.lo - 4 && j < f.hi; }  // (scores outside were not written)

// Their weights of the rows, x(r) their scores of row r, PRE of which come from `pre`; into the cached keys' scores.
template <int PRE, class X>
__device__ __forceinline__ void weigh4(const WeightArgs& a, const Few& f, int j, const Keys4& k, const float2* stat, const f32x4* pre, X&& x) {
    if (j >= f.rq.kcap || (unsigned)k.page >= (unsigned)a.n_pages) return;
    f32x4 w = {0.f, 0.f, 0.f, 0.f};
    if (some_seen(f, j)) {
        int t = 0, g = 0;
        auto add = [&](int r, f32x4 x) INL {
            const float2 st = stat[r];
            const int jlo = a.from(f.p0 + t), jhi = min(f.p0 + t + 1, f.hi);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const bool keep = (j + e >= jlo) & (j + e < jhi);
                w[e] += keep ? exp2_fast(x[e] - st.x) * st.y : 0.f;
            }
            if (++g == a.G) g = 0, t++;
        };
#pragma unroll
        for (int r = 0; r < PRE; r++)
            if (r < f.nrows) add(r, pre[r]);
#pragma unroll 4
        for (int r = PRE; r < f.nrows; r++) add(r, x(r));
    }
    if (j <= min(f.rq.p0, f.rq.kcap) - 4) {
        f32x4u y;
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = a.decay != 0.f ? __builtin_fmaf(a.decay, k.old[e], w[e]) : w[e];
        *reinterpret_cast<f32x4u*>(a.out + k.at) = y;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++)
            if (j + e < f.rq.kcap) put_weight(a, f.rq, k.at + e, j + e, w[e]);
    }
}

// The weights of the few rows' splits, from their scores: 4 keys per thread, after every workgroup has joined the rows' parts.
__global__ __launch_bounds__(256) void k_weights_few_sum(WeightArgs a) {
    constexpr int PRE = 4;
    __shared__ float2 stat[32];
    const int tid = threadIdx.x, kh = blockIdx.x % a.HK, b = a.first + blockIdx.y;
    const size_t bh = (size_t)blockIdx.y * a.HK + kh;
    const int c0 = blockIdx.x / a.HK * 1024, step = gridDim.x / a.HK * 1024;  // (with 8 heads a head's scores stay with one XCD's L2)
    const Few f = few_of(a, b);
    const int nrows = f.nrows;
    if (nrows == 0 || nrows > a.few || c0 >= f.rq.kcap) return;
    const float* const S = a.S + bh * a.rw * a.kvp;
    struct Keys {
        Keys4 k;
        f32x4 x[PRE];  // the scores of the first PRE rows
    };
    auto load = [&](int j) INL {
        Keys k;
        k.k = keys4(a, f, kh, j, page_of(a, b, j));
#pragma unroll
        for (int r = 0; r < PRE; r++) {
            k.x[r] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (some_seen(f, j) && r < nrows) k.x[r] = *reinterpret_cast<const f32x4*>(S + (size_t)r * a.kvp + j);
        }
        return k;
    };
    Keys k = load(c0 + 4 * tid);  // (on their way while the rows are joined)
    {
        const float2* const ml = a.few_ml + bh * a.few_ks * a.rw;
        if (nrows <= 4) {
            const float2 st = join_parts<64>(ml + min(tid >> 6, nrows - 1), a.rw, a.few_ks, 1.f);
            if ((tid & 63) == 0) stat[tid >> 6] = st;
        } else {
            const float2 st = join_parts<8>(ml + min(tid >> 3, nrows - 1), a.rw, a.few_ks, 1.f);
            if ((tid & 7) == 0) stat[tid >> 3] = st;
        }
    }
    __syncthreads();
    for (int j0 = c0;; j0 += step) {
        const int j = j0 + 4 * tid;
        const Keys now = k;
        const bool more = step < f.rq.kcap - j0;
        if (more) k = load(j + step);
        weigh4<PRE>(a, f, j, now.k, stat, now.x, [&](int r) { return *reinterpret_cast<const f32x4*>(S + (size_t)r * a.kvp + j); });
        if (!more) break;
    }
}

// Short caches: a (request, kv head) per workgroup, its scores in LDS, in one launch.  64 requests of 1000 to 8191 keys, 8 heads
// of 128 dims: 70 us for 400 MB of keys, 5.7 TB/s, the longest first (as they come 83, in splits 97); 4 waves level, 16 slower.
constexpr int ONE_W = 8, ONE_LDS = 136 << 10, ONE_KEYS = 8192;  // waves; bytes of scores, and keys, at most
constexpr int ONE_ORDER = 64 * ONE_W;  // requests up to which they are taken by length
template <class T, int HD, int NR, bool ONCE>
__global__ __launch_bounds__(64 * ONE_W, HD * NR <= 128 ? 4 : 2) void k_weights_few_one(const T* __restrict__ Q, const T* __restrict__ Kp, WeightArgs a) {
    constexpr int R = 16 * NR, KN = ONE_KEYS / (256 * ONE_W);
    constexpr bool EARLY = HD * NR == 256;
    extern __shared__ __align__(16) float S[];
    __shared__ float Ms[ONE_W * R], Ls[ONE_W * R];
    __shared__ float2 stat[R];
    __shared__ __align__(16) uint32_t by_length[ONE_ORDER];
    __shared__ int nth;
    const int tid = threadIdx.x, kh = blockIdx.x;
    int b = blockIdx.y;
    if (a.ordered) {  // the longest first: the b-th of them
        uint32_t own = 0;
        if (tid < a.B) own = (uint32_t)min(max(a.kv_lens[tid], 0), ONE_KEYS) * ONE_ORDER + tid;
        by_length[tid] = own;
        __syncthreads();
        if (tid < a.B) {
            int longer = 0;
#pragma unroll 4
            for (int i = 0; i < a.B; i += 4) {
                const u32x4 x = *reinterpret_cast<const u32x4*>(by_length + i);
#pragma unroll
                for (int e = 0; e < 4; e++) longer += x[e] > own;
            }
            if (longer == b) nth = tid;
        }
        __syncthreads();
        b = __builtin_amdgcn_readfirstlane(nth);
    }
    const Few f = few_of(a, b);
    if (f.nrows == 0 || f.nrows > a.few) return;
    int page[KN];  // (what the keys have is on its way meanwhile too, where no second workgroup fits the CU's registers anyway)
    Keys4 k[KN];
#pragma unroll
    for (int i = 0; i < KN; i++) {
        const int j = 4 * (tid + 64 * ONE_W * i);
        page[i] = page_of(a, b, j);
        if (EARLY) k[i] = keys4(a, f, kh, j, page[i]);
    }
    few_scores<T, HD, NR, ONCE, ONE_W, HD == 64 ? 3 : 2>(Q, Kp, a, f, b, kh, f.lo >> 5, (f.hi + 31) >> 5, S, a.kvp, Ms, Ls);
#pragma unroll
    for (int i = 0; i < KN; i++)
        if (!EARLY) k[i] = keys4(a, f, kh, 4 * (tid + 64 * ONE_W * i), page[i]);
    __syncthreads();
    if (tid < f.nrows) {
        float mx = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < ONE_W; w++) mx = fmaxf(mx, Ms[w * R + tid]);
#pragma unroll
        for (int w = 0; w < ONE_W; w++) sum += Ls[w * R + tid] * part_weight(Ms[w * R + tid], mx);
        stat[tid] = make_float2(base_of(mx), inverse_of(sum));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < KN; i++) {
        const int j = 4 * (tid + 64 * ONE_W * i);
        weigh4<0>(a, f, j, k[i], stat, nullptr, [&](int r) { return *reinterpret_cast<const f32x4*>(S + r * a.kvp + j); });
    }
}

// ---- many rows ----

constexpr int ROW_TILE = 128, KEY_TILE = 128;

__device__ __forceinline__ int many_rows(const WeightArgs& a, int b) {  // of request b, 0 where they are few
    const int n = observed(request(a.cu, a.kv_lens, b, a.rows, a.max_new, a.kcap), a.observers).n * a.G;
    return n > a.few ? n : 0;
}
// Tile x of those that `which` says, `of(b)` of request b, as find_tile numbers them; in the index, which holds them in the
// requests' order, by the lanes' steps through it, and by theirs through the step.
enum { ROW_TILES, KEY_PARTS, KEY_TILES };
template <class F>
__device__ __forceinline__ Tile tile_of(const WeightArgs& a, int which, int x, F&& of) {
    if (!a.index) return find_tile(a.B, x, of);
    const int* const first = a.index + which * (a.B + 1);
    const int lane = threadIdx.x & 63, step = (a.B + 63) >> 6;  // (128 at most)
    const int total = first[a.B], y = first[min(lane * step, a.B)];
    if (x >= total) return {-1, 0, 0};
    const int n = total - 1 - x;
    const int b0 = (__popcll(__ballot(lane * step < a.B && y <= n)) - 1) * step, b1 = min(b0 + step, a.B);
    const int u = first[min(b0 + lane, a.B)], v = first[min(b0 + 64 + lane, a.B)];
    const int at = __popcll(__ballot(b0 + lane < b1 && u <= n)) + __popcll(__ballot(b0 + 64 + lane < b1 && v <= n)) - 1;
    return {b0 + at, n - (at < 64 ? __builtin_amdgcn_readlane(u, at) : __builtin_amdgcn_readlane(v, at - 64)), n};
}
__device__ __forceinline__ int row_tiles(const WeightArgs& a, int b) { return (many_rows(a, b) + ROW_TILE - 1) / ROW_TILE; }
__device__ __forceinline__ Tile row_tile(const WeightArgs& a, int x) {
    return tile_of(a, ROW_TILES, x, [&](int b) { return row_tiles(a, b); });
}

// A tile's rows, the keys that some of them see, and this split's blocks of those.
struct RowTile {
    Req rq;
    Seen ob;
    int nrows, r0, r1, lo, hi, blk0, blk1;
};
__device__ __forceinline__ RowTile row_tile_of(const WeightArgs& a, const Tile& tl, int z) {
    RowTile t;
    t.rq = request(a.cu, a.kv_lens, tl.b, a.rows, a.max_new, a.kcap);
    t.ob = observed(t.rq, a.observers);
    t.nrows = t.ob.n * a.G;
    t.r0 = tl.i * ROW_TILE;
    t.r1 = min(t.nrows, t.r0 + ROW_TILE);
    const int p = t.rq.p0 + t.ob.t0;
    t.hi = min(p + (t.r1 - 1) / a.G + 1, t.rq.kcap);
    t.lo = max(0, a.from(p + t.r0 / a.G));
    t.blk0 = (t.lo >> 5) + z * a.span;
    t.blk1 = min((t.hi + 31) >> 5, t.blk0 + a.span);
    return t;
}

// A ring of blocks in LDS, NB of them: block i is in buffer i % NB, and while it is worked on the NB - 1 after it are on their
// way.  (An array per buffer: the compiler then sees that the DMAs into one never alias the reads of another.)  With 256 dims two
// are enough, since the CU then has room for four workgroups, which cover each other's waits.
#define RING(X)                                                                                          \
    __shared__ __align__(1024) uint8_t X##0[Rg::BYTES], X##1[Rg::BYTES], X##2[NB > 2 ? Rg::BYTES : 16], \
        X##3[NB > 3 ? Rg::BYTES : 16];
// turn(i, its buffer, the buffer that block i + NB - 1 goes to) for n blocks.
#define RING_START(X, fetch)        \
    fetch(0, X##0);                 \
    if (NB > 2) fetch(1, X##1);     \
    if (NB > 3) fetch(2, X##2);
#define RING_LOOP(X, n)                                               \
    for (int i = 0;;) {                                               \
        turn(i, X##0, NB == 4 ? X##3 : NB == 3 ? X##2 : X##1);        \
        if (++i >= n) break;                                          \
        turn(i, X##1, X##0);                                          \
        if (++i >= n) break;                                          \
        if (NB > 2) {                                                 \
            turn(i, X##2, X##1);                                      \
            if (++i >= n) break;                                      \
        }                                                             \
        if (NB > 3) {                                                 \
            turn(i, X##3, X##2);                                      \
            if (++i >= n) break;                                      \
        }                                                             \
    }

// Blocks of 32 rows x HD of a ring in LDS: [HD / 32][32 rows][64 bytes], the 16-byte pieces of each row at p ^ (row / 4) % 4,
// so that neither the DMAs' writes nor the fragments' reads meet a bank twice.
template <int HD>
struct Ring {
    static constexpr int BYTES = HD * 64, IW = BYTES / 4096, NB = HD == 256 ? 2 : HD == 128 ? 3 : 4;  // of a block; its DMAs per wave
    static __device__ __forceinline__ u32x4 read(const uint8_t* buf, int st, int c, int g) {
        return *reinterpret_cast<const u32x4*>(buf + (st >> 1) * 2048 + c * 64 + (((2 * (st & 1) + g) ^ ((c >> 2) & 3)) << 4));
    }
};

// The key of a block that is register e of S^T in the lanes of half g, less 4 g.
__device__ __forceinline__ constexpr int key_of(int e) { return 8 * (e >> 2) + (e & 3); }

// Keys lo to hi of a block, as a test of the constants key_of(e) that takes no register for each: one subtraction and an
// unsigned comparison.
struct Within {
    uint32_t from, span;
    __device__ __forceinline__ Within(int lo, int hi) {
        lo = max(lo, 0);
        from = hi < lo ? 1u << 30 : (uint32_t)lo, span = hi < lo ? 0u : (uint32_t)(hi - lo);
    }
    __device__ __forceinline__ bool has(int k) const { return (uint32_t)k - from <= span; }
};

// Maxima and sums of 128 rows over a split of their keys: each wave has 32 rows' queries in registers, and all four share
// blocks of 32 keys that arrive by LDS DMA, in a ring.  A lane keeps its own maximum and sum of the half of each block that it
// has; the two halves meet at the end.
//
// A block is one chain: reads from LDS, products, maximum, exponentials.  Four workgroups on a CU cover each other's, so a wave
// may take 128 registers.  A prompt of 4096 (8 query heads on 2, 256 dims) 51 us where the products alone would take 29: CUs are
// busy for three quarters of it, and of those cycles products have 43 %, vector instructions 40 %.  On 32 rows of 2
// caches of 60 to 131 thousand keys 32 us, 4.3 TB/s.  Measured and slower: 64 rows a wave with two workgroups on a CU, the
// rows of a short question in LDS with waves by themselves, fragments read four ahead, two accumulators in turn, 256 to 1024
// keys a workgroup less or more, tiles in the other order, the last split of each tile at the end (level).
template <class T, int HD>
__global__ __launch_bounds__(256, 4) void k_weights_rows(const T* __restrict__ Q, const T* __restrict__ Kp, WeightArgs a) {
    typedef typename Vec8<T>::type T8;
    typedef Ring<HD> Rg;
    constexpr int NS = HD / 16, NB = Rg::NB, IW = Rg::IW, PART = Rg::BYTES / 4;
    RING(K)
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, g = lane >> 5;
    // The split changes slowest, and by an odd number of tiles: an XCD has every eighth workgroup, late splits have no keys for
    // most tiles, and there are fewer tiles than their bound.
    const int kh = blockIdx.x % a.HK, tiles = a.tiles | 1, z = blockIdx.x / (a.HK * tiles), x = blockIdx.x / a.HK % tiles;
    if (x >= a.tiles) return;
    const Tile tl = row_tile(a, x);
    if (tl.b < 0 || tl.x >= a.tiles) return;  // (more tiles than rows make: row starts that do not ascend)
    const RowTile t = row_tile_of(a, tl, z);
    const int nb = t.blk1 - t.blk0;
    if (nb <= 0) return;
    const int w0 = t.r0 + 32 * wv, w1 = min(w0 + 32, t.r1);
    const bool live = w0 < t.r1;
    const int p0 = t.rq.p0 + t.ob.t0;
    const int all0 = a.from(p0 + (w1 - 1) / a.G), all1 = min(p0 + w0 / a.G + 1, t.hi);
    const int lbpp = a.lps - 5;
    const int* const tb = a.table + (size_t)tl.b * a.max_blocks;
    auto entries = [&](int i) { return tb[min((t.blk0 + i + lane) >> lbpp, a.max_blocks - 1)]; };  // lane l: of block i + l
    int win = 0, ids = entries(0), ids2 = entries(32);
    auto there = [&](int i, int& page) INL {
        page = __builtin_amdgcn_readlane(ids, i - win);
        return i < nb && (unsigned)page < (unsigned)a.n_pages;
    };
    const uint32_t dlane = (uint32_t)((lane >> 2) * 64 + (((lane & 3) ^ ((lane >> 4) & 3)) << 4));
    auto fetch = [&](int i, uint8_t* buf) INL {  // (the same number of DMAs always: of what is not there, of zeros)
        int page;
        const bool ok = there(i, page);
        const int blk = t.blk0 + i;
        const size_t at = ok ? (size_t)page * a.pstride + ((size_t)(kh << lbpp) + (blk & ((1 << lbpp) - 1))) * (HD * 32) : 0;
        const Rsrc rs = make_rsrc(Kp + at, ok ? Rg::BYTES : 0);
#pragma unroll
        for (int u = 0; u < IW; u++) buf_lds16(rs, dlane, wv * PART + u * 1024, buf + wv * PART + u * 1024);
    };
    T8 qf[NS];
    const int r = min(w0 + c, t.r1 - 1), tok = t.ob.t0 + r / a.G;
    const int jlo = a.from(t.rq.p0 + tok), jhi = min(t.rq.p0 + tok + 1, t.hi);
    {
        const T* const q = Q + ((size_t)(t.rq.q0 + tok) * a.HQ + kh * a.G + r % a.G) * HD + 8 * g;
#pragma unroll
        for (int s = 0; s < NS; s++) qf[s] = *reinterpret_cast<const T8*>(q + 16 * s);
    }
    float m = -INFINITY;
    LongSum l;
    auto turn = [&](int i, const uint8_t* K, uint8_t* Kx) INL {
        wait_loads<vmcnt_imm((NB - 2) * IW)>();
        lds_barrier();  // block i is there for every wave, the one before is done with
        if (i >= win + 32) win += 32, ids = ids2, ids2 = entries(win + 32);
        fetch(i + NB - 1, Kx);
        if (!live) return;
        f32x16 s;
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = 0.f;
#pragma unroll
        for (int st = 0; st < NS; st++) s = Num<T>::mfma32(__builtin_bit_cast(T8, Rg::read(K, st, c, g)), qf[st], s);
        const int j0 = (t.blk0 + i) * 32;
        int page;
        const bool ok = there(i, page);
        if (!(ok && j0 >= all0 && j0 + 32 <= all1)) {
            const Within keep(max(jlo, 0) - j0 - 4 * g, ok ? max(jhi, 0) - 1 - j0 - 4 * g : -1);
#pragma unroll
            for (int e = 0; e < 16; e++) s[e] = keep.has(key_of(e)) ? s[e] : -INFINITY;
        }
        float top = s[0];
#pragma unroll
        for (int e = 1; e < 16; e++) top = fmaxf(top, s[e]);
        const float mn = fmaxf(m, top), base = base_of(mn);
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; e++) x[e] = exp2_fast((s[e] - base) * a.c);
        l.add(exp2_fast((m - base) * a.c), sum_pairs(x));
        m = mn;
    };
    RING_START(K, fetch)
    RING_LOOP(K, nb)
    wait_loads<vmcnt_imm(0)>();  // (no DMA outlives the workgroup whose LDS it writes)
    const float mx = max_halves(m);
    float sum = l.sum * part_of(m, mx, a.c);
    sum += __shfl_xor(sum, 32);
    if (!live || g || w0 + c >= t.r1) return;
    if (a.ks == 1) a.stat[stat_at(a, t.rq, t.ob, kh) + r] = make_float2(base_of(mx), inverse_of(sum));
    else a.ml[(((size_t)z * a.tiles + tl.x) * a.HK + kh) * ROW_TILE + 32 * wv + c] = make_float2(mx, sum);
}

// Joins the splits of the rows: N threads per row.
template <int N>
__global__ __launch_bounds__(256) void k_weights_join(WeightArgs a) {
    constexpr int ROWS = 256 / N, PER = ROW_TILE / ROWS;
    const int kh = blockIdx.x / PER % a.HK;
    const Tile tl = row_tile(a, blockIdx.x / (PER * a.HK));
    if (tl.b < 0 || tl.x >= a.tiles) return;
    const RowTile t = row_tile_of(a, tl, 0);
    const int i = blockIdx.x % PER * ROWS + threadIdx.x / N, r = t.r0 + i;
    if (r >= t.r1) return;
    const int n = min(a.ks, (((t.hi + 31) >> 5) - t.blk0 + a.span - 1) / a.span);
    const float2 st = join_parts<N>(a.ml + ((size_t)tl.x * a.HK + kh) * ROW_TILE + i, (size_t)a.tiles * a.HK * ROW_TILE, n, a.c);
    if (threadIdx.x % N == 0) a.stat[stat_at(a, t.rq, t.ob, kh) + r] = st;
}

// (key tile, part of the rows) x of the requests', numbered through.
__device__ __forceinline__ int key_tiles(const WeightArgs& a, const Req& rq) { return (rq.kcap + KEY_TILE - 1) / KEY_TILE; }
__device__ __forceinline__ int parts_of(const WeightArgs& a, int tokens) { return a.parts == 1 ? 1 : (tokens + a.part - 1) / a.part; }
__device__ __forceinline__ int key_parts(const WeightArgs& a, int b) {
    const Req rq = request(a.cu, a.kv_lens, b, a.rows, a.max_new, a.kcap);
    const int n = observed(rq, a.observers).n;
    return n * a.G > a.few ? parts_of(a, n) * key_tiles(a, rq) : 0;
}
__device__ __forceinline__ Tile key_tile(const WeightArgs& a, int x) {
    return tile_of(a, KEY_PARTS, x, [&](int b) { return key_parts(a, b); });
}
__device__ __forceinline__ int split_key_tiles(const WeightArgs& a, int b) {  // of a request with several parts
    const Req rq = request(a.cu, a.kv_lens, b, a.rows, a.max_new, a.kcap);
    const int n = observed(rq, a.observers).n;
    return n * a.G > a.few && parts_of(a, n) > 1 ? key_tiles(a, rq) : 0;
}
// The first of a request's parts in `col`: `parts` for each request, or, where that is more than the step's rows can need, by
// its first row: two slots per part's tokens, since a request of r > 1 parts' tokens has ceil(r) <= floor(2 r) parts.
__device__ __forceinline__ int slot_of(const WeightArgs& a, const Req& rq, int b) {
    return (long long)a.B * a.parts <= a.slots ? b * a.parts : (int)(2 * (unsigned)rq.q0 / (unsigned)a.part);
}
// The index: one workgroup.  (Sums are cut at 2^24, which row starts that do not ascend could pass.)
constexpr int INDEX_T = 1024;
__global__ __launch_bounds__(INDEX_T) void k_weights_index(WeightArgs a) {
    __shared__ int ws[3][INDEX_T / 64];
    const int tid = threadIdx.x, wv = tid >> 6, per = (a.B + INDEX_T - 1) / INDEX_T, b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    auto cut = [](int x) { return min(x, 1 << 24); };
    int own[3] = {0, 0, 0}, at[3];
    for (int b = b0; b < b1; b++) {
        own[ROW_TILES] = cut(own[ROW_TILES] + row_tiles(a, b));
        own[KEY_PARTS] = cut(own[KEY_PARTS] + key_parts(a, b));
        own[KEY_TILES] = cut(own[KEY_TILES] + split_key_tiles(a, b));
    }
#pragma unroll
    for (int k = 0; k < 3; k++) {
        at[k] = lanes_upto(own[k]);
        if ((tid & 63) == 63) ws[k][wv] = cut(at[k]);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; k++) {
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < INDEX_T / 64; w++) before += w < wv ? ws[k][w] : 0, all += ws[k][w];
        at[k] += before - own[k];
        if (tid == 0) a.index[k * (a.B + 1) + a.B] = cut(all);
    }
    for (int b = b0; b < b1; b++) {
#pragma unroll
        for (int k = 0; k < 3; k++) a.index[k * (a.B + 1) + b] = cut(at[k]);
        at[ROW_TILES] = cut(at[ROW_TILES] + row_tiles(a, b));
        at[KEY_PARTS] = cut(at[KEY_PARTS] + key_parts(a, b));
        at[KEY_TILES] = cut(at[KEY_TILES] + split_key_tiles(a, b));
    }
}
// The tokens [lo, hi) of a request that see some key of [j0, j0 + 128).
__device__ __forceinline__ void tokens_of(const WeightArgs& a, const Req& rq, const Seen& ob, int j0, int& lo, int& hi) {
    const long long p0 = (long long)rq.p0 + ob.t0;
    lo = (int)min((long long)ob.n, max(0ll, j0 - p0));
    hi = a.window ? (int)max(0ll, min((long long)ob.n, j0 + 127ll + a.window - p0)) : ob.n;
}

// The sum of 16 keys' weights over the 32 rows' lanes, halving the registers at each step: lane c has key c / 2.  The partners of
// the first step are 16 lanes away, then 8, 4 of 7 - c, 2 and 1: each differs in the bit that says which half a lane keeps.
template <int CTRL>
__device__ __forceinline__ float from_lane(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float sum_rows(const f32x16& acc) {
#if defined(__HIP_DEVICE_COMPILE__)
    const int c = threadIdx.x & 31;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {  // (one swap of two registers' halves: each lane then has what it keeps, and the other's)
        const float x = acc[e], y = acc[e + 8];
        const auto sw = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y), false, false);
        const uint32_t lo = sw[0], hi = sw[1];
        v[e] = __builtin_bit_cast(float, lo) + __builtin_bit_cast(float, hi);
    }
    auto halve = [&](auto n, auto ctrl) INL {
        constexpr int N = decltype(n)::value;
        const bool up = c & 2 * N;
#pragma unroll
        for (int e = 0; e < N; e++) {
            const float x = v[e], y = v[e + N];
            v[e] = (up ? y : x) + from_lane<decltype(ctrl)::value>(up ? x : y);
        }
    };
    using std::integral_constant;
    halve(integral_constant<int, 4>(), integral_constant<int, 0x128>());  // 8 lanes on in each row of 16
    halve(integral_constant<int, 2>(), integral_constant<int, 0x141>());  // lane 7 - c of each 8
    halve(integral_constant<int, 1>(), integral_constant<int, 0x4E>());   // c ^ 2
    return v[0] + from_lane<0xB1>(v[0]);                                  // c ^ 1
#else
    return acc[0];
#endif
}

// Weights of 128 keys from a part of the rows: each wave has 32 keys in registers, and all four share blocks of 32 rows of queries
// that arrive by LDS DMA, in a ring.  A lane adds its row's weights to its 16 keys' sums, in registers; the 32 lanes meet at the
// end.  What changes from block to block is scalar: a block's first token and head, and offsets into Q and the statistics.
// As above 51 us for the prompt and 34 for the long caches; 64 keys a wave (two workgroups on a CU) took 80.  With 256 dims its
// registers allow three workgroups on a CU.  LOOP: a workgroup takes several (key tile, part)s; the loop's own registers cost 8 to
// 10 % of the times above, so calls of few workgroups go without.
template <class T, int HD, bool LOOP>
__global__ __launch_bounds__(256, HD == 256 ? 3 : 4) void k_weights_keys(const T* __restrict__ Q, const T* __restrict__ Kp, WeightArgs a) {
    typedef typename Vec8<T>::type T8;
    typedef Ring<HD> Rg;
    constexpr int NS = HD / 16, NB = Rg::NB, IW = Rg::IW;
    RING(Q)
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int c = lane & 31, g = lane >> 5;
    const int kh = blockIdx.x % a.HK;
    for (int unit = blockIdx.x / a.HK; unit < a.units; unit += gridDim.x / a.HK) {
        if (LOOP && unit >= (int)gridDim.x / a.HK) lds_barrier();  // (the last one's blocks are done with)
        const Tile tl = key_tile(a, unit);
        if (tl.b < 0 || tl.x >= a.units) return;  // (as above)
        const Req rq = request(a.cu, a.kv_lens, tl.b, a.rows, a.max_new, a.kcap);
        const Seen ob = observed(rq, a.observers);
        const int parts = parts_of(a, ob.n), p0 = rq.p0 + ob.t0;
        const bool sole = parts == 1;  // this workgroup's sums are the keys' weights
        const int z = sole ? 0 : tl.i % parts, tile = sole ? tl.i : tl.i / parts, j0 = tile * KEY_TILE;
        const int slot = sole ? 0 : slot_of(a, rq, tl.b) + z;
        int t0, t1;  // the part's tokens that see some of the keys
        tokens_of(a, rq, ob, j0, t0, t1);
        t0 = max(t0, z * a.part), t1 = min(t1, sole ? ob.n : (z + 1) * a.part);
        if (!sole && (t1 <= t0 || slot >= a.slots)) {  // (slots: row starts that do not ascend)
            if (LOOP) continue;
            return;
        }
        const int nr = max(0, t1 - t0) * a.G, nb = (nr + 31) >> 5;  // rows, and blocks of them
        const int jw = j0 + 32 * wv, lbpp = a.lps - 5, blk = jw >> 5;
        const int page = a.table[(size_t)tl.b * a.max_blocks + min(blk >> lbpp, a.max_blocks - 1)];
        const bool there = jw < rq.kcap && (unsigned)page < (unsigned)a.n_pages;
        f32x16 acc;
#pragma unroll
        for (int e = 0; e < 16; e++) acc[e] = 0.f;
        if (nb > 0) {
            u32x4 kf[NS];
            {
                const size_t at = there ? (size_t)page * a.pstride + ((size_t)(kh << lbpp) + (blk & ((1 << lbpp) - 1))) * (HD * 32) : 0;
                const Rsrc rk = make_rsrc(Kp + at, there ? HD * 64u : 0u);
#pragma unroll
                for (int x = 0; x < NS; x++) kf[x] = buf_b128(rk, c * 64 + (2 * (x & 1) + g) * 16, (x >> 1) * 2048);
            }
            // row 32 i + x of the part is token t + (g0 + x) / G, head (g0 + x) % G, counted from its first token: t tf, g0 gf
            const uint32_t row = (uint32_t)a.HQ * HD * 2;  // bytes (a part's are fewer than 2^31)
            const size_t q0 = (size_t)rq.q0 + ob.t0 + t0, left = (a.rows - q0) * row - (size_t)kh * a.G * HD * 2;
            const Rsrc rs = make_rsrc(Q + (q0 * a.HQ + (size_t)kh * a.G) * HD, (uint32_t)min(left, (size_t)0x7FFFFFFF));
            const Rsrc rst = make_rsrc(a.stat + stat_at(a, rq, ob, kh) + (size_t)t0 * a.G, (uint32_t)nr * 8);
            int gf = 0;         // of the block that is fetched next
            uint32_t qoff = 0;  // its token's rows, in Q
            const uint32_t piece = (((lane & 3) ^ ((lane >> 4) & 3)) << 4);
            uint32_t off0, off1;  // of the lane's rows of the two halves of a block, or of the wave's one
            auto token_of = [&](int x) INL { return a.G == 1 ? (uint32_t)x : __umulhi((uint32_t)x, a.magic); };
            auto offset = [&](int x) INL {
                const uint32_t t = token_of(x);
                return t * row + (x - t * a.G) * (HD * 2) + piece;
            };
            auto offsets = [&]() INL {
                off0 = offset(gf + (IW == 1 ? 16 * (wv & 1) : 0) + (lane >> 2));
                if (IW > 1) off1 = offset(gf + 16 + (lane >> 2));
            };
            offsets();
            auto fetch = [&](int, uint8_t* buf) INL {  // the next block (rows past the last are other rows, or zeros past Q's end: no matter)
                if (a.dg) offsets();
#pragma unroll
                for (int u = 0; u < IW; u++) {
                    const int x = wv * IW + u;  // half x % 2 of dims 32 (x / 2) ..
                    buf_lds16(rs, (u & 1 ? off1 : off0) + qoff, (x >> 1) * 64, buf + x * 1024);  // (a row in range is there whole)
                }
                qoff += a.dt * row, gf += a.dg;
                if (gf >= a.G) gf -= a.G, qoff += row;
                qoff = min(qoff, 0x7FFFFFFFu - 0xFFFFu);  // (blocks past the last)
            };
            auto stat = [&](int i) INL { return __builtin_bit_cast(float2, buf_b64(rst, c * 8 + i * 256, 0)); };  // (0 past the last row)
            float2 st = stat(0);
            int tb = t0, gb = 0;  // the first row's of the block that is worked on
            RING_START(Q, fetch)
            auto turn = [&](int i, const uint8_t* buf, uint8_t* bufx) INL {
                wait_loads<vmcnt_imm((NB - 2) * IW)>();
                lds_barrier();
                const float2 now = st;
                st = stat(i + 1);
                fetch(i + NB - 1, bufx);
                f32x16 s;
#pragma unroll
                for (int e = 0; e < 16; e++) s[e] = 0.f;
#pragma unroll
                for (int x = 0; x < NS; x++)
                    s = Num<T>::mfma32(__builtin_bit_cast(T8, kf[x]), __builtin_bit_cast(T8, Rg::read(buf, x, c, g)), s);
                // every row sees every key: the first token's causally, the last one's through the window
                const bool open = there && jw + 32 <= rq.kcap && 32 * i + 32 <= nr && p0 + tb >= jw + 31 &&
                                  (!a.window || p0 + tb + a.dt + 1 - jw < a.window);
                if (__builtin_expect(open, 1)) {
#pragma unroll
                    for (int e = 0; e < 16; e++) acc[e] = __builtin_fmaf(exp2_fast((s[e] - now.x) * a.c), now.y, acc[e]);
                } else {
                    const int p = max(p0 + tb + (int)token_of(gb + c), -1), j = jw + 4 * g;
                    const Within keep(max(a.from(p), 0) - j, there && 32 * i + c < nr ? p - j : -1);
#pragma unroll
                    for (int e = 0; e < 16; e++) {
                        const float w = exp2_fast((s[e] - now.x) * a.c) * now.y;
                        acc[e] += keep.has(key_of(e)) ? w : 0.f;
                    }
                }
                tb += a.dt, gb += a.dg;
                if (gb >= a.G) gb -= a.G, tb++;
            };
            RING_LOOP(Q, nb)
            wait_loads<vmcnt_imm(0)>();  // (no DMA outlives the workgroup whose LDS it writes)
        }
        const float w = sum_rows(acc);
        const int x = key_of(c >> 1) + 4 * g, j = jw + x;
        if (!(c & 1)) {
            if (!sole) a.col[(((size_t)tile * a.slots + slot) * a.HK + kh) * KEY_TILE + 32 * wv + x] = w;
            else if (there && j < rq.kcap) put_weight(a, rq, mark_at(page, a.HK, kh, j, a.lps), j, w);
        }
        if (!LOOP) return;
    }
}

// Adds up the parts of 128 keys, in their order: every fourth by a group of 128 threads, then the groups' sums.  (64 parts of
// 4096 keys, 2 heads: 5.3 us; by one group 6.5)
constexpr int SUM_G = 4;
template <bool LOOP>
__global__ __launch_bounds__(SUM_G * KEY_TILE) void k_weights_sum(WeightArgs a, int units) {
    __shared__ float part[SUM_G][KEY_TILE];
    const int kh = blockIdx.x % a.HK, i = threadIdx.x % KEY_TILE, grp = threadIdx.x / KEY_TILE;
    for (int unit = blockIdx.x / a.HK; unit < units; unit += gridDim.x / a.HK) {
        const Tile tl = tile_of(a, KEY_TILES, unit, [&](int b) { return split_key_tiles(a, b); });
        if (tl.b < 0) return;
        const Req rq = request(a.cu, a.kv_lens, tl.b, a.rows, a.max_new, a.kcap);
        const Seen ob = observed(rq, a.observers);
        const int parts = parts_of(a, ob.n), j0 = tl.i * KEY_TILE, j = j0 + i, slot = slot_of(a, rq, tl.b);
        if (slot + parts > a.slots) {  // (row starts that do not ascend)
            if (LOOP) continue;
            return;
        }
        const int page = a.table[(size_t)tl.b * a.max_blocks + min(j >> a.lps, a.max_blocks - 1)];
        int t0, t1;
        tokens_of(a, rq, ob, j0, t0, t1);
        float w = 0.f;
        const float* const col = a.col + (((size_t)tl.i * a.slots + slot) * a.HK + kh) * KEY_TILE + i;
        if (t1 > t0) {
#pragma unroll 8
            for (int z = t0 / a.part + grp; z <= (t1 - 1) / a.part; z += SUM_G) w += col[(size_t)z * a.HK * KEY_TILE];
        }
        part[grp][i] = w;
        __syncthreads();
        if (!grp && j < rq.kcap && (unsigned)page < (unsigned)a.n_pages) {
#pragma unroll
            for (int g = 1; g < SUM_G; g++) w += part[g][i];
            put_weight(a, rq, mark_at(page, a.HK, kh, j, a.lps), j, w);
        }
        if (!LOOP) return;
        __syncthreads();
    }
}

// ---- the rows that go -----------------------------------------------------------------------------------------------
//
// Of a (request, kv head)'s n rows the m of the highest ranks stay: a rank is 32 bits, its order the scores', protected
// rows above all.  The m-th is found by digits of 11, 11 and 10 bits from the highest down: a histogram in LDS of the rows
// whose digits above match, and a scan of its counts.  Rows above that rank stay, and of those that have it the first.
// Up to 32768 rows one workgroup does it all, with every row's rank in registers, read once.  512 heads of 4113 rows under a
// bound of 8192, 17 MB without positions: 8.5 us in a row of calls (8.7 with them), 11 to 12 by itself; a chain of 16 barriers, two
// workgroups to a CU.

// A score's place in the order, ascending: NaN, and a row in a hole, before all numbers; -0 is 0.
__device__ __forceinline__ uint32_t rank_of(float s) {
    if (s != s) return 0;
    const uint32_t u = __builtin_bit_cast(uint32_t, s + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int EVICT_T = 1024, BINS = 2048;
constexpr int EVICT_ONE = 32768;  // rows up to which one workgroup does a head

// The sum over the threads before this one, and over all; `ws` holds EVICT_T / 64 sums.
__device__ __forceinline__ int scan(int x, int* ws, int& total) {
    const int wv = threadIdx.x >> 6, v = lanes_upto(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) ws[wv] = v;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < EVICT_T / 64; w++) {
        const int y = ws[w];
        before += w < wv ? y : 0, all += y;
    }
    total = all;
    return before + v - x;
}

struct EvictArgs {
    const float* scores;
    const int *kpos, *table, *kv_lens, *budgets;
    int max_blocks, B, max_kv, HK, lps, n_pages, sink, recent, W;
    int *new_lens, *moves, *counts;
    // heads of more than EVICT_ONE rows: their chunks
    int chunks, groups;  // at most; workgroups of a head
    int* newest;  // [B][HK][groups]
    int* hist;    // [B][HK][3][BINS]
    int* cuts;    // [B][HK][2][4]: the first two digits' cuts, as found by the launch after theirs
    int* parts;   // [B][HK][chunks][4]: rows of the m-th rank and above it, below m and from m on
};

// One head's part in a launch.  over: rows go.
struct Head {
    int b, h, n, m;
    bool over;
    const int* tb;
    size_t bh;
};
__device__ __forceinline__ Head head_of(const EvictArgs& a, int h, int b) {
    Head x;
    x.b = b, x.h = h;
    x.tb = a.table + (size_t)b * a.max_blocks;
    x.bh = (size_t)b * a.HK + h;
    return x;
}
__device__ __forceinline__ void lengths(const EvictArgs& a, Head& x) {
    x.n = a.kv_lens[x.b];
    const int budget = a.budgets[x.b];
    x.over = x.n <= a.max_kv && budget >= 0 && x.n > budget;
    x.m = x.over ? budget : x.n;
}


// 4 rows from j on (a multiple of 4: they lie on end), as loaded.  Their page comes first, whatever the request's length:
// the two loads of the lengths and of the table are then on their way together.
struct Four {
    f32x4u s;
    i32x4 p;
    bool there;
};
__device__ __forceinline__ int page_of(const EvictArgs& a, const Head& x, int j) { return x.tb[min(j >> a.lps, a.max_blocks - 1)]; }
__device__ __forceinline__ Four load4(const EvictArgs& a, const Head& x, int j, int page) {
    Four r;
    r.there = j < x.n && (unsigned)page < (unsigned)a.n_pages;
    const size_t at = mark_at(r.there ? page : 0, a.HK, x.h, r.there ? j : 0, a.lps);
    r.s = *reinterpret_cast<const f32x4u*>(a.scores + at);
    if (a.kpos) r.p = *reinterpret_cast<const i32x4*>(a.kpos + at);
    else r.p = i32x4{j, j + 1, j + 2, j + 3};
    return r;
}
__device__ __forceinline__ int newest_of(const Four& v, const Head& x, int j) {
    int most = INT_MIN;
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (v.there && j + e < x.n) most = max(most, v.p[e]);
    return most;
}
__device__ __forceinline__ uint32_t rank4(const EvictArgs& a, const Four& v, int e, long long keep_from) {
    if (!v.there) return 0;
    return v.p[e] < a.sink || v.p[e] > keep_from ? 0xFFFFFFFFu : min(rank_of(v.s[e]), 0xFFFFFFFEu);
}

__device__ __forceinline__ int max_all(int x, int* ws) {  // over the workgroup
    auto take = [&](auto ctrl, auto rows) {
        x = max(x, __builtin_amdgcn_update_dpp(x, x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false));
    };
    using std::integral_constant;
    take(integral_constant<int, 0x111>(), integral_constant<int, 0xF>());  // as in lanes_upto
    take(integral_constant<int, 0x112>(), integral_constant<int, 0xF>());
    take(integral_constant<int, 0x114>(), integral_constant<int, 0xF>());
    take(integral_constant<int, 0x118>(), integral_constant<int, 0xF>());
    take(integral_constant<int, 0x142>(), integral_constant<int, 0xA>());
    take(integral_constant<int, 0x143>(), integral_constant<int, 0xC>());
    if ((threadIdx.x & 63) == 63) ws[threadIdx.x >> 6] = x;
    __syncthreads();
    int r = ws[0];
#pragma unroll
    for (int w = 1; w < EVICT_T / 64; w++) r = max(r, ws[w]);
    return r;
}

// A histogram in LDS: COPIES counters side by side for each digit, a thread's by its number, since many rows have one digit (all
// of them where scores are equal), and adds to one address go one by one.  (us with 1, 2, 4 and 8 of them: 512 heads of 4113
// rows 9.0 9.1 9.0 9.9 where scores differ, 31.3 21.6 17.3 17.6 where they are equal; of 8000 rows 17.1 16.6 16.9 17.3 and
// 52.9 32.9 23.6 21.5)
constexpr int COPIES = 4;
__device__ __forceinline__ void clear_bins(int* hist) {
#pragma unroll
    for (int i = 0; i < COPIES * BINS / (4 * EVICT_T); i++) reinterpret_cast<i32x4*>(hist)[i * EVICT_T + threadIdx.x] = i32x4{0, 0, 0, 0};
}
__device__ __forceinline__ void count_digit(int* hist, int d) { atomicAdd(&hist[d * COPIES + (threadIdx.x & (COPIES - 1))], 1); }

// Digit t of a rank, and the bits above it.
constexpr int SHIFT[3] = {21, 10, 0};
__device__ __forceinline__ int digit(uint32_t r, int shift) { return r >> shift & (shift ? BINS - 1 : 1023); }

// Of a histogram's rows the `left` of the largest digits stay: the digit of the last of them, `left` less those above it,
// and how many have it.  Two bins a thread; all threads get the answer, behind a barrier since the histogram and since
// ws were used.  (left 0: the largest digit, of which none stays)
struct Cut {
    int digit, left, count;
};
template <int R>  // copies of the histogram
__device__ __forceinline__ Cut cut_at(const int* hist, int left, int* ws, int* found) {
    const int tid = threadIdx.x, d1 = BINS - 1 - 2 * tid, d0 = d1 - 1;  // (from the largest digit down)
    int c1 = 0, c0 = 0;
#pragma unroll
    for (int i = 0; i < R; i++) c1 += hist[d1 * R + i], c0 += hist[d0 * R + i];
    // (a scan as above, its first barrier done: the histogram's)
    const int wv = tid >> 6, to = lanes_upto(c1 + c0);
    if ((tid & 63) == 63) ws[wv] = to;
    __syncthreads();
    int before = to - c1 - c0;
#pragma unroll
    for (int w = 0; w < EVICT_T / 64; w++) before += w < wv ? ws[w] : 0;
    if (left == 0 ? tid == 0 : before < left && left <= before + c1 + c0) {
        const bool first = left == 0 || left <= before + c1;
        found[0] = first ? d1 : d0;
        found[1] = left - before - (first ? 0 : c1);
        found[2] = first ? c1 : c0;
    }
    __syncthreads();
    return {found[0], found[1], found[2]};
}

// One workgroup per (request, kv head), N times 4 rows a thread.  Where a digit leaves up to CANDIDATES rows, each of them
// counts those before it, and the m-th is found at once.
constexpr int CANDIDATES = 512;
template <int N>
__global__ __launch_bounds__(EVICT_T, N <= 2 ? 8 : 4) void k_page_evict(EvictArgs a) {  // (two to a CU, where registers allow)
    constexpr int WV = EVICT_T / 64;
    __shared__ __align__(16) int hist[COPIES * BINS];
    __shared__ int ws[WV], found[3], at_last;
    __shared__ uint32_t sums[N * WV], rank_last;
    __shared__ __align__(16) unsigned long long cand[CANDIDATES];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    Head x = head_of(a, blockIdx.x, blockIdx.y);
    int page[N];
#pragma unroll
    for (int i = 0; i < N; i++) page[i] = page_of(a, x, (i * EVICT_T + tid) * 4);
    lengths(a, x);
    if (x.h == 0 && tid == 0) a.new_lens[x.b] = x.m;
    if (!x.over) {
        if (tid == 0) a.counts[x.bh] = 0;
        return;
    }
    uint32_t rank[4 * N];
    {
        Four v[N];
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = load4(a, x, (i * EVICT_T + tid) * 4, page[i]);
        clear_bins(hist);
        int most = INT_MIN;
#pragma unroll
        for (int i = 0; i < N; i++) most = max(most, newest_of(v[i], x, (i * EVICT_T + tid) * 4));
        const long long keep_from = (long long)max_all(most, ws) - a.recent;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) rank[4 * i + e] = rank4(a, v[i], e, keep_from);
    }
    auto at = [&](int k) { return ((k >> 2) * EVICT_T + tid) * 4 + (k & 3); };  // the row of rank[k]
    auto any = [&](int i) { return (i * EVICT_T + 64 * wv) * 4 < x.n; };        // the wave has some of rank[4 i ..]
    // Rows above `prefix` stay, and those up to `last` that have it.
    uint32_t prefix = 0;
    int left = x.m, count = 0, last = INT_MAX;
    bool done = false;
#pragma unroll
    for (int t = 0; t < 3; t++) {
        const int shift = SHIFT[t], above = t ? SHIFT[t - 1] : 0;
        if (done) break;
        if (t) {
            __syncthreads();
            clear_bins(hist);
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (!any(i)) break;
#pragma unroll
            for (int k = 4 * i; k < 4 * i + 4; k++)
                if (at(k) < x.n && (t == 0 || rank[k] >> above == prefix >> above)) count_digit(hist, digit(rank[k], shift));
        }
        if (tid == 0) at_last = 0;
        __syncthreads();
        const Cut c = cut_at<COPIES>(hist, left, ws, found);
        prefix |= (uint32_t)c.digit << shift;
        left = c.left, count = c.count;
        if (left == count) {  // all of them (none where m is 0: nothing has the last digit of all)
            done = true;
            if (left == 0) last = -1;
        } else if (left && count <= CANDIDATES) {
            done = true;
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (!any(i)) break;
#pragma unroll
                for (int k = 4 * i; k < 4 * i + 4; k++)
                    if (at(k) < x.n && rank[k] >> shift == prefix >> shift)
                        cand[atomicAdd(&at_last, 1)] = (unsigned long long)rank[k] << 32 | ~(uint32_t)at(k);
            }
            __syncthreads();
            if (tid < count) {
                const unsigned long long own = cand[tid];
                int before = 0;
#pragma unroll 8
                for (int i = 0; i < count; i++) before += cand[i] > own;
                if (before == left - 1) rank_last = (uint32_t)(own >> 32), found[0] = (int)~(uint32_t)own;
            }
            __syncthreads();
            prefix = rank_last, last = found[0];
        }
    }
    if (!done) {  // the first `left` of the rows that have the m-th rank
        __syncthreads();
        if (tid == 0) found[0] = -1;
        int before = 0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            int ties = 0, total;
#pragma unroll
            for (int e = 0; e < 4; e++) ties += at(4 * i + e) < x.n && rank[4 * i + e] == prefix;
            int nth = before + scan(ties, ws, total);
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (at(4 * i + e) < x.n && rank[4 * i + e] == prefix && ++nth == left) found[0] = at(4 * i + e);
            before += total;
        }
        __syncthreads();
        last = found[0];
    }
    auto stays = [&](int k) { return rank[k] > prefix || (rank[k] == prefix && at(k) <= last); };
    uint32_t own[N];  // holes of the thread's 4 rows, and rows times 2^16; first numbered in their wave
#pragma unroll
    for (int i = 0; i < N; i++) {
        uint32_t c = 0;
        if (any(i)) {
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int k = 4 * i + e, j = at(k);
                const bool s = stays(k);
                c += j < x.m ? !s : s && j < x.n ? 0x10000u : 0u;
            }
        }
        const uint32_t to = lanes_upto(c);
        own[i] = to - c;
        if (lane == 63) sums[i * WV + wv] = to;
    }
    __syncthreads();
    if (wv == 0) {  // (at most 32768 of each: 2^16 holds both)
        uint32_t carry = 0;
        for (int i = 0; i < N * WV; i += 64) {
            const uint32_t y = i + lane < N * WV ? sums[i + lane] : 0, to = lanes_upto(y);
            if (i + lane < N * WV) sums[i + lane] = carry + to - y;
            carry += __builtin_amdgcn_readlane(to, 63);
        }
        if (lane == 0) a.counts[x.bh] = carry >> 16;
    }
    __syncthreads();
    int* const mv = a.moves + x.bh * a.W * 2;
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (!any(i)) break;
        uint32_t no = sums[i * WV + wv] + own[i];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const int k = 4 * i + e, j = at(k);
            const bool s = stays(k);
            if (j < x.m && !s) mv[2 * (no & 0xFFFF)] = j, no += 1;
            if (j >= x.m && s && j < x.n) mv[2 * (no >> 16) + 1] = j, no += 0x10000u;
        }
    }
}

// ---- heads of more rows: the same in chunks, a launch for each step that needs all of them ----
//
// 4 heads of 90 to 131 thousand rows: 3.2, 4.1, 4.9, 4.6, 5.7 and 7.0 us, launches of 128 workgroups that are latency
// alone (lengths, pages, rows, histogram in series); the bytes of one pass would take 1.

// (rows of a chunk: 4 CN a thread, CN 1 where few heads leave CUs idle.  us with 1 and 2: 4 heads of 131 thousand rows of which 33
// thousand stay 30.5 33, 64 heads of 40 thousand 57 52, 512 heads of 40 thousand 204 199)
template <int CN>
constexpr int chunk_rows() { return EVICT_T * 4 * CN; }

template <int CN>
__device__ __forceinline__ void chunk_pages(const EvictArgs& a, const Head& x, int c, int (&page)[CN]) {
#pragma unroll
    for (int i = 0; i < CN; i++) page[i] = page_of(a, x, c * chunk_rows<CN>() + (i * EVICT_T + threadIdx.x) * 4);
}

// A head has gridDim.x workgroups, each of which takes every gridDim.x-th chunk: where the lengths lie far below max_kv, few
// find none.  each(chunk, its pages) for those that there are; the first one's pages are on their way with the lengths.
template <int CN, class F>
__device__ __forceinline__ void chunks_of(const EvictArgs& a, const Head& x, int (&page)[CN], F&& each) {
    const int last = (x.n - 1) / chunk_rows<CN>();
    for (int c = blockIdx.x;;) {
        each(c);
        if (last - c < (int)gridDim.x) break;
        c += gridDim.x;
        chunk_pages(a, x, c, page);
    }
}
template <int CN>
__device__ __forceinline__ bool has_chunk(const Head& x) { return x.over && blockIdx.x <= (x.n - 1) / chunk_rows<CN>(); }

// The latest position that each workgroup finds, and the histograms cleared.
template <int CN>
__global__ __launch_bounds__(EVICT_T) void k_evict_newest(EvictArgs a) {
    __shared__ int ws[EVICT_T / 64];
    const int tid = threadIdx.x;
    Head x = head_of(a, blockIdx.y, blockIdx.z);
    int page[CN];
    chunk_pages(a, x, blockIdx.x, page);
    lengths(a, x);
    if (blockIdx.x == 0 && tid == 0) {
        if (x.h == 0) a.new_lens[x.b] = x.m;
        if (!x.over) a.counts[x.bh] = 0;
    }
    if (!x.over) return;
    for (int i = blockIdx.x * EVICT_T + tid; i < 3 * BINS; i += gridDim.x * EVICT_T) a.hist[x.bh * 3 * BINS + i] = 0;
    int most = INT_MIN;
    if (has_chunk<CN>(x))
        chunks_of<CN>(a, x, page, [&](int c) INL {
#pragma unroll
            for (int i = 0; i < CN; i++) {
                const int j = c * chunk_rows<CN>() + (i * EVICT_T + tid) * 4;
                most = max(most, newest_of(load4(a, x, j, page[i]), x, j));
            }
        });
    most = max_all(most, ws);
    if (tid == 0) a.newest[x.bh * a.groups + blockIdx.x] = most;
}

// A chunk's rows, as loaded, and their ranks; row 4 i + e of a thread is row e of the 4 that it loads i-th.
template <int CN>
struct Chunk {
    Four v[CN];
    uint32_t rank[4 * CN];
    __device__ __forceinline__ void load(const EvictArgs& a, const Head& x, int c, const int (&page)[CN]) {
#pragma unroll
        for (int i = 0; i < CN; i++) v[i] = load4(a, x, c * chunk_rows<CN>() + (i * EVICT_T + threadIdx.x) * 4, page[i]);
    }
    __device__ __forceinline__ void ranks(const EvictArgs& a, long long keep_from) {
#pragma unroll
        for (int i = 0; i < CN; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) rank[4 * i + e] = rank4(a, v[i], e, keep_from);
    }
};
template <int CN>
__device__ __forceinline__ int chunk_row(int c, int k) { return c * chunk_rows<CN>() + ((k >> 2) * EVICT_T + threadIdx.x) * 4 + (k & 3); }

__device__ __forceinline__ long long keep_from_of(const EvictArgs& a, const Head& x, int* ws) {
    int most = INT_MIN;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += EVICT_T) most = max(most, a.newest[x.bh * a.groups + i]);
    return (long long)max_all(most, ws) - a.recent;
}
// The digits of the m-th rank that the first T histograms give, and how many of those that have them stay.
struct Prefix {
    uint32_t rank;
    int left;
};
template <int T>
__device__ __forceinline__ Prefix prefix_of(const EvictArgs& a, const Head& x, int* ws, int* found) {
    Prefix p{0, x.m};
    // (the cut before the last is in memory since the last launch)
#pragma unroll
    for (int t = 0; t < T; t++) {
        Cut cut;
        int* const kept = a.cuts + (x.bh * 2 + t) * 4;
        if (t + 1 < T) {
            cut = {kept[0], kept[1], kept[2]};
        } else {
            __syncthreads();
            cut = cut_at<1>(a.hist + (x.bh * 3 + t) * BINS, p.left, ws, found);
            if (t < 2 && blockIdx.x == 0 && threadIdx.x == 0) kept[0] = cut.digit, kept[1] = cut.left, kept[2] = cut.count;
        }
        p.rank |= (uint32_t)cut.digit << SHIFT[t];
        p.left = cut.left;
    }
    return p;
}

// The histogram of digit T, of all chunks.  (Whole numbers: their sum has no order.)
template <int T, int CN>
__global__ __launch_bounds__(EVICT_T) void k_evict_digit(EvictArgs a) {
    __shared__ __align__(16) int hist[COPIES * BINS];
    __shared__ int ws[EVICT_T / 64], found[3];
    const int tid = threadIdx.x;
    Head x = head_of(a, blockIdx.y, blockIdx.z);
    int page[CN];
    chunk_pages(a, x, blockIdx.x, page);
    lengths(a, x);
    if (!has_chunk<CN>(x)) return;
    Chunk<CN> k;
    k.load(a, x, blockIdx.x, page);  // (on their way meanwhile)
    clear_bins(hist);
    const long long keep_from = keep_from_of(a, x, ws);
    const Prefix p = prefix_of<T>(a, x, ws, found);
    __syncthreads();
    chunks_of<CN>(a, x, page, [&](int c) INL {
        if (c != (int)blockIdx.x) k.load(a, x, c, page);
        k.ranks(a, keep_from);
#pragma unroll
        for (int i = 0; i < 4 * CN; i++)
            if (chunk_row<CN>(c, i) < x.n && (T == 0 || k.rank[i] >> SHIFT[T ? T - 1 : 0] == p.rank >> SHIFT[T ? T - 1 : 0]))
                count_digit(hist, digit(k.rank[i], SHIFT[T]));
    });
    __syncthreads();
    for (int i = tid; i < BINS; i += EVICT_T) {
        const i32x4 n = reinterpret_cast<const i32x4*>(hist)[i];
        const int sum = (n[0] + n[1]) + (n[2] + n[3]);
        if (sum) atomicAdd(&a.hist[(x.bh * 3 + T) * BINS + i], sum);
    }
}

// How many rows of each chunk have the m-th rank, and how many are above it, on either side of m.
template <int CN>
__global__ __launch_bounds__(EVICT_T) void k_evict_count(EvictArgs a) {
    __shared__ int ws[EVICT_T / 64], found[3], n[4];
    const int tid = threadIdx.x;
    Head x = head_of(a, blockIdx.y, blockIdx.z);
    int page[CN];
    chunk_pages(a, x, blockIdx.x, page);
    lengths(a, x);
    if (!has_chunk<CN>(x)) return;
    Chunk<CN> k;
    k.load(a, x, blockIdx.x, page);
    const long long keep_from = keep_from_of(a, x, ws);
    const Prefix p = prefix_of<3>(a, x, ws, found);
    chunks_of<CN>(a, x, page, [&](int c) INL {
        if (c != (int)blockIdx.x) k.load(a, x, c, page);
        k.ranks(a, keep_from);
        uint32_t below = 0, from = 0;  // ties, and rows above times 2^16
#pragma unroll
        for (int i = 0; i < 4 * CN; i++) {
            const int j = chunk_row<CN>(c, i);
            const uint32_t w = j >= x.n ? 0u : k.rank[i] == p.rank ? 1u : k.rank[i] > p.rank ? 0x10000u : 0u;
            if (j < x.m) below += w;
            else from += w;
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) below += __shfl_xor(below, o), from += __shfl_xor(from, o);
        __syncthreads();  // (the last chunk's are written)
        if (tid < 4) n[tid] = 0;
        __syncthreads();
        if ((tid & 63) == 0) {
            atomicAdd(&n[0], (int)(below & 0xFFFF));
            atomicAdd(&n[1], (int)(below >> 16));
            atomicAdd(&n[2], (int)(from & 0xFFFF));
            atomicAdd(&n[3], (int)(from >> 16));
        }
        __syncthreads();
        if (tid < 4) a.parts[(x.bh * a.chunks + c) * 4 + tid] = n[tid];
    });
}

// Each chunk's moves, numbered behind those of the chunks before it.
template <int CN>
__global__ __launch_bounds__(EVICT_T) void k_evict_moves(EvictArgs a) {
    __shared__ int ws[EVICT_T / 64], found[3];
    __shared__ int before[3];  // ties, holes and rows of the chunks before
    const int tid = threadIdx.x;
    Head x = head_of(a, blockIdx.y, blockIdx.z);
    int page[CN];
    chunk_pages(a, x, blockIdx.x, page);
    lengths(a, x);
    if (!has_chunk<CN>(x)) return;
    Chunk<CN> k;
    k.load(a, x, blockIdx.x, page);
    const long long keep_from = keep_from_of(a, x, ws);
    const Prefix p = prefix_of<3>(a, x, ws, found);
    int* const mv = a.moves + x.bh * a.W * 2;
    int upto = 0, ties0 = 0, holes0 = 0, rows0 = 0;  // (in the first wave: those of the chunks before chunk `upto`)
    chunks_of<CN>(a, x, page, [&](int c) INL {
        if (c != (int)blockIdx.x) k.load(a, x, c, page);
        k.ranks(a, keep_from);
        if (tid < 64) {  // 64 chunks at a time: their ties from the first on stay until `left` are used up
            for (; upto < c; upto = min(c, upto + 64)) {
                const int i = upto + tid;
                i32x4 n = {0, 0, 0, 0};
                if (i < c) n = *reinterpret_cast<const i32x4*>(a.parts + (x.bh * a.chunks + i) * 4);
                const int to = lanes_upto(n[0] + n[2]);
                const int first = ties0 + to - n[0] - n[2];
                const int kept0 = min(max(p.left - first, 0), n[0]), kept1 = min(max(p.left - first - n[0], 0), n[2]);
                int h = i < c ? max(0, min(chunk_rows<CN>(), x.m - i * chunk_rows<CN>())) - n[1] - kept0 : 0, r = n[3] + kept1;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) h += __shfl_xor(h, o), r += __shfl_xor(r, o);
                holes0 += h, rows0 += r;
                ties0 += __shfl(to, 63);
            }
            if (tid == 0) before[0] = ties0, before[1] = holes0, before[2] = rows0;
        }
        __syncthreads();
        int ties = before[0], holes = before[1], rows = before[2];
#pragma unroll
        for (int i = 0; i < CN; i++) {
            int t = 0, total;
#pragma unroll
            for (int e = 0; e < 4; e++) t += chunk_row<CN>(c, 4 * i + e) < x.n && k.rank[4 * i + e] == p.rank;
            int nth = ties + scan(t, ws, total);
            ties += total;
            bool hole[4], row[4];
            int mine = 0;  // holes, and rows times 2^16
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int j = chunk_row<CN>(c, 4 * i + e);
                const uint32_t r = k.rank[4 * i + e];
                const bool stays = j < x.n && (r > p.rank || (r == p.rank && nth < p.left));
                nth += j < x.n && r == p.rank;
                hole[e] = j < x.m && !stays, row[e] = j >= x.m && stays;
                mine += hole[e] + (row[e] ? 0x10000 : 0);
            }
            const int no = scan(mine, ws, total);
            int h = holes + (no & 0xFFFF), r = rows + (no >> 16);
            holes += total & 0xFFFF, rows += total >> 16;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                if (hole[e]) mv[2 * h++] = chunk_row<CN>(c, 4 * i + e);
                if (row[e]) mv[2 * r++ + 1] = chunk_row<CN>(c, 4 * i + e);
            }
        }
        if (tid == 0 && c == (x.n - 1) / chunk_rows<CN>()) a.counts[x.bh] = rows;
    });
}

// ---- their pages ----------------------------------------------------------------------------------------------------

constexpr int RELEASE_T = 1024;

__device__ __forceinline__ long long scan(long long x, long long* ws, long long& total) {  // as above
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    long long v = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long long y = __shfl_up(v, o);
        if (lane >= o) v += y;
    }
    __syncthreads();
    if (lane == 63) ws[wv] = v;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < RELEASE_T / 64; w++) before += w < wv ? ws[w] : 0, all += ws[w];
    total = all;
    return before + v - x;
}

// One workgroup: the requests' pages that go numbered through by a scan over the requests, then pushed in that order, a
// round of 1024 entries at a time, those out of range left out.  64 requests, a page each: 4.3 us; 2 that drop 500 to 770 pages
// 5.1: lengths, a scan, table and stack in series.
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
//
// Sources lie behind all places that are written, so moves run in any order.  Bound by memory: K's rows are pieces of 64
// bytes, but a row of V is one element of each of HD runs of 32 rows.  Moves ascend on both sides, so many of them on end touch
// few blocks: lane l takes move l % N of N, and a wave's load of a dim, or its store, falls into one or two runs.  Where a
// head has few moves, each a block of its own, smaller N spread them over more workgroups.
//
// 15 rows of each of 512 heads of 128 dims: 18 us, 13 of them V's stores: 983 thousand single elements, each in 64 bytes of its
// own, which memory takes as masked writes of 32 bytes.  96 thousand rows of 256 dims: 107 us; 268 MB read and 125 written for
// the 196 that move, 3.7 TB/s; without V 44, without its stores 77, without its loads 74.
constexpr int MOVES = 32;  // that a workgroup does at a time, at most

template <int HD, int N>
__device__ __forceinline__ void move_rows(const int* mv, int n, const int* tb, size_t h, int HK, int lps, int max_blocks, int n_pages,
                                          size_t pstride, uint16_t* Kp, uint16_t* Vp, float* scores, int* kpos,
                                          size_t (&off)[2][MOVES], int (&row)[2][MOVES]) {
    const int tid = threadIdx.x, l = tid % N;
    const long long rows = (long long)max_blocks << lps;
    // Groups of N moves: an XCD (every eighth workgroup) takes adjacent ones, which share blocks in its L2.
    const int groups = (n + N - 1) / N, X = min((int)gridDim.x, 8), per = (groups + X - 1) / X, x0 = blockIdx.x % X * per;
    const int wgs = (gridDim.x - blockIdx.x % X + X - 1) / X;  // of this XCD
    for (int y = blockIdx.x / X; y < per && x0 + y < groups; y += wgs) {
        const int i0 = (x0 + y) * N;
        __syncthreads();
        if (tid < 2 * N) {  // (in the first wave: lane l has move l's place, lane N + l its row)
            const int side = tid / N, j = i0 + l < n ? mv[2 * (i0 + l) + side] : -1;
            const bool in = j >= 0 && j < rows;
            const int page = in ? tb[j >> lps] : -1;
            const bool there = (unsigned)page < (unsigned)n_pages;
            const int other = __shfl_xor((int)there, N);  // (all lanes: not behind a branch)
            const bool both = there && other;
            off[side][l] = (size_t)(there ? page : 0) * pstride + ((h << (lps - 5)) + ((j & ((1 << lps) - 1)) >> 5)) * (HD * 32);
            row[side][l] = both ? j & 31 : -1;
            const size_t at = mark_at(there ? page : 0, HK, (int)h, j, lps);
            const size_t to = __shfl(at, l);
            if (side && both) {
                if (scores) scores[to] = scores[at];
                if (kpos) kpos[to] = kpos[at];
            }
        }
        __syncthreads();
        constexpr int P = HD / 8, KN = (N * P + 255) / 256;  // 16-byte pieces of a row of K; those of a thread
        u32x4 k[KN];
#pragma unroll
        for (int x = 0; x < KN; x++) {
            const int i = (tid + 256 * x) / P, p = (tid + 256 * x) % P;
            if (i < N && row[1][i] >= 0) k[x] = *reinterpret_cast<const u32x4*>(Kp + off[1][i] + (p >> 2) * 1024 + row[1][i] * 32 + (p & 3) * 8);
        }
        constexpr int STEP = 256 / N, VN = (HD + STEP - 1) / STEP;  // dims side by side; dims of a thread
        uint16_t v[VN];
        const bool mine = row[0][l] >= 0 && tid / N < HD;
        const uint16_t* const from = Vp + off[1][l] + row[1][l] + tid / N * 32;
        uint16_t* const to = Vp + off[0][l] + row[0][l] + tid / N * 32;
        if (mine) {
#pragma unroll
            for (int x = 0; x < VN; x++) v[x] = from[x * STEP * 32];
        }
#pragma unroll
        for (int x = 0; x < KN; x++) {
            const int i = (tid + 256 * x) / P, p = (tid + 256 * x) % P;
            if (i < N && row[0][i] >= 0) *reinterpret_cast<u32x4*>(Kp + off[0][i] + (p >> 2) * 1024 + row[0][i] * 32 + (p & 3) * 8) = k[x];
        }
        if (mine) {
#pragma unroll
            for (int x = 0; x < VN; x++) to[x * STEP * 32] = v[x];
        }
    }
}

template <int HD>
__global__ __launch_bounds__(256) void k_paged_move(const int* __restrict__ moves, const int* __restrict__ counts,
                                                    const int* __restrict__ table, int max_blocks, int W, int HK, int lps,
                                                    int n_pages, size_t pstride, uint16_t* Kp, uint16_t* Vp, float* scores,
                                                    int* kpos) {
    __shared__ size_t off[2][MOVES];  // of a move's place and row: their blocks, in a cache
    __shared__ int row[2][MOVES];     // and the rows there; -1: no move
    const int h = blockIdx.y, b = blockIdx.z;
    const size_t bh = (size_t)b * HK + h;
    const int n = min(counts[bh], W), each = n / (int)gridDim.x;
    const int* const mv = moves + bh * W * 2;
    const int* const tb = table + (size_t)b * max_blocks;
    auto run = [&](auto c) INL {
        move_rows<HD, decltype(c)::value>(mv, n, tb, h, HK, lps, max_blocks, n_pages, pstride, Kp, Vp, scores, kpos, off, row);
    };
    if (each >= 12) run(std::integral_constant<int, 32>());
    else if (each >= 4) run(std::integral_constant<int, 8>());
    else run(std::integral_constant<int, 4>());
}

// Requests up to which each workgroup finds its tile by itself; from there on a launch before makes an index.  (us without and with
// it, 20 new rows on 300 keys each, 8 and 2 heads of 128 dims: 128 requests 25 27.6, 192 34.2 34.9, 256 42.7 41.5, 1024
// 134 94, 8192 4020 768; 16 on 2000 keys, 32 and 8 heads: 128 requests 247 236, 256 522 477, 1024 2415 1790)
constexpr int INDEX_B = 128;

// Workgroups of a pass over keys from which on 8192 take several (key tile, part)s each, so that bounds far above the lengths cost
// little.  (us so, and with a workgroup for each, 8 heads of 128 dims: 64 requests of 20 new rows on 300 keys under 32768 45 104;
// 200, one of them 600 rows on 20000 keys, under 131072 486 897; 256, one of 3841 rows 2468 2890; where nearly all have work, 100
// requests of 20 rows on 16000 keys, 1650 1615)
constexpr int LOOP_FROM = 131072, LOOP_WGS = 8192;

// How a call runs, from its sizes alone (the lengths themselves are on the device).
struct WeightPlan {
    int nr = 0, few = 0, few_ks = 1, few_span = 1, kvp = 0;  // nr: 16-row groups of k_weights_few, 0: not launched
    int tiles = 0, ks = 1, span = 1, part = 1, parts = 1, units = 0, slots = 0;  // tiles 0: no many rows
    bool once = false, one = false, ordered = false;  // keys read past the last-level cache; k_weights_few_one, by length
    size_t ml = 0, stat = 0, col = 0, index = 0;  // floats and ints of the workspace
    size_t S = 0, few_ml = 0;                     // and of each request whose few rows' splits run in one launch
    size_t least() const { return (ml + stat + col + index + S + few_ml) * 4; }  // bytes for one such request, and for B of them
    size_t whole(int B) const { return (ml + stat + col + index + B * (S + few_ml)) * 4; }
    int few_at_once(int B, size_t bytes) const {
        return S ? (int)std::min<size_t>(B, (bytes / 4 - ml - stat - col - index) / (S + few_ml)) : B;
    }
};

WeightPlan plan_weights(const PagedShape& s, int B, int rows, int max_new, int max_kv, int observers) {
    const int G = s.HQ / s.HK;
    const int tokens = std::min({max_new, rows, observers ? observers : INT_MAX});
    const long long most = (long long)tokens * G;
    WeightPlan p;
    const int nb = (int)(((long long)max_kv + 31) / 32);
    if (most <= 32) p.few = (int)most;
    else if (G <= 32 && rows < (long long)max_new * B) p.few = G;
    if (p.few) {
        p.nr = p.few <= 16 ? 1 : 2;
        p.kvp = (int)std::min<long long>((long long)nb * 32, INT_MAX);
        // One workgroup per head where there are enough of them, or few bytes of keys for each: one launch, and no scores in memory.
        // us in splits and so, at n keys of each request:
        // 2 heads, 256 dims: 300 8.5 7.6, 700 8.1 10.3; 8 heads, 128 dims: 700 8.1 7.4, 1200 8.2 9.2, 2000 8.1 11.8
        // 128 heads, 256 dims: 700 16.4 12.4, 2000 27.8 23.4, 1000 to 8100 58 79; 128 dims: 2000 18.9 13.9, 1000 to 8100 31.2 33.4
        // 256 heads: 128 dims, 1000 to 8100 60 52; 256 dims 101 98
        // 512 heads, 128 dims: 1200 32.7 27.9, 3800 105 83, 8100 220 183, 1000 to 8100 113 78; 64 dims: 1200 21.8 16.3, 8100 118 92
        const size_t each = (size_t)nb * s.HD * 64;
        p.one = (long long)nb * 32 <= ONE_KEYS && (size_t)p.few * p.kvp * 4 <= ONE_LDS &&
                (B * s.HK >= 256 || each <= (size_t(B * s.HK >= 128 ? 1024 : 256) << 10));
        // By length, the longest first, where not all run at once and a head's keys outweigh every workgroup's look at all lengths
        // (which nothing hides where a CU has one workgroup).  us without and with it, lengths between the two (in logarithms):
        // 8 heads, 128 dims: 64 requests of 100 to 1200 keys 15.9 15.5, of 1000 to 8100 96 79; 128 of 100 to 2000 38.0 36.2, of 500 to
        // 8100 150 134; 200 of 100 to 2000 52.9 56.1, to 4000 92 88; 500 of 100 to 1000 76 125
        // 64 dims: 128 of 100 to 2000 20.8 23.1, of 500 to 4000 46.9 43.5.  256 dims: 64 of 50 to 300 14.0 14.7, of 1000 to 8100 183
        // 148, 100 of 100 to 1000 40 40, 200 of 100 to 2000 103 118
        p.ordered = p.one && B <= ONE_ORDER && B * s.HK > 256 && each >= (size_t)B * (s.HD * p.nr > 128 ? 8192 : 4096);
        p.once = (size_t)B * nb * s.HK * s.HD * 64 > (size_t(256) << 20);
        if (!p.one) {
            const int want = std::max(1, std::min(256, 8192 / (B * s.HK)));
            p.few_span = std::max(FEW_W, (nb + want - 1) / want);
            p.few_ks = (nb + p.few_span - 1) / p.few_span;
            p.S = (size_t)s.HK * p.few * p.kvp;
            p.few_ml = (size_t)s.HK * p.few_ks * p.few * 2;
        }
    }
    if (most > p.few) {
        const long long all = std::min((long long)rows, (long long)B * tokens) * G;  // rows that are counted
        const long long reqs = std::min((long long)B, all / (p.few + 1));
        p.tiles = (int)(all / ROW_TILE + reqs);
        const int want = (int)std::min(128ll, std::max(1ll, 2048 / (std::max(1ll, all / ROW_TILE) * s.HK)));
        p.span = std::max(8, (nb + want - 1) / want);
        p.ks = (nb + p.span - 1) / p.span;
        const int nkb = (int)(((long long)max_kv + KEY_TILE - 1) / KEY_TILE);
        // parts of at least 256 rows, so many that there are 4096 workgroups; of at most 16384 (a lane then adds up 512 weights on
        // end), and of fewer than 2^30 bytes of Q
        const long long wanted = std::max(1ll, 4096ll / ((long long)nkb * s.HK));
        p.part = (int)((std::min(16384ll, std::max(256ll, (all + wanted - 1) / wanted)) + G - 1) / G);
        p.part = (int)std::min<long long>(p.part, std::max(1ll, (1ll << 29) / ((long long)s.HQ * s.HD)));
        p.parts = (tokens + p.part - 1) / p.part;
        const long long units = (long long)nkb * std::min(reqs * p.parts, all / G / p.part + reqs);
        if (units >= 1 << 24 || (long long)(p.tiles | 1) * s.HK * (p.ks > 1 ? std::max(p.ks, 32) : 1) >= 1 << 24)
            throw Error("sd_op_paged_weights: too many rows and keys for one launch");
        p.units = (int)units;
        p.slots = p.parts == 1 ? 0 : (int)std::min((long long)B * p.parts, B == 1 ? p.parts : 2ll * rows / p.part);
        p.ml = p.ks > 1 ? (size_t)p.ks * p.tiles * s.HK * ROW_TILE * 2 : 0;
        p.stat = (size_t)rows * s.HQ * 2;
        p.col = (size_t)p.slots * nkb * s.HK * KEY_TILE;
        p.index = B > INDEX_B ? 3 * ((size_t)B + 1) : 0;
    }
    for (size_t* x : {&p.ml, &p.stat, &p.col, &p.index, &p.S, &p.few_ml}) *x = (*x + 3) & ~size_t(3);
    return p;
}

template <class T, int HD>
void weights_as(const PagedShape& s, const PagedWeights& a, hipStream_t st) {
    const WeightPlan p = plan_weights(s, a.B, a.rows, a.max_new, a.max_kv, a.observers);
    const int G = s.HQ / s.HK;
    float* const ws = static_cast<float*>(a.ws);
    WeightArgs g{a.table, a.cu, a.kv_lens, a.pos, a.max_blocks, a.B, a.rows, s.HQ, s.HK, G, log2i(s.PS), s.n_pages, a.max_new,
                 a.max_kv, a.window, a.observers, p.few, p.few_ks, p.few_span, p.few, p.kvp, 0, p.tiles, p.ks, p.span, p.part,
                 p.parts, p.units, p.slots, p.ordered, 32 / G, 32 % G, (uint32_t)((1ull << 32) / G + 1), a.scale * LOG2E, a.decay, s.pstride, a.scores, a.out, a.kpos};
    g.ml = reinterpret_cast<float2*>(ws);
    g.stat = reinterpret_cast<float2*>(ws + p.ml);
    g.col = ws + p.ml + p.stat;
    g.index = p.index ? reinterpret_cast<int*>(g.col + p.col) : nullptr;
    const int at_once = p.few_at_once(a.B, a.ws_bytes);
    g.S = g.col + p.col + p.index;
    g.few_ml = reinterpret_cast<float2*>(g.S + at_once * p.S);
    const T *Q = static_cast<const T*>(a.Q), *K = static_cast<const T*>(a.Kp);
    auto launch = [&](auto kernel, dim3 grid, int threads, auto... args) {
        hipLaunchKernelGGL(kernel, grid, dim3(threads), 0, st, args...);
        launched("paged_weights");
    };
    if (p.tiles) {
        const int looping = std::max(1, LOOP_WGS / s.HK);  // workgroups of a head
        const bool loop = (long long)p.units * s.HK >= LOOP_FROM;
        const dim3 rows((p.tiles | 1) * s.HK * p.ks), keys((loop ? looping : p.units) * s.HK);
        if (p.index) launch(k_weights_index, dim3(1), INDEX_T, g);
        launch(k_weights_rows<T, HD>, rows, 256, Q, K, g);
        if (p.ks > 16) launch(k_weights_join<64>, dim3(p.tiles * s.HK * (ROW_TILE / 4)), 256, g);
        else if (p.ks > 1) launch(k_weights_join<8>, dim3(p.tiles * s.HK * (ROW_TILE / 32)), 256, g);
        if (loop) launch(k_weights_keys<T, HD, true>, keys, 256, Q, K, g);
        else launch(k_weights_keys<T, HD, false>, keys, 256, Q, K, g);
        if (p.parts > 1) {
            const long long nkb = ((long long)a.max_kv + KEY_TILE - 1) / KEY_TILE;
            const int tiles = (int)std::min<long long>(std::min(a.B, p.slots) * nkb, p.units);
            if (tiles > 2 * looping) launch(k_weights_sum<true>, dim3(2 * looping * s.HK), SUM_G * KEY_TILE, g, tiles);
            else launch(k_weights_sum<false>, dim3(tiles * s.HK), SUM_G * KEY_TILE, g, tiles);
        }
    }
    if (p.nr) {
        auto few = [&](auto nr, auto once) {
            constexpr int NR = decltype(nr)::value;
            constexpr bool ONCE = decltype(once)::value;
            if (p.one) {
                hipLaunchKernelGGL((k_weights_few_one<T, HD, NR, ONCE>), dim3(s.HK, a.B), dim3(64 * ONE_W), p.few * p.kvp * 4, st, Q, K, g);
                launched("paged_weights");
                return;
            }
            const long long chunks = ((long long)a.max_kv + 1023) / 1024;  // of 1024 keys; at most so many workgroups that each has some
            for (g.first = 0; g.first < a.B; g.first += at_once) {  // (so many requests in turn as the workspace holds scores for)
                const int n = std::min(at_once, a.B - g.first);
                launch(k_weights_few<T, HD, NR, ONCE>, dim3(s.HK * p.few_ks, n), 64 * FEW_W, Q, K, g);
                launch(k_weights_few_sum, dim3((unsigned)std::min(chunks, std::max(1ll, 16384ll / (s.HK * n))) * s.HK, n), 256, g);
            }
        };
        auto once = [&](auto nr) {
            if (p.once) few(nr, std::true_type());
            else few(nr, std::false_type());
        };
        if (p.nr == 1) once(std::integral_constant<int, 1>());
        else once(std::integral_constant<int, 2>());
    }
}

}  // namespace

WeightsWs paged_weights_ws(const PagedShape& s, int B, int rows, int max_new, int max_kv, int observers) {
    const WeightPlan p = plan_weights(s, B, rows, max_new, max_kv, observers);
    return {p.whole(B), p.least()};
}

void paged_weights(const PagedShape& s, const PagedWeights& a, hipStream_t st) {
    by_type(s, [&](auto t, auto hd) { weights_as<decltype(t), decltype(hd)::value>(s, a, st); });
}

namespace {
struct EvictWs {
    int cn = 0, groups = 0;
    size_t chunks = 0, newest = 0, hist = 0, cuts = 0, parts = 0;  // ints
};
EvictWs evict_ws(int B, int max_kv, int HK) {
    EvictWs w;
    if (max_kv <= EVICT_ONE) return w;
    const size_t heads = (size_t)B * HK;
    w.cn = heads <= 16 ? 1 : 2;
    const size_t rows = w.cn == 1 ? chunk_rows<1>() : chunk_rows<2>();
    w.chunks = ((size_t)max_kv + rows - 1) / rows;
    // (us with 512, 1024 and 2048 workgroups in all: 512 heads of 4113 rows under a bound of 131072 44 86 154, and a workgroup for
    // each chunk of the bound 438; of 40000 rows 199 223 306; 64 heads of 100000 98 116 -)
    w.groups = (int)std::min(w.chunks, std::max(size_t(1), 512 / heads));
    w.newest = (heads * w.groups + 3) & ~size_t(3);
    w.hist = heads * 3 * BINS;
    w.cuts = heads * 8;
    w.parts = heads * w.chunks * 4;
    return w;
}
}  // namespace

size_t page_evict_ws(int B, int max_kv, int HK) {
    const EvictWs w = evict_ws(B, max_kv, HK);
    return (w.newest + w.hist + w.cuts + w.parts) * 4;
}

void page_evict(const PageEvict& a, hipStream_t st) {
    const EvictWs w = evict_ws(a.B, a.max_kv, a.HK);
    EvictArgs g{a.scores, a.kpos, a.table, a.kv_lens, a.budgets, a.max_blocks, a.B, a.max_kv, a.HK, log2i(a.PS), a.n_pages,
                a.sink, a.recent, std::max(a.max_kv / 2, 1), a.new_lens, a.moves, a.counts, (int)w.chunks, w.groups};
    auto launch = [&](auto kernel, dim3 grid) {
        hipLaunchKernelGGL(kernel, grid, dim3(EVICT_T), 0, st, g);
        launched("page_evict");
    };
    if (!w.chunks) {
        const dim3 grid(a.HK, a.B);
        if (a.max_kv <= 4096) launch(k_page_evict<1>, grid);
        else if (a.max_kv <= 8192) launch(k_page_evict<2>, grid);
        else if (a.max_kv <= 16384) launch(k_page_evict<4>, grid);
        else launch(k_page_evict<8>, grid);
        return;
    }
    g.newest = static_cast<int*>(a.ws);
    g.hist = g.newest + w.newest;
    g.cuts = g.hist + w.hist;
    g.parts = g.cuts + w.cuts;
    const dim3 grid((unsigned)w.groups, a.HK, a.B);
    auto all = [&](auto cn) {
        constexpr int CN = decltype(cn)::value;
        launch(k_evict_newest<CN>, grid);
        launch(k_evict_digit<0, CN>, grid);
        launch(k_evict_digit<1, CN>, grid);
        launch(k_evict_digit<2, CN>, grid);
        launch(k_evict_count<CN>, grid);
        launch(k_evict_moves<CN>, grid);
    };
    if (w.cn == 1) all(std::integral_constant<int, 1>());
    else all(std::integral_constant<int, 2>());
}

void page_release(const PageRelease& a, hipStream_t st) {
    hipLaunchKernelGGL(k_page_release, dim3(1), dim3(RELEASE_T), 0, st, a.kv_lens, a.new_lens, a.dropped, a.table, a.max_blocks,
                       a.B, log2i(a.PS), a.n_pages, a.free_pages, a.n_free, a.dropped_out, a.n_free_out);
    launched("page_release");
}

void paged_move(const PagedShape& s, const PagedMove& a, hipStream_t st) {
    const int W = std::max(a.max_kv / 2, 1);
    auto launch = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3(std::min((W + 3) / 4, std::max(1, 2048 / (s.HK * a.B))), s.HK, a.B), dim3(256), 0, st, a.moves,
                           a.counts, a.table, a.max_blocks, W, s.HK, log2i(s.PS), s.n_pages, s.pstride,
                           static_cast<uint16_t*>(a.Kp), static_cast<uint16_t*>(a.Vp), a.scores, a.kpos);
    };
    if (s.HD == 64) launch(k_paged_move<64>);
    else if (s.HD == 128) launch(k_paged_move<128>);
    else launch(k_paged_move<256>);
    launched("paged_move");
}

}  // namespace sd
