// Log-probabilities of given tokens, the distribution's entropy and its top alternatives, in
// one pass over the logits (exl3b200_token_logprobs).
//
//   lse = M + log sum_i exp(x_i - M)     logprob(t) = (x_t - M) - log S
//   H   = lse - sum_i p_i x_i            = log S - T / S   with y_i = x_i - M,
//                                          S = sum exp(y_i), T = sum y_i exp(y_i)
//
// the sums in base 2.  M is subtracted before anything is rounded - x log2(e) less a reference
// is one fused multiply-add, as is the reference less M log2(e) by which the sums are rescaled
// to M itself - so that logits with a large common offset lose no accuracy (rounding M log2(e)
// on one side alone cost 9e-5 at logits around 3000).  A row of 16-bit or fp32 logits is cut into
// units of 256 vectors of 8 elements and is one CTA's, or - when rows are few - a cluster's
// of up to 8 CTAs, whose first joins the pieces through distributed shared memory in a fixed
// order.
//
// Alternatives: each thread keeps the maximum of the vectors it saw and the vector that held
// it, and the second largest vector maximum.  The k-th largest of the threads' maxima is a
// lower bound of the k-th largest element; only the vectors of the k threads above it hold
// candidates, and of those only the ones that the second maximum says so need to be read
// again.  Elements are ordered by (value, lower index first) as unique 64-bit keys, so that
// equal logits come in the order of their ids.
//
// Bound by HBM where rows are many: 2048 x 128256 bf16 (525 MB) take 92 us, 5.7 TB/s, in a
// burst (a long run of calls settles at 102 to 106, 5 TB/s); what is left is the exponential
// (16 a clock and SM, 60 us of it here) beside nearly seven other instructions an element.
// Whole rows to a CTA beat equal runs of units over all rows joined by a second kernel (107
// us; 500 x 151936 fp32: 57 instead of 77 us): a row's finish costs more than an uneven last
// wave.  Few rows are a chain of latencies: 1 x 128256 9 us, 80 x 151936 fp32 with 20
// alternatives 18 us (48.6 MB).
#include <algorithm>
#include <climits>

#include <cooperative_groups.h>

#include "exl3_common.cuh"
#include "exl3_capi_internal.h"
#include "exl3_grouped_dev.cuh"

namespace exl3b200 {

namespace cg = cooperative_groups;

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpVec = 8;                       // elements of a thread's vector
constexpr int kLpUnit = kLpThreads * kLpVec;    // elements of a unit
constexpr int kLpCluster = 8;                   // most CTAs of a row
// CTAs of a launch with clusters: 4 fit on an SM, but clusters do not pack a GPC's slots
// fully. 568 are resident as clusters of 8, 546 as 7, 558 to 568 as 3 to 6, 592 as pairs; 480
// fit at every size, with rounding down to whole clusters counted.  80 rows of 151936 fp32 as
// clusters of 7 (560 CTAs) took two waves: 27.5 us instead of 18.0 as 6; 80 of 128256 bf16
// 20.3 instead of 14.2.  (Limits of 400 and 560 for 50 to 240 rows: up to 6 us slower at 400,
// up to 3 faster at 560 where its clusters fit.)
constexpr int kLpClusterCtas = 480;
constexpr int kLpMaxTop = EXL3B200_LOGPROBS_MAX_TOP;
constexpr int kLpBuffer = 1024;                 // candidates kept before they are cut back to the best 32
constexpr float kLpLog2e = 1.4426950408889634f;
constexpr float kLpLn2 = 0.6931471805599453f;
// The running reference of the exponents is raised only when an element exceeds it by 2^8:
// sums of 2^31 terms below 2^8 stay far inside fp32.  T's terms y e are rounded at up to 8 times
// their weight before the rescale to M takes that back (raised at 2^16 the entropies of 2048 x
// 128256 were off by 3.5e-7 of their size, 5.5 times what the plain fp32 form is, now by 1.0e-7;
// 92 us either way, at 2^2 93).
constexpr float kLpSlack = 8.f;

typedef unsigned long long u64;

struct LogprobArgs {
    const void* logits;
    const long long* tokens;
    float* logprob;
    float* entropy;
    float* top_logprob;   // [rows][top]
    long long* top_ids;   // [rows][top]
    long long row_stride;
    int rows, vocab, top, row_units;
    int row_ctas;         // CTAs of a row: a cluster
};

__device__ __forceinline__ float lp_ex2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
// a lower bound of -200 on an exponent that lets a NaN through
__device__ __forceinline__ float lp_bound(float y)
{
    float r;
    asm("max.NaN.f32 %0, %1, 0fC3480000;" : "=f"(r) : "f"(y));
    return r;
}
// two fp32 operations in one instruction
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 lp_pair(float a, float b)
{
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void lp_unpair(f32x2 v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ f32x2 lp_fma2(f32x2 a, f32x2 b, f32x2 c)
{
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 lp_add2(f32x2 a, f32x2 b)
{
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// max of packed 16-bit pairs; the NaN form lets a NaN through
template <typename T> __device__ __forceinline__ uint32_t lp_max2(uint32_t a, uint32_t b)
{
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("max.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    else asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
template <typename T> __device__ __forceinline__ uint32_t lp_low2(uint32_t a)
{
    uint32_t r;
    if constexpr (std::is_same<T, __half>::value) asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0xFBFFFBFFu));
    else asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0xF149F149u));
    return r;
}
__device__ __forceinline__ float lp_low(float x)
{
    float r;
    asm("max.NaN.f32 %0, %1, 0fF149F2CA;" : "=f"(r) : "f"(x));  // -1e30
    return r;
}
// A thread's first reference (base 2): so far above what -inf is lifted to that a lifted
// element's exponent gives 0 (fp16: -65504 log2 e = -94502.3, 502 below), and below every
// logit that counts - where a row's maximum is itself that far down lp_far holds.
template <typename T> __device__ __forceinline__ constexpr float lp_start() { return std::is_same<T, __half>::value ? -9.4e4f : -1e30f; }
template <typename T> __device__ __forceinline__ float2 lp_float2(uint32_t w)
{
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
// order of the values as unsigned integers (0 is below every value; -0 counts as 0)
__device__ __forceinline__ unsigned lp_order(float x)
{
    const unsigned u = __float_as_uint(x + 0.f);
    return u ^ ((unsigned) ((int) u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float lp_value(unsigned o)
{
    return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ u64 lp_key(float x, int idx) { return (u64) lp_order(x) << 32 | (unsigned) ~idx; }
__device__ __forceinline__ u64 lp_swap(u64 v, int j, bool larger)
{
    const u64 o = __shfl_xor_sync(~0u, v, j);
    return (v > o) == larger ? v : o;
}
// a warp's 32 keys in descending order
__device__ __forceinline__ u64 lp_sort(u64 v, int lane)
{
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j; j >>= 1) v = lp_swap(v, j, ((lane & j) == 0) == ((lane & k) == 0));
    return v;
}
// the 32 largest of two descending lists, descending
__device__ __forceinline__ u64 lp_merge(u64 a, u64 b, int lane)
{
    const u64 r = __shfl_sync(~0u, b, 31 - lane);
    u64 v = a > r ? a : r;
#pragma unroll
    for (int j = 16; j; j >>= 1) v = lp_swap(v, j, (lane & j) == 0);
    return v;
}
// the 32 largest of every warp's list (descending), in warp 0
__device__ __forceinline__ u64 lp_merge_warps(u64 v, u64 (*lists)[32], int warp, int lane)
{
#pragma unroll
    for (int n = kLpWarps / 2; n; n >>= 1) {
        if (warp >= n && warp < 2 * n) lists[warp][lane] = v;
        __syncthreads();
        if (warp < n) v = lp_merge(v, lists[warp + n][lane], lane);
    }
    return v;
}

// a vector's eight elements in fp32; elements outside the row are -inf
template <typename T> __device__ __forceinline__ float lp_float(T x) { return (float) x; }
template <> __device__ __forceinline__ float lp_float<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float lp_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> struct LpVec {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p)
    {
#pragma unroll
        for (int i = 0; i < (int) sizeof(T) / 2; ++i)
            asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w)
                         : "l"(reinterpret_cast<const uint4*>(p) + i));
    }
    __device__ __forceinline__ void get(float (&f)[8]) const
    {
#pragma unroll
        for (int i = 0; i < (int) sizeof(T) / 2; ++i) {
            const uint32_t u[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (sizeof(T) == 4) f[4 * i + j] = __uint_as_float(u[j]);
                else if constexpr (std::is_same<T, __nv_bfloat16>::value) {
                    f[2 * j] = __uint_as_float(u[j] << 16);
                    f[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
                } else {
                    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
                    f[2 * j] = t.x, f[2 * j + 1] = t.y;
                }
            }
        }
    }
};

// A row as vectors that begin on 16-byte boundaries: vector 0 begins `shift` elements before
// the row, the last one may end behind it; both are read element by element.
template <typename T> struct LpRow {
    const T* p;      // the row's first element, less shift
    int shift, end;  // element e of the row is p[e + shift], e + shift < end
    __device__ __forceinline__ LpRow(const LogprobArgs& a, int row)
    {
        const T* r = reinterpret_cast<const T*>(a.logits) + (long long) row * a.row_stride;
        shift = (int) (((uintptr_t) r & 15) / sizeof(T));
        p = r - shift;
        end = shift + a.vocab;
    }
    __device__ __forceinline__ bool inside(int v) const { return v * kLpVec >= shift && (v + 1) * kLpVec <= end; }
    __device__ __forceinline__ void edge(int v, float (&f)[8]) const
    {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = v * kLpVec + i;
            f[i] = e >= shift && e < end ? lp_float<T>(p[e]) : -INFINITY;
        }
    }
    __device__ __forceinline__ void read(int v, float (&f)[8]) const
    {
        if (inside(v)) {
            LpVec<T> x;
            x.load(p + v * kLpVec);
            x.get(f);
        } else {
            edge(v, f);
        }
    }
    __device__ __forceinline__ int vectors() const { return (end + kLpVec - 1) / kLpVec; }
};

// A row's finite maximum for which the sums are taken again from (x - M): its product with
// log2 e might overflow, or it is near the bound to which the main loop lifts -inf (so that
// y e is 0 and not NaN): -1e30, in fp16 the lowest value.
template <typename T> __device__ __forceinline__ bool lp_far(float M)
{
    return (fabsf(M) > 1e29f && fabsf(M) < INFINITY) || (std::is_same<T, __half>::value && M < -3e4f && M > -INFINITY);
}

// A row's results from its maximum M, S and T (relative to M) and warp 0's descending keys.
template <typename T>
__device__ __forceinline__ void lp_write(const LogprobArgs& a, int row, float M, float S, float Tt, u64 key, int tid)
{
    const float ls = log2f(S);
    auto of = [&](float x) { return fmaf(-ls, kLpLn2, x - M); };
    if (tid == 0) {
        const long long t = a.tokens[row];
        float lp = -INFINITY;  // an id outside the vocabulary has no probability
        if (t >= 0 && t < a.vocab) {
            const float x = lp_float<T>(reinterpret_cast<const T*>(a.logits)[(long long) row * a.row_stride + t]);
            lp = of(x);
        }
        a.logprob[row] = lp;
        a.entropy[row] = (ls - Tt / S) * kLpLn2;
    }
    if (tid < a.top) {
        a.top_logprob[(long long) row * a.top + tid] = of(lp_value((unsigned) (key >> 32)));
        a.top_ids[(long long) row * a.top + tid] = (long long) (unsigned) ~(unsigned) key;
    }
}

// A row of several pieces: part(p) is {M, S, T} of piece p, keys(p) its descending keys.
template <typename T, typename Part, typename Keys>
__device__ __forceinline__ void lp_join(const LogprobArgs& a, int row, int pieces, Part part, Keys keys, u64 (*lists)[32])
{
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    float M = -INFINITY, S = 0.f, Tt = 0.f;
    if (warp == 0) {
        for (int p = lane; p < pieces; p += 32) M = fmaxf(M, part(p).x);
#pragma unroll
        for (int i = 16; i; i >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, i));
        for (int p = lane; p < pieces; p += 32) {
            const float4 q = part(p);
            const float d = (q.x - M) * kLpLog2e, k = lp_ex2(d);
            S += q.y * k;
            Tt += k == 0.f ? 0.f : (q.z + d * q.y) * k;
        }
#pragma unroll
        for (int i = 16; i; i >>= 1) {
            S += __shfl_xor_sync(~0u, S, i);
            Tt += __shfl_xor_sync(~0u, Tt, i);
        }
    }
    u64 key = 0;
    if (a.top > 0) {
        const int n = pieces * a.top;
        for (int b = warp * 32; b < n; b += kLpThreads) {
            const int i = b + lane;
            key = lp_merge(key, lp_sort(i < n ? keys(i / a.top)[i % a.top] : 0, lane), lane);
        }
        key = lp_merge_warps(key, lists, warp, lane);
    }
    if (warp == 0) lp_write<T>(a, row, M, S, Tt, key, tid);
}

template <typename T>
__global__ __launch_bounds__(kLpThreads, 4) void exl3_logprobs_kernel(const __grid_constant__ LogprobArgs a)
{
    __shared__ u64 lists[kLpWarps][32];
    __shared__ u64 buffer[kLpBuffer + kLpThreads * kLpVec];
    __shared__ float red[kLpWarps][3];
    __shared__ u64 sh_bound;
    __shared__ int sh_count, sh_cols, cols[kLpThreads];
    __shared__ int best_vec[kLpThreads];
    __shared__ float4 sh_part;
    __shared__ u64 sh_keys[32];
    griddep_launch();
    griddep_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int row = blockIdx.x / a.row_ctas, part = blockIdx.x - row * a.row_ctas;
    // units of the row: this CTA's piece
    const int c0 = (int) ((long long) part * a.row_units / a.row_ctas), c1 = (int) ((long long) (part + 1) * a.row_units / a.row_ctas);
    const LpRow<T> r(a, row);
    const int nv = r.vectors();
    const int v0 = c0 * kLpThreads + tid, v1 = min(nv, c1 * kLpThreads);  // vectors v0, v0 + 256, ... of this thread
    float best = -INFINITY, second = -INFINITY, ref = lp_start<T>();
    f32x2 s2 = lp_pair(0.f, 0.f), t2 = s2;
    int bv = v0;
    // vectors b .. b + n of the row into L2, one request of one thread
    auto prefetch = [&](int b, int n) {
        const int lo = max(b, r.inside(0) ? 0 : 1), hi = min(b + n, min(v1, r.end / kLpVec));
        if (tid == 0 && hi > lo) {
            const char* p = reinterpret_cast<const char*>(r.p + (long long) lo * kLpVec);
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p), "r"((hi - lo) * kLpVec * (int) sizeof(T)) : "memory");
        }
    };
    auto raise = [&](float cm) {  // before elements of at most cm are added
        const float c2 = cm * kLpLog2e;
        if (c2 > ref + kLpSlack) {
            const float d = ref - c2, k = lp_ex2(d);
            float s0, s1, t0, t1;
            lp_unpair(s2, s0, s1);
            lp_unpair(t2, t0, t1);
            t2 = lp_pair((t0 + d * s0) * k, (t1 + d * s1) * k);
            s2 = lp_pair(s0 * k, s1 * k);
            ref = c2;
        }
    };
    auto rank = [&](float cm, int v) {  // a vector's maximum among this thread's
        second = fmaxf(second, fminf(best, cm));
        bv = cm > best ? v : bv;
        best = fmaxf(best, cm);
    };
    auto add = [&](float x0, float x1) {  // finite or NaN
        const f32x2 y = lp_fma2(lp_pair(x0, x1), lp_pair(kLpLog2e, kLpLog2e), lp_pair(-ref, -ref));
        float y0, y1;
        lp_unpair(y, y0, y1);
        const f32x2 e = lp_pair(lp_ex2(y0), lp_ex2(y1));
        s2 = lp_add2(s2, e);
        t2 = lp_fma2(y, e, t2);
    };
    auto max8 = [](const float (&f)[8]) {
        return fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
    };
    auto largest = [&](const LpVec<T>& x) {
        if constexpr (sizeof(T) == 4) {
            float f[8];
            x.get(f);
            return max8(f);
        } else {
            const uint4 w = x.w[0];
            const float2 m = lp_float2<T>(lp_max2<T>(lp_max2<T>(w.x, w.y), lp_max2<T>(w.z, w.w)));
            return fmaxf(m.x, m.y);
        }
    };
    auto add8 = [&](const LpVec<T>& x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                const uint4 w = x.w[i >> 1];
                add(lp_low(__uint_as_float(i & 1 ? w.z : w.x)), lp_low(__uint_as_float(i & 1 ? w.w : w.y)));
            } else {
                const uint4 w = x.w[0];
                const float2 f = lp_float2<T>(lp_low2<T>(i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w));
                add(f.x, f.y);
            }
        }
    };
    auto take_any = [&](int v) {
        float f[8];
        r.read(v, f);
        const float cm = max8(f);
        raise(cm);
        rank(cm, v);
#pragma unroll
        for (int i = 0; i < 8; i += 2) add(lp_low(f[i]), lp_low(f[i + 1]));
    };
    {
        constexpr int kAhead = sizeof(T) == 4 ? 2 : 4;
        constexpr int kFar = 2;
        prefetch(c0 * kLpThreads, kFar * kAhead * kLpThreads);
        int v = v0;
        if (v < v1 && !r.inside(v)) {
            take_any(v);
            v += kLpThreads;
        }
        for (; v + (kAhead - 1) * kLpThreads < v1 && r.inside(v + (kAhead - 1) * kLpThreads); v += kAhead * kLpThreads) {
            prefetch(v - tid + kFar * kAhead * kLpThreads, kAhead * kLpThreads);
            LpVec<T> x[kAhead];
            float cm[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) x[i].load(r.p + (long long) (v + i * kLpThreads) * kLpVec);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) cm[i] = largest(x[i]);
            float all = cm[0];
#pragma unroll
            for (int i = 1; i < kAhead; ++i) all = fmaxf(all, cm[i]);
            raise(all);
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                rank(cm[i], v + i * kLpThreads);
                add8(x[i]);
            }
        }
        for (; v < v1; v += kLpThreads) take_any(v);
    }
    float s, t;
    {
        float s1, t1;
        lp_unpair(s2, s, s1);
        lp_unpair(t2, t, t1);
        s += s1;
        t += t1;
    }

    // M, S, T of the piece
    float M = best;
#pragma unroll
    for (int i = 16; i; i >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, i));
    if (lane == 0) red[warp][0] = M;
    if (tid == 0) sh_count = sh_cols = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kLpWarps; ++i) M = fmaxf(M, red[i][0]);
    if (lp_far<T>(M)) {  // logits whose product with log2 e leaves fp32's exact range, as a mask of the type's lowest value
        s = t = 0.f;
        for (int v = v0; v < v1; v += kLpThreads) {
            float f[8];
            r.read(v, f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float y = lp_bound((f[i] - M) * kLpLog2e), e = lp_ex2(y);
                s += e;
                t = fmaf(y, e, t);
            }
        }
    } else {
        const float d = fmaf(-M, kLpLog2e, ref), k = s == 0.f ? 0.f : lp_ex2(d);
        t = s == 0.f ? 0.f : (t + d * s) * k;
        s *= k;
    }
    {
#pragma unroll
        for (int i = 16; i; i >>= 1) {
            s += __shfl_xor_sync(~0u, s, i);
            t += __shfl_xor_sync(~0u, t, i);
        }
        if (lane == 0) red[warp][1] = s, red[warp][2] = t;
    }
    u64 key = 0;
    if (a.top > 0) {
        float f[8];
        if (v0 < v1) {
            r.read(bv, f);
#pragma unroll
            for (int i = 7; i >= 0; --i) {
                const int e = bv * kLpVec + i;
                if (f[i] == best && e >= r.shift && e < r.end) key = lp_key(best, e - r.shift);
            }
            if (key == 0) {  // NaN alone: an id of the vocabulary all the same
                const int i = max(r.shift - bv * kLpVec, 0);
                key = lp_key(__uint_as_float(0x7fffffffu), bv * kLpVec + i - r.shift);
            }
        }
        best_vec[tid] = bv;
        const u64 mine = key;
        if (a.top == 1) {  // the largest of the threads' largest
#pragma unroll
            for (int i = 16; i; i >>= 1) {
                const u64 o = __shfl_xor_sync(~0u, key, i);
                key = o > key ? o : key;
            }
            if (lane == 0) lists[0][warp] = key;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kLpWarps; ++i) key = lists[0][i] > key ? lists[0][i] : key;
        } else {
            key = lp_merge_warps(lp_sort(key, lane), lists, warp, lane);
            if (warp == 0 && lane == a.top - 1) sh_bound = key;
            __syncthreads();
            u64 bound = sh_bound;
            auto push = [&](const float (&x)[8], int v) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = v * kLpVec + i;
                    if (e >= r.shift && e < r.end) {
                        const u64 k = lp_key(x[i], e - r.shift);
                        if (k >= bound) buffer[atomicAdd(&sh_count, 1)] = k;
                    }
                }
            };
            // the best vectors of the threads above the bound (at most 32 of them, unless
            // the piece has fewer threads with elements than alternatives)
            if (v0 < v1 && mine >= bound) {
                push(f, bv);
                if (v0 + kLpThreads < v1 && lp_order(second) >= (unsigned) (bound >> 32)) cols[atomicAdd(&sh_cols, 1)] = tid;
            }
            __syncthreads();
            const int units = (v1 - c0 * kLpThreads + kLpThreads - 1) / kLpThreads;  // vectors of a column, at most
            const int again = sh_cols * units;
            for (int i0 = 0;; i0 += kLpThreads) {
                const int n = sh_count;
                __syncthreads();  // every thread has read it
                if (n > kLpBuffer) {  // cut back to the best 32, raise the bound
                    if (warp == 0) {
                        u64 l = 0;
                        for (int b = 0; b < n; b += 32) l = lp_merge(l, lp_sort(b + lane < n ? buffer[b + lane] : 0, lane), lane);
                        buffer[lane] = l;
                        if (lane == a.top - 1) sh_bound = l;
                        if (lane == 0) sh_count = 32;
                    }
                    __syncthreads();
                    bound = sh_bound;
                }
                if (i0 >= again) break;
                if (i0 + tid < again) {
                    const int col = cols[(i0 + tid) / units];
                    const int v = c0 * kLpThreads + col + ((i0 + tid) % units) * kLpThreads;
                    if (v < v1 && v != best_vec[col]) {
                        float x[8];
                        r.read(v, x);
                        push(x, v);
                    }
                }
                __syncthreads();
            }
            if (warp == 0) {
                key = 0;
                const int n = sh_count;
                for (int b = 0; b < n; b += 32) key = lp_merge(key, lp_sort(b + lane < n ? buffer[b + lane] : 0, lane), lane);
            }
        }
    }
    __syncthreads();
    if (warp == 0) {
        float S = 0.f, Tt = 0.f;
#pragma unroll
        for (int i = 0; i < kLpWarps; ++i) S += red[i][1], Tt += red[i][2];
        if (a.row_ctas == 1) {
            lp_write<T>(a, row, M, S, Tt, key, tid);
        } else {
            if (lane == 0) sh_part = make_float4(M, S, Tt, 0.f);
            sh_keys[lane] = key;
        }
    }
    if (a.row_ctas > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        if (cluster.block_rank() == 0)
            lp_join<T>(a, row, a.row_ctas,
                       [&](int p) { return *cluster.map_shared_rank(&sh_part, p); },
                       [&](int p) { return (const u64*) cluster.map_shared_rank(sh_keys, p); }, lists);
        cluster.sync();  // the pieces stay until they are read
    }
}

// (a row that does not begin on a 16-byte boundary reaches over one vector more)
static int lp_row_units(int vocab) { return (int) (((long long) vocab + kLpVec - 1 + kLpUnit - 1) / kLpUnit); }

template <typename T> static int lp_launch(const LogprobArgs& a, cudaStream_t st)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned) (a.rows * a.row_ctas));
    cfg.blockDim = dim3(kLpThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned) a.row_ctas;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.row_ctas > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, exl3_logprobs_kernel<T>, a) == cudaSuccess ? kOk : kErrLaunch;
}

}  // namespace exl3b200

using namespace exl3b200;

extern "C" int exl3b200_token_logprobs(const void* logits, long long row_stride, int rows, int vocab, int dtype,
                                       const long long* tokens, int top, float* logprob, float* entropy,
                                       float* top_logprobs, long long* top_ids, void* stream)
{
    if (!logits || !tokens || !logprob || !entropy || (top > 0 && (!top_logprobs || !top_ids))) return kErrNullPointer;
    if (rows < 1 || vocab < 1 || vocab > (1 << 30) || top < 0 || top > kLpMaxTop || top > vocab || (rows > 1 && row_stride < vocab))
        return kErrBadShape;
    if (dtype != EXL3B200_DTYPE_F16 && dtype != EXL3B200_DTYPE_BF16 && dtype != EXL3B200_DTYPE_F32) return kErrBadArgument;
    if ((uintptr_t) logits % (dtype == EXL3B200_DTYPE_F32 ? 4 : 2)) return kErrUnaligned;
    LogprobArgs a = {};
    a.logits = logits, a.tokens = tokens, a.logprob = logprob, a.entropy = entropy;
    a.top_logprob = top_logprobs, a.top_ids = top_ids;
    a.row_stride = row_stride, a.rows = rows, a.vocab = vocab, a.top = top, a.row_units = lp_row_units(vocab);
    a.row_ctas = std::max(1, std::min({kLpClusterCtas / rows, kLpCluster, a.row_units}));
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (dtype == EXL3B200_DTYPE_F16) return lp_launch<__half>(a, st);
    if (dtype == EXL3B200_DTYPE_BF16) return lp_launch<__nv_bfloat16>(a, st);
    return lp_launch<float>(a, st);
}
