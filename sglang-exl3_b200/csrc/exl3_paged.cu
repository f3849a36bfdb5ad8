// Paged key-value cache: the append of new tokens with the position rotation applied
// on the way (exl3b200_rope_append), and the attention of a few new tokens per sequence
// over its pages (exl3b200_paged_attention).
//
// A cache is [pages][page_size][kv_heads][head_dim] in any stride order whose last
// dimension is contiguous, 16 bit or e4m3 with one fp32 scale per kv head.
#include <atomic>
#include <cfloat>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <utility>

#include <cuda_fp8.h>

#include "exl3_common.cuh"
#include "exl3_capi_internal.h"
#include "exl3_grouped_dev.cuh"

namespace exl3b200 {

constexpr int kSms = 148;

// ---------------------------------------------------------------------------
// append
// ---------------------------------------------------------------------------

enum PagedDtype { kF16 = EXL3B200_DTYPE_F16, kBf16 = EXL3B200_DTYPE_BF16, kF32 = EXL3B200_DTYPE_F32,
                  kE4m3 = EXL3B200_DTYPE_E4M3 };

struct AppendArgs {
    const void* q;
    const void* k;
    const void* v;
    void* q_out;
    unsigned char* k_cache;
    unsigned char* v_cache;
    const long long* positions;
    const long long* slots;
    const float* inv_freq;
    const float* k_scale;
    const float* v_scale;
    int* status;
    long long q_tok, q_head, k_tok, k_head, v_tok, v_head, qo_tok, qo_head;  // elements
    long long c_page, c_pos, c_head;                                        // bytes
    long long num_slots;
    int tokens, q_heads, kv_heads, page_size, rotary;
};

constexpr int kAppThreads = 256;
constexpr int kAppMaxTile = 4;   // tokens of a CTA
constexpr int kAppMaxHalf = 64;  // rotated pairs of a head

template <typename T> struct Vec8;  // eight values of an input row
template <> struct Vec8<__half> {
    uint4 w;
    __device__ __forceinline__ void load(const __half* p)
    {
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(p) : "memory");
    }
    __device__ __forceinline__ void get(float (&f)[8]) const
    {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
            f[2 * i] = t.x, f[2 * i + 1] = t.y;
        }
    }
};
template <> struct Vec8<__nv_bfloat16> {
    uint4 w;
    __device__ __forceinline__ void load(const __nv_bfloat16* p)
    {
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "l"(p) : "memory");
    }
    __device__ __forceinline__ void get(float (&f)[8]) const
    {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(u[i] << 16);
            f[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
        }
    }
};
template <> struct Vec8<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p)
    {
        asm volatile("ld.global.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(a.x), "=f"(a.y), "=f"(a.z), "=f"(a.w) : "l"(p) : "memory");
        asm volatile("ld.global.L1::no_allocate.v4.f32 {%0, %1, %2, %3}, [%4];"
                     : "=f"(b.x), "=f"(b.y), "=f"(b.z), "=f"(b.w) : "l"(p + 4) : "memory");
    }
    __device__ __forceinline__ void get(float (&f)[8]) const
    {
        f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
    }
};

// two fp32 -> one packed pair, one rounding to nearest
__device__ __forceinline__ uint32_t pack2(float a, float b, __half)
{
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T> __device__ __forceinline__ void store8(void* p, const float (&f)[8])
{
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(f[0], f[1], T()), pack2(f[2], f[3], T()),
                                              pack2(f[4], f[5], T()), pack2(f[6], f[7], T()));
}
// e4m3, rounded to nearest even and saturated at 448 (a NaN stays one)
__device__ __forceinline__ void store8_e4m3(void* p, const float (&f)[8], float scale)
{
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_fp8x2_storage_t t = __nv_cvt_float2_to_fp8x2(
            make_float2(__fdiv_rn(f[2 * i], scale), __fdiv_rn(f[2 * i + 1], scale)), __NV_SATFINITE, __NV_E4M3);
        w[i >> 1] |= (uint32_t) t << (16 * (i & 1));
    }
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

// One CTA: a tile of tokens, all their heads.  The tile's cosines and sines are computed
// once into shared memory: the angle p * w_i (a position of up to 2^31 times an fp32
// frequency) is a product of two doubles taken to a fraction of pi before it is rounded
// to fp32, so that a far position turns by as exact an angle as a near one.  A thread
// then takes 16-element units of a head: elements [a, a+8) and [b, b+8), whose pairs
// turn together - half-split pairs (i, i + r/2) sit in the two vectors, adjacent pairs
// inside each.  Units beyond the rotated part, and v, are copied.
// Bound by HBM: 16384 tokens of 64 + 2 x 8 heads of 128 in fp16 (671 MB) take 115 us,
// 5.8 TB/s.  Tiles of four tokens (one: 138 us, two: 122, eight: 118) share the angles and
// the launch; few tokens take one each, to reach every SM (one token: 3.5 us, a launch).
template <typename IN, typename QO, bool E4M3, int D, bool AHEAD>
__global__ __launch_bounds__(kAppThreads, AHEAD ? 4 : 5) void exl3_rope_append_kernel(const __grid_constant__ AppendArgs a, int tile,
                                                                       int interleaved)
{
    constexpr int kUnits = D / 16;                       // units of a head
    constexpr int kHeadsPerPass = kAppThreads / kUnits;  // heads that the CTA takes at once
    __shared__ float2 turn[kAppMaxTile][kAppMaxHalf];    // (cos, sin)
    __shared__ long long at[kAppMaxTile];                // the token's byte offset in the cache, -1: not written
    // No griddep_launch: what follows starts when the cache is written.  The dense decode attention
    // reads rows of earlier steps before its dependency wait, and with an early trigger here it
    // could be resident, behind kernels that trigger early too, while its rows are still being
    // written (a prompt appended through a view of a dense cache).  One token:
    // 3.7 -> 3.8 us, 16384: 115.5 -> 115.8.
    griddep_wait();
    const int t0 = blockIdx.x * tile;
    const int nt = min(tile, a.tokens - t0);
    const int half = a.rotary >> 1;
    for (int i = threadIdx.x; i < nt * half; i += kAppThreads) {
        const int t = i / half, f = i - t * half;
        const double x = (double) a.positions[t0 + t] * (double) a.inv_freq[f] * 0.31830988618379067154;
        float s, c;
        sincospif((float) (x - 2.0 * rint(x * 0.5)), &s, &c);
        turn[t][f] = make_float2(c, s);
    }
    if (threadIdx.x < nt) {
        const long long slot = a.slots[t0 + threadIdx.x];
        long long off = -1;
        if (slot >= a.num_slots) {
            if (a.status) atomicCAS(a.status, 0, (int) kErrBadArgument);
        } else if (slot >= 0) {
            const long long page = slot / a.page_size;
            off = page * a.c_page + (slot - page * a.page_size) * a.c_pos;
        }
        at[threadIdx.x] = off;
    }
    __syncthreads();
    const int u = threadIdx.x % kUnits;
    const bool rot_unit = 16 * u < a.rotary;
    const bool split = rot_unit && !interleaved;
    const int ea = split ? 8 * u : 16 * u, eb = split ? half + 8 * u : 16 * u + 8;
    const int heads = a.q_heads + 2 * a.kv_heads;
    // AHEAD (tiles of several tokens): a unit is read while the one before it is turned and
    // written, 118 -> 115 us for 16384 tokens of 64 + 2 x 8 heads of 128; a single token's few
    // units would only pay for the registers (1357 tokens of 48 heads of 64: 7.0 -> 8.2 us)
    struct Unit {
        Vec8<IN> a, b;
        int t, h;
    };
    auto fetch = [&](Unit& x, int t, int h) {  // false: behind the tile; a row that is not written is not read
        while (h >= heads) h -= heads, ++t;
        x.t = t, x.h = h;
        if (t >= nt) return false;
        if (h >= a.q_heads && at[t] < 0) return true;
        const long long tok = t0 + t;
        const IN* src = h < a.q_heads ? reinterpret_cast<const IN*>(a.q) + tok * a.q_tok + h * a.q_head
                        : h < a.q_heads + a.kv_heads
                            ? reinterpret_cast<const IN*>(a.k) + tok * a.k_tok + (h - a.q_heads) * a.k_head
                            : reinterpret_cast<const IN*>(a.v) + tok * a.v_tok + (h - a.q_heads - a.kv_heads) * a.v_head;
        x.a.load(src + ea);
        x.b.load(src + eb);
        return true;
    };
    Unit now, next;
    bool have = fetch(now, 0, threadIdx.x / kUnits);
    while (have) {
        if (AHEAD) have = fetch(next, now.t, now.h + kHeadsPerPass);
        const int kind = now.h < a.q_heads ? 0 : now.h < a.q_heads + a.kv_heads ? 1 : 2;  // q, k, v
        const long long off = at[now.t];
        if (kind == 0 || off >= 0) {
            float x[8], y[8];
            now.a.get(x);
            now.b.get(y);
            if (kind != 2 && rot_unit) {
                const float2* cs = &turn[now.t][8 * u];
                if (!interleaved) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const float2 w = cs[i];
                        const float p = x[i] * w.x - y[i] * w.y;
                        y[i] = y[i] * w.x + x[i] * w.y;
                        x[i] = p;
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 w = cs[i], z = cs[i + 4];
                        float p = x[2 * i] * w.x - x[2 * i + 1] * w.y;
                        x[2 * i + 1] = x[2 * i + 1] * w.x + x[2 * i] * w.y;
                        x[2 * i] = p;
                        p = y[2 * i] * z.x - y[2 * i + 1] * z.y;
                        y[2 * i + 1] = y[2 * i + 1] * z.x + y[2 * i] * z.y;
                        y[2 * i] = p;
                    }
                }
            }
            if (kind == 0) {
                QO* dst = reinterpret_cast<QO*>(a.q_out) + (t0 + now.t) * a.qo_tok + now.h * a.qo_head;
                store8<QO>(dst + ea, x);
                store8<QO>(dst + eb, y);
            } else {
                const int hh = now.h - a.q_heads - (kind == 2 ? a.kv_heads : 0);
                unsigned char* dst = (kind == 1 ? a.k_cache : a.v_cache) + off + hh * a.c_head;
                if constexpr (E4M3) {
                    const float* sp = kind == 1 ? a.k_scale : a.v_scale;
                    const float sc = sp ? sp[hh] : 1.f;
                    store8_e4m3(dst + ea, x, sc);
                    store8_e4m3(dst + eb, y, sc);
                } else {
                    store8<QO>(dst + 2 * ea, x);
                    store8<QO>(dst + 2 * eb, y);
                }
            }
        }
        if (AHEAD) now = next;
        else have = fetch(now, now.t, now.h + kHeadsPerPass);
    }
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------

struct AttnArgs {
    const void* q;
    const unsigned char* k;
    const unsigned char* v;
    const int* table;
    const int* lens;
    const float* k_scale;
    const float* v_scale;
    void* out;
    float* lse;
    int4* desc;       // [ctas]: {sequence, head block, pieces, 0} of the split item that begins in the CTA's range
    float* part_o;    // [2 ctas][mrows][D]: unnormalised partial outputs
    float2* part_ml;  // [2 ctas][mrows]: their row maximum (base 2, less kRef) and sum
    int* status;
    long long q_row, q_head, out_row, out_head;  // elements
    long long c_page, c_pos, c_head;             // bytes
    long long table_row;
    int seqs, rows, group, kv_heads, mblocks, mrows, mtotal;  // rows per sequence; m = row * group + head of the group
    int page_size, num_pages, capacity;
    unsigned page_mul;
    int page_sh1, page_sh2;
    int window;
    float scale, softcap;
};

constexpr int kAttnWarps = 4;
constexpr int kStages = 3;
constexpr int kMaxTiles = 5;   // row tiles of 8 of an item
constexpr int kItemRows = 8 * kMaxTiles;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                 "{%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <> __device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
                 "{%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void pg_ldsm4(uint32_t (&r)[4], unsigned s)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s) : "memory");
}
__device__ __forceinline__ void pg_ldsm4t(uint32_t (&r)[4], unsigned s)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(s) : "memory");
}
__device__ __forceinline__ void pg_cp16(unsigned s, const void* g, int bytes)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(s), "l"(g), "r"(bytes) : "memory");
}
// four e4m3 values as two fp16 pairs (exact)
__device__ __forceinline__ void e4m3x4_f16x2(uint32_t w, uint32_t& lo, uint32_t& hi)
{
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n cvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(lo), "=r"(hi) : "r"(w));
}
// weights as 16-bit hi + lo pairs: together about twice the type's significant bits, so
// that rounding the weights costs nothing beside the rounding of the output (single fp16
// weights for e4m3 caches under bf16 queries: verify 57.5 us instead of 61.7, but 9 % of its
// outputs a step of bf16 away from the rounded definition; pairs: 0.05 %)
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo, __nv_bfloat16)
{
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const float2 f = __bfloat1622float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack2(a - f.x, b - f.y, __nv_bfloat16());
}
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo, __half)
{
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack2(a - f.x, b - f.y, __half());
}

// 2^x to 2 ulp, 0 for -inf
__device__ __forceinline__ float ex2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// movmatrix: an 8x8 matrix of 16-bit elements, transposed across the warp
__device__ __forceinline__ uint32_t pg_transpose(uint32_t x)
{
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
    return r;
}
__device__ __forceinline__ float rcp(float x)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Weights are 2^(score - reference + kRef), a score at most 2^kSlack above the reference.
// fp16 weights reach 2^14 so that small ones keep their bits: what is lost of a weight is
// under 2^-31 of the largest.
constexpr float kSlack = 8.f;
// a positive factor of the scores, kept from 0, with which a masked -inf would become NaN, and from
// infinity, with which a score of 0 would (a NaN stays one)
__device__ __forceinline__ float in_range(float x) { return x < FLT_MIN ? FLT_MIN : x > FLT_MAX ? FLT_MAX : x; }
constexpr float kNone = -1e30f;  // the reference of a row that has seen nothing (finite: no case of its own in the loop)
template <typename MT> __host__ __device__ constexpr float weight_ref() { return std::is_same<MT, __half>::value ? 6.f : 0.f; }

template <int D, bool F8> struct AttnShape {
    static constexpr int kRowBytes = D * (F8 ? 1 : 2);
    static constexpr int kChunks = kRowBytes / 16;           // 16-byte pieces of a row
    static constexpr int kPos = kRowBytes == 256 ? 16 : 32;  // positions of a warp's stage
    static constexpr int kUnit = kAttnWarps * kPos;          // positions of a CTA's stage
    static constexpr int kSlot = 2 * kPos * kRowBytes;       // bytes of K and V
    static constexpr int kQPitch = 2 * D + 16;               // bytes of a row of q in shared memory
    static_assert(kSlot >= 16 * D * 4 && (kSlot & (kSlot - 1)) == 0, "a stage holds 16 rows of a warp's partial output at the end of an item");
    // 16-byte piece c of row r, so that eight rows of a piece column lie in distinct banks
    static __device__ __forceinline__ int at(int r, int c)
    {
        const int x = kRowBytes >= 128 ? (r & 7) : ((r >> 1) & 3);
        return r * kRowBytes + ((c ^ x) << 4);
    }
    // q in shared memory (more than 16 rows) follows the ring
    static constexpr int smem(int tiles) { return kAttnWarps * kStages * kSlot + (tiles > 2 ? 8 * tiles * kQPitch : 0); }
};

// A position in the launch's sequence of units: (sequence, kv head and row block, unit of
// the sequence's visible positions).  Every CTA owns a contiguous run of units.
template <int UNIT> struct Walk {
    int s, h, c, n, c0, lo, len;
    // `tokens`: the sequence's length, cut to what its pages hold
    __device__ __forceinline__ void sequence(const AttnArgs& a, int tokens)
    {
        len = tokens;
        lo = a.window > 0 ? max(0, len - a.rows + 1 - a.window) : 0;
        c0 = lo / UNIT;
        n = max(1, (len + UNIT - 1) / UNIT - c0);  // a sequence without tokens has one (masked) unit: its rows are written too
    }
    template <typename Length> __device__ __forceinline__ void next(const AttnArgs& a, Length length)
    {
        if (++c == n) {
            c = 0;
            if (++h == a.kv_heads * a.mblocks) {
                h = 0;
                s = min(s + 1, a.seqs - 1);  // (past the last sequence: nothing follows)
                sequence(a, length(s));
            }
        }
    }
};
__device__ __forceinline__ int attn_length(const AttnArgs& a, int s) { return min(max(__ldg(a.lens + s), 0), a.capacity); }

// One CTA: its run of units, warp w the positions w * kPos .. of each, through a ring of
// stages of its own (no barrier within an item).  The cache is the MMAs' A operand and
// the query rows (heads of the group, rows of the sequence) their N, so that 8 heads fill an
// MMA without padding: S^T = K Q^T, its columns' running maxima and sums, the weights
// transposed in registers (movmatrix) and O^T = V^T P^T.  (The query rows as the MMA's M,
// padded to 16, took 459 us instead of 397 for the first size below.)
//
// Every position is read once for all query rows of a kv head, by 16-byte asynchronous
// copies three stages deep; pages are looked up a stage ahead.  Bound by HBM where the cache
// is large: 64 sequences of up to 16384 (2.69 GB, bf16, 64 / 8 heads of 128) take 397 us with
// the join, 6.8 TB/s.  With e4m3 caches or 64-wide heads half the bytes carry the same
// instructions: 16 x 16384 e4m3, 32 / 4 heads, 53 us, 5.1 TB/s.  40 query rows (5 rows of 8
// heads) hold 160 accumulators a thread: 255 registers (of which 100 bytes spill), two warps
// a scheduler and nothing to hide their latencies with, 1.95 TB/s (137 us; as two items of
// 20 rows, the cache read twice, the same 137 us, but 176 instead of 141 over a bf16 cache).
// Small batches are a chain of latencies: 1 x 2049, 64 / 8 heads, 12 us in two kernels.
template <int D, typename QT, bool F8, int NT>
__global__ __launch_bounds__(32 * kAttnWarps, 2) void exl3_paged_attn_kernel(const __grid_constant__ AttnArgs a)
{
    using S = AttnShape<D, F8>;
    using MT = typename std::conditional<F8, __half, QT>::type;      // the MMAs' type
    constexpr float kRef = weight_ref<MT>();
    constexpr bool kRowScale = F8 && !std::is_same<QT, __half>::value;  // bf16 queries taken into fp16's range row by row
    constexpr bool kQShared = NT > 2;
    constexpr int kBlocks = S::kPos == 32 && NT <= 3 ? 2 : 1;  // 16-position blocks of a step (e4m3, 24 rows: 92.9 -> 78.2 us for 16 x 16384)
    extern __shared__ __align__(1024) unsigned char smem[];
    __shared__ float sh_m[kAttnWarps][8 * NT], sh_l[kAttnWarps][8 * NT];
    __shared__ int sh_start[3], sh_len[32 * kAttnWarps];
    __shared__ __align__(8) float sh_rs[kRowScale ? 8 * NT : 1];
    __shared__ long long sh_q[8 * NT];                // the item's rows: offset in q,
    __shared__ int sh_out[8 * NT];                    // row * q_heads + head,
    __shared__ __align__(8) int sh_end[8 * NT];       // and the positions below which are seen
    griddep_launch();
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, c = lane & 3;
    const int items = a.kv_heads * a.mblocks;  // of a sequence

    // Units of all sequences, and where this CTA's run begins: by the first warp, and the
    // lengths from there on through a window in shared memory, so that the warps never differ
    // about where an item ends - not even if a caller wrongly changes lengths under the kernel.
    Walk<S::kUnit> w;
    if (warp == 0) {
        int total = 0;
        for (w.s = lane; w.s < a.seqs; w.s += 32) {
            w.sequence(a, attn_length(a, w.s));
            total += w.n * items;
            if (blockIdx.x == 0 && __ldg(a.lens + w.s) > a.capacity) atomicCAS(a.status, 0, (int) kErrBadArgument);
        }
        total = __reduce_add_sync(~0u, total);
        const int grid = min((int) gridDim.x, total);
        const int u0 = (int) ((long long) blockIdx.x * total / grid);
        int first = a.seqs - 1, in = 0;
        for (int base = 0, s0 = 0; s0 < a.seqs && (int) blockIdx.x < grid; s0 += 32) {
            w.s = s0 + lane;
            int n = 0;
            if (w.s < a.seqs) {
                w.sequence(a, attn_length(a, w.s));
                n = w.n * items;
            }
            int inc = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int t = __shfl_up_sync(~0u, inc, d);
                if (lane >= d) inc += t;
            }
            const unsigned past = __ballot_sync(~0u, u0 < base + inc);
            if (past) {
                const int l = __ffs(past) - 1;
                first = s0 + l;
                in = u0 - base - __shfl_sync(~0u, inc - n, l);
                break;
            }
            base += __shfl_sync(~0u, inc, 31);
        }
        if (lane == 0) sh_start[0] = total, sh_start[1] = first, sh_start[2] = in;
    }
    __syncthreads();
    const int total = sh_start[0], grid = min((int) gridDim.x, total);
    if ((int) blockIdx.x >= grid) {
        if (tid == 0) a.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
        return;
    }
    const int u0 = (int) ((long long) blockIdx.x * total / grid), u1 = (int) ((long long) (blockIdx.x + 1) * total / grid);
    w.s = sh_start[1];
    int len_base = w.s;  // the window's first sequence
    auto read_lengths = [&] { sh_len[tid] = attn_length(a, min(len_base + tid, a.seqs - 1)); };
    auto length = [&](int s) { return sh_len[s - len_base]; };
    read_lengths();
    __syncthreads();
    w.sequence(a, length(w.s));
    w.h = min(sh_start[2] / w.n, items - 1);
    w.c = min(sh_start[2] - w.h * w.n, w.n - 1);

    const unsigned ring = (unsigned) __cvta_generic_to_shared(smem) + warp * (kStages * S::kSlot);
    const unsigned qsh = (unsigned) __cvta_generic_to_shared(smem) + kAttnWarps * kStages * S::kSlot;
    // a lane's position in a stage, its index in the block table, and whether a query row may see it
    auto locate = [&](const Walk<S::kUnit>& x, int& pos, int& pi) {
        pos = (x.c0 + x.c) * S::kUnit + warp * S::kPos + (lane & (S::kPos - 1));
        const unsigned t = __umulhi(a.page_mul, (unsigned) pos);
        pi = (int) ((t + (((unsigned) pos - t) >> a.page_sh1)) >> a.page_sh2);
        return pos >= x.lo && pos < x.len;
    };
    // its page, read a stage ahead of the stage's copies
    auto page_of = [&](const Walk<S::kUnit>& x) {
        int pos, pi;
        return locate(x, pos, pi) ? __ldg(a.table + x.s * a.table_row + pi) : -1;
    };
    // the copies of a stage: 8 (or 4) lanes a row; rows that no query row sees are zeroed
    auto stage = [&](const Walk<S::kUnit>& x, int slot, int page) {
        int pos, pi;
        bool ok = locate(x, pos, pi);
        long long off = 0;
        if (ok) {
            if ((unsigned) page >= (unsigned) a.num_pages) {
                ok = false;
                atomicCAS(a.status, 0, (int) kErrBadArgument);
            } else {
                off = page * a.c_page + (pos - pi * a.page_size) * a.c_pos + (x.h / a.mblocks) * a.c_head;
            }
        }
        const unsigned valid = __ballot_sync(~0u, ok);
        const unsigned base = ring + slot * S::kSlot;
        constexpr int kLanes = S::kChunks >= 8 ? 8 : S::kChunks;  // lanes of a row
        constexpr int kRows = 32 / kLanes;
        const int r0 = lane / kLanes, ch = lane % kLanes;
#pragma unroll
        for (int i = 0; i < S::kPos / kRows; ++i) {
            const int row = i * kRows + r0;
            const long long o = __shfl_sync(~0u, off, row) + ch * 16;
            const int bytes = (valid >> row) & 1 ? 16 : 0;
            const unsigned dst = base + S::at(row, ch);
#pragma unroll
            for (int x2 = 0; x2 < S::kChunks; x2 += kLanes) {
                pg_cp16(dst + 16 * x2, a.k + o + 16 * x2, bytes);
                pg_cp16(dst + 16 * x2 + S::kPos * S::kRowBytes, a.v + o + 16 * x2, bytes);
            }
        }
    };

    // first stages
    Walk<S::kUnit> f = w;  // runs ahead of w
    int fu = u0;
    int page = page_of(f);
    auto fill = [&](int slot) {
        if (fu < u1) {
            const Walk<S::kUnit> x = f;
            f.next(a, length);
            const int next = ++fu < u1 ? page_of(f) : -1;
            stage(x, slot, page);
            page = next;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fill(i);

    const int k_row = (lane & 7) + (((lane >> 3) & 1) << 3), v_row = F8 ? k_row : (lane & 7) + ((lane >> 4) << 3);
    uint32_t qf[kQShared ? 1 : D / 16][NT][2];  // B fragments of q
    float o[D / 16][NT][4];                     // O^T: dims g, g + 8 of a 16-dim tile x rows 2c, 2c + 1
    float rm[NT][2], rl[NT][2];                 // rows 2c, 2c + 1 of a tile: running maximum (base 2), this lane's sum
    float ks = 0.f;                             // the scores' scale, to base 2
    int mbase = 0, mcount = 0, item_u = u0, slot = 0;
    bool fresh = true;
    for (int u = u0; u < u1; ++u) {
        if (fresh) {  // a new item: its rows of q
            fresh = false;
            item_u = u;
            const int kvh = w.h / a.mblocks, mb = w.h - kvh * a.mblocks;
            mbase = mb * a.mrows;
            mcount = min(a.mrows, a.mtotal - mbase);
            ks = in_range(((F8 && a.k_scale) ? a.scale * __ldg(a.k_scale + kvh) : a.scale) * kLog2e);
            if (tid < 8 * NT) {  // (rows past the item's last repeat it and are not written)
                const int mm = mbase + min(tid, mcount - 1), j = mm / a.group;
                const int row = w.s * a.rows + j, head = kvh * a.group + mm - j * a.group;
                sh_q[tid] = row * a.q_row + head * a.q_head;
                sh_out[tid] = row * (a.kv_heads * a.group) + head;
                sh_end[tid] = w.len - a.rows + 1 + j;
            }
            __syncthreads();
            auto q_row = [&](int m) { return reinterpret_cast<const QT*>(a.q) + sh_q[m]; };
            // An e4m3 cache meets q in fp16, to which e4m3 converts exactly; a bf16 row is taken
            // into fp16's range by a power of two that the scores' scale takes back.  Four bytes
            // of a cache row come to a lane: dims 4c .. 4c + 3 of each 16 are its k slots.
            auto power = [&](float amax, float* down) {
                // amax 2^-e in [2^13, 2^14); zeros, infinities and NaN stay
                int e = (int) (__float_as_uint(amax) >> 23) - 127 - 13;
                if (amax == 0.f || !(amax < INFINITY)) e = 0;
                e = min(max(e, -100), 115);
                *down = __uint_as_float((unsigned) (127 - e) << 23);
                return __uint_as_float((unsigned) (127 + e) << 23);
            };
            auto lo16 = [](uint32_t x) { return __uint_as_float(x << 16); };
            auto hi16 = [](uint32_t x) { return __uint_as_float(x & 0xffff0000u); };
            if constexpr (!kQShared) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const QT* qr = q_row(8 * nt + g);
                    if constexpr (!F8) {
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk) {
                            qf[kk][nt][0] = *reinterpret_cast<const uint32_t*>(qr + 16 * kk + 2 * c);
                            qf[kk][nt][1] = *reinterpret_cast<const uint32_t*>(qr + 16 * kk + 8 + 2 * c);
                        }
                    } else {
                        float amax = 0.f;
#pragma unroll
                        for (int kk = 0; kk < D / 16; ++kk) {
                            const uint2 t = *reinterpret_cast<const uint2*>(qr + 16 * kk + 4 * c);
                            qf[kk][nt][0] = t.x, qf[kk][nt][1] = t.y;
                            if constexpr (kRowScale)
                                amax = fmaxf(amax, fmaxf(fmaxf(fabsf(lo16(t.x)), fabsf(hi16(t.x))), fmaxf(fabsf(lo16(t.y)), fabsf(hi16(t.y)))));
                        }
                        if constexpr (kRowScale) {
                            amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 1));
                            amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, 2));
                            float down;
                            const float up = power(amax, &down);
                            if (warp == 0 && c == 0) sh_rs[8 * nt + g] = in_range(ks * up);
#pragma unroll
                            for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
                                for (int i = 0; i < 2; ++i)
                                    qf[kk][nt][i] = pack2(lo16(qf[kk][nt][i]) * down, hi16(qf[kk][nt][i]) * down, __half());
                        }
                    }
                }
            } else {
                // eight lanes a row, D / 8 dims each; all rows read at once
                constexpr int kPer = D / 16;                                  // pairs of a lane and row
                constexpr int kMine = (8 * NT + 4 * kAttnWarps - 1) / (4 * kAttnWarps);
                uint32_t t[kMine][kPer];
                const int r0 = 4 * warp + (lane >> 3), l8 = lane & 7;
#pragma unroll
                for (int k = 0; k < kMine; ++k) {
                    const QT* qr = q_row(min(r0 + 4 * kAttnWarps * k, 8 * NT - 1)) + 2 * kPer * l8;
#pragma unroll
                    for (int i = 0; i < kPer; i += 4) *reinterpret_cast<uint4*>(&t[k][i]) = *reinterpret_cast<const uint4*>(qr + 2 * i);
                }
#pragma unroll
                for (int k = 0; k < kMine; ++k) {
                    const int m = r0 + 4 * kAttnWarps * k;
                    float down = 1.f, up = 1.f;
                    if constexpr (kRowScale) {
                        float amax = 0.f;
#pragma unroll
                        for (int i = 0; i < kPer; ++i) amax = fmaxf(amax, fmaxf(fabsf(lo16(t[k][i])), fabsf(hi16(t[k][i]))));
#pragma unroll
                        for (int i = 4; i; i >>= 1) amax = fmaxf(amax, __shfl_xor_sync(~0u, amax, i));
                        up = power(amax, &down);
                    }
                    if (m >= 8 * NT) continue;
                    if (kRowScale && l8 == 0) sh_rs[m] = in_range(ks * up);
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        const uint32_t x = kRowScale ? pack2(lo16(t[k][i]) * down, hi16(t[k][i]) * down, __half()) : t[k][i];
                        const int d = 2 * (kPer * l8 + i);
                        // e4m3: dims 4c, 4c + 1 of a 16 go to slots 2c, 2c + 1, dims 4c + 2, 4c + 3 to 8 + 2c, 9 + 2c
                        const int at = F8 ? (d & ~15) + ((d & 2) ? 8 : 0) + ((d & 12) >> 1) : d;
                        asm volatile("st.shared.u32 [%0], %1;" ::"r"(qsh + m * S::kQPitch + 2 * at), "r"(x) : "memory");
                    }
                }
            }
            if constexpr (kQShared || kRowScale) __syncthreads();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                rm[nt][0] = rm[nt][1] = kNone;
                rl[nt][0] = rl[nt][1] = 0.f;
#pragma unroll
                for (int j = 0; j < D / 16; ++j) o[j][nt][0] = o[j][nt][1] = o[j][nt][2] = o[j][nt][3] = 0.f;
            }
        }

        asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
        __syncwarp();
        fill(slot == 0 ? kStages - 1 : slot - 1);
        const int p0 = (w.c0 + w.c) * S::kUnit + warp * S::kPos;
        const unsigned kb = ring + slot * S::kSlot, vb = kb + S::kPos * S::kRowBytes;
#pragma unroll 1
        for (int sb = 0; sb < S::kPos / 16; sb += kBlocks) {
            const int ps = p0 + 16 * sb;
            if (ps >= w.len || ps + 16 * kBlocks <= w.lo) continue;  // warp-uniform
            // this lane's row and first piece of a tile of K and of V; other pieces differ in the
            // pieces' bits alone (a row begins on a boundary of its pieces)
            const unsigned ka0 = kb + S::at(16 * sb + k_row, lane >> 4);
            const unsigned va0 = vb + S::at(16 * sb + v_row, F8 ? lane >> 4 : (lane >> 3) & 1);
            // scores: positions g, g + 8 x rows 2c, 2c + 1 of every tile
            float s[kBlocks][NT][4];
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) s[b][nt][0] = s[b][nt][1] = s[b][nt][2] = s[b][nt][3] = 0.f;
            float s2[4] = {0.f, 0.f, 0.f, 0.f};  // one tile of one block: a second chain of accumulations
#pragma unroll
            for (int kk = 0; kk < D / 16; kk += 2)
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) {
                const unsigned ka = ka0 + b * 16 * S::kRowBytes;
                uint32_t k0[4], k1[4];
                if constexpr (F8) {
                    uint32_t r[4];
                    pg_ldsm4(r, ka ^ (16 * kk));
                    e4m3x4_f16x2(r[0], k0[0], k0[2]);
                    e4m3x4_f16x2(r[1], k0[1], k0[3]);
                    e4m3x4_f16x2(r[2], k1[0], k1[2]);
                    e4m3x4_f16x2(r[3], k1[1], k1[3]);
                } else {
                    pg_ldsm4(k0, ka ^ (32 * kk));
                    pg_ldsm4(k1, ka ^ (32 * kk + 32));
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    if constexpr (kQShared) {
                        uint32_t r[4];
                        pg_ldsm4(r, qsh + (8 * nt + (lane & 7)) * S::kQPitch + 32 * kk + 16 * (lane >> 3));
                        mma16816<MT>(s[b][nt], k0, r[0], r[1]);
                        mma16816<MT>(s[b][nt], k1, r[2], r[3]);
                    } else {
                        mma16816<MT>(s[b][nt], k0, qf[kk][nt][0], qf[kk][nt][1]);
                        mma16816<MT>(NT == 1 && kBlocks == 1 ? s2 : s[b][nt], k1, qf[kk + 1][nt][0], qf[kk + 1][nt][1]);
                    }
                }
            }
            if (NT == 1 && kBlocks == 1)
#pragma unroll
                for (int i = 0; i < 4; ++i) s[0][0][i] += s2[i];
            // cap and mask
            const bool open = ps >= w.lo && ps + 16 * kBlocks <= w.len - a.rows + 1 && (a.window <= 0 || ps >= w.len - a.window);
            // the factors that take rows 2c, 2c + 1 of a tile to base 2 (positive)
            auto factor = [&](int nt) {
                float2 t = make_float2(ks, ks);
                if constexpr (kRowScale) t = *reinterpret_cast<const float2*>(&sh_rs[8 * nt + 2 * c]);
                return t;
            };
            const bool capped = a.softcap > 0.f;
            if (capped) {
                // cap tanh(t), t = x / cap: cap (1 - 2 / (1 + exp(2 t))), near 0 (where that cancels) x (1 - t^2 / 3 + 2 t^4 / 15)
                const float capl = a.softcap * kLog2e, icap = 2.f / a.softcap, tcap = kLn2 / a.softcap;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float2 f = factor(nt);
#pragma unroll
                    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float y = s[b][nt][i] * ((i & 1) ? f.y : f.x), t = y * tcap, t2 = t * t;
                            const float far = fmaf(-2.f * capl, rcp(1.f + ex2(y * icap)), capl);
                            s[b][nt][i] = fabsf(t) < 0.06f ? y * fmaf(t2, fmaf(t2, 2.f / 15.f, -1.f / 3.f), 1.f) : far;
                        }
                }
            }
            if (!open) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int end = sh_end[8 * nt + 2 * c + (i & 1)];
#pragma unroll
                        for (int b = 0; b < kBlocks; ++b) {
                            const int pos = ps + 16 * b + g + 8 * (i >> 1);
                            if (pos >= end || (a.window > 0 && pos < end - a.window)) s[b][nt][i] = -INFINITY;
                        }
                    }
            }
            // The weights' reference is a maximum seen, raised only when a score exceeds it by
            // 2^kSlack: the outputs so far are rescaled in few of the steps.
            auto largest = [&](int nt, int i) {  // of the lane's scores in row 2c + i
                float x = fmaxf(s[0][nt][i], s[0][nt][2 + i]);
                if constexpr (kBlocks == 2) x = fmaxf(x, fmaxf(s[1][nt][i], s[1][nt][2 + i]));
                return x;
            };
            float top = -INFINITY;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float2 t = factor(nt);
                if (capped) t = make_float2(1.f, 1.f);
                top = fmaxf(top, fmaxf(fmaf(largest(nt, 0), t.x, -rm[nt][0]), fmaf(largest(nt, 1), t.y, -rm[nt][1])));
            }
            if (__any_sync(~0u, top > kSlack)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    float2 t = factor(nt);
                    if (capped) t = make_float2(1.f, 1.f);
                    float al[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float x = largest(nt, i) * (i ? t.y : t.x);
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 4));
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 8));
                        x = fmaxf(x, __shfl_xor_sync(~0u, x, 16));
                        x = fmaxf(x, rm[nt][i]);
                        al[i] = ex2(rm[nt][i] - x);
                        rm[nt][i] = x;
                        rl[nt][i] *= al[i];
                    }
#pragma unroll
                    for (int j = 0; j < D / 16; ++j) {
                        o[j][nt][0] *= al[0], o[j][nt][1] *= al[1];
                        o[j][nt][2] *= al[0], o[j][nt][3] *= al[1];
                    }
                }
            }
            // weights, as B fragments (rows x positions)
            uint32_t hi[kBlocks][NT][2], lo[kBlocks][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float2 t = factor(nt);
                if (capped) t = make_float2(1.f, 1.f);
                const float f0 = kRef - rm[nt][0], f1 = kRef - rm[nt][1];
#pragma unroll
                for (int bh = 0; bh < 2 * kBlocks; ++bh) {
                    const int b = bh >> 1, hf = bh & 1;
                    const float x = ex2(fmaf(s[b][nt][2 * hf], t.x, f0)), y = ex2(fmaf(s[b][nt][2 * hf + 1], t.y, f1));
                    rl[nt][0] += x;
                    rl[nt][1] += y;
                    split2(x, y, hi[b][nt][hf], lo[b][nt][hf], MT());
                    hi[b][nt][hf] = pg_transpose(hi[b][nt][hf]);
                    lo[b][nt][hf] = pg_transpose(lo[b][nt][hf]);
                }
            }
            if constexpr (F8) {
                // 16 dims of V: rows g of the A fragment are dims 2g, rows g + 8 dims 2g + 1
#pragma unroll
                for (int j = 0; j < D / 16; j += 2)
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    uint32_t r[4];
                    pg_ldsm4t(r, (va0 + b * 16 * S::kRowBytes) ^ (16 * j));
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        uint32_t v[4];
                        e4m3x4_f16x2(__byte_perm(r[2 * i], r[2 * i + 1], 0x6420), v[0], v[2]);
                        e4m3x4_f16x2(__byte_perm(r[2 * i], r[2 * i + 1], 0x7531), v[1], v[3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma16816<MT>(o[j + i][nt], v, hi[b][nt][0], hi[b][nt][1]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma16816<MT>(o[j + i][nt], v, lo[b][nt][0], lo[b][nt][1]);
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < D / 16; ++j)
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    uint32_t v[4];
                    pg_ldsm4t(v, (va0 + b * 16 * S::kRowBytes) ^ (32 * j));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816<MT>(o[j][nt], v, hi[b][nt][0], hi[b][nt][1]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma16816<MT>(o[j][nt], v, lo[b][nt][0], lo[b][nt][1]);
                }
            }
        }

        if (w.c == w.n - 1 || u == u1 - 1) {
            // the end of the item's piece: join the warps, 16 rows at a time, through the stage just read
            float* mine = reinterpret_cast<float*>(smem + warp * (kStages * S::kSlot) + slot * S::kSlot);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    rl[nt][i] += __shfl_xor_sync(~0u, rl[nt][i], 4);
                    rl[nt][i] += __shfl_xor_sync(~0u, rl[nt][i], 8);
                    rl[nt][i] += __shfl_xor_sync(~0u, rl[nt][i], 16);
                    if (g == 0) sh_m[warp][8 * nt + 2 * c + i] = rm[nt][i] > kNone ? rm[nt][i] : -INFINITY, sh_l[warp][8 * nt + 2 * c + i] = rl[nt][i];
                }
            const bool whole = w.c == w.n - 1 && u - item_u == w.n - 1;
            const bool starts = w.c == u - item_u;  // the piece holds the item's first unit
            const int kvh = w.h / a.mblocks;
            const long long part = 2ll * blockIdx.x + (starts ? 1 : 0);
            const float vs = (F8 && a.v_scale) ? __ldg(a.v_scale + kvh) : 1.f;
            // element (r, d) of the 16 x D tile: d ^ 8 (r / 2 % 4), so that a warp's stores meet distinct banks
#pragma unroll
            for (int n0 = 0; n0 < NT; n0 += 2) {
                if (8 * n0 >= mcount) break;
                __syncwarp();  // the stage has been read
#pragma unroll
                for (int nt = n0; nt < NT && nt < n0 + 2; ++nt)
#pragma unroll
                    for (int j = 0; j < D / 16; ++j)
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            float* row = mine + (8 * (nt - n0) + 2 * c + i) * D;
                            if constexpr (F8) {
                                *reinterpret_cast<float2*>(row + ((16 * j + 2 * g) ^ (8 * c))) = make_float2(o[j][nt][i], o[j][nt][2 + i]);
                            } else {
                                row[(16 * j + g) ^ (8 * c)] = o[j][nt][i];
                                row[(16 * j + 8 + g) ^ (8 * c)] = o[j][nt][2 + i];
                            }
                        }
                __syncthreads();
                constexpr int kVec = D / 4;  // threads of a row
                for (int e = tid; e < min(16, mcount - 8 * n0) * kVec; e += 32 * kAttnWarps) {
                    const int r = e / kVec, d = (e - r * kVec) * 4;
                    const int m = 8 * n0 + r;
                    float M = sh_m[0][m];
#pragma unroll
                    for (int i = 1; i < kAttnWarps; ++i) M = fmaxf(M, sh_m[i][m]);
                    float L = 0.f;
                    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < kAttnWarps; ++i) {
                        const float mi = sh_m[i][m], li = sh_l[i][m];
                        const float4 t = *reinterpret_cast<const float4*>(smem + i * (kStages * S::kSlot) + slot * S::kSlot +
                                                                          4 * (r * D + (d ^ (8 * ((r >> 1) & 3)))));
                        if (mi != -INFINITY || li != 0.f) {  // (a warp that saw only NaN: a sum, no maximum)
                            const float k = mi == -INFINITY ? 1.f : ex2(mi - M);
                            L += k * li;
                            y.x += k * t.x, y.y += k * t.y, y.z += k * t.z, y.w += k * t.w;
                        }
                    }
                    if (whole) {
                        const int at = sh_out[m], row = at / (a.kv_heads * a.group), head = at - row * (a.kv_heads * a.group);
                        const float inv = L == 0.f ? 0.f : vs / L;
                        QT* dst = reinterpret_cast<QT*>(a.out) + row * a.out_row + head * a.out_head + d;
                        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2(y.x * inv, y.y * inv, QT()), pack2(y.z * inv, y.w * inv, QT()));
                        if (a.lse && d == 0) a.lse[at] = L == 0.f ? -INFINITY : (M - kRef + log2f(L)) * kLn2;
                    } else {
                        *reinterpret_cast<float4*>(a.part_o + (part * a.mrows + m) * D + d) = y;
                        if (d == 0) a.part_ml[part * a.mrows + m] = make_float2(M, L);
                    }
                }
                __syncthreads();  // the stage may be filled again
            }
            if (u == u1 - 1 && tid == 0) {
                // a split item that begins here: how many CTAs hold it
                int pieces = 0;
                if (starts && !whole) {
                    const long long last = (long long) u + (w.n - 1 - w.c);  // the item's last unit
                    pieces = min((int) (((last + 1) * grid - 1) / total), grid - 1) - (int) blockIdx.x + 1;
                }
                a.desc[blockIdx.x] = make_int4(w.s, w.h, pieces, 0);
            }
            fresh = true;
        }
        w.next(a, length);
        if (fresh && w.s - len_base >= 16 * kAttnWarps) {  // half of the window is behind (f is two units ahead at most)
            __syncthreads();
            len_base = w.s;
            read_lengths();
            __syncthreads();
        }
        slot = slot == kStages - 1 ? 0 : slot + 1;
    }
}

// Joins the pieces of the items that the CTAs' runs split: block (x, y) takes the item that
// begins in the run of CTA x and its rows 8y .. 8y + 7, a warp each, in the order of the
// pieces (so that a result does not depend on timing).  A chain of loads: the first pieces
// are read along with the descriptor that says how many there are, the others eight at a
// time (1 x 2049, 33 pieces: 14.1 -> 12.0 us for both kernels).
constexpr int kJoinWarps = 8;
template <int D, typename QT, bool F8>
__global__ __launch_bounds__(32 * kJoinWarps) void exl3_paged_join_kernel(const __grid_constant__ AttnArgs a)
{
    constexpr float kRef = weight_ref<typename std::conditional<F8, __half, QT>::type>();
    constexpr int V = D / 32, kFirst = 4, kBatch = 8;
    griddep_launch();
    const int lane = threadIdx.x & 31;
    const int m = blockIdx.y * kJoinWarps + (threadIdx.x >> 5);
    if (m >= a.mrows) return;
    const int most = (int) (gridDim.x - 1 - blockIdx.x);  // pieces after the first, at most
    auto piece = [&](int p) { return (p == 0 ? 2ll * blockIdx.x + 1 : 2ll * (blockIdx.x + p)) * a.mrows + m; };
    auto load = [&](int p, float (&t)[V]) {
        const float* src = a.part_o + piece(p) * D + lane * V;
        if constexpr (V == 4) *reinterpret_cast<float4*>(t) = *reinterpret_cast<const float4*>(src);
        else *reinterpret_cast<float2*>(t) = *reinterpret_cast<const float2*>(src);
    };
    griddep_wait();
    const int4 d = a.desc[blockIdx.x];
    float2 ml = a.part_ml[piece(min(lane, most))];
    float first[kFirst][V];
#pragma unroll
    for (int i = 0; i < kFirst; ++i) load(min(i, most), first[i]);
    const int kvh = d.y / a.mblocks, mbase = (d.y - kvh * a.mblocks) * a.mrows;
    if (d.z == 0 || m >= a.mtotal - mbase) return;
    float M = lane < d.z ? ml.x : -INFINITY;
    for (int p = lane + 32; p < d.z; p += 32) M = fmaxf(M, a.part_ml[piece(p)].x);
#pragma unroll
    for (int i = 16; i; i >>= 1) M = fmaxf(M, __shfl_xor_sync(~0u, M, i));
    float L = 0.f, y[V];
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = 0.f;
    for (int p0 = 0; p0 < d.z; p0 += 32) {
        if (p0 > 0 && p0 + lane < d.z) ml = a.part_ml[piece(p0 + lane)];
        float k = 0.f;
        if (p0 + lane < d.z) {
            k = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : ex2(ml.x - M);
            L += k * ml.y;
        }
        const int n = min(32, d.z - p0);
        int i0 = 0;
        if (p0 == 0) {
#pragma unroll
            for (int i = 0; i < kFirst; ++i) {
                const float ki = __shfl_sync(~0u, k, i);
                if (i < n)
#pragma unroll
                    for (int e = 0; e < V; ++e) y[e] += ki * first[i][e];
            }
            i0 = kFirst;
        }
        for (int i = i0; i < n; i += kBatch) {  // (past the last piece it is read again, with weight 0)
            float t[kBatch][V];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) load(p0 + min(i + b, n - 1), t[b]);
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const float kb = __shfl_sync(~0u, k, (i + b) & 31), ki = i + b < n ? kb : 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] += ki * t[b][e];
            }
        }
    }
#pragma unroll
    for (int i = 16; i; i >>= 1) L += __shfl_xor_sync(~0u, L, i);
    const int mm = mbase + m, j = mm / a.group;
    const long long row = (long long) d.x * a.rows + j;
    const int head = kvh * a.group + mm - j * a.group;
    const float vs = (F8 && a.v_scale) ? __ldg(a.v_scale + kvh) : 1.f;
    const float inv = L == 0.f ? 0.f : vs / L;
    QT* dst = reinterpret_cast<QT*>(a.out) + row * a.out_row + head * a.out_head + lane * V;
#pragma unroll
    for (int e = 0; e < V; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack2(y[e] * inv, y[e + 1] * inv, QT());
    if (a.lse && lane == 0)
        a.lse[row * (a.kv_heads * a.group) + head] = L == 0.f ? -INFINITY : (M - kRef + log2f(L)) * kLn2;
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

template <typename Kern, typename... Args>
static int paged_launch(Kern kern, dim3 grid, int block, int smem, cudaStream_t stream, Args... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned) block);
    cfg.dynamicSmemBytes = (size_t) smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, args...) == cudaSuccess ? kOk : kErrLaunch;
}

static bool misaligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n != 0; }

// whether two of an output's n0 x n1 rows of d elements share an address (an expanded view):
// several CTAs would write it
static bool overlapping(long long n0, long long s0, long long n1, long long s1, int d)
{
    s0 = std::abs(s0), s1 = std::abs(s1);
    if (n0 <= 1 || n1 <= 1) return (n0 > 1 && s0 < d) || (n1 > 1 && s1 < d);
    if (s0 < s1) std::swap(s0, s1), std::swap(n0, n1);
    return s1 < d || s0 < (n1 - 1) * s1 + d;
}

// the strides of a cache, in bytes; false: a row would not begin on a 16-byte boundary
static bool cache_strides(const exl3b200_paged_cache& c, long long* page, long long* pos, long long* head)
{
    const int e = c.dtype == kE4m3 ? 1 : 2;
    *page = c.page_stride * e, *pos = c.pos_stride * e, *head = c.head_stride * e;
    return !(misaligned(c.k, 16) || misaligned(c.v, 16) || *page % 16 || *pos % 16 || *head % 16);
}

static int check_cache(const exl3b200_paged_cache& c)
{
    if (!c.k || !c.v) return kErrNullPointer;
    if (c.pages < 1 || c.page_size < 1 || c.kv_heads < 1 || (c.head_dim != 64 && c.head_dim != 128)) return kErrBadShape;
    if (c.page_stride < 0 || c.pos_stride < 0 || c.head_stride < 0) return kErrBadShape;
    if (c.dtype != kF16 && c.dtype != kBf16 && c.dtype != kE4m3) return kErrBadArgument;
    return kOk;
}

template <typename IN, typename QO, bool E4M3>
static int append_launch(const AppendArgs& a, int head_dim, int tile, int interleaved, cudaStream_t st)
{
    const dim3 grid((unsigned) ((a.tokens + tile - 1) / tile));
    if (head_dim == 128)
        return tile > 1 ? paged_launch(exl3_rope_append_kernel<IN, QO, E4M3, 128, true>, grid, kAppThreads, 0, st, a, tile, interleaved)
                        : paged_launch(exl3_rope_append_kernel<IN, QO, E4M3, 128, false>, grid, kAppThreads, 0, st, a, tile, interleaved);
    return tile > 1 ? paged_launch(exl3_rope_append_kernel<IN, QO, E4M3, 64, true>, grid, kAppThreads, 0, st, a, tile, interleaved)
                    : paged_launch(exl3_rope_append_kernel<IN, QO, E4M3, 64, false>, grid, kAppThreads, 0, st, a, tile, interleaved);
}

template <typename IN>
static int append_types(const AppendArgs& a, int q_out, int cache, int head_dim, int tile, int interleaved, cudaStream_t st)
{
    if (cache == kE4m3)
        return q_out == kF16 ? append_launch<IN, __half, true>(a, head_dim, tile, interleaved, st)
                             : append_launch<IN, __nv_bfloat16, true>(a, head_dim, tile, interleaved, st);
    return q_out == kF16 ? append_launch<IN, __half, false>(a, head_dim, tile, interleaved, st)
                         : append_launch<IN, __nv_bfloat16, false>(a, head_dim, tile, interleaved, st);
}

template <int D, typename QT, bool F8, int NT>
static int attn_launch(const AttnArgs& a, int ctas, cudaStream_t st)
{
    constexpr int smem = AttnShape<D, F8>::smem(NT);
    static std::atomic<bool> done[64];  // threads that race on the first call set the same value
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return kErrLaunch;
    auto kern = exl3_paged_attn_kernel<D, QT, F8, NT>;
    if (!done[dev].load(std::memory_order_acquire)) {
        if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return kErrLaunch;
        done[dev].store(true, std::memory_order_release);
    }
    const int rc = paged_launch(kern, dim3((unsigned) ctas), 32 * kAttnWarps, smem, st, a);
    if (rc != kOk) return rc;
    return paged_launch(exl3_paged_join_kernel<D, QT, F8>, dim3((unsigned) ctas, (unsigned) ((a.mrows + kJoinWarps - 1) / kJoinWarps)),
                        32 * kJoinWarps, 0, st, a);
}

template <int D, typename QT, bool F8>
static int attn_tiles(const AttnArgs& a, int ctas, cudaStream_t st)
{
    const int tiles = (a.mrows + 7) / 8;
    if (tiles == 1) return attn_launch<D, QT, F8, 1>(a, ctas, st);
    if (tiles == 2) return attn_launch<D, QT, F8, 2>(a, ctas, st);
    if (tiles == 3) return attn_launch<D, QT, F8, 3>(a, ctas, st);
    return attn_launch<D, QT, F8, 5>(a, ctas, st);
}

template <typename QT>
static int attn_types(const AttnArgs& a, int head_dim, bool f8, int ctas, cudaStream_t st)
{
    if (head_dim == 128) return f8 ? attn_tiles<128, QT, true>(a, ctas, st) : attn_tiles<128, QT, false>(a, ctas, st);
    return f8 ? attn_tiles<64, QT, true>(a, ctas, st) : attn_tiles<64, QT, false>(a, ctas, st);
}

// How the rows of a (sequence, kv head) go into items: up to 40 at once, more in blocks of
// equal size.
struct AttnSplit {
    int mtotal, mblocks, mrows, ctas;
    size_t o_bytes, ml_bytes, desc_bytes;
};
static AttnSplit attn_split(int rows, int group, int head_dim)
{
    AttnSplit s;
    s.mtotal = rows * group;
    s.mblocks = (s.mtotal + kItemRows - 1) / kItemRows;
    s.mrows = (s.mtotal + s.mblocks - 1) / s.mblocks;
    s.ctas = 2 * kSms;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    s.o_bytes = up((size_t) 2 * s.ctas * s.mrows * head_dim * 4);
    s.ml_bytes = up((size_t) 2 * s.ctas * s.mrows * 8);
    s.desc_bytes = up((size_t) s.ctas * 16);
    return s;
}

}  // namespace exl3b200

using namespace exl3b200;

extern "C" int exl3b200_rope_append(const exl3b200_rope_append_args* p, void* stream)
{
    if (!p) return kErrNullPointer;
    const exl3b200_paged_cache& c = p->cache;
    if (const int rc = check_cache(c)) return rc;
    if (!p->q || !p->k || !p->v || !p->q_out || !p->positions || !p->slots || (p->rotary > 0 && !p->inv_freq)) return kErrNullPointer;
    if (p->tokens < 1 || p->q_heads < 1 || p->rotary < 0 || p->rotary > c.head_dim || p->rotary % 16) return kErrBadShape;
    if (p->in_dtype != kF16 && p->in_dtype != kBf16 && p->in_dtype != kF32) return kErrBadArgument;
    if (p->q_out_dtype != kF16 && p->q_out_dtype != kBf16) return kErrBadArgument;
    if (c.dtype != kE4m3 && c.dtype != p->q_out_dtype) return kErrBadArgument;
    if (p->interleaved != 0 && p->interleaved != 1) return kErrBadArgument;
    const long long vec = p->in_dtype == kF32 ? 4 : 8;  // elements of 16 bytes
    const long long in[] = {p->q_stride, p->q_head_stride, p->k_stride, p->k_head_stride, p->v_stride, p->v_head_stride};
    for (long long s : in)
        if (s % vec) return kErrUnaligned;
    if (p->q_out_stride % 8 || p->q_out_head_stride % 8) return kErrUnaligned;
    if (misaligned(p->q, 16) || misaligned(p->k, 16) || misaligned(p->v, 16) || misaligned(p->q_out, 16)) return kErrUnaligned;
    if (overlapping(p->tokens, p->q_out_stride, p->q_heads, p->q_out_head_stride, c.head_dim)) return kErrBadShape;
    AppendArgs a = {};
    if (!cache_strides(c, &a.c_page, &a.c_pos, &a.c_head)) return kErrUnaligned;
    a.q = p->q, a.k = p->k, a.v = p->v, a.q_out = p->q_out;
    a.k_cache = reinterpret_cast<unsigned char*>(c.k), a.v_cache = reinterpret_cast<unsigned char*>(c.v);
    a.positions = p->positions, a.slots = p->slots, a.inv_freq = p->inv_freq;
    a.k_scale = c.k_scale, a.v_scale = c.v_scale;
    a.q_tok = p->q_stride, a.q_head = p->q_head_stride, a.k_tok = p->k_stride, a.k_head = p->k_head_stride;
    a.v_tok = p->v_stride, a.v_head = p->v_head_stride, a.qo_tok = p->q_out_stride, a.qo_head = p->q_out_head_stride;
    a.num_slots = (long long) c.pages * c.page_size;
    a.tokens = p->tokens, a.q_heads = p->q_heads, a.kv_heads = c.kv_heads, a.page_size = c.page_size, a.rotary = p->rotary;
    a.status = exl3_status_dev_ptr();
    if (!a.status) return kErrLaunch;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const int tile = p->tokens >= 8 * kSms * kAppMaxTile ? kAppMaxTile : 1;
    if (p->in_dtype == kF16) return append_types<__half>(a, p->q_out_dtype, c.dtype, c.head_dim, tile, p->interleaved, st);
    if (p->in_dtype == kBf16) return append_types<__nv_bfloat16>(a, p->q_out_dtype, c.dtype, c.head_dim, tile, p->interleaved, st);
    return append_types<float>(a, p->q_out_dtype, c.dtype, c.head_dim, tile, p->interleaved, st);
}

extern "C" size_t exl3b200_paged_attention_scratch_size(int rows_per_seq, int q_heads, int kv_heads, int head_dim)
{
    if (rows_per_seq < 1 || kv_heads < 1 || q_heads < kv_heads || q_heads % kv_heads || (head_dim != 64 && head_dim != 128)) return 0;
    if ((long long) rows_per_seq * (q_heads / kv_heads) > EXL3B200_PAGED_MAX_ROWS) return 0;
    const AttnSplit s = attn_split(rows_per_seq, q_heads / kv_heads, head_dim);
    return s.o_bytes + s.ml_bytes + s.desc_bytes;
}

extern "C" int exl3b200_paged_attention(const exl3b200_paged_attention_args* p, void* scratch, size_t scratch_bytes, void* stream)
{
    if (!p) return kErrNullPointer;
    const exl3b200_paged_cache& c = p->cache;
    if (const int rc = check_cache(c)) return rc;
    if (!p->q || !p->out || !p->block_table || !p->seq_lens || !scratch) return kErrNullPointer;
    if (p->seqs < 1 || p->max_pages < 1 || p->table_stride < p->max_pages || p->window < 0) return kErrBadShape;
    const size_t need = exl3b200_paged_attention_scratch_size(p->rows_per_seq, p->q_heads, c.kv_heads, c.head_dim);
    if (need == 0) return kErrBadShape;
    if (p->dtype != kF16 && p->dtype != kBf16) return kErrBadArgument;
    if (c.dtype != kE4m3 && c.dtype != p->dtype) return kErrBadArgument;
    if (!(p->softcap == 0.f || p->softcap >= 1e-6f) || !std::isfinite(p->softcap) || !(p->scale > 0.f) || !std::isfinite(p->scale)) return kErrBadArgument;
    if (scratch_bytes < need) return kErrWorkspace;
    if (misaligned(scratch, 256) || misaligned(p->q, 16) || misaligned(p->out, 16)) return kErrUnaligned;
    if (p->q_stride % 8 || p->q_head_stride % 8 || p->out_stride % 8 || p->out_head_stride % 8) return kErrUnaligned;
    if (overlapping((long long) p->seqs * p->rows_per_seq, p->out_stride, p->q_heads, p->out_head_stride, c.head_dim)) return kErrBadShape;
    AttnArgs a = {};
    if (!cache_strides(c, &a.c_page, &a.c_pos, &a.c_head)) return kErrUnaligned;
    const AttnSplit sp = attn_split(p->rows_per_seq, p->q_heads / c.kv_heads, c.head_dim);
    // positions are 32-bit, a length less the rows and a window and one rounded up to units among
    // them, and so is the number of units of a launch
    const long long capacity = std::min((long long) p->max_pages * c.page_size, (long long) INT_MAX - 2 * EXL3B200_PAGED_MAX_ROWS);
    if (((capacity + 63) / 64 + 1) * p->seqs * c.kv_heads * sp.mblocks > INT_MAX ||
        (long long) p->seqs * p->rows_per_seq * p->q_heads > INT_MAX)
        return kErrBadShape;
    a.q = p->q, a.out = p->out, a.lse = p->lse;
    a.k = reinterpret_cast<const unsigned char*>(c.k), a.v = reinterpret_cast<const unsigned char*>(c.v);
    a.table = p->block_table, a.lens = p->seq_lens, a.table_row = p->table_stride;
    a.k_scale = c.k_scale, a.v_scale = c.v_scale;
    unsigned char* w = reinterpret_cast<unsigned char*>(scratch);
    a.part_o = reinterpret_cast<float*>(w);
    a.part_ml = reinterpret_cast<float2*>(w + sp.o_bytes);
    a.desc = reinterpret_cast<int4*>(w + sp.o_bytes + sp.ml_bytes);
    a.q_row = p->q_stride, a.q_head = p->q_head_stride, a.out_row = p->out_stride, a.out_head = p->out_head_stride;
    a.seqs = p->seqs, a.rows = p->rows_per_seq, a.group = p->q_heads / c.kv_heads, a.kv_heads = c.kv_heads;
    a.mblocks = sp.mblocks, a.mrows = sp.mrows, a.mtotal = sp.mtotal;
    a.page_size = c.page_size, a.num_pages = c.pages, a.capacity = (int) capacity;
    // position / page_size as a multiplication (unsigned division by an invariant, Granlund and Montgomery)
    int l = 0;
    while (l < 31 && (1u << l) < (unsigned) c.page_size) ++l;
    a.page_mul = (unsigned) ((((1ull << l) - (unsigned) c.page_size) << 32) / (unsigned) c.page_size + 1);
    a.page_sh1 = std::min(l, 1), a.page_sh2 = std::max(l - 1, 0);
    a.window = p->window >= capacity ? 0 : p->window, a.scale = p->scale, a.softcap = p->softcap;
    a.status = exl3_status_dev_ptr();
    if (!a.status) return kErrLaunch;
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    const bool f8 = c.dtype == kE4m3;
    return p->dtype == kF16 ? attn_types<__half>(a, c.head_dim, f8, sp.ctas, st)
                            : attn_types<__nv_bfloat16>(a, c.head_dim, f8, sp.ctas, st);
}
