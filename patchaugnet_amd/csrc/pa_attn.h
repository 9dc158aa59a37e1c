// Shared device code of the windowed / paged attention kernels (window_attention.hip, window_attention_bwd.hip, paged_attention.hip).
//
// All of them multiply with 32 x 32 MFMA tiles and keep the same register layouts:
//   operand fragment  lane l holds row l % 32, contraction slots 8 (l / 32) + e, e = 0..7 of 16
//   accumulator       lane l holds column l % 32, rows 8 (r / 4) + 4 (l / 32) + r % 4, r = 0..15
// 16-bit types contract 16 slots with one v_mfma_f32_32x32x16; float32 contracts them with eight v_mfma_f32_32x32x2, MFMA e taking slots e and 8 + e.
//
// Eight accumulator registers of a lane (r = 8 u .. 8 u + 7) ARE an operand fragment whose slot 8 h + e stands for row 16 u + 4 h + e (e < 4) or
// 16 u + 8 + 4 h + e - 4: a product computed into registers feeds the next one without leaving them, if the other operand lists its contraction
// index in the same order (ldt below).
#pragma once
#include <initializer_list>

#include "pa_common.h"

typedef float pa_f16v __attribute__((ext_vector_type(16)));
typedef float pa_f8 __attribute__((ext_vector_type(8)));
typedef float pa_f4 __attribute__((ext_vector_type(4)));
typedef __bf16 pa_bf8 __attribute__((ext_vector_type(8)));
typedef __bf16 pa_bf4 __attribute__((ext_vector_type(4)));
typedef _Float16 pa_h8 __attribute__((ext_vector_type(8)));
typedef _Float16 pa_h4 __attribute__((ext_vector_type(4)));
typedef short pa_s4 __attribute__((ext_vector_type(4)));
typedef u32 pa_u4 __attribute__((ext_vector_type(4), may_alias));

enum { PA_DT_F32 = 0, PA_DT_F16 = 1, PA_DT_BF16 = 2 };

namespace pa_attn {

constexpr int MAXLEN = 1 << 28;          // tokens of a sequence, rows of a key head: their sums and those with a window side stay inside 32 bits
constexpr int UNBOUNDED = 1 << 29;       // window side without a limit
constexpr int NOWHERE = 0x7fffffff;      // a position that no key reaches

// Workgroups go to the eight XCDs in turn; each XCD has an L2 of its own.  Work item for workgroup x of n, such that an XCD's workgroups own one
// contiguous run of items: neighbours, which share keys and values, meet in one L2.
__device__ __forceinline__ long xcd_item(long x, long n)
{
    const long k = x & 7, each = n >> 3, rest = n & 7;
    return k * each + (k < rest ? k : rest) + (x >> 3);
}

template <typename T> struct Frag;
template <> struct Frag<float> { typedef pa_f8 type; };
template <> struct Frag<_Float16> { typedef pa_h8 type; };
template <> struct Frag<__bf16> { typedef pa_bf8 type; };

__device__ __forceinline__ void mma(pa_f16v &c, const pa_bf8 &a, const pa_bf8 &b) { c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ void mma(pa_f16v &c, const pa_h8 &a, const pa_h8 &b) { c = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ void mma(pa_f16v &c, const pa_f8 &a, const pa_f8 &b)
{
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
}

// the larger of two scores, NaN if one is: v_maximum3_f32 takes three without the canonicalising moves that fmaxf needs on a product's registers
__device__ __forceinline__ float larger(float a, float b) { return __builtin_elementwise_maximum(a, b); }
__device__ __forceinline__ float ex2(float x) { return __builtin_amdgcn_exp2f(x); }

// value of the lane with the other l / 32
__device__ __forceinline__ float other_half(float x)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// A tile of rows in LDS: 16-byte chunks, chunk c of row r at place c ^ swz(r).  The swizzle makes both kinds of reads free of bank conflicts for
// every row width (multiples of 64 bytes): 16 rows at one chunk (operand fragments) and 4 rows at 4 neighbouring chunks (transposed fragments).
template <typename T, int DT> struct Tile {
    static constexpr int RB = DT * (int)sizeof(T);           // bytes of a row
    static constexpr int CH = RB / 16;                       // chunks of a row
    static constexpr int EC = 16 / (int)sizeof(T);           // elements of a chunk

    __device__ static __forceinline__ int swz(int r)
    {
        const int low = (r >> 2) & 3;
        if (RB % 256 == 0) return ((r & 3) << 2) | low;
        if (RB % 128 == 0) return ((r & 2) << 1) | low;
        return low;
    }
    __device__ static __forceinline__ int at(int r, int c) { return r * RB + ((c ^ swz(r)) << 4); }

    // operand fragment: row r0 + l % 32, elements 16 kk + 8 (l / 32) ..
    __device__ static __forceinline__ typename Frag<T>::type ld(const char *s, int r0, int kk)
    {
        const int l = threadIdx.x & 63, r = r0 + (l & 31), h = l >> 5;
        typename Frag<T>::type f;
        if constexpr (sizeof(T) == 2) {
            f = *reinterpret_cast<const typename Frag<T>::type *>(s + at(r, 2 * kk + h));
        } else {
            const pa_f4 a = *reinterpret_cast<const pa_f4 *>(s + at(r, 4 * kk + 2 * h)), b = *reinterpret_cast<const pa_f4 *>(s + at(r, 4 * kk + 2 * h + 1));
            f = (pa_f8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        }
        return f;
    }

    // transposed fragment: "row" = element c0 + l % 32, contraction slots over the rows r0 .. r0 + 15 in the accumulators' order
    // (slot 8 h + e: row r0 + 4 h + e, e < 4, or r0 + 8 + 4 h + e - 4).  16-bit: ds_read_b64_tr_b16, where lane s of 16 passes the address of four
    // elements of row s / 4 and receives one element of each of the four rows.
    __device__ static __forceinline__ typename Frag<T>::type ldt(const char *s, int r0, int c0)
    {
        const int l = threadIdx.x & 63, h = l >> 5;
        if constexpr (sizeof(T) == 2) {
            const int q = l & 15, c = c0 + (l & 16) + 4 * (q & 3);
            const int ra = r0 + 4 * h + (q >> 2), rb = ra + 8;
            typedef __attribute__((address_space(3))) pa_s4 *lp;
            const pa_s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(s + at(ra, c >> 3) + (c & 4) * 2));
            const pa_s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(s + at(rb, c >> 3) + (c & 4) * 2));
            typedef short s8 __attribute__((ext_vector_type(8)));
            const s8 z = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
            return __builtin_bit_cast(typename Frag<T>::type, z);
        } else {
            pa_f8 f;
            const int c = c0 + (l & 31);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = r0 + 4 * h + (e & 3) + 8 * (e >> 2);
                f[e] = *reinterpret_cast<const float *>(s + at(r, c >> 2) + (c & 3) * 4);
            }
            return f;
        }
    }
};

// 16 bytes of a row from global memory, zeros when `ok` is false (the address is not touched then)
__device__ __forceinline__ pa_u4 ldg16(const void *p, bool ok)
{
    pa_u4 z = {0, 0, 0, 0};
    if (ok) z = *reinterpret_cast<const pa_u4 *>(p);
    return z;
}

// A per-thread offset, fixed for the whole kernel, at the place of its use.  Without this the compiler (ROCm 7.2) keeps the 64-bit form of the offset
// across the loop and, where one way of a fetch is masked, computes it in some lanes only: the other lanes then load from anywhere.
__device__ __forceinline__ u32 here(u32 x)
{
    asm volatile("" : "+v"(x));
    return x;
}

__device__ const pa_u4 pa_zeros = {0, 0, 0, 0};

// R rows of a tensor straight from memory into an LDS tile by NT threads (global_load_lds, 16 bytes a lane): no registers on the way, one load per chunk
// at (uniform base of the tile) + (32-bit offset of the thread, the same for every tile).  A wave's lanes fill 64 neighbouring places, so the swizzle is in which chunk a lane asks for; rows from `valid` on and elements from d on are asked of a block of zeros.
// The data is there for all waves after arrived() and a barrier.
template <typename T, int DT, int R, int NT> struct Direct {
    typedef Tile<T, DT> L;
    static constexpr int ALL = R * L::CH, N = (ALL + NT - 1) / NT;
    u32 off[N];

    __device__ static __forceinline__ int row(int u) { return (int)(threadIdx.x + u * NT) / L::CH; }
    __device__ static __forceinline__ int chunk(int u) { return ((int)(threadIdx.x + u * NT) - row(u) * L::CH) ^ L::swz(row(u)); }
    __device__ __forceinline__ void strided(long stride)
    {
#pragma unroll
        for (int u = 0; u < N; ++u) off[u] = ((u32)row(u) * (u32)stride + chunk(u) * L::EC) * (u32)sizeof(T);
    }
    __device__ __forceinline__ void fetch(char *tile, const T *base, int valid, int d) const
    {
        typedef const __attribute__((address_space(1))) void *gp;
        typedef __attribute__((address_space(3))) void *lp;
        const char *p = reinterpret_cast<const char *>(base);
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        if (valid >= R && d == DT) {
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (ALL % NT == 0 || wave * 64 + u * NT < ALL) __builtin_amdgcn_global_load_lds((gp)(p + here(off[u])), (lp)(tile + (u * NT + wave * 64) * 16), 16, 0, 0);
        } else {
#pragma unroll
            for (int u = 0; u < N; ++u)
                if (ALL % NT == 0 || wave * 64 + u * NT < ALL) {
                    const bool ok = row(u) < valid && chunk(u) * L::EC < d;
                    const u32 o = here(off[u]);
                    const char *g = ok ? p + o : reinterpret_cast<const char *>(&pa_zeros);
                    __builtin_amdgcn_global_load_lds((gp)g, (lp)(tile + (u * NT + wave * 64) * 16), 16, 0, 0);
                }
        }
    }
};
__device__ __forceinline__ void arrived() { __builtin_amdgcn_s_waitcnt(0x0f70); }      // vmcnt(0): this wave's loads into LDS

// eight accumulator registers as an operand fragment (one rounding to the operand type)
template <typename T> __device__ __forceinline__ typename Frag<T>::type pack(const pa_f16v &a, int u)
{
    typename Frag<T>::type f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (T)a[8 * u + e];
    return f;
}

// what pack() rounded away, as a fragment of its own: with it a product takes the registers to twice the type's digits
template <typename T> __device__ __forceinline__ typename Frag<T>::type pack_rest(const pa_f16v &a, const typename Frag<T>::type &f, int u)
{
    typename Frag<T>::type g;
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = (T)(a[8 * u + e] - (float)f[e]);
    return g;
}

// fragment of a row held in global memory: elements 16 kk + 8 h .. of `row`, zeros past d (a multiple of 8)
template <typename T> __device__ __forceinline__ typename Frag<T>::type ldrow(const T *row, int kk, int h, int d, bool ok)
{
    const int e0 = 16 * kk + 8 * h;
    ok = ok && e0 < d;
    if constexpr (sizeof(T) == 2) {
        return __builtin_bit_cast(typename Frag<T>::type, ldg16(row + e0, ok));
    } else {
        const pa_f4 a = __builtin_bit_cast(pa_f4, ldg16(row + e0, ok)), b = __builtin_bit_cast(pa_f4, ldg16(row + e0 + 4, ok));
        return (pa_f8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    }
}

// four floats as four elements of a row
template <typename T> __device__ __forceinline__ void st4(T *p, float a, float b, float c, float d)
{
    typedef T t4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<t4 *>(p) = (t4){(T)a, (T)b, (T)c, (T)d};
}

// x / g for 0 <= x < 2^31 by one multiplication with m = ceil(2^32 / g): the excess x (m g - 2^32) / (g 2^32) is below 1/2, so the product is the
// quotient or one more, and one comparison settles it
struct Div {
    u32 g, m;
    __host__ __device__ Div() : g(1), m(0) {}
    explicit __host__ Div(int d) : g((u32)d), m((u32)((0x100000000ull + (u32)d - 1) / (u32)d)) {}
    __device__ __forceinline__ int div(int x) const
    {
        if (g == 1) return x;
        u32 q = __umulhi((u32)x, m);
        if (q * g > (u32)x) --q;
        return (int)q;
    }
};

// What a query sees.  Query i of sequence b stands at position p = start_b + i; key j is in view if j < len_b, j <= p + right, and j >= p - left or
// j < sinks.  A query at p >= len_b is padding and sees nothing.  Both device values are clamped to the buffer, so that no value faults.
struct View {
    int m, left, right, sinks;
    const int *start, *length;

    __device__ __forceinline__ int len(int b) const { return length ? min(max(length[b], 0), m) : m; }
    __device__ __forceinline__ int first(int b) const { return start ? min(max(start[b], 0), m) : 0; }
};

// keys in view of one row as [lo, lo + span] and [0, sink); nothing: lo out of reach
struct Keys {
    int lo, sink;
    u32 span;
    bool ok;

    __device__ __forceinline__ Keys(const View &v, int p, int len, bool there)
    {
        ok = there && p < len;
        const int hi = min(p + v.right, len - 1);
        lo = ok ? max(p - v.left, 0) : NOWHERE;
        span = ok ? (u32)(hi - lo) : 0u;
        sink = ok ? min(v.sinks, hi + 1) : 0;
    }
    __device__ __forceinline__ bool sees(int j) const { return (u32)(j - lo) <= span || j < sink; }
};

// the KT-key tiles that rows at positions p0 .. p1 walk: nsk tiles of first tokens, then [lo, hi)
template <int KT> struct TileList {
    int nsk, lo, n;

    __device__ __forceinline__ TileList(const View &v, int p0, int p1, int len)
    {
        nsk = lo = n = 0;
        p1 = min(p1, len - 1);
        if (p0 > p1) return;                                   // padding rows only
        const int hi = min(p1 + v.right, len - 1) + 1;
        lo = max(p0 - v.left, 0) / KT;
        nsk = min((min(v.sinks, hi) + KT - 1) / KT, lo);
        n = nsk + (hi + KT - 1) / KT - lo;
    }
    __device__ __forceinline__ int tile(int i) const { return i < nsk ? i : lo + i - nsk; }
};

// Waves of a workgroup, each with 32 rows (forward, dq) or 32 keys (dk and dv).  Four share a tile's way into LDS; with two, the keys (rows) that a workgroup
// walks reach less beyond its own and float32 needs fewer registers for tiles on their way.  Measured, us with four / two waves:
//   rows, bf16 forward, 8 x 4096 tokens, keys in reach 64 / 128 / 256 / 512: 8 heads of 64: 34, 34, 43, 63 / 31, 35, 45, 67; 16 of 128 over 4: 115, 125, 151, 209 /
//   119, 132, 160, 226.  What two gain at a reach of 64 with as many key heads they lose elsewhere, so 16-bit rows take four.  float32 4 x 2048 x 8 of 64 and
//   128, window 256: 64 / 60 and 142 / 127.
//   keys, dk and dv: float32, the same two: 209 / 184 and 454 / 447; fp16 8 x 4096 x 8 of 96 with 64 keys either side 122 / 103; bf16 4 x 2048 x 16 of 64, all
//   keys: 193 / 236.
constexpr int row_waves(int es) { return es == 4 ? 2 : 4; }
static inline int key_waves(int es, long reach) { return es == 4 || reach < 256 ? 2 : 4; }

// 16-bit training passes over few (query, key) pairs multiply weights and dS as the sum of their rounding and the rest's.  Rounded once, dS adds as much to
// the error of dq and dk as their own rounding does (1.41 times it together) where many pairs average out; up to 1.53 times it was seen below 2^22
// pairs, and 1.97 for sequences of two or three tokens.  The second part costs 1.0 and 1.6 us (dq 8.0, dk and dv 9.8) at 2^20 pairs, 32 wide, 1.5 and 2.3 us
// of 13 at 2^22, 64 wide; at 2^24 it would be 2.9 of 20.7 and 4.7 of 31.4, where it gains nothing.
static inline bool few_pairs(long heads, long n, long m, long reach) { return heads * n * (m < reach ? m : reach) <= (1l << 22); }

// waves on a SIMD that the registers are held down to
template <typename T, int DT> constexpr int waves_per_simd() { return sizeof(T) == 2 ? 2 : DT <= 32 ? 3 : DT <= 64 ? 2 : 1; }

// Keys of a tile of the kernels that own rows: two-wave workgroups with 64 keys would fill the LDS before the registers (float32 18 x 1024, 8 heads of 32,
// 128 keys either side: forward 88 us, dq 121; with 32 keys 76 and 109).
template <typename T, int DT, int NW> constexpr int key_tile() { return NW == 2 ? 32 : 64; }

// a launch holds fewer than 2^32 threads along a dimension
static inline bool launchable(long workgroups, int threads) { return workgroups < (1l << 32) / threads; }

static inline int width(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : 128; }      // padded head width

}  // namespace pa_attn

// argument checks that forward and backward share
static inline int window_attention_check(const char *name, int dtype, int b, int n, int m, int h, int hk, int d, int left, int right, int sinks, float scale)
{
    PA_REQUIRE(dtype >= PA_DT_F32 && dtype <= PA_DT_BF16, "%s: dtype %d is none of 0 (float32), 1 (float16), 2 (bfloat16)", name, dtype);
    PA_REQUIRE(b >= 0 && n >= 0 && m >= 0 && n <= pa_attn::MAXLEN && m <= pa_attn::MAXLEN, "%s: bad sizes b=%d n=%d m=%d (up to 2^28 tokens)", name, b, n, m);
    PA_REQUIRE(h > 0 && hk > 0 && h % hk == 0, "%s: %d query heads do not share %d key heads evenly", name, h, hk);
    PA_REQUIRE((long)n * (h / hk) <= pa_attn::UNBOUNDED, "%s: n (h / hk) = %ld rows exceed 2^29", name, (long)n * (h / hk));
    PA_REQUIRE(d > 0 && d <= 128 && d % 8 == 0, "%s: head width %d is not a multiple of 8 up to 128", name, d);
    PA_REQUIRE(left >= -1 && right >= -1 && left <= pa_attn::MAXLEN && right <= pa_attn::MAXLEN && sinks >= 0, "%s: bad window left=%d right=%d sinks=%d", name, left,
               right, sinks);
    PA_REQUIRE(scale > 0.f && scale <= 0x1p127f, "%s: the scale has to be in (0, 2^127]", name);
    return PA_OK;
}

// largest power of two up to 16 that divides every address and every stride (in bytes)
static inline long alignment_of(int es, std::initializer_list<const void *> ps, std::initializer_list<long> ss)
{
    unsigned long m = 16;
    for (const void *p : ps) m |= (unsigned long)(uintptr_t)p;
    for (long s : ss) m |= (unsigned long)(s * es);
    return (long)(m & -m);
}

// a tile's rows are addressed by 32-bit offsets: 64 tokens and 64 heads of 4-byte elements stay below 2^32 bytes
constexpr long PA_ATTN_MAXSTRIDE = 1l << 22;

// element type and padded head width as template arguments of F: runs F(T, DT)
#define PA_ATTN_WIDTH(T, d, F)                                                  \
    do {                                                                        \
        if ((d) <= 32) { F(T, 32); }                                            \
        else if ((d) <= 64) { F(T, 64); }                                       \
        else if ((d) <= 96) { F(T, 96); }                                       \
        else { F(T, 128); }                                                     \
    } while (0)
#define PA_ATTN_DISPATCH(dtype, d, F)                                           \
    do {                                                                        \
        if ((dtype) == PA_DT_F32) PA_ATTN_WIDTH(float, d, F);                   \
        else if ((dtype) == PA_DT_F16) PA_ATTN_WIDTH(_Float16, d, F);           \
        else PA_ATTN_WIDTH(__bf16, d, F);                                       \
    } while (0)
