// Attention of one new token per sequence over a paged key / value cache, and the writes into that cache.
//
//     o_h = softmax_j(scale q_h . k_j) v_j  over the keys in view of the last position p = len - 1:  j >= p - left or j < sinks
//
// Key j of sequence b lies in page table[b][j / page] at row j % page.  An entry outside the pool holds no keys (they are left out like keys out of
// view), so pages behind the window may be taken away and marked -1.
//
// Every visible row of K and V is read once, which is the bound (HBM).  The cache of a (sequence, key head) is cut into runs of TPC tiles of 32 keys,
// one workgroup each; a workgroup's four waves take its tiles in turn and never wait for each other until the end: a wave has one row of keys per
// lane pair straight from memory as the operand of S^T = K Q^T (Q: the heads that share the key head, up to 32 rows), and V goes through 32 rows of
// LDS of its own to be read transposed.  The next tile is requested before the present one is used.  Waves join in LDS, runs in a second launch --
// none when one run covers the cache.
//
// Measured: 48 sequences of 4096 to 16384 tokens, 32 heads of 128 over 8, bf16, pages of 64: 381 + 7 us for 1.95 GB = 5.0 TB/s (a 2 GiB copy: 4.9, read and
// written).  With one wave per SIMD (290 registers) and a branch around every load it was 525 us.  100 tokens, 8 heads of 64 over 2: 5.3 us, one launch.
// float32, 24 of them: 473 + 8 us = 4.1 TB/s (208 registers and four tiles of 16 KB in LDS: one wave per SIMD).
// P is rounded to the type of V for the second product (16-bit types), relative to a running maximum as in the forward pass: out is off by 1.2 to 1.45 times its own
// rounding.
// append: 16 prompts of up to 2048 tokens, 8 heads of 128: 147 MB in 25 us = 5.9 TB/s; one token of 32 sequences 3.2 us.
#include "pa_attn.h"

using namespace pa_attn;

namespace {

constexpr int KT = 32;

struct PagedArgs {
    const void *q, *k, *v;
    const int *table, *length;
    void *out;
    float *part;
    long qb, qh, kp, kt, kh, vp, vt, vh, tb;
    int B, H, Hk, D, G, ngt, pages, page, cap, left, sinks, tpc, runs;
    float c;
    Div pg;
};

__device__ __forceinline__ View view_of(const PagedArgs &a)
{
    View v;
    v.m = a.cap; v.left = a.left; v.right = 0; v.sinks = a.sinks; v.start = nullptr; v.length = a.length;
    return v;
}

template <typename T, int DT>
__global__ __launch_bounds__(256, (waves_per_simd<T, DT>())) void paged_kernel(const PagedArgs a)
{
    typedef Tile<T, DT> L;
    typedef typename Frag<T>::type F;
    constexpr int NK = DT / 16, NP = (int)sizeof(T) / 2;       // fragments of a row, 16-byte pieces of a fragment
    extern __shared__ __attribute__((aligned(16))) char smem[];      // [4] V tile of a wave; then the join
    const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63, h = l >> 5;
    const int gt = blockIdx.x % a.ngt, bh = blockIdx.x / a.ngt, b = bh / a.Hk, hk = bh - b * a.Hk;
    const View view = view_of(a);
    const int len = view.len(b);
    const TileList<KT> tiles(view, len - 1, len - 1, len);     // none when the sequence is empty
    const int t0 = blockIdx.y * a.tpc, t1 = min(t0 + a.tpc, tiles.n);
    if (t0 >= t1 && a.runs > 1) return;                        // nothing in this run: the join knows

    const int g = gt * 32 + (l & 31);                          // this lane's head of the group
    F qf[NK];
    {
        const T *qp = (const T *)a.q + b * a.qb + (hk * a.G + min(g, a.G - 1)) * a.qh;
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) qf[kk] = ldrow<T>(qp, kk, h, a.D, g < a.G);
    }
    const int lo = max(len - 1 - a.left, 0);
    const T *kbase = (const T *)a.k + hk * a.kh, *vbase = (const T *)a.v + hk * a.vh;
    const int *table = a.table + b * a.tb;
    F kf[NK];
    pa_u4 pv[NK * NP];
    u32 mask = 0;
    auto fetch = [&](int t) __attribute__((always_inline)) {
        const int j = tiles.tile(t) * KT + (l & 31);
        bool ok = j < len && (j >= lo || j < a.sinks);
        int page = 0, at = 0;
        if (ok) {
            const int e = a.pg.div(j);
            at = j - e * a.page;
            page = table[e];
            ok = (u32)page < (u32)a.pages;
        }
        mask = (u32)__ballot(ok);
        const T *kr = kbase + (long)page * a.kp + (long)at * a.kt, *vr = vbase + (long)page * a.vp + (long)at * a.vt;
        if (mask == 0xffffffffu && a.D == DT) {                 // the rule: no lane leaves anything out
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) kf[kk] = ldrow<T>(kr, kk, h, DT, true);
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
#pragma unroll
                for (int u = 0; u < NP; ++u) pv[kk * NP + u] = *reinterpret_cast<const pa_u4 *>(vr + 16 * kk + 8 * h + u * L::EC);
            return;
        }
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) kf[kk] = ldrow<T>(kr, kk, h, a.D, ok);
#pragma unroll
        for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int u = 0; u < NP; ++u) {
                const int e0 = 16 * kk + 8 * h + u * L::EC;
                pv[kk * NP + u] = ldg16(vr + e0, ok && e0 < a.D);
            }
    };

    pa_f16v o[DT / 32];
#pragma unroll
    for (int ct = 0; ct < DT / 32; ++ct) o[ct] = (pa_f16v)(0.f);
    float m_run = -INFINITY, l_run = 0.f;
    char *vs = smem + wave * KT * L::RB;

    if (t0 + wave < t1) fetch(t0 + wave);
    for (int t = t0 + wave; t < t1; t += 4) {
#pragma unroll
        for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int u = 0; u < NP; ++u) *reinterpret_cast<pa_u4 *>(vs + L::at(l & 31, (2 * kk + h) * NP + u)) = pv[kk * NP + u];
        pa_f16v s = (pa_f16v)(0.f);
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) mma(s, kf[kk], qf[kk]);
        const u32 seen = mask;
        if (t + 4 < t1) fetch(t + 4);
        if (seen != 0xffffffffu) {
            const u32 mine = seen >> (4 * h);
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = (mine >> (8 * (r >> 2) + (r & 3))) & 1 ? s[r] : -INFINITY;
        }
        float mt = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) mt = larger(mt, s[r]);
        mt = larger(mt, other_half(mt)) * a.c;
        if (__any(mt > m_run + 8.f)) {
            const float mn = fmaxf(m_run, mt), sc = mn > -INFINITY ? ex2(m_run - mn) : 0.f;
#pragma unroll
            for (int ct = 0; ct < DT / 32; ++ct)
#pragma unroll
                for (int r = 0; r < 16; ++r) o[ct][r] *= sc;
            l_run *= sc;
            m_run = mn;
        }
        const float mref = m_run > -INFINITY ? m_run : 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = ex2(__builtin_fmaf(s[r], a.c, -mref));
            l_run += s[r];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront"); // the wave's own stores above; LDS serves one wave in order
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const F p = pack<T>(s, u);
#pragma unroll
            for (int ct = 0; ct < DT / 32; ++ct) mma(o[ct], L::ldt(vs, 16 * u, ct * 32), p);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    l_run += other_half(l_run);

    // the four waves: common maximum, then one after the other adds its rows
    float *ob = reinterpret_cast<float *>(smem), *mb = ob + 32 * (DT + 4);       // [32][DT + 4] sums, [4][32] maxima, [4][32] sums of weights
    __syncthreads();
    if (h == 0) {
        mb[wave * 32 + l] = m_run;
        mb[128 + wave * 32 + l] = l_run;
    }
    __syncthreads();
    float m = -INFINITY, lt = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, mb[w * 32 + (l & 31)]);
    const float mref = m > -INFINITY ? m : 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) lt += ex2(mb[w * 32 + (l & 31)] - mref) * mb[128 + w * 32 + (l & 31)];
    const float sc = ex2(m_run - mref);
    for (int w = 0; w < 4; ++w) {
        if (wave == w && g < a.G) {
#pragma unroll
            for (int ct = 0; ct < DT / 32; ++ct)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    pa_f4 *p = reinterpret_cast<pa_f4 *>(ob + (l & 31) * (DT + 4) + ct * 32 + 8 * u + 4 * h);
                    pa_f4 x = (pa_f4){o[ct][4 * u] * sc, o[ct][4 * u + 1] * sc, o[ct][4 * u + 2] * sc, o[ct][4 * u + 3] * sc};
                    if (w > 0) x += *p;
                    *p = x;
                }
        }
        __syncthreads();
    }
    const int ng = min(32, a.G - gt * 32);
    if (a.runs > 1) {
        const size_t all = (size_t)a.B * a.H, row = (size_t)b * a.H + hk * a.G + gt * 32;
        float *po = a.part + ((size_t)blockIdx.y * all + row) * DT, *pm = a.part + (size_t)a.runs * all * DT + ((size_t)blockIdx.y * all + row) * 2;
        for (int i = tid; i < ng * (DT / 4); i += 256) {
            const int r = i / (DT / 4), c = (i - r * (DT / 4)) * 4;
            *reinterpret_cast<pa_f4 *>(po + (size_t)r * DT + c) = *reinterpret_cast<const pa_f4 *>(ob + r * (DT + 4) + c);
        }
        if (wave == 0 && l < ng) {
            pm[l * 2] = m;
            pm[l * 2 + 1] = lt;
        }
        return;
    }
    __syncthreads();
    if (wave == 0 && h == 0) mb[l] = lt;
    __syncthreads();
    for (int i = tid; i < ng * (a.D / 4); i += 256) {
        const int r = i / (a.D / 4), c = (i - r * (a.D / 4)) * 4;
        const float t = mb[r], inv = t != 0.f ? 1.0f / t : 0.f;
        const pa_f4 x = *reinterpret_cast<const pa_f4 *>(ob + r * (DT + 4) + c);
        st4<T>((T *)a.out + ((size_t)b * a.H + hk * a.G + gt * 32 + r) * a.D + c, x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
    }
}

// the runs of a row
template <typename T, int DT>
__global__ __launch_bounds__(256) void paged_join_kernel(const PagedArgs a)
{
    constexpr int TR = DT / 4;
    const size_t all = (size_t)a.B * a.H;
    const size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) / TR;
    const int c = (int)(((size_t)blockIdx.x * 256 + threadIdx.x) % TR) * 4;
    if (at >= all) return;
    const int b = (int)(at / a.H);
    const View view = view_of(a);
    const int len = view.len(b);
    const TileList<KT> tiles(view, len - 1, len - 1, len);
    const int runs = (tiles.n + a.tpc - 1) / a.tpc;
    const float *pm = a.part + (size_t)a.runs * all * DT;
    float m = -INFINITY, l = 0.f;
#pragma unroll 8
    for (int s = 0; s < runs; ++s) m = fmaxf(m, pm[(s * all + at) * 2]);
    const float mref = m > -INFINITY ? m : 0.f;
    pa_f4 o = (pa_f4)(0.f);
#pragma unroll 8
    for (int s = 0; s < runs; ++s) {
        const float w = ex2(pm[(s * all + at) * 2] - mref);
        l += w * pm[(s * all + at) * 2 + 1];
        o += w * *reinterpret_cast<const pa_f4 *>(a.part + (s * all + at) * DT + c);
    }
    const float inv = l != 0.f ? 1.0f / l : 0.f;
    if (c < a.D) st4<T>((T *)a.out + at * a.D + c, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
}

struct Runs {
    int tpc, runs;
};

// Tiles per workgroup.  About 2048 workgroups (eight per CU, for lengths that differ) but at least 8 tiles each (two per wave): shorter runs cost more
// in joins than they gain.  A cache of up to 16 tiles is one run, one launch.
Runs runs_of(int B, int Hk, int G, int cap, int left, int sinks)
{
    const long whole = pa_div_up(cap, KT), near = pa_div_up((long)left + 1, KT) + 1 + pa_div_up(sinks, KT);
    const long tiles = whole < near ? whole : near;            // most tiles of a sequence
    Runs r;
    if (tiles <= 16) {
        r.tpc = tiles > 0 ? (int)tiles : 1;
        r.runs = 1;
        return r;
    }
    long per = tiles * B * Hk * pa_div_up(G, 32) / 2048;
    per = per < 8 ? 8 : (per + 3) / 4 * 4;
    if (pa_div_up(tiles, per) > 65535) per = pa_div_up(tiles, 65535);
    r.tpc = (int)(per < tiles ? per : tiles);
    r.runs = pa_div_up(tiles, r.tpc);
    return r;
}

template <typename T, int DT>
int launch_paged(const PagedArgs &a, hipStream_t st)
{
    constexpr int lv = 4 * KT * DT * (int)sizeof(T), lj = (32 * (DT + 4) + 256) * 4, lds = lv > lj ? lv : lj;
    hipLaunchKernelGGL((paged_kernel<T, DT>), dim3((unsigned)((long)a.B * a.Hk * a.ngt), (unsigned)a.runs), dim3(256), lds, st, a);
    if (a.runs > 1) {
        const long threads = (long)a.B * a.H * (DT / 4);
        hipLaunchKernelGGL((paged_join_kernel<T, DT>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a);
    }
    return 0;
}

// A thread copies 16 bytes of a new row of K and of V, pieces first .. total of all.
__global__ __launch_bounds__(256) void append_kernel(long first, long total, int tokens, int hk, int chunks, int es, const char *__restrict__ k, const char *__restrict__ v, long kb,
                                                     long kn, long kh, long vb, long vn, long vh, char *__restrict__ kpages, char *__restrict__ vpages, long kp,
                                                     long kt, long kph, long vp, long vt, long vph, const int *__restrict__ table, long tb, int pages, int page,
                                                     int cap, const int *__restrict__ starts, const int *__restrict__ counts)
{
    const long id = first + (long)blockIdx.x * 256 + threadIdx.x;
    if (id >= total) return;
    const int c = (int)(id % chunks);
    const long rest = id / chunks;
    const int g = (int)(rest % hk), t = (int)(rest / hk % tokens), b = (int)(rest / hk / tokens);
    const long j = (long)starts[b] + t;
    if ((counts && t >= counts[b]) || j < 0 || j >= cap) return;
    const int e = (int)j / page, at = (int)j - e * page, p = table[b * tb + e];
    if ((u32)p >= (u32)pages) return;
    *reinterpret_cast<pa_u4 *>(kpages + (p * kp + at * kt + g * kph) * es + c * 16) = *reinterpret_cast<const pa_u4 *>(k + (b * kb + t * kn + g * kh) * es + c * 16);
    *reinterpret_cast<pa_u4 *>(vpages + (p * vp + at * vt + g * vph) * es + c * 16) = *reinterpret_cast<const pa_u4 *>(v + (b * vb + t * vn + g * vh) * es + c * 16);
}

int paged_check(const char *name, int dtype, int b, int hk, int d, int pages, int page, int width)
{
    PA_REQUIRE(dtype >= PA_DT_F32 && dtype <= PA_DT_BF16, "%s: dtype %d is none of 0 (float32), 1 (float16), 2 (bfloat16)", name, dtype);
    PA_REQUIRE(b >= 0 && hk > 0 && pages >= 0 && page > 0 && width >= 0, "%s: bad sizes b=%d hk=%d pages=%d page=%d width=%d", name, b, hk, pages, page, width);
    PA_REQUIRE(d > 0 && d <= 128 && d % 8 == 0, "%s: head width %d is not a multiple of 8 up to 128", name, d);
    PA_REQUIRE((long)width * page <= MAXLEN, "%s: a table of %d pages of %d tokens exceeds 2^28 tokens", name, width, page);
    return PA_OK;
}

}  // namespace

PA_API long pa_paged_attention_scratch_floats(int b, int h, int hk, int d, int page, int width_, int left, int sinks)
{
    if (b <= 0 || h <= 0 || hk <= 0 || h % hk != 0 || page <= 0 || width_ < 0 || sinks < 0) return 0;
    const int cap = (int)((long)width_ * page > MAXLEN ? MAXLEN : (long)width_ * page);
    const Runs r = runs_of(b, hk, h / hk, cap, left < 0 ? UNBOUNDED : left, sinks < cap ? sinks : cap);
    return r.runs <= 1 ? 0 : (long)r.runs * b * h * (width(d) + 2);
}

PA_API int pa_paged_attention(int dtype, int b, int h, int hk, int d, const void *q, long qb, long qh, const void *k_pages, long kp, long kt, long kh,
                              const void *v_pages, long vp, long vt, long vh, int pages, int page, const int *table, int width_, const int *length, int left,
                              int sinks, float scale, void *out, float *scratch, pa_stream_t stream)
{
    int rc = paged_check("pa_paged_attention", dtype, b, hk, d, pages, page, width_);
    if (rc != PA_OK) return rc;
    PA_REQUIRE(h > 0 && h % hk == 0, "pa_paged_attention: %d query heads do not share %d key heads evenly", h, hk);
    PA_REQUIRE(left >= -1 && left <= MAXLEN && sinks >= 0, "pa_paged_attention: bad window left=%d sinks=%d", left, sinks);
    PA_REQUIRE(scale > 0.f && scale <= 0x1p127f, "pa_paged_attention: the scale has to be in (0, 2^127]");
    if (b == 0) return PA_OK;
    PA_REQUIRE(q && out && length && (width_ == 0 || table) && (pages == 0 || (k_pages && v_pages)), "pa_paged_attention: null tensor");
    PA_REQUIRE(alignment_of(dtype == PA_DT_F32 ? 4 : 2, {q, k_pages, v_pages, out, scratch}, {qb, qh, kp, kt, kh, vp, vt, vh}) == 16,
               "pa_paged_attention: addresses and strides have to be multiples of 16 bytes");
    PagedArgs a;
    a.q = q; a.k = k_pages; a.v = v_pages; a.table = table; a.length = length; a.out = out; a.part = scratch;
    a.qb = qb; a.qh = qh; a.kp = kp; a.kt = kt; a.kh = kh; a.vp = vp; a.vt = vt; a.vh = vh; a.tb = width_;
    a.B = b; a.H = h; a.Hk = hk; a.D = d; a.G = h / hk; a.ngt = pa_div_up(a.G, 32);
    a.pages = pages; a.page = page; a.cap = width_ * page;
    a.left = left < 0 ? UNBOUNDED : left;
    a.sinks = sinks < a.cap ? sinks : a.cap;
    a.c = scale * 1.4426950408889634f;
    a.pg = Div(page);
    const Runs r = runs_of(b, hk, a.G, a.cap, a.left, a.sinks);
    a.tpc = r.tpc;
    a.runs = r.runs;
    PA_REQUIRE(launchable((long)b * hk * a.ngt, 256) && launchable(((long)b * h * (width(d) / 4) + 255) / 256, 256), "pa_paged_attention: too many workgroups");
    PA_REQUIRE(a.runs == 1 || scratch, "pa_paged_attention: this size needs pa_paged_attention_scratch_floats() of scratch");
    hipStream_t st = (hipStream_t)stream;
#define PAGED(T, DT) launch_paged<T, DT>(a, st)
    PA_ATTN_DISPATCH(dtype, d, PAGED);
#undef PAGED
    PA_CHECK_LAUNCH("pa_paged_attention");
    return PA_OK;
}

PA_API int pa_paged_append(int dtype, int b, int tokens, int hk, int d, const void *k, long kb, long kn, long kh, const void *v, long vb, long vn, long vh,
                           void *k_pages, long kp, long kt, long kph, void *v_pages, long vp, long vt, long vph, int pages, int page, const int *table, int width_,
                           const int *starts, const int *counts, pa_stream_t stream)
{
    int rc = paged_check("pa_paged_append", dtype, b, hk, d, pages, page, width_);
    if (rc != PA_OK) return rc;
    PA_REQUIRE(tokens >= 0, "pa_paged_append: %d tokens", tokens);
    if (b == 0 || tokens == 0 || pages == 0 || width_ == 0) return PA_OK;
    PA_REQUIRE(k && v && k_pages && v_pages && table && starts, "pa_paged_append: null tensor");
    const int es = dtype == PA_DT_F32 ? 4 : 2, chunks = d * es / 16;
    PA_REQUIRE(alignment_of(es, {k, v, k_pages, v_pages}, {kb, kn, kh, vb, vn, vh, kp, kt, kph, vp, vt, vph}) == 16,
               "pa_paged_append: addresses and strides have to be multiples of 16 bytes");
    const long total = (long)b * tokens * hk * chunks;
    constexpr long most = 1l << 31;                            // pieces of a launch
    for (long first = 0; first < total; first += most) {
        const long n = total - first < most ? total - first : most;
        hipLaunchKernelGGL(append_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream, first, total, tokens, hk, chunks, es, (const char *)k,
                           (const char *)v, kb, kn, kh, vb, vn, vh, (char *)k_pages, (char *)v_pages, kp, kt, kph, vp, vt, vph, table, (long)width_, pages, page,
                           width_ * page, starts, counts);
    }
    PA_CHECK_LAUNCH("pa_paged_append");
    return PA_OK;
}
