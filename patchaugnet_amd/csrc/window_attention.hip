// Attention with a sliding window and a few first tokens that stay in view, forward.
//
//     o_i = sum_j P_ij v_j,   P_ij = exp(s_ij) / sum_j exp(s_ij),   s_ij = scale q_i . k_j   over the keys j in view of row i (View, pa_attn.h)
//
// One pass over the keys with a running maximum and sum: O(window) work and nothing N x M in memory.  A workgroup owns 128 (float32: 64) rows -- the N
// queries of the G heads that share a key head, query-major, so that one tile of keys serves all of them -- and walks the tiles of 64 (32) keys that its rows can
// see: the tiles of the first tokens, then one contiguous range.  A wave owns 32 rows.  S^T = K Q^T puts one row into a lane's registers (maximum and
// sum need one exchange between the two half waves), and the registers of P^T feed O^T += V^T P^T without leaving the lane; V is read transposed
// from LDS.  Tiles go straight from memory into the other half of a double buffer while the present one is used, one barrier a tile.
//
// Roundings: s, maximum, sum and o are 32-bit; P is rounded to the type of V for the second product (16-bit types), with P <= 2^8 by the running
// maximum, which is only moved when a row's maximum grows by more than 2^8 (the quotient is the same for any reference value).  Where a backward pass
// follows, its delta is a difference that magnifies the error of o: what the rounding of o leaves is handed on beside it, and for heads of 8 and 16 (their
// dq is off by up to 1.58 times the rounding of the result, wider heads' by 1.5) and few pairs (few_pairs()) P is multiplied as the sum of its rounding and
// the rest's -- without gradients too, so that out has the same bits with and without.  4 x 4096 tokens, 16 heads over 4 in a tile 32 wide, window 512:
// 45 us, in two parts 60.
//
// Measured: bf16 4 x 16384 tokens, 16 heads of 128 over 4, window 1024: 665 us = 805 TFLOP/s of visible pairs (a library product of that type: 1219;
// 12 % of the work is keys of tiles that a row does not see); 4 x 4096, 16 heads of 64 over 4, window 512: 60 us = 540 (68 with what the rounding of out
// leaves, for a backward pass); all keys of 4 x 2048, 16 heads of 64: 91 us = 755.
// Bound, by counters: matrix and vector work of the two waves of a SIMD mostly follow one another.  Width 128, window 1024: matrix units busy 39 % of the
// time, vector units 46 %, LDS 20 % and free of bank conflicts, 1.9 waves per SIMD; 133 vector and 59 scalar instructions for a 32 x 32 part of 16 MFMA.
// Width 64, window 512: vector 50 %, matrix 21 %, LDS 10 %; 136 vector and 66 scalar instructions for a part of 8 MFMA.  Reading ahead by one product
// within a wave (scores of the next part beside the exponentials of this one) cost more in registers than it hid (80 against 65 us at width 64).
// float32 72 x 1024, 8 heads of 64, all keys: 1245 us = 124 of the 153 TFLOP/s of a library product; 18 x 1024, 8 heads of 32, 128 keys either side: 76 us =
// 60: a quarter of the keys in its parts are out of view, and it is 4.5 waves per SIMD in all, whose start and end nothing covers (matrix units busy 45 %,
// vector 17 %, LDS 4 %).
#include "pa_attn.h"

using namespace pa_attn;

namespace {

struct FwdArgs {
    const void *q, *k, *v;
    void *out, *low;
    float *lse, *part;
    long qb, qn, qh, kb, kn, kh, vb, vn, vh;
    int B, N, H, Hk, D, G, splits, nqt;
    bool few;
    float c;                  // scale log2(e)
    View view;
    Div g;
};

// four elements of the output and, for the backward pass, what their rounding left
template <typename T> __device__ __forceinline__ void store_out(T *out, T *low, pa_f4 x)
{
    st4<T>(out, x[0], x[1], x[2], x[3]);
    if (low) st4<T>(low, x[0] - (float)(T)x[0], x[1] - (float)(T)x[1], x[2] - (float)(T)x[2], x[3] - (float)(T)x[3]);
}

// FINE: the product with V takes P in two parts
template <typename T, int DT, int NW, bool SPLIT, bool FINE>
__global__ __launch_bounds__(64 * NW, (waves_per_simd<T, DT>())) void fwd_kernel(const FwdArgs a)
{
    typedef Tile<T, DT> L;
    typedef typename Frag<T>::type F;
    constexpr int KT = key_tile<T, DT, NW>(), TB = KT * L::RB, QT = 32 * NW;
    __shared__ __attribute__((aligned(16))) char k0[TB], k1[TB], v0[TB], v1[TB];       // apart, so that loads into one hold up no reads of another
    const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63, h = l >> 5;

    const int item = (int)xcd_item(blockIdx.x, gridDim.x);
    const int qt = item % a.nqt, bh = item / a.nqt, b = bh / a.Hk, hk = bh - b * a.Hk;
    const int rows = a.N * a.G, len = a.view.len(b), start = a.view.first(b);
    const int r0 = qt * QT;
    const TileList<KT> tiles(a.view, start + a.g.div(r0), start + a.g.div(min(r0 + QT, rows) - 1), len);
    int t0 = 0, t1 = tiles.n;
    if (SPLIT) {
        t0 = (int)((long)tiles.n * blockIdx.y / a.splits);
        t1 = (int)((long)tiles.n * (blockIdx.y + 1) / a.splits);
    }

    // this lane's row
    const int row = r0 + wave * 32 + (l & 31), i = a.g.div(min(row, rows - 1)), hq = hk * a.G + min(row, rows - 1) - i * a.G;
    const Keys keys(a.view, start + i, len, row < rows);
    F qf[DT / 16];
    {
        const T *qp = (const T *)a.q + b * a.qb + i * a.qn + hq * a.qh;
#pragma unroll
        for (int kk = 0; kk < DT / 16; ++kk) qf[kk] = ldrow<T>(qp, kk, h, a.D, keys.ok);        // padding rows are zeros
    }
    // the wave's rows: positions of the first and of the last one that is not padding
    const int wr = __builtin_amdgcn_readfirstlane(r0 + wave * 32);
    const int wp0 = start + a.g.div(min(wr, rows - 1)), wp1 = min(start + a.g.div(min(wr + 31, rows - 1)), len - 1);
    const bool wave_on = wr < rows && wp0 < len;
    const int wlo = max(wp0 - a.view.left, 0), whi = min(wp1 + a.view.right, len - 1);                  // some row sees [wlo, whi]
    const int flo = max(wp1 - a.view.left, 0), fhi = min(wp0 + a.view.right, len - 1);                  // every row sees [flo, fhi]

    const T *kp = (const T *)a.k + b * a.kb + hk * a.kh, *vp = (const T *)a.v + b * a.vb + hk * a.vh;
    Direct<T, DT, KT, 64 * NW> sk, sv;
    sk.strided(a.kn);
    sv.strided(a.vn);
    auto fetch = [&](int t, char *ks, char *vs) __attribute__((always_inline)) {              // rows behind the sequence are zeros: what they hold never meets a product
        sk.fetch(ks, kp + (long)t * KT * a.kn, len - t * KT, a.D);
        sv.fetch(vs, vp + (long)t * KT * a.vn, len - t * KT, a.D);
    };

    pa_f16v o[DT / 32];
#pragma unroll
    for (int ct = 0; ct < DT / 32; ++ct) o[ct] = (pa_f16v)(0.f);
    float m_run = -INFINITY, l_run = 0.f;

    if (t0 < t1) fetch(tiles.tile(t0), k0, v0);
    auto step = [&](int it, char *ks, char *vs, char *kn, char *vn) __attribute__((always_inline)) {
        arrived();
        __syncthreads();                                       // the tile is there, and everyone is done with the one before it
        const int j0 = tiles.tile(it) * KT;
        if (it + 1 < t1) fetch(tiles.tile(it + 1), kn, vn);
        if (!wave_on) return;
#pragma unroll
        for (int sub = 0; sub < KT / 32; ++sub) {
            const int js = j0 + sub * 32;
            if (!((js <= whi && js + 31 >= wlo) || js < min(a.view.sinks, whi + 1))) continue;
            pa_f16v s = (pa_f16v)(0.f);
#pragma unroll
            for (int kk = 0; kk < DT / 16; ++kk) mma(s, L::ld(ks, sub * 32, kk), qf[kk]);
            if (!(js >= flo && js + 31 <= fhi)) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = keys.sees(js + 8 * (r >> 2) + 4 * h + (r & 3)) ? s[r] : -INFINITY;
            }
            float mt = s[0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mt = larger(mt, s[r]);
            mt = larger(mt, other_half(mt)) * a.c;
            if (__any(mt > m_run + 8.f)) {                     // -inf + 8 = -inf: the first visible key of a row always moves it
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
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const F p = pack<T>(s, u);
                F rest;
                if constexpr (FINE) rest = pack_rest<T>(s, p, u);
#pragma unroll
                for (int ct = 0; ct < DT / 32; ++ct) {
                    const F v = L::ldt(vs, sub * 32 + 16 * u, ct * 32);
                    mma(o[ct], v, p);
                    if constexpr (FINE) mma(o[ct], v, rest);
                }
            }
        }
    };
    for (int it = t0; it < t1; it += 2) {                      // two halves of LDS, two copies of the step: places in LDS are constants
        step(it, k0, v0, k1, v1);
        if (it + 1 < t1) step(it + 1, k1, v1, k0, v0);
    }

    l_run += other_half(l_run);
    if (row >= rows) return;
    if (SPLIT) {
        const size_t all = (size_t)a.B * a.Hk * rows, at = (size_t)blockIdx.y * all + (size_t)bh * rows + row;
        float *po = a.part + at * DT, *pm = a.part + (size_t)a.splits * all * DT + at * 2;
#pragma unroll
        for (int ct = 0; ct < DT / 32; ++ct)
#pragma unroll
            for (int u = 0; u < 4; ++u)
                *reinterpret_cast<pa_f4 *>(po + ct * 32 + 8 * u + 4 * h) = (pa_f4){o[ct][4 * u], o[ct][4 * u + 1], o[ct][4 * u + 2], o[ct][4 * u + 3]};
        if (h == 0) {
            pm[0] = m_run;
            pm[1] = l_run;
        }
        return;
    }
    const bool some = keys.ok && l_run != 0.f;                 // padding rows take part where their wave's other rows see everything: 0, whatever came out
    const float inv = 1.0f / l_run;
    const size_t place = (((size_t)b * a.N + i) * a.H + hq) * a.D;
    T *op = (T *)a.out + place, *low = a.low ? (T *)a.low + place : nullptr;
#pragma unroll
    for (int ct = 0; ct < DT / 32; ++ct)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int c = ct * 32 + 8 * u + 4 * h;
            pa_f4 x = (pa_f4)(0.f);
            if (some) x = (pa_f4){o[ct][4 * u] * inv, o[ct][4 * u + 1] * inv, o[ct][4 * u + 2] * inv, o[ct][4 * u + 3] * inv};
            if (c < a.D) store_out<T>(op + c, low ? low + c : nullptr, x);
        }
    if (a.lse && h == 0) a.lse[((size_t)b * a.H + hq) * a.N + i] = some ? m_run + __builtin_amdgcn_logf(l_run) : INFINITY;
}

// The rows of a split launch: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s.  A thread owns four elements of a row.
template <typename T, int DT>
__global__ __launch_bounds__(256) void join_kernel(const FwdArgs a)
{
    constexpr int TR = DT / 4;
    const int rows = a.N * a.G;
    const size_t all = (size_t)a.B * a.Hk * rows;
    const size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) / TR;
    const int c = (int)(((size_t)blockIdx.x * 256 + threadIdx.x) % TR) * 4;
    if (at >= all) return;
    const float *pm = a.part + (size_t)a.splits * all * DT;
    float m = -INFINITY, l = 0.f;
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, pm[(s * all + at) * 2]);
    const float mref = m > -INFINITY ? m : 0.f;
    pa_f4 o = (pa_f4)(0.f);
#pragma unroll 8
    for (int s = 0; s < a.splits; ++s) {
        const float w = ex2(pm[(s * all + at) * 2] - mref);
        l += w * pm[(s * all + at) * 2 + 1];
        o += w * *reinterpret_cast<const pa_f4 *>(a.part + (s * all + at) * DT + c);
    }
    const int bh = (int)(at / rows), row = (int)(at - (size_t)bh * rows), b = bh / a.Hk, hk = bh - b * a.Hk;
    const int i = a.g.div(row), hq = hk * a.G + row - i * a.G;
    const bool some = a.view.first(b) + i < a.view.len(b) && l != 0.f;      // padding rows: 0
    if (some) o *= 1.0f / l;
    else o = (pa_f4)(0.f);
    const size_t place = (((size_t)b * a.N + i) * a.H + hq) * a.D + c;
    if (c < a.D) store_out<T>((T *)a.out + place, a.low ? (T *)a.low + place : nullptr, o);
    if (a.lse && c == 0) a.lse[((size_t)b * a.H + hq) * a.N + i] = some ? m + __builtin_amdgcn_logf(l) : INFINITY;
}

struct Shape {
    int waves, nqt, splits;
};

// Work is split over the keys when the rows alone leave the chip idle: fewer than 256 workgroups (one per CU).  Two per CU are aimed at, each with
// at least four tiles, because a part costs one round trip of its rows in 32 bits.
Shape shape_of(int B, int N, int M, int H, int Hk, int es, int left, int right, int sinks)
{
    const long G = H / Hk, rows = (long)N * G;
    Shape s;
    s.waves = row_waves(es);
    s.nqt = pa_div_up(rows, 32 * s.waves);
    s.splits = 1;
    const long wgs = (long)B * Hk * s.nqt;
    if (wgs >= 256) return s;
    const long span = (long)left + right + 32 * s.waves / G + 1;             // longest range of keys of one workgroup
    const long tiles = pa_div_up(M < span ? M : span, 64) + (left < M ? pa_div_up(sinks < M ? sinks : M, 64) : 0);
    const long want = 512 / wgs, most = tiles / 4;
    const long n = want < most ? want : most;
    s.splits = n < 1 ? 1 : (n > 64 ? 64 : (int)n);
    return s;
}

template <typename T, int DT, int NW, bool SPLIT, bool FINE>
void launch_rows(const FwdArgs &a, hipStream_t st)
{
    hipLaunchKernelGGL((fwd_kernel<T, DT, NW, SPLIT, FINE>), dim3((unsigned)((long)a.nqt * a.B * a.Hk), (unsigned)a.splits), dim3(64 * NW), 0, st, a);
}

template <typename T, int DT>
int launch_fwd(const FwdArgs &a, hipStream_t st)
{
    constexpr int NW = row_waves(sizeof(T));
    const bool fine = a.few || a.D <= 16;
    if (a.splits > 1) {
        if (fine) launch_rows<T, DT, NW, true, sizeof(T) == 2>(a, st);
        else launch_rows<T, DT, NW, true, false>(a, st);
        const long threads = (long)a.B * a.Hk * a.N * a.G * (DT / 4);
        hipLaunchKernelGGL((join_kernel<T, DT>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, st, a);
    } else {
        if (fine) launch_rows<T, DT, NW, false, sizeof(T) == 2>(a, st);
        else launch_rows<T, DT, NW, false, false>(a, st);
    }
    return 0;
}

}  // namespace

PA_API long pa_window_attention_scratch_floats(int b, int n, int m, int h, int hk, int d, int left, int right, int sinks)
{
    if (b <= 0 || n <= 0 || h <= 0 || hk <= 0 || h % hk != 0) return 0;
    const int l = left < 0 ? UNBOUNDED : left, r = right < 0 ? UNBOUNDED : right;
    const int s2 = shape_of(b, n, m, h, hk, 2, l, r, sinks).splits, s4 = shape_of(b, n, m, h, hk, 4, l, r, sinks).splits, s = s2 > s4 ? s2 : s4;
    return s <= 1 ? 0 : (long)s * b * n * h * (width(d) + 2);
}

PA_API int pa_window_attention(int dtype, int b, int n, int m, int h, int hk, int d, const void *q, long qb, long qn, long qh, const void *k, long kb, long kn,
                               long kh, const void *v, long vb, long vn, long vh, int left, int right, int sinks, float scale, const int *start,
                               const int *length, void *out, void *low, float *lse, float *scratch, pa_stream_t stream)
{
    int rc = window_attention_check("pa_window_attention", dtype, b, n, m, h, hk, d, left, right, sinks, scale);
    if (rc != PA_OK) return rc;
    if (b == 0 || n == 0) return PA_OK;
    PA_REQUIRE(q && out && (m == 0 || (k && v)), "pa_window_attention: null tensor");
    PA_REQUIRE(alignment_of(dtype == PA_DT_F32 ? 4 : 2, {q, k, v, out, low}, {qb, qn, qh, kb, kn, kh, vb, vn, vh}) == 16,
               "pa_window_attention: addresses and strides have to be multiples of 16 bytes");
    FwdArgs a;
    a.q = q; a.k = k; a.v = v; a.out = out; a.low = low; a.lse = lse; a.part = scratch;
    a.qb = qb; a.qn = qn; a.qh = qh; a.kb = kb; a.kn = kn; a.kh = kh; a.vb = vb; a.vn = vn; a.vh = vh;
    a.B = b; a.N = n; a.H = h; a.Hk = hk; a.D = d; a.G = h / hk;
    a.view.m = m; a.view.left = left < 0 ? UNBOUNDED : left; a.view.right = right < 0 ? UNBOUNDED : right; a.view.sinks = sinks < m ? sinks : m;
    a.view.start = start; a.view.length = length;
    a.c = scale * 1.4426950408889634f;
    a.g = Div(a.G);
    const Shape sh = shape_of(b, n, m, h, hk, dtype == PA_DT_F32 ? 4 : 2, a.view.left, a.view.right, sinks);
    a.nqt = sh.nqt;
    a.few = few_pairs((long)b * h, n, m, (long)a.view.left + a.view.right + 1);
    a.splits = sh.splits;
    PA_REQUIRE(kn >= 0 && vn >= 0 && kn <= PA_ATTN_MAXSTRIDE && vn <= PA_ATTN_MAXSTRIDE, "pa_window_attention: tokens are more than 2^22 elements apart");
    PA_REQUIRE(launchable((long)a.nqt * b * hk, 256), "pa_window_attention: too many workgroups");
    PA_REQUIRE(a.splits == 1 || scratch, "pa_window_attention: this size needs pa_window_attention_scratch_floats() of scratch");
    hipStream_t st = (hipStream_t)stream;
#define FWD(T, DT) launch_fwd<T, DT>(a, st)
    PA_ATTN_DISPATCH(dtype, d, FWD);
#undef FWD
    PA_CHECK_LAUNCH("pa_window_attention");
    return PA_OK;
}
