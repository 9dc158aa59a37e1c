// Gradients of the attention with a sliding window and first tokens that stay in view (window_attention.hip).
//
//     P_ij = exp(s_ij - lse_i)            delta_i = do_i . o_i            dS_ij = P_ij (do_i . v_j - delta_i)
//     dq_i = scale sum_j dS_ij k_j        dk_j = scale sum_i dS_ij q_i        dv_j = sum_i P_ij do_i       (i over all rows that share key head)
//
// Two kernels recompute the scores from q, k and the forward's lse (log2 units): one owns rows and walks keys (dq, and delta, which it leaves for the
// other), one owns keys and walks rows (dk, dv).  That is 7 products where one kernel with both would need 5, but every gradient is summed by one
// owner in a fixed order: no atomics, the same bits every run.  The registers of P and dS feed the second products as they are (pa_attn.h); q, do
// and k are read from LDS both as rows and transposed.
//
// The first tokens are seen by every later row, N / window times more rows than see any other key.  The rows behind their window are walked by
// workgroups of their own, 32 keys each: there the waves share the keys and take the rows in turn.  They write 32-bit partial sums, joined with the
// window's by a second launch; all walks are cut into such slices when the keys alone do not fill the chip.
//
// Roundings: P and dS are rounded to the operand type for the second products (16-bit types; the sum of two parts for few pairs, few_pairs()); the scale
// is applied to the 32-bit sums, so that dS is rounded before it gets smaller.  delta takes o as the forward pass had it before it was rounded
// (out + low): dP - delta is small beside delta, and with the rounded o alone dq and dk were off by 1.6 times the rounding of the result, now 1.4 to 1.5 (heads of 8: up to 1.58).
// float16 has its P and dS lifted into its range besides (lifted()), which costs 5 to 8 % of such a pass; without it gradients of 1e-3 had dq and dk off by 1.5 to 11.
//
// Measured, dq / dk and dv / join: bf16 4 x 4096 tokens, 16 heads of 64 over 4, window 512: 81 / 113 / 5 us (600 / 575 TFLOP/s of visible pairs); all keys of
// 4 x 2048, 16 heads of 64: 114 / 157 us (900 / 870; a library product: 1219); 2 x 8192, 16 of 128 over 4, window 1024: 226 / 437 / 7 us; float32
// 18 x 1024, 8 heads of 32, 128 keys either side: 110 / 158 / 9 us; fp16 4 x 4096 tokens, 16 heads of 64 over 4, window 512: 89 / 124 / 5.
// Bound, by counters.  dq as the forward pass: at width 64 and window 512 vector units busy 46 %, matrix units 28 %, LDS 14 %, 2.2 waves per SIMD.  dk, dv there:
// 1.6 waves per SIMD, which wait 45 % of their time; vector 32 %, matrix 25 %, LDS 20 %.  At width 128 it holds 390 registers, one wave per SIMD: nothing hides a
// wave's exponentials and reads (matrix 24 %, vector 20 %, LDS 15 %, 47 % waiting), and its rate is 580.  float32: matrix 44 to 47 %, vector 12, LDS 4 to 6.
#include "pa_attn.h"

using namespace pa_attn;

namespace {

// dk, dv: rows of a tile, fewer where they are wide (registers on their way into LDS)
template <typename T, int DT> constexpr int row_tile() { return DT * (int)sizeof(T) >= 512 ? 32 : 64; }

// float16 has its full digits from 2^-14 to 65504.  P, about 1 / keys, and dS, which has the size of the incoming gradient besides, are lifted by powers of
// two before they are packed, and the 32-bit sums are brought back.  In dv P takes 2^12 (a factor of 2^3 is left for what the rounding of a large lse
// adds).  In dq a row's factor puts its first |dS| below 2^10 and is lowered when one passes 2^15, like the running maximum of the forward pass; the largest
// |dS| of every 32 rows is left for dk, where the rows that a workgroup walks share the factor that puts the largest of them below 2^15.  So dS keeps all digits
// down to 2^-24 of the largest one of its row (dq), 2^-28 of the largest one in its workgroup's rows (dk).
template <typename T> constexpr bool lifted() { return false; }
template <> constexpr bool lifted<_Float16>() { return true; }
constexpr float P_LIFT = 12.f;
constexpr int MAX_LIFT = 80;           // 2^80 times the largest dP - delta (2^39) stays inside 32 bits' exponents

__device__ __forceinline__ float pow2(int e) { return __builtin_ldexpf(1.f, e); }
__device__ __forceinline__ int exponent(float x) { return __builtin_amdgcn_frexp_expf(x); }        // x in [2^(e-1), 2^e)

struct BwdArgs {
    const void *q, *k, *v, *out, *low, *dout;
    const float *lse;
    float *delta, *peak, *part;         // peak: largest |dS| of every 32 rows (float16)
    void *dq, *dk, *dv;
    long qb, qn, qh, kb, kn, kh, vb, vn, vh, gb, gn, gh;
    int B, N, H, Hk, D, G, nqt;
    int nkt, slices;                   // key tiles, slices of their walks
    int nst, groups, fars;             // key tiles with first tokens, groups of 32 first tokens that have far rows, slices of their walks
    int rt;                            // rows of a tile: as many whole queries as fit
    bool few;
    float c, scale;
    View view;
    Div g;
};

// FINE: the second products take P and dS in two parts
template <typename T, int DT, int NW, bool FINE>
__global__ __launch_bounds__(64 * NW, (waves_per_simd<T, DT>())) void dq_kernel(const BwdArgs a)
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

    const int row = r0 + wave * 32 + (l & 31), i = a.g.div(min(row, rows - 1)), hq = hk * a.G + min(row, rows - 1) - i * a.G;
    const Keys keys(a.view, start + i, len, row < rows);
    const size_t at = ((size_t)b * a.H + hq) * a.N + i;
    F qf[DT / 16], gf[DT / 16];
    float delta = 0.f;
    {
        const T *qp = (const T *)a.q + b * a.qb + i * a.qn + hq * a.qh, *gp = (const T *)a.dout + b * a.gb + i * a.gn + hq * a.gh;
        const size_t place = (((size_t)b * a.N + i) * a.H + hq) * a.D;
        const T *op = (const T *)a.out + place, *lp = a.low ? (const T *)a.low + place : op;
        F of[DT / 16], lf[DT / 16];
#pragma unroll
        for (int kk = 0; kk < DT / 16; ++kk) {
            qf[kk] = ldrow<T>(qp, kk, h, a.D, keys.ok);
            gf[kk] = ldrow<T>(gp, kk, h, a.D, keys.ok);
            of[kk] = ldrow<T>(op, kk, h, a.D, keys.ok);
            lf[kk] = ldrow<T>(lp, kk, h, a.D, keys.ok && a.low);
        }
#pragma unroll
        for (int kk = 0; kk < DT / 16; ++kk)
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = __builtin_fmaf((float)gf[kk][e], (float)of[kk][e] + (float)lf[kk][e], delta);
        delta += other_half(delta);
    }
    const float lse = keys.ok ? a.lse[at] : INFINITY;
    if (h == 0 && row < rows) a.delta[at] = delta;

    const int wr = __builtin_amdgcn_readfirstlane(r0 + wave * 32);
    const int wp0 = start + a.g.div(min(wr, rows - 1)), wp1 = min(start + a.g.div(min(wr + 31, rows - 1)), len - 1);
    const bool wave_on = wr < rows && wp0 < len;
    const int wlo = max(wp0 - a.view.left, 0), whi = min(wp1 + a.view.right, len - 1);
    const int flo = max(wp1 - a.view.left, 0), fhi = min(wp0 + a.view.right, len - 1);

    const T *kp = (const T *)a.k + b * a.kb + hk * a.kh, *vp = (const T *)a.v + b * a.vb + hk * a.vh;
    Direct<T, DT, KT, 64 * NW> sk, sv;
    sk.strided(a.kn);
    sv.strided(a.vn);
    auto fetch = [&](int t, char *ks, char *vs) __attribute__((always_inline)) {
        sk.fetch(ks, kp + (long)t * KT * a.kn, len - t * KT, a.D);
        sv.fetch(vs, vp + (long)t * KT * a.vn, len - t * KT, a.D);
    };

    pa_f16v dq[DT / 32];
#pragma unroll
    for (int ct = 0; ct < DT / 32; ++ct) dq[ct] = (pa_f16v)(0.f);
    int e = 0;                                                 // lifted types: sums are 2^e dq, most the largest |2^e dS| so far
    float f = 1.f, fdelta = delta, most = 0.f, top = 0.f;

    const TileList<KT> tiles(a.view, start + a.g.div(r0), start + a.g.div(min(r0 + QT, rows) - 1), len);
    if (tiles.n) fetch(tiles.tile(0), k0, v0);
    auto step = [&](int it, char *ks, char *vs, char *kn, char *vn) __attribute__((always_inline)) {
        arrived();
        __syncthreads();                                       // the tile is there, and everyone is done with the one before it
        const int j0 = tiles.tile(it) * KT;
        if (it + 1 < tiles.n) fetch(tiles.tile(it + 1), kn, vn);
        if (!wave_on) return;
#pragma unroll
        for (int sub = 0; sub < KT / 32; ++sub) {
            const int js = j0 + sub * 32;
            if (!((js <= whi && js + 31 >= wlo) || js < min(a.view.sinks, whi + 1))) continue;
            pa_f16v s = (pa_f16v)(0.f), dp = (pa_f16v)(0.f);
#pragma unroll
            for (int kk = 0; kk < DT / 16; ++kk) mma(s, L::ld(ks, sub * 32, kk), qf[kk]);
            if (!(js >= flo && js + 31 <= fhi)) {
#pragma unroll
                for (int r = 0; r < 16; ++r) s[r] = keys.sees(js + 8 * (r >> 2) + 4 * h + (r & 3)) ? s[r] : -INFINITY;
            }
#pragma unroll
            for (int kk = 0; kk < DT / 16; ++kk) mma(dp, L::ld(vs, sub * 32, kk), gf[kk]);              // meanwhile the exponentials
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = ex2(__builtin_fmaf(s[r], a.c, -lse)) * (lifted<T>() ? __builtin_fmaf(dp[r], f, -fdelta) : dp[r] - delta);
            if constexpr (lifted<T>()) {
                float mx = fabsf(s[0]);
#pragma unroll
                for (int r = 1; r < 16; ++r) mx = larger(mx, fabsf(s[r]));
                mx = larger(mx, other_half(mx));
                most = fmaxf(most, mx);                        // NaN is passed over
                if (__any(mx > top)) {                         // the first dS that is not 0, or one that passes 2^15
                    const int up = mx > top ? min(e + 10 - exponent(mx), MAX_LIFT) : e;
                    const float by = pow2(up - e);
#pragma unroll
                    for (int ct = 0; ct < DT / 32; ++ct)
#pragma unroll
                        for (int r = 0; r < 16; ++r) dq[ct][r] *= by;
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[r] *= by;
                    top = mx > top ? 0x1p15f : top;
                    most *= by;
                    e = up;
                    f = pow2(e);
                    fdelta = delta * f;
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const F ds = pack<T>(s, u);
                F rest;
                if constexpr (FINE) rest = pack_rest<T>(s, ds, u);
#pragma unroll
                for (int ct = 0; ct < DT / 32; ++ct) {
                    const F kt = L::ldt(ks, sub * 32 + 16 * u, ct * 32);
                    mma(dq[ct], kt, ds);
                    if constexpr (FINE) mma(dq[ct], kt, rest);
                }
            }
        }
    };
    for (int it = 0; it < tiles.n; it += 2) {
        step(it, k0, v0, k1, v1);
        if (it + 1 < tiles.n) step(it + 1, k1, v1, k0, v0);
    }
    if constexpr (lifted<T>()) {
        most = most < INFINITY ? most * pow2(-e) : 0.f;        // a row that is lost already does not decide for the others
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) most = fmaxf(most, __shfl_xor(most, o));
        if (l == 0) a.peak[((size_t)bh * a.nqt + qt) * NW + wave] = most;
    }
    if (row >= rows) return;
    T *dp = (T *)a.dq + (((size_t)b * a.N + i) * a.H + hq) * a.D;
    if (!keys.ok) {                                            // padding rows: 0, whatever the sequence's keys hold
#pragma unroll
        for (int ct = 0; ct < DT / 32; ++ct) dq[ct] = (pa_f16v)(0.f);
    }
    const float back = lifted<T>() ? a.scale * pow2(-e) : a.scale;
#pragma unroll
    for (int ct = 0; ct < DT / 32; ++ct)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int c = ct * 32 + 8 * u + 4 * h;
            if (c < a.D) st4<T>(dp + c, dq[ct][4 * u] * back, dq[ct][4 * u + 1] * back, dq[ct][4 * u + 2] * back, dq[ct][4 * u + 3] * back);
        }
}

// What a workgroup of the dk, dv launch owns: a slice of a key tile's window, or (behind them in the launch: they are short and fill its last round) a
// slice of the far rows of 32 first tokens.
struct Walk {
    int bh, k0, slice, slices;          // keys from k0
    bool far;
    long slot;                          // place of its partial sums, in keys; < 0: it writes the gradients itself

    __device__ __forceinline__ Walk(const BwdArgs &a, long id, int kb, int nw)
    {
        const long nwin = (long)a.B * a.Hk * a.nkt * a.slices, nfar = (long)a.B * a.Hk * a.groups * a.fars;
        far = id >= nwin;
        if (far) {
            id -= nwin;
            slot = id * 32 * nw;
            slices = a.fars;
            slice = (int)(id % slices);
            id /= slices;
            k0 = (int)(id % a.groups) * 32;
            bh = (int)(id / a.groups);
        } else {
            id = xcd_item(id, nwin);
            const long at = id;
            slices = a.slices;
            slice = (int)(id % slices);
            id /= slices;
            const int tile = (int)(id % a.nkt);
            k0 = tile * kb;
            bh = (int)(id / a.nkt);
            slot = slices > 1 ? at : a.groups > 0 && tile < a.nst ? (long)bh * a.nst + tile : -1;
            if (slot >= 0) slot = nfar * 32 * nw + slot * kb;
        }
    }
};

template <typename T, int DT, int NW, bool FINE>
__global__ __launch_bounds__(64 * NW, sizeof(T) == 2 && DT <= 64 ? 2 : 1) void dkv_kernel(const BwdArgs a)
{
    typedef Tile<T, DT> L;
    typedef typename Frag<T>::type F;
    constexpr int KB = 32 * NW, RT = row_tile<T, DT>(), TB = RT * L::RB;
    __shared__ __attribute__((aligned(16))) char q0[TB], q1[TB], g0[TB], g1[TB];
    __shared__ __attribute__((aligned(16))) float r0[3][RT], r1[3][RT];                // of the tile's rows: lse, delta, position
    const int tid = threadIdx.x, wave = tid >> 6, l = tid & 63, h = l >> 5;
    const Walk w(a, blockIdx.x, KB, NW);
    const int b = w.bh / a.Hk, hk = w.bh - b * a.Hk;
    const int len = a.view.len(b), start = a.view.first(b);

    // rows that see the tile's keys k0 .. k1 in their window: positions k0 - right .. k1 + left; behind them the far rows of first tokens
    int ra = 0, rb = 0;
    {
        const int k0 = w.k0 / KB * KB, k1 = min(k0 + KB, len) - 1;
        const int last = min(a.N - 1, len - 1 - start), ib = k1 + a.view.left - start;
        const int ia = max(w.far ? ib + 1 : k0 - a.view.right - start, 0), iz = w.far ? last : min(last, ib);
        if (k0 <= k1 && ia <= iz) {
            ra = ia * a.G;
            rb = (iz + 1) * a.G;
        }
    }
    const int all = (rb - ra + a.rt - 1) / a.rt;
    const int t0 = (int)((long)all * w.slice / w.slices), t1 = (int)((long)all * (w.slice + 1) / w.slices);

    int e = 0;                                                 // lifted types: sums are 2^e dk and 2^P_LIFT dv
    if constexpr (lifted<T>()) {
        if (t0 < t1) {
            const float *peak = a.peak + (size_t)w.bh * a.nqt * row_waves(sizeof(T));       // one of every wave of the dq launch
            float most = 0.f;
            const int last = (min(ra + t1 * a.rt, rb) - 1) / 32;
            for (int x = (ra + t0 * a.rt) / 32 + l; x <= last; x += 64) most = fmaxf(most, peak[x]);
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) most = fmaxf(most, __shfl_xor(most, o));
            e = most > 0.f ? min(15 - exponent(most), MAX_LIFT) : 0;
        }
    }
    const float f = lifted<T>() ? pow2(e - (int)P_LIFT) : 1.f;

    const int wk = __builtin_amdgcn_readfirstlane(w.far ? w.k0 : w.k0 + wave * 32), wk1 = min(wk + 31, len - 1);
    const bool wave_on = wk < len;
    const int j = wk + (l & 31);
    // this lane's key is seen from positions plo .. plo + span
    const int plo = j < len ? j - a.view.right : NOWHERE;
    const u32 span = j >= len ? 0u : j < a.view.sinks ? 0x7fffffffu : (u32)a.view.left + (u32)a.view.right;
    F kf[DT / 16], vf[DT / 16];
    {
        const T *kp = (const T *)a.k + b * a.kb + hk * a.kh + (long)j * a.kn, *vp = (const T *)a.v + b * a.vb + hk * a.vh + (long)j * a.vn;
#pragma unroll
        for (int kk = 0; kk < DT / 16; ++kk) {
            kf[kk] = ldrow<T>(kp, kk, h, a.D, j < len);
            vf[kk] = ldrow<T>(vp, kk, h, a.D, j < len);
        }
    }

    // A tile is a.rt rows: whole queries, so that a thread's rows have the same head and the same distance from the tile's first query every time.
    // (More than RT heads a group: RT rows from anywhere, decoded each time.)
    Direct<T, DT, RT, 64 * NW> sq, sg;
    const bool whole = a.G <= RT;
    float pl = 0.f, pd = 0.f;
    int pp = 0;
    const T *qp = (const T *)a.q + b * a.qb + (long)hk * a.G * a.qh, *gp = (const T *)a.dout + b * a.gb + (long)hk * a.G * a.gh;
    auto place = [&](int first) __attribute__((always_inline)) {                              // offsets of the tile's rows from query first / G
#pragma unroll
        for (int u = 0; u < sq.N; ++u) {
            const int x = first + sq.row(u), i = a.g.div(x), g = x - i * a.G;
            sq.off[u] = ((u32)i * (u32)a.qn + (u32)g * (u32)a.qh + sq.chunk(u) * L::EC) * (u32)sizeof(T);
            sg.off[u] = ((u32)i * (u32)a.gn + (u32)g * (u32)a.gh + sq.chunk(u) * L::EC) * (u32)sizeof(T);
        }
    };
    place(0);
    const int li = a.g.div(tid), lg = hk * a.G + tid - li * a.G;       // row tid of a tile: query and head (threads below RT)
    auto fetch = [&](int t, char *qs, char *gs) __attribute__((always_inline)) {
        const int first = ra + t * a.rt, i0 = a.g.div(first), valid = min(a.rt, rb - first);
        if (!whole) place(first - i0 * a.G);
        sq.fetch(qs, qp + (long)i0 * a.qn, valid, a.D);        // padding rows are behind rb
        sg.fetch(gs, gp + (long)i0 * a.gn, valid, a.D);
        if (tid < RT) {
            int i = i0 + li, hq = lg;
            if (!whole) {
                i = a.g.div(first + tid);
                hq = hk * a.G + first + tid - i * a.G;
            }
            const size_t at = ((size_t)b * a.H + hq) * a.N + i;
            pl = tid < valid ? a.lse[at] - (lifted<T>() ? P_LIFT : 0.f) : INFINITY;
            pd = tid < valid ? a.delta[at] * f : 0.f;
            pp = start + i;
        }
    };

    pa_f16v dk[DT / 32], dv[DT / 32];
#pragma unroll
    for (int ct = 0; ct < DT / 32; ++ct) dk[ct] = dv[ct] = (pa_f16v)(0.f);

    if (t0 < t1) fetch(t0, q0, g0);
    auto step = [&](int t, char *qs, char *gs, float (&rs)[3][RT], char *qn, char *gn) __attribute__((always_inline)) {
        const float *ls = rs[0], *ds = rs[1];
        const int *ps = reinterpret_cast<const int *>(rs[2]);
        if (tid < RT) {
            rs[0][tid] = pl;
            rs[1][tid] = pd;
            rs[2][tid] = __int_as_float(pp);
        }
        arrived();
        __syncthreads();
        if (t + 1 < t1) fetch(t + 1, qn, gn);
        if (!wave_on) return;
#pragma unroll
        for (int sub = 0; sub < RT / 32; ++sub) {
            const int rf = ra + t * a.rt + sub * 32, re = min(min(rf + 31, ra + t * a.rt + a.rt - 1), rb - 1);
            if (rf > re || (w.far && (t * (RT / 32) + sub) % NW != wave)) continue;
            const int p0 = start + a.g.div(rf), p1 = start + a.g.div(re);
            if (!(p1 >= wk - a.view.right && (p0 <= wk1 + a.view.left || wk < a.view.sinks))) continue;
            pa_f16v s = (pa_f16v)(0.f), dp = (pa_f16v)(0.f);
#pragma unroll
            for (int kk = 0; kk < DT / 16; ++kk) mma(s, L::ld(qs, sub * 32, kk), kf[kk]);
            if (!(p0 >= wk + 31 - a.view.right && p1 <= wk + a.view.left && wk + 31 < len)) {           // some row does not see some key
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int4 pos = *reinterpret_cast<const int4 *>(ps + sub * 32 + 8 * u + 4 * h);
                    const int pe[4] = {pos.x, pos.y, pos.z, pos.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[4 * u + e] = (u32)pe[e] - (u32)plo <= span ? s[4 * u + e] : -INFINITY;
                }
            }
#pragma unroll
            for (int kk = 0; kk < DT / 16; ++kk) mma(dp, L::ld(gs, sub * 32, kk), vf[kk]);              // meanwhile the exponentials
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int rr = sub * 32 + 8 * u + 4 * h;
                const pa_f4 lse = *reinterpret_cast<const pa_f4 *>(ls + rr), delta = *reinterpret_cast<const pa_f4 *>(ds + rr);
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int r = 4 * u + x;
                    s[r] = ex2(__builtin_fmaf(s[r], a.c, -lse[x]));
                    dp[r] = s[r] * (lifted<T>() ? __builtin_fmaf(dp[r], f, -delta[x]) : dp[r] - delta[x]);
                }
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const F pf = pack<T>(s, u), df = pack<T>(dp, u);
                F pr, dr;
                if constexpr (FINE) {
                    pr = pack_rest<T>(s, pf, u);
                    dr = pack_rest<T>(dp, df, u);
                }
#pragma unroll
                for (int ct = 0; ct < DT / 32; ++ct) {
                    const F gt = L::ldt(gs, sub * 32 + 16 * u, ct * 32), qt = L::ldt(qs, sub * 32 + 16 * u, ct * 32);
                    mma(dv[ct], gt, pf);
                    mma(dk[ct], qt, df);
                    if constexpr (FINE) {
                        mma(dv[ct], gt, pr);
                        mma(dk[ct], qt, dr);
                    }
                }
            }
        }
    };
    for (int t = t0; t < t1; t += 2) {
        step(t, q0, g0, r0, q1, g1);
        if (t + 1 < t1) step(t + 1, q1, g1, r1, q0, g0);
    }
    if (w.far && j >= a.view.sinks) return;                     // nobody reads those
    if (j >= len) {                                             // padding keys: 0, whatever the sequence's rows hold
#pragma unroll
        for (int ct = 0; ct < DT / 32; ++ct) dk[ct] = dv[ct] = (pa_f16v)(0.f);
    }
    if constexpr (lifted<T>()) {
        const float bk = pow2(-e), bv = pow2(-(int)P_LIFT);
#pragma unroll
        for (int ct = 0; ct < DT / 32; ++ct)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                dk[ct][r] *= bk;
                dv[ct][r] *= bv;
            }
    }
    if (w.slot >= 0) {
        float *po = a.part + ((size_t)w.slot + wave * 32 + (l & 31)) * (2 * DT);
#pragma unroll
        for (int ct = 0; ct < DT / 32; ++ct)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int c = ct * 32 + 8 * u + 4 * h;
                *reinterpret_cast<pa_f4 *>(po + c) = (pa_f4){dk[ct][4 * u], dk[ct][4 * u + 1], dk[ct][4 * u + 2], dk[ct][4 * u + 3]};
                *reinterpret_cast<pa_f4 *>(po + DT + c) = (pa_f4){dv[ct][4 * u], dv[ct][4 * u + 1], dv[ct][4 * u + 2], dv[ct][4 * u + 3]};
            }
        return;
    }
    if (j >= a.view.m) return;
    const size_t at = (((size_t)b * a.view.m + j) * a.Hk + hk) * a.D;
    T *ko = (T *)a.dk + at, *vo = (T *)a.dv + at;
#pragma unroll
    for (int ct = 0; ct < DT / 32; ++ct)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int c = ct * 32 + 8 * u + 4 * h;
            if (c < a.D) {
                st4<T>(ko + c, dk[ct][4 * u] * a.scale, dk[ct][4 * u + 1] * a.scale, dk[ct][4 * u + 2] * a.scale, dk[ct][4 * u + 3] * a.scale);
                st4<T>(vo + c, dv[ct][4 * u], dv[ct][4 * u + 1], dv[ct][4 * u + 2], dv[ct][4 * u + 3]);
            }
        }
}

// dk, dv of the key tiles that left partial sums: the window's slices, then the far rows' (slice by slice, wave by wave).  A workgroup owns a key;
// DT / 2 threads hold a row of dk and dv, four elements each, the 512 / DT groups of such threads take the sums in turn and are added in order.
template <typename T, int DT, int NW>
__global__ __launch_bounds__(256) void dkv_join_kernel(const BwdArgs a, int tiles, long first)
{
    constexpr int C = DT / 2, P = 256 / C, KB = 32 * NW;
    __shared__ pa_f4 red[P][C];
    const int c = (int)threadIdx.x % C * 4, part = (int)threadIdx.x / C;
    const long tile = first + blockIdx.x / KB;
    const int r = (int)(blockIdx.x % KB);
    const int bh = (int)(tile / tiles), t = (int)(tile % tiles), b = bh / a.Hk, hk = bh - b * a.Hk, j = t * KB + r;
    if (j >= a.view.m) return;
    const size_t nfar = (size_t)a.B * a.Hk * a.groups * a.fars * 32 * NW;
    const float *p = a.part + (nfar + (size_t)tile * a.slices * KB + r) * (2 * DT) + c;
    pa_f4 s = (pa_f4)(0.f);
#pragma unroll 4
    for (int i = part; i < a.slices; i += P) s += *reinterpret_cast<const pa_f4 *>(p + (size_t)i * KB * 2 * DT);
    if (j < a.view.sinks && a.groups > 0) {
        p = a.part + (((size_t)bh * a.groups + j / 32) * a.fars * 32 * NW + (j & 31)) * (2 * DT) + c;
#pragma unroll 8
        for (int i = part; i < a.fars * NW; i += P) s += *reinterpret_cast<const pa_f4 *>(p + (size_t)i * 32 * 2 * DT);
    }
    if (part < P) red[part][c / 4] = s;
    __syncthreads();
    if (part > 0) return;
#pragma unroll
    for (int i = 1; i < P; ++i) s += red[i][c / 4];
    const size_t at = (((size_t)b * a.view.m + j) * a.Hk + hk) * a.D;
    if (c < DT) {
        if (c < a.D) st4<T>((T *)a.dk + at + c, s[0] * a.scale, s[1] * a.scale, s[2] * a.scale, s[3] * a.scale);
    } else if (c - DT < a.D) {
        st4<T>((T *)a.dv + at + c - DT, s[0], s[1], s[2], s[3]);
    }
}

struct Shape {
    int qwaves, nqt, kwaves, nkt, slices, nst, groups, fars, rt;
    long slots(long bh) const                                  // keys of partial sums
    {
        return bh * groups * fars * 32 * kwaves + (slices > 1 ? bh * nkt * slices : groups > 0 ? bh * nst : 0) * 32 * kwaves;
    }
    int joined() const { return slices > 1 ? nkt : groups > 0 ? nst : 0; }      // key tiles with partial sums
};

// Slices: keys that do not fill the chip (fewer than 2048 waves, two per SIMD) have their walks cut, each slice with at least four row tiles;
// far rows are cut into slices of 16 row tiles, more where the slices alone would fill the chip several times (2048 of them).
Shape shape_of(int B, int N, int M, int H, int Hk, int d, int es, int left, int right, int sinks, bool started)
{
    Shape s;
    const long G = H / Hk, bh = (long)B * Hk, rows = (long)N * G;
    s.qwaves = row_waves(es);
    s.nqt = pa_div_up(rows, 32 * s.qwaves);
    s.kwaves = key_waves(es, (long)left + right);
    const int kb = 32 * s.kwaves, rt = width(d) * es >= 512 ? 32 : 64;
    s.rt = G <= rt ? rt / (int)G * (int)G : rt;
    s.nkt = pa_div_up(M, kb);
    const long wgs = bh * s.nkt, reach = (long)left + right + kb, walk = pa_div_up((N < reach ? N : reach) * G, s.rt);
    long n = wgs ? 2048 / s.kwaves / wgs : 1;
    if (n > walk / 4) n = walk / 4;
    s.slices = n < 1 ? 1 : n > 64 ? 64 : (int)n;
    const int first = sinks < M ? sinks : M;
    const bool far = N > 0 && first > 0 && (started ? left < M : left < N - 1);        // rows behind the window of the first tokens
    s.groups = far ? pa_div_up(first, 32) : 0;
    s.nst = pa_div_up(first, kb);
    long f = (rows + 16 * s.rt - 1) / (16 * s.rt);
    const long most = s.groups ? 2048 / (bh * s.groups) : 0;
    f = f > most ? most : f;
    s.fars = far ? (f > 64 ? 64 : f < 1 ? 1 : (int)f) : 1;
    return s;
}

template <typename T, int DT, int NW, bool FINE>
void launch_dq(const BwdArgs &a, hipStream_t st)
{
    hipLaunchKernelGGL((dq_kernel<T, DT, NW, FINE>), dim3((unsigned)((long)a.nqt * a.B * a.Hk)), dim3(64 * NW), 0, st, a);
}

template <typename T, int DT, int NW, bool FINE>
void launch_dkv(const BwdArgs &a, int joined, hipStream_t st)
{
    const long bh = (long)a.B * a.Hk;
    hipLaunchKernelGGL((dkv_kernel<T, DT, NW, FINE>), dim3((unsigned)(bh * a.groups * a.fars + bh * a.nkt * a.slices)), dim3(64 * NW), 0, st, a);
    constexpr long most = (1l << 23) / (32 * NW);              // tiles of a launch: 2^31 threads
    for (long first = 0; first < bh * joined; first += most) {
        const long n = bh * joined - first < most ? bh * joined - first : most;
        hipLaunchKernelGGL((dkv_join_kernel<T, DT, NW>), dim3((unsigned)(n * 32 * NW)), dim3(256), 0, st, a, joined, first);
    }
}

template <typename T, int DT>
int launch_bwd(const BwdArgs &a, const Shape &s, hipStream_t st)
{
    if constexpr (sizeof(T) == 4) {
        if (a.nqt) launch_dq<T, DT, row_waves(4), false>(a, st);
        if (a.nkt) launch_dkv<T, DT, 2, false>(a, s.joined(), st);
    } else {
        if (a.nqt) {
            if (a.few) launch_dq<T, DT, row_waves(2), true>(a, st);
            else launch_dq<T, DT, row_waves(2), false>(a, st);
        }
        if (a.nkt) {
            if (s.kwaves == 2 && a.few) launch_dkv<T, DT, 2, true>(a, s.joined(), st);
            else if (s.kwaves == 2) launch_dkv<T, DT, 2, false>(a, s.joined(), st);
            else if (a.few) launch_dkv<T, DT, 4, true>(a, s.joined(), st);
            else launch_dkv<T, DT, 4, false>(a, s.joined(), st);
        }
    }
    return 0;
}

}  // namespace

// floats of scratch: delta (B H N), the largest |dS| of every 32 rows, then the partial sums of sliced walks
static long front_floats(int b, int n, int h, int hk) { return pa_div_up((long)b * h * n, 4) * 4l + (long)b * hk * pa_div_up((long)n * (h / hk), 32 * row_waves(2)) * row_waves(2); }

PA_API long pa_window_attention_backward_scratch_floats(int b, int n, int m, int h, int hk, int d, int left, int right, int sinks)
{
    if (b <= 0 || n <= 0 || h <= 0 || hk <= 0 || h % hk != 0 || m < 0 || sinks < 0) return 0;
    const long bh = (long)b * hk;
    long most = 0;                                              // of both element sizes, with and without q_start
    for (int i = 0; i < 4; ++i) {
        const long k = shape_of(b, n, m, h, hk, d, i & 1 ? 4 : 2, left < 0 ? UNBOUNDED : left, right < 0 ? UNBOUNDED : right, sinks, i & 2).slots(bh);
        most = k > most ? k : most;
    }
    return front_floats(b, n, h, hk) + most * 2 * width(d);
}

PA_API long pa_window_attention_backward_plan_floats(int dtype, int b, int n, int m, int h, int hk, int d, int left, int right, int sinks, int started)
{
    const Shape s = shape_of(b, n, m, h, hk, d, dtype == PA_DT_F32 ? 4 : 2, left < 0 ? UNBOUNDED : left, right < 0 ? UNBOUNDED : right, sinks, started != 0);
    const long slots = s.nkt ? s.slots((long)b * hk) : 0;
    return front_floats(b, n, h, hk) + slots * 2 * width(d);
}

PA_API int pa_window_attention_backward(int dtype, int b, int n, int m, int h, int hk, int d, const void *q, long qb, long qn, long qh, const void *k, long kb,
                                        long kn, long kh, const void *v, long vb, long vn, long vh, const void *out, const void *low, const float *lse, const void *dout, long gb,
                                        long gn, long gh, int left, int right, int sinks, float scale, const int *start, const int *length, void *dq, void *dk,
                                        void *dv, float *scratch, pa_stream_t stream)
{
    int rc = window_attention_check("pa_window_attention_backward", dtype, b, n, m, h, hk, d, left, right, sinks, scale);
    if (rc != PA_OK) return rc;
    if (b == 0 || (n == 0 && m == 0)) return PA_OK;
    PA_REQUIRE((n == 0 || (q && out && lse && dout && dq && scratch)) && (m == 0 || (k && v && dk && dv)), "pa_window_attention_backward: null tensor");
    PA_REQUIRE(alignment_of(dtype == PA_DT_F32 ? 4 : 2, {q, k, v, out, low, dout, dq, dk, dv, scratch}, {qb, qn, qh, kb, kn, kh, vb, vn, vh, gb, gn, gh}) == 16,
               "pa_window_attention_backward: addresses and strides have to be multiples of 16 bytes");
    BwdArgs a;
    a.q = q; a.k = k; a.v = v; a.out = out; a.low = low; a.dout = dout; a.lse = lse; a.dq = dq; a.dk = dk; a.dv = dv;
    a.delta = scratch;
    a.peak = scratch + pa_div_up((long)b * h * n, 4) * 4l;
    a.part = scratch + front_floats(b, n, h, hk);
    a.qb = qb; a.qn = qn; a.qh = qh; a.kb = kb; a.kn = kn; a.kh = kh; a.vb = vb; a.vn = vn; a.vh = vh; a.gb = gb; a.gn = gn; a.gh = gh;
    a.B = b; a.N = n; a.H = h; a.Hk = hk; a.D = d; a.G = h / hk;
    a.view.m = m; a.view.left = left < 0 ? UNBOUNDED : left; a.view.right = right < 0 ? UNBOUNDED : right; a.view.sinks = sinks < m ? sinks : m;
    a.view.start = start; a.view.length = length;
    a.scale = scale;
    a.c = scale * 1.4426950408889634f;
    a.g = Div(a.G);
    const Shape s = shape_of(b, n, m, h, hk, d, dtype == PA_DT_F32 ? 4 : 2, a.view.left, a.view.right, sinks, start != nullptr);
    a.few = few_pairs((long)b * h, n, m, (long)a.view.left + a.view.right + 1);
    a.nqt = s.nqt; a.nkt = s.nkt; a.slices = s.slices; a.nst = s.nst; a.groups = s.groups; a.fars = s.fars; a.rt = s.rt;
    PA_REQUIRE(kn >= 0 && vn >= 0 && kn <= PA_ATTN_MAXSTRIDE && vn <= PA_ATTN_MAXSTRIDE && qn >= 0 && qh >= 0 && gn >= 0 && gh >= 0 && qn <= PA_ATTN_MAXSTRIDE &&
                   gn <= PA_ATTN_MAXSTRIDE && qh <= PA_ATTN_MAXSTRIDE && gh <= PA_ATTN_MAXSTRIDE,
               "pa_window_attention_backward: tokens or heads are more than 2^22 elements apart");
    PA_REQUIRE(a.G <= 32 || (long)a.G * (qh > gh ? qh : gh) * 4 < (1l << 31), "pa_window_attention_backward: the heads of a group span 2^31 bytes");
    PA_REQUIRE(launchable((long)a.nqt * b * hk, 256) && launchable((long)b * hk * ((long)s.groups * s.fars + (long)s.nkt * s.slices), 256),
               "pa_window_attention_backward: too many workgroups");
    PA_REQUIRE(s.slots((long)b * hk) == 0 || scratch, "pa_window_attention_backward: this size needs pa_window_attention_backward_scratch_floats() of scratch");
    hipStream_t st = (hipStream_t)stream;
#define BWD(T, DT) launch_bwd<T, DT>(a, s, st)
    PA_ATTN_DISPATCH(dtype, d, BWD);
#undef BWD
    PA_CHECK_LAUNCH("pa_window_attention_backward");
    return PA_OK;
}
