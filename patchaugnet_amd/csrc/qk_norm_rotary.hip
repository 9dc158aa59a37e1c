// Norm of every query and key head with the position rotation in the same pass, forward and backward.
//
//     r = (mean_d x_d^2 + eps)^-1/2,   n = x r,   t = n w,   y = R(position) t
//     R turns the pair (u, v) number a F + f of the first 2 A F elements by position_a inv_freq[a][f]; the other elements stay as they are.
//     Pairs: (t_i, t_{i + A F}), or (t_{2 i}, t_{2 i + 1}) when interleaved.
// Gradients:
//     s = R^T dy,   dw = sum s n,   t = s w,   dx = r (t - n mean(t n))
//
// Bound: bytes -- x and y (backward: x, dy and dx) once.  A few lanes hold a row: a lane has the two V-element pieces of its pairs (one row of 128
// 16-bit elements: 8 lanes with 2 x 16 bytes each), so the mean square is the only exchange between lanes.  The rotation's sines and cosines are the
// expensive part (64-bit range reduction: positions of 10^6 keep full accuracy); a workgroup computes those of its tokens once, into LDS, for all
// query and key heads.  Everything between load and store is 32-bit, rounded once.
//
// The weight gradients are sums over all tokens and heads: per lane in registers over a workgroup's tokens, then across the workgroup, then by a
// second launch over the workgroups' rows, always in the same order.
#include <initializer_list>

#include "pa_common.h"

namespace {

enum { F32 = 0, F16 = 1, BF16 = 2 };
constexpr int MAXD = 512, MAXTOK = 16;

struct NormArgs {
    const void *q, *k, *gq, *gk;        // gq, gk: gradients of the outputs (backward)
    void *oq, *ok;                      // outputs (forward) / input gradients (backward), contiguous
    const void *qw, *kw;
    const void *pos;
    const float *freq;
    float *part;                        // (workgroups, 2, D) partial weight gradients
    long qb, qn, qh, kb, kn, kh, gqb, gqn, gqh, gkb, gkn, gkh, pb;
    long tokens;
    int N, H, Hk, D, axes, per, pairs, interleaved, wtype, ptype;
    int tb, units, lpr;                 // tokens of a workgroup's turn, units of a row, lanes of a row (a power of two)
    float eps;
};

template <typename T> __device__ __forceinline__ float weight_at(const void *w, int f32, int i)
{
    return w == nullptr ? 1.f : f32 ? ((const float *)w)[i] : (float)((const T *)w)[i];
}

__device__ __forceinline__ double position_at(const NormArgs &a, int b, int n, int axis)
{
    const long i = b * a.pb + (long)n * a.axes + axis;
    return a.ptype == 0 ? (double)((const int *)a.pos)[i] : a.ptype == 1 ? (double)((const long long *)a.pos)[i] : (double)((const float *)a.pos)[i];
}

// cos and sin of position * frequency: reduced in 64 bits to an eighth of a turn either side of a quarter turn, where 32 bits are enough
__device__ __forceinline__ float2 turn(double x)
{
    const double q = x * 0.63661977236758134308;                // quarter turns
    const double n = __builtin_rint(q);
    // x / (pi / 2) is rounded at 2^-53 of its size; the frequencies are 32-bit numbers, so x itself is exact
    const float f = (float)(q - n);
    float s, c;
    sincospif(0.5f * f, &s, &c);
    const int k = (int)(n - 4.0 * __builtin_floor(n * 0.25));
    return k == 0 ? make_float2(c, s) : k == 1 ? make_float2(-s, c) : k == 2 ? make_float2(-c, -s) : make_float2(s, -c);
}

template <typename T, int V> struct Vec {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T> struct Vec<T, 1> {
    typedef T type;
};
template <typename T, int V> __device__ __forceinline__ void load(float *x, const T *p)
{
    const typename Vec<T, V>::type v = *reinterpret_cast<const typename Vec<T, V>::type *>(p);
    if constexpr (V == 1) x[0] = (float)v;
    else
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (float)v[i];
}
template <typename T, int V> __device__ __forceinline__ void store(T *p, const float *x)
{
    typename Vec<T, V>::type v;
    if constexpr (V == 1) v = (T)x[0];
    else
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (T)x[i];
    *reinterpret_cast<typename Vec<T, V>::type *>(p) = v;
}

// A row as units of two V-element pieces: the pairs' two halves, then the unrotated rest.  The last piece of an odd rest does not exist (V = 1 only).
template <int V> struct Unit {
    int o1, o2, pair;                   // pair < 0: not rotated
    bool on, two;

    __device__ __forceinline__ Unit(const NormArgs &a, int u)
    {
        const int rot = a.pairs / V;
        on = u < a.units;
        pair = u < rot ? u * V : -1;
        if (u < rot && !a.interleaved) {
            o1 = u * V;
            o2 = a.pairs + u * V;
        } else {
            o1 = 2 * u * V;
            o2 = o1 + V;
        }
        two = on && o2 < a.D;
    }
};

template <int V> __device__ __forceinline__ void rotate(float *x, const Unit<V> &t, int interleaved, const float *cs, const float *sn, float sign)
{
    if (t.pair < 0) return;
    if (interleaved) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float c = cs[t.pair + i], s = sign * sn[t.pair + i], u = x[2 * i], v = x[2 * i + 1];
            x[2 * i] = u * c - v * s;
            x[2 * i + 1] = u * s + v * c;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float c = cs[t.pair + i], s = sign * sn[t.pair + i], u = x[i], v = x[V + i];
            x[i] = u * c - v * s;
            x[V + i] = u * s + v * c;
        }
    }
}

// UPL: units a lane can hold (1 for the wide pieces, up to 4 for the narrow ones: 64 lanes x 4 units x 2 elements = MAXD)
template <typename T, int V, int UPL, bool BWD>
__global__ __launch_bounds__(256) void norm_kernel(const NormArgs a)
{
    extern __shared__ __attribute__((aligned(16))) float sh[];       // [tb][pairs] cosines, [tb][pairs] sines; backward: then the join of 2 D sums
    const int tid = threadIdx.x, lane = tid & (a.lpr - 1), slot = tid / a.lpr, slots = 256 / a.lpr;
    const int heads = a.H + a.Hk;
    float wq[UPL][2 * V], wk[UPL][2 * V], sq[UPL][2 * V], sk[UPL][2 * V];
#pragma unroll
    for (int p = 0; p < UPL; ++p) {
        const Unit<V> t(a, lane + p * a.lpr);
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) {
            const int e = (i < V ? t.o1 + i : t.o2 + i - V);
            const bool in = t.on && (i < V || t.two);
            wq[p][i] = in ? weight_at<T>(a.qw, a.wtype, e) : 0.f;
            wk[p][i] = in ? weight_at<T>(a.kw, a.wtype, e) : 0.f;
            sq[p][i] = sk[p][i] = 0.f;
        }
    }
    const float inv_d = 1.0f / (float)a.D;
    for (long t0 = (long)blockIdx.x * a.tb; t0 < a.tokens; t0 += (long)gridDim.x * a.tb) {
        const int nt = (int)(a.tokens - t0 < a.tb ? a.tokens - t0 : a.tb);
        if (a.pairs > 0) {
            if (BWD) __syncthreads();                           // readers of the previous turn's angles
            for (int i = tid; i < nt * a.pairs; i += 256) {
                const int tok = i / a.pairs, pr = i - tok * a.pairs, axis = pr / a.per;
                const long at = t0 + tok;
                const int b = (int)(at / a.N), n = (int)(at - (long)b * a.N);
                const float2 cs = turn(position_at(a, b, n, axis) * (double)a.freq[pr]);
                sh[tok * a.pairs + pr] = cs.x;
                sh[(a.tb + tok) * a.pairs + pr] = cs.y;
            }
            __syncthreads();
        }
        for (int row = slot; row < nt * heads; row += slots) {
            const int tok = row / heads, hd = row - tok * heads;
            const long at = t0 + tok;
            const int b = (int)(at / a.N), n = (int)(at - (long)b * a.N);
            const bool isq = hd < a.H;
            const int g = isq ? hd : hd - a.H;
            const T *x = isq ? (const T *)a.q + b * a.qb + n * a.qn + g * a.qh : (const T *)a.k + b * a.kb + n * a.kn + g * a.kh;
            T *y = isq ? (T *)a.oq + (at * a.H + g) * a.D : (T *)a.ok + (at * a.Hk + g) * a.D;
            float v[UPL][2 * V], gr[BWD ? UPL : 1][2 * V], ss = 0.f;
            const float *cs = sh + tok * a.pairs, *sn = sh + (a.tb + tok) * a.pairs;
#pragma unroll
            for (int p = 0; p < UPL; ++p) {
                const Unit<V> t(a, lane + p * a.lpr);
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) v[p][i] = 0.f;
                if (t.on) load<T, V>(&v[p][0], x + t.o1);
                if (t.two) load<T, V>(&v[p][V], x + t.o2);
                if (BWD) {
                    const T *gp = isq ? (const T *)a.gq + b * a.gqb + n * a.gqn + g * a.gqh : (const T *)a.gk + b * a.gkb + n * a.gkn + g * a.gkh;
#pragma unroll
                    for (int i = 0; i < 2 * V; ++i) gr[p][i] = 0.f;
                    if (t.on) load<T, V>(&gr[p][0], gp + t.o1);
                    if (t.two) load<T, V>(&gr[p][V], gp + t.o2);
                }
            }
#pragma unroll
            for (int p = 0; p < UPL; ++p)
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) ss = __builtin_fmaf(v[p][i], v[p][i], ss);
            for (int o = 1; o < a.lpr; o <<= 1) ss += __shfl_xor(ss, o);
            const float r = 1.0f / __builtin_sqrtf(__builtin_fmaf(ss, inv_d, a.eps));
            if (!BWD) {
#pragma unroll
                for (int p = 0; p < UPL; ++p) {
                    const Unit<V> t(a, lane + p * a.lpr);
#pragma unroll
                    for (int i = 0; i < 2 * V; ++i) v[p][i] = v[p][i] * r * (isq ? wq[p][i] : wk[p][i]);
                    rotate<V>(v[p], t, a.interleaved, cs, sn, 1.f);
                    if (t.on) store<T, V>(y + t.o1, &v[p][0]);
                    if (t.two) store<T, V>(y + t.o2, &v[p][V]);
                }
            } else {
                float dot = 0.f;
#pragma unroll
                for (int p = 0; p < UPL; ++p) {
                    const Unit<V> t(a, lane + p * a.lpr);
                    rotate<V>(gr[p], t, a.interleaved, cs, sn, -1.f);
#pragma unroll
                    for (int i = 0; i < 2 * V; ++i) {
                        v[p][i] *= r;                           // n
                        const float d = gr[p][i] * v[p][i];
                        sq[p][i] += isq ? d : 0.f;
                        sk[p][i] += isq ? 0.f : d;
                        gr[p][i] *= isq ? wq[p][i] : wk[p][i];
                        dot = __builtin_fmaf(gr[p][i], v[p][i], dot);
                    }
                }
                for (int o = 1; o < a.lpr; o <<= 1) dot += __shfl_xor(dot, o);
                dot *= inv_d;
#pragma unroll
                for (int p = 0; p < UPL; ++p) {
                    const Unit<V> t(a, lane + p * a.lpr);
#pragma unroll
                    for (int i = 0; i < 2 * V; ++i) gr[p][i] = r * (gr[p][i] - v[p][i] * dot);
                    if (t.on) store<T, V>(y + t.o1, &gr[p][0]);
                    if (t.two) store<T, V>(y + t.o2, &gr[p][V]);
                }
            }
        }
    }
    if (!BWD || a.part == nullptr) return;
    // sums of this workgroup: over the rows of a wave by exchanges, over the waves through LDS
    __syncthreads();
#pragma unroll
    for (int p = 0; p < UPL; ++p)
#pragma unroll
        for (int i = 0; i < 2 * V; ++i)
            for (int o = a.lpr; o < 64; o <<= 1) {
                sq[p][i] += __shfl_xor(sq[p][i], o);
                sk[p][i] += __shfl_xor(sk[p][i], o);
            }
    for (int w = 0; w < 4; ++w) {
        if ((tid >> 6) == w && (tid & 63) < a.lpr) {
#pragma unroll
            for (int p = 0; p < UPL; ++p) {
                const Unit<V> t(a, lane + p * a.lpr);
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) {
                    const int e = (i < V ? t.o1 + i : t.o2 + i - V);
                    if (!t.on || (i >= V && !t.two)) continue;
                    sh[e] = (w ? sh[e] : 0.f) + sq[p][i];
                    sh[a.D + e] = (w ? sh[a.D + e] : 0.f) + sk[p][i];
                }
            }
        }
        __syncthreads();
    }
    for (int i = tid; i < 2 * a.D; i += 256) a.part[(size_t)blockIdx.x * 2 * a.D + i] = sh[i];
}

// dw: the workgroups' rows of 2 D sums.  A workgroup owns 16 columns, 16 threads walk the rows of each.
__global__ __launch_bounds__(256) void weight_kernel(const float *__restrict__ part, int rows, int d, float *__restrict__ dqw, float *__restrict__ dkw)
{
    __shared__ float red[16][17];
    const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4, c = blockIdx.x * 16 + cx;
    float s = 0.f;
    if (c < 2 * d)
        for (int r = ry; r < rows; r += 16) s += part[(size_t)r * 2 * d + c];
    red[ry][cx] = s;
    __syncthreads();
    if (ry == 0 && c < 2 * d) {
        for (int r = 1; r < 16; ++r) s += red[r][cx];
        if (c < d) {
            if (dqw) dqw[c] = s;
        } else if (dkw) dkw[c - d] = s;
    }
}

// widest piece that every row start and every piece of a row is a multiple of
int piece(int dtype, int d, int pairs, int interleaved, long mask)
{
    const int most = dtype == F32 ? 4 : 8;
    const long es = dtype == F32 ? 4 : 2;
    for (int v = most; v > 1; v >>= 1)
        if (pairs % v == 0 && (d - 2 * pairs) % (2 * v) == 0 && mask % (v * es) == 0) return v;
    return 1;
}

int groups_of(long tokens, int tb) { return (int)((tokens + tb - 1) / tb < 1024 ? (tokens + tb - 1) / tb : 1024); }

// Tokens of a workgroup's turn: four rows per row slot, so that the angles are shared and loads overlap, while there are workgroups enough (four per
// CU) -- else fewer, down to one token.
int turn_tokens(long tokens, int heads, int lpr)
{
    long tb = pa_div_up(4 * (256 / lpr), heads);
    while (tb > 1 && tokens / tb < 1024) tb >>= 1;
    return tb < 1 ? 1 : tb > MAXTOK ? MAXTOK : (int)tb;
}

template <typename T, bool BWD>
void launch_norm(const NormArgs &a, int v, dim3 grid, size_t lds, hipStream_t st)
{
    if constexpr (sizeof(T) == 2) {
        if (v == 8) { hipLaunchKernelGGL((norm_kernel<T, 8, 1, BWD>), grid, dim3(256), lds, st, a); return; }
    }
    if (v == 4) hipLaunchKernelGGL((norm_kernel<T, 4, 1, BWD>), grid, dim3(256), lds, st, a);
    else if (v == 2) hipLaunchKernelGGL((norm_kernel<T, 2, 2, BWD>), grid, dim3(256), lds, st, a);
    else hipLaunchKernelGGL((norm_kernel<T, 1, 4, BWD>), grid, dim3(256), lds, st, a);
}

int norm_check(const char *name, int dtype, int b, int n, int h, int hk, int d, int axes, int per, int ptype, float eps, const void *pos, const void *freq)
{
    PA_REQUIRE(dtype >= F32 && dtype <= BF16, "%s: dtype %d is none of 0 (float32), 1 (float16), 2 (bfloat16)", name, dtype);
    PA_REQUIRE(b >= 0 && n >= 0 && h >= 0 && hk >= 0 && h + hk > 0 && h <= 65536 && hk <= 65536, "%s: bad sizes b=%d n=%d h=%d hk=%d", name, b, n, h, hk);
    PA_REQUIRE(d > 0 && d <= MAXD, "%s: head width %d is not in 1..%d", name, d, MAXD);
    PA_REQUIRE(axes >= 0 && per >= 0 && axes <= MAXD && per <= MAXD && 2 * axes * per <= d, "%s: %d axes of %d frequencies rotate more than %d elements", name, axes, per, d);
    PA_REQUIRE(axes * per == 0 || (pos && freq), "%s: null positions / frequencies", name);
    PA_REQUIRE(ptype >= 0 && ptype <= 2, "%s: position type %d is none of 0 (int32), 1 (int64), 2 (float32)", name, ptype);
    PA_REQUIRE(eps >= 0.f && eps < INFINITY, "%s: eps has to be finite and not negative", name);
    return PA_OK;
}

// fills sizes, piece width and launch shape; returns the piece width
int norm_plan(NormArgs &a, int dtype, int b, long mask)
{
    a.pairs = a.axes * a.per;
    a.tokens = (long)b * a.N;
    const int v = piece(dtype, a.D, a.pairs, a.interleaved, mask);
    a.units = pa_div_up(a.D, 2 * v);
    a.lpr = 1;
    while (a.lpr < a.units && a.lpr < 64) a.lpr <<= 1;
    a.tb = turn_tokens(a.tokens, a.H + a.Hk, a.lpr);
    return v;
}

}  // namespace

// q (b, n, h, d) and k (b, n, hk, d) with strides in elements, unit stride in d; mask: the bitwise or of every address and of every stride in bytes
static long mask_of(int es, std::initializer_list<const void *> ps, std::initializer_list<long> ss)
{
    unsigned long m = 16;
    for (const void *p : ps) m |= (unsigned long)(uintptr_t)p;
    for (long s : ss) m |= (unsigned long)(s * es);
    return (long)(m & -m);                                      // largest power of two that divides all of them
}

PA_API int pa_qk_norm_rotary(int dtype, int b, int n, int h, int hk, int d, const void *q, long qb, long qn, long qh, const void *k, long kb, long kn, long kh,
                             const void *qw, const void *kw, int w_f32, const void *pos, int ptype, long pb, const float *freq, int axes, int per, float eps,
                             int interleaved, void *q_out, void *k_out, pa_stream_t stream)
{
    int rc = norm_check("pa_qk_norm_rotary", dtype, b, n, h, hk, d, axes, per, ptype, eps, pos, freq);
    if (rc != PA_OK) return rc;
    if (b == 0 || n == 0) return PA_OK;
    PA_REQUIRE((h == 0 || (q && q_out)) && (hk == 0 || (k && k_out)), "pa_qk_norm_rotary: null tensor");
    NormArgs a = {};
    a.q = q; a.k = k; a.oq = q_out; a.ok = k_out; a.qw = qw; a.kw = kw; a.pos = pos; a.freq = freq;
    a.qb = qb; a.qn = qn; a.qh = qh; a.kb = kb; a.kn = kn; a.kh = kh; a.pb = pb;
    a.N = n; a.H = h; a.Hk = hk; a.D = d; a.axes = axes; a.per = per; a.interleaved = interleaved; a.wtype = w_f32; a.ptype = ptype; a.eps = eps;
    const int es = dtype == F32 ? 4 : 2;
    const int v = norm_plan(a, dtype, b, mask_of(es, {q, k, q_out, k_out}, {qb, qn, qh, kb, kn, kh, d}));
    const long groups = (a.tokens + a.tb - 1) / a.tb;
    PA_REQUIRE(groups < (1l << 31), "pa_qk_norm_rotary: too many workgroups");
    const size_t lds = (size_t)2 * a.tb * a.pairs * 4;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == F32) launch_norm<float, false>(a, v, dim3((unsigned)groups), lds, st);
    else if (dtype == F16) launch_norm<_Float16, false>(a, v, dim3((unsigned)groups), lds, st);
    else launch_norm<__bf16, false>(a, v, dim3((unsigned)groups), lds, st);
    PA_CHECK_LAUNCH("pa_qk_norm_rotary");
    return PA_OK;
}

PA_API long pa_qk_norm_rotary_backward_scratch_floats(int b, int n, int d) { return b <= 0 || n <= 0 || d <= 0 ? 0 : ((long)b * n < 1024 ? (long)b * n : 1024) * 2 * d; }

PA_API int pa_qk_norm_rotary_backward(int dtype, int b, int n, int h, int hk, int d, const void *q, long qb, long qn, long qh, const void *k, long kb, long kn,
                                      long kh, const void *qw, const void *kw, int w_f32, const void *pos, int ptype, long pb, const float *freq, int axes,
                                      int per, float eps, int interleaved, const void *gq, long gqb, long gqn, long gqh, const void *gk, long gkb, long gkn,
                                      long gkh, void *dq, void *dk, float *dqw, float *dkw, float *scratch, pa_stream_t stream)
{
    int rc = norm_check("pa_qk_norm_rotary_backward", dtype, b, n, h, hk, d, axes, per, ptype, eps, pos, freq);
    if (rc != PA_OK) return rc;
    if (b == 0 || n == 0) return PA_OK;
    PA_REQUIRE((h == 0 || (q && gq && dq)) && (hk == 0 || (k && gk && dk)) && (!(dqw || dkw) || scratch), "pa_qk_norm_rotary_backward: null tensor");
    NormArgs a = {};
    a.q = q; a.k = k; a.gq = gq; a.gk = gk; a.oq = dq; a.ok = dk; a.qw = qw; a.kw = kw; a.pos = pos; a.freq = freq;
    a.qb = qb; a.qn = qn; a.qh = qh; a.kb = kb; a.kn = kn; a.kh = kh; a.gqb = gqb; a.gqn = gqn; a.gqh = gqh; a.gkb = gkb; a.gkn = gkn; a.gkh = gkh; a.pb = pb;
    a.N = n; a.H = h; a.Hk = hk; a.D = d; a.axes = axes; a.per = per; a.interleaved = interleaved; a.wtype = w_f32; a.ptype = ptype; a.eps = eps;
    a.part = dqw || dkw ? scratch : nullptr;
    const int es = dtype == F32 ? 4 : 2;
    const int v = norm_plan(a, dtype, b, mask_of(es, {q, k, gq, gk, dq, dk}, {qb, qn, qh, kb, kn, kh, gqb, gqn, gqh, gkb, gkn, gkh, d}));
    const int groups = groups_of(a.tokens, a.tb);
    size_t lds = (size_t)2 * a.tb * a.pairs * 4;
    if (lds < (size_t)2 * d * 4) lds = (size_t)2 * d * 4;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == F32) launch_norm<float, true>(a, v, dim3(groups), lds, st);
    else if (dtype == F16) launch_norm<_Float16, true>(a, v, dim3(groups), lds, st);
    else launch_norm<__bf16, true>(a, v, dim3(groups), lds, st);
    if (a.part) hipLaunchKernelGGL(weight_kernel, dim3(pa_div_up(2 * d, 16)), dim3(256), 0, st, a.part, groups, d, dqw, dkw);
    PA_CHECK_LAUNCH("pa_qk_norm_rotary_backward");
    return PA_OK;
}
