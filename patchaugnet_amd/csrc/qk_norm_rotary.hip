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
// expensive part (64-bit range reduction: angles up to 2^27 keep full accuracy); a workgroup computes those of its tokens once, into LDS, for all
// query and key heads.  Everything between load and store is 32-bit, rounded once.
//
// Measured, forward / backward / weights: bf16 8 x 4096 tokens, 16 + 4 heads of 128: 75 / 129 / 5 us (336 and 503 MB: 4.5 and 3.9 TB/s; a copy: 4.9);
// float32 18 x 1024, 8 + 8 heads of 64, three axes: 28 / 47 / 4 us.  Addresses and angles once per token (64-bit products per row cost 224 us backward),
// the next row in flight.  A piece is 16 bytes wide; where the number of pairs is no multiple of that, lanes keep pieces of consecutive elements and the
// pairs are exchanged through LDS (1.5 to 3.5 TB/s); where the rows themselves do not start at 16 bytes, pieces are narrower (16-bit heads of 66, 33 pairs: 2 bytes,
// 0.7 TB/s).
//
// The weight gradients are sums over all tokens and heads: per lane in registers over a workgroup's tokens, then across the workgroup, then by a
// second launch over the workgroups' rows, always in the same order.
#include "pa_attn.h"

using pa_attn::Div;

namespace {

enum { F32 = PA_DT_F32, F16 = PA_DT_F16, BF16 = PA_DT_BF16 };
constexpr int MAXD = 512, MAXTOK = 16;
constexpr long MAXTURNS = 1l << 22;    // workgroups of the forward pass (2^30 threads); more turns go round
constexpr int MAXGROUPS = 768;         // workgroups of the backward pass: three per CU are resident at its registers, one round

struct Side {                           // the queries, or the keys
    const void *x, *g, *w;              // input, gradient of the output (backward), weights
    void *y;                            // output (forward) / input gradient (backward), contiguous
    long xb, xn, xh, gb, gn, gh;
    int heads;
    Div d;
};

struct NormArgs {
    Side side[2];
    const void *pos;
    const float *freq;
    float *part;                        // (workgroups, 2, D) partial weight gradients
    long pb;
    int tokens, N, D, axes, per, pairs, interleaved, wtype, ptype;
    int exchange, pitch;                // pairs exchanged through LDS; angles of a token in LDS
    int tb, units, lpr;                 // tokens of a workgroup's turn, units of a row, lanes of a row (a power of two)
    float eps;
    Div dn, dpairs, dper;
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
    // x and x / (pi / 2) are each rounded at 2^-53 of their size: the angle is off by 2^-52 |x|, less than 32 bits resolve up to |x| = 2^27
    const float f = (float)(q - n);
    float s, c;
    sincospif(0.5f * f, &s, &c);
    const int k = (int)(n - 4.0 * __builtin_floor(n * 0.25));
    return k == 0 ? make_float2(c, s) : k == 1 ? make_float2(-s, c) : k == 2 ? make_float2(-c, -s) : make_float2(s, -c);
}

template <typename T, int V> struct Vec {
    typedef T type __attribute__((ext_vector_type(V)));
    __device__ static __forceinline__ float get(const type &v, int i) { return (float)v[i]; }
    __device__ static __forceinline__ void set(type &v, int i, float x) { v[i] = (T)x; }
};
template <typename T> struct Vec<T, 1> {
    typedef T type;
    __device__ static __forceinline__ float get(const type &v, int) { return (float)v; }
    __device__ static __forceinline__ void set(type &v, int, float x) { v = (T)x; }
};
template <typename T, int V> __device__ __forceinline__ void store(T *p, const float *x)
{
    typename Vec<T, V>::type v;
#pragma unroll
    for (int i = 0; i < V; ++i) Vec<T, V>::set(v, i, x[i]);
    *reinterpret_cast<typename Vec<T, V>::type *>(p) = v;
}

// A row as units of two V-element pieces: the pairs' two halves, then the unrotated rest.  The last piece of an odd rest does not exist (V = 1 only).
template <int V, bool EX> struct Unit {
    int o1, o2, pair;                   // pair < 0: not rotated
    bool on, two;

    __device__ __forceinline__ Unit(const NormArgs &a, int u)
    {
        const int rot = EX ? 0 : a.pairs / V;
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

template <int V> __device__ __forceinline__ void rotate(float *x, const Unit<V, false> &t, int interleaved, const float *cs, const float *sn, float sign)
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

// Place of element (or pair) e in LDS: lanes read 2 V apart, the skip spreads them over the banks.
__device__ __forceinline__ int skip(int e) { return e + (e >> 4); }

// The rotation where the pairs' second halves do not start at a whole piece: lanes keep pieces of consecutive elements, every element's partner comes
// through the row's place in LDS.  A row is a wave's own, so LDS serves its stores and loads in order: first the pieces of all its units, then the partners
// (a partner may lie in another unit of a lane).
template <int V, int UPL> __device__ __forceinline__ void exchange(float (&x)[UPL][2 * V], const NormArgs &a, int lane, float *row, const float *cs, const float *sn, float sign)
{
#pragma unroll
    for (int p = 0; p < UPL; ++p) {
        const Unit<V, true> t(a, lane + p * a.lpr);
        int e0 = t.o1;
        asm volatile("" : "+v"(e0));                            // the places are worked out here, not kept for 2 V elements over all rows
        if (t.on) {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) row[skip(e0 + i)] = x[p][i];
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
    for (int p = 0; p < UPL; ++p) {
        const Unit<V, true> t(a, lane + p * a.lpr);
        int e0 = t.o1;
        asm volatile("" : "+v"(e0));
        if (t.on) {
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) {
                const int e = e0 + i;
                const bool first = a.interleaved ? (e & 1) == 0 : e < a.pairs;
                const int other = a.interleaved ? e ^ 1 : first ? e + a.pairs : e - a.pairs, pr = a.interleaved ? e >> 1 : first ? e : other;
                if (e < 2 * a.pairs) {
                    const float y = row[skip(other)], c = cs[skip(pr)], s = sign * sn[skip(pr)];
                    x[p][i] = first ? x[p][i] * c - y * s : y * s + x[p][i] * c;
                }
            }
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// 1 / sqrt(x), 2^-126 <= x < 2^127: v_rsq_f32 and a Newton step
__device__ __forceinline__ float rsqrt32(float x)
{
    const float r = __builtin_amdgcn_rsqf(x);
    return r * __builtin_fmaf(-0.5f * x * r, r, 1.5f);
}

// The rows of one side in a workgroup's turn of nt tokens from t0: row slot by row slot, the next one fetched while this one is computed.  where:
// offsets of the turn's tokens in x and in g; cos, sin: their angles.  acc: this lane's sums for the weights' gradient.
template <typename T, int V, int UPL, bool BWD, bool EX>
__device__ __forceinline__ void side_rows(const NormArgs &a, const Side &sd, int t0, int nt, const long *where, const float *cos, const float *sin, float *mine,
                                          const float (&w)[UPL][2 * V], float (&acc)[BWD ? UPL : 1][2 * V])
{
    typedef typename Vec<T, V>::type P;
    const int tid = threadIdx.x, lane = tid & (a.lpr - 1), slot = tid / a.lpr, slots = 256 / a.lpr, rows = nt * sd.heads;
    const float inv_d = 1.0f / (float)a.D;
    struct Row {
        P x[UPL][2], g[BWD ? UPL : 1][2];
        T *y;
        int tok;
    } cur, nxt;
    auto fetch = [&](Row &r, int row) {
        r.tok = sd.d.div(row);
        const int hd = row - r.tok * sd.heads;
        const T *x = (const T *)sd.x + where[r.tok] + hd * sd.xh, *dy = BWD ? (const T *)sd.g + where[MAXTOK + r.tok] + hd * sd.gh : nullptr;
        r.y = (T *)sd.y + ((long)t0 * sd.heads + row) * a.D;
#pragma unroll
        for (int p = 0; p < UPL; ++p) {
            const Unit<V, EX> t(a, lane + p * a.lpr);
            r.x[p][0] = r.x[p][1] = 0;
            if (t.on) r.x[p][0] = *reinterpret_cast<const P *>(x + t.o1);
            if (t.two) r.x[p][1] = *reinterpret_cast<const P *>(x + t.o2);
            if (BWD) {
                r.g[p][0] = r.g[p][1] = 0;
                if (t.on) r.g[p][0] = *reinterpret_cast<const P *>(dy + t.o1);
                if (t.two) r.g[p][1] = *reinterpret_cast<const P *>(dy + t.o2);
            }
        }
    };
    if (slot < rows) fetch(cur, slot);
    for (int row = slot; row < rows; row += slots) {
        if (row + slots < rows) fetch(nxt, row + slots);
        float v[UPL][2 * V], gr[BWD ? UPL : 1][2 * V], ss = 0.f;
        const float *cs = cos + cur.tok * a.pitch, *sn = sin + cur.tok * a.pitch;
#pragma unroll
        for (int p = 0; p < UPL; ++p)
#pragma unroll
            for (int i = 0; i < 2 * V; ++i) {
                v[p][i] = Vec<T, V>::get(cur.x[p][i / V], i % V);
                if (BWD) gr[p][i] = Vec<T, V>::get(cur.g[p][i / V], i % V);
                ss = __builtin_fmaf(v[p][i], v[p][i], ss);
            }
        for (int o = 1; o < a.lpr; o <<= 1) ss += __shfl_xor(ss, o);
        float mean = __builtin_fmaf(ss, inv_d, a.eps), r = rsqrt32(mean);
        if (!(mean >= 0x1p-100f && mean < 0x1p126f)) {          // squares that leave 32 bits: the root from the row times a power of two
            const float lift = mean < 1.f ? 0x1p100f : 0x1p-75f;
            ss = 0.f;
#pragma unroll
            for (int p = 0; p < UPL; ++p)
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) {
                    const float y = v[p][i] * lift;
                    ss = __builtin_fmaf(y, y, ss);
                }
            for (int o = 1; o < a.lpr; o <<= 1) ss += __shfl_xor(ss, o);
            mean = __builtin_fmaf(ss, inv_d, a.eps * lift * lift);
            r = mean == INFINITY ? 0.f : rsqrt32(mean) * lift;
        }
        if (!BWD) {
#pragma unroll
            for (int p = 0; p < UPL; ++p)
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) v[p][i] = v[p][i] * r * w[p][i];
            if constexpr (EX) exchange<V>(v, a, lane, mine, cs, sn, 1.f);
#pragma unroll
            for (int p = 0; p < UPL; ++p) {
                const Unit<V, EX> t(a, lane + p * a.lpr);
                if constexpr (!EX) rotate<V>(v[p], t, a.interleaved, cs, sn, 1.f);
                if (t.on) store<T, V>(cur.y + t.o1, &v[p][0]);
                if (t.two) store<T, V>(cur.y + t.o2, &v[p][V]);
            }
        } else {
            float dot = 0.f;
            if constexpr (EX) exchange<V>(gr, a, lane, mine, cs, sn, -1.f);
#pragma unroll
            for (int p = 0; p < UPL; ++p) {
                const Unit<V, EX> t(a, lane + p * a.lpr);
                if constexpr (!EX) rotate<V>(gr[p], t, a.interleaved, cs, sn, -1.f);
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) {
                    v[p][i] *= r;                               // n
                    acc[p][i] = __builtin_fmaf(gr[p][i], v[p][i], acc[p][i]);
                    gr[p][i] *= w[p][i];
                    dot = __builtin_fmaf(gr[p][i], v[p][i], dot);
                }
            }
            for (int o = 1; o < a.lpr; o <<= 1) dot += __shfl_xor(dot, o);
            dot *= inv_d;
#pragma unroll
            for (int p = 0; p < UPL; ++p) {
                const Unit<V, EX> t(a, lane + p * a.lpr);
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) gr[p][i] = r * __builtin_fmaf(-v[p][i], dot, gr[p][i]);
                if (t.on) store<T, V>(cur.y + t.o1, &gr[p][0]);
                if (t.two) store<T, V>(cur.y + t.o2, &gr[p][V]);
            }
        }
        cur = nxt;
    }
}

// UPL: units a lane can hold (1 for the wide pieces, up to 4 for the narrow ones: 64 lanes x 4 units x 2 elements = MAXD)
template <typename T, int V, int UPL, bool BWD, bool EX>
__global__ __launch_bounds__(256, BWD ? 3 : 4) void norm_kernel(const NormArgs a)
{
    extern __shared__ __attribute__((aligned(16))) float sh[];       // [tb][pitch] cosines, [tb][pitch] sines, exchanges; backward: then the join of 2 D sums
    __shared__ long where[2][2][MAXTOK];
    const int tid = threadIdx.x, lane = tid & (a.lpr - 1);
    float *mine = sh + 2 * a.tb * a.pitch + tid / a.lpr * (skip(a.D) + 1);       // this row slot's place for exchanges
    float w[2][UPL][2 * V], acc[2][BWD ? UPL : 1][2 * V];
#pragma unroll
    for (int p = 0; p < UPL; ++p) {
        const Unit<V, EX> t(a, lane + p * a.lpr);
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) {
            const int e = (i < V ? t.o1 + i : t.o2 + i - V);
            const bool in = t.on && (i < V || t.two);
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                w[s][p][i] = in ? weight_at<T>(a.side[s].w, a.wtype, e) : 0.f;
                if (BWD) acc[s][p][i] = 0.f;
            }
        }
    }
    for (int t0 = blockIdx.x * a.tb; t0 < a.tokens; t0 += gridDim.x * a.tb) {
        const int nt = min(a.tokens - t0, a.tb);
        if (t0 != (int)blockIdx.x * a.tb) __syncthreads();      // readers of the previous turn's table and angles
        if (tid < 4 * MAXTOK && (tid & (MAXTOK - 1)) < nt) {
            const int s = tid / (2 * MAXTOK), g = tid / MAXTOK & 1, tok = tid & (MAXTOK - 1), b = a.dn.div(t0 + tok), n = t0 + tok - b * a.N;
            const Side &sd = s ? a.side[1] : a.side[0];
            where[s][g][tok] = g ? b * sd.gb + n * sd.gn : b * sd.xb + n * sd.xn;
        }
        for (int i = tid; i < nt * a.pairs; i += 256) {
            const int tok = a.dpairs.div(i), pr = i - tok * a.pairs, at = t0 + tok, b = a.dn.div(at);
            const float2 cs = turn(position_at(a, b, at - b * a.N, a.dper.div(pr)) * (double)a.freq[pr]);
            const int at_pr = tok * a.pitch + (EX ? skip(pr) : pr);
            sh[at_pr] = cs.x;
            sh[a.tb * a.pitch + at_pr] = cs.y;
        }
        __syncthreads();
        side_rows<T, V, UPL, BWD, EX>(a, a.side[0], t0, nt, where[0][0], sh, sh + a.tb * a.pitch, mine, w[0], acc[0]);
        side_rows<T, V, UPL, BWD, EX>(a, a.side[1], t0, nt, where[1][0], sh, sh + a.tb * a.pitch, mine, w[1], acc[1]);
    }
    if (!BWD || a.part == nullptr) return;
    // sums of this workgroup: over the rows of a wave by exchanges, over the waves through LDS
    __syncthreads();
#pragma unroll
    for (int p = 0; p < UPL; ++p)
#pragma unroll
        for (int i = 0; i < 2 * V; ++i)
            for (int o = a.lpr; o < 64; o <<= 1) {
                acc[0][p][i] += __shfl_xor(acc[0][p][i], o);
                acc[1][p][i] += __shfl_xor(acc[1][p][i], o);
            }
    for (int w = 0; w < 4; ++w) {
        if ((tid >> 6) == w && (tid & 63) < a.lpr) {
#pragma unroll
            for (int p = 0; p < UPL; ++p) {
                const Unit<V, EX> t(a, lane + p * a.lpr);
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) {
                    const int e = (i < V ? t.o1 + i : t.o2 + i - V);
                    if (!t.on || (i >= V && !t.two)) continue;
                    sh[e] = (w ? sh[e] : 0.f) + acc[0][p][i];
                    sh[a.D + e] = (w ? sh[a.D + e] : 0.f) + acc[1][p][i];
                }
            }
        }
        __syncthreads();
    }
    for (int i = tid; i < 2 * a.D; i += 256) a.part[(size_t)blockIdx.x * 2 * a.D + i] = sh[i];
}

// dw: the workgroups' rows of 2 D sums.  A workgroup owns 16 columns, 64 threads walk the rows of each.
__global__ __launch_bounds__(1024) void weight_kernel(const float *__restrict__ part, int rows, int d, float *__restrict__ dqw, float *__restrict__ dkw)
{
    __shared__ float red[64][17];
    const int cx = threadIdx.x & 15, ry = threadIdx.x >> 4, c = blockIdx.x * 16 + cx;
    float s = 0.f;
    if (c < 2 * d) {
#pragma unroll 4
        for (int r = ry; r < rows; r += 64) s += part[(size_t)r * 2 * d + c];
    }
    red[ry][cx] = s;
    __syncthreads();
    if (ry < 4) {
        s = 0.f;
        for (int r = 0; r < 16; ++r) s += red[ry * 16 + r][cx];
    }
    __syncthreads();
    if (ry < 4) red[ry][cx] = s;
    __syncthreads();
    if (ry == 0 && c < 2 * d) {
        s = (red[0][cx] + red[1][cx]) + (red[2][cx] + red[3][cx]);
        if (c < d) {
            if (dqw) dqw[c] = s;
        } else if (dkw) dkw[c - d] = s;
    }
}

// Widest piece that every row start is a multiple of and a row (pairs: their two halves and the rest) consists of.
int piece(int dtype, int d, int pairs, long align)
{
    const int most = dtype == F32 ? 4 : 8;
    const long es = dtype == F32 ? 4 : 2;
    for (int v = most; v > 1; v >>= 1)
        if (pairs % v == 0 && (d - 2 * pairs) % (2 * v) == 0 && align % (v * es) == 0) return v;
    return 1;
}

// Tokens of a workgroup's turn: ten rows per row slot, so that the angles and the barriers are shared and loads overlap, while there are workgroups
// enough (four per CU) -- else fewer, down to one token.  Backward: turns of one size that deal the tokens evenly to the resident workgroups.
int turn_tokens(long tokens, int heads, int lpr, bool bwd)
{
    long tb = pa_div_up(10 * (256 / lpr), heads);
    tb = tb > MAXTOK ? MAXTOK : tb;
    if (bwd) {
        const long each = (tokens + MAXGROUPS - 1) / MAXGROUPS, turns = (each + tb - 1) / tb;
        return (int)((each + turns - 1) / turns);
    }
    while (tb > 1 && tokens / tb < 1024) tb >>= 1;
    return (int)tb;
}

int groups_of(long tokens, int tb) { return (int)((tokens + tb - 1) / tb < MAXGROUPS ? (tokens + tb - 1) / tb : MAXGROUPS); }

template <typename T, bool BWD, bool EX>
void launch_pieces(const NormArgs &a, int v, dim3 grid, size_t lds, hipStream_t st)
{
    if constexpr (sizeof(T) == 2) {
        if (v == 8) { hipLaunchKernelGGL((norm_kernel<T, 8, 1, BWD, EX>), grid, dim3(256), lds, st, a); return; }
    }
    if (v == 4) hipLaunchKernelGGL((norm_kernel<T, 4, 1, BWD, EX>), grid, dim3(256), lds, st, a);
    else if (v == 2) hipLaunchKernelGGL((norm_kernel<T, 2, 2, BWD, EX>), grid, dim3(256), lds, st, a);
    else if constexpr (!EX) hipLaunchKernelGGL((norm_kernel<T, 1, 4, BWD, EX>), grid, dim3(256), lds, st, a);
}

template <typename T, bool BWD>
void launch_norm(const NormArgs &a, int v, dim3 grid, size_t lds, hipStream_t st)
{
    if (a.exchange) launch_pieces<T, BWD, true>(a, v, grid, lds, st);
    else launch_pieces<T, BWD, false>(a, v, grid, lds, st);
}

int norm_check(const char *name, int dtype, int b, int n, int h, int hk, int d, int axes, int per, int ptype, float eps, const void *pos, const void *freq)
{
    PA_REQUIRE(dtype >= F32 && dtype <= BF16, "%s: dtype %d is none of 0 (float32), 1 (float16), 2 (bfloat16)", name, dtype);
    PA_REQUIRE(b >= 0 && n >= 0 && h >= 0 && hk >= 0 && h + hk > 0 && h <= 65536 && hk <= 65536, "%s: bad sizes b=%d n=%d h=%d hk=%d", name, b, n, h, hk);
    PA_REQUIRE((long)b * n <= (1l << 30), "%s: %ld tokens exceed 2^30", name, (long)b * n);
    PA_REQUIRE(d > 0 && d <= MAXD, "%s: head width %d is not in 1..%d", name, d, MAXD);
    PA_REQUIRE(axes >= 0 && per >= 0 && axes <= MAXD && per <= MAXD && 2 * axes * per <= d, "%s: %d axes of %d frequencies rotate more than %d elements", name, axes, per, d);
    PA_REQUIRE(axes * per == 0 || (pos && freq), "%s: null positions / frequencies", name);
    PA_REQUIRE(ptype >= 0 && ptype <= 2, "%s: position type %d is none of 0 (int32), 1 (int64), 2 (float32)", name, ptype);
    PA_REQUIRE(eps >= 0.f && eps < INFINITY, "%s: eps has to be finite and not negative", name);
    return PA_OK;
}

// fills sizes, piece width and launch shape; returns the piece width
int norm_plan(NormArgs &a, int dtype, int b, bool bwd, long mask)
{
    a.pairs = a.axes * a.per;
    a.tokens = (int)((long)b * a.N);
    a.dn = Div(a.N > 0 ? a.N : 1);
    for (Side &s : a.side) s.d = Div(s.heads > 0 ? s.heads : 1);
    a.dpairs = Div(a.pairs > 0 ? a.pairs : 1);
    a.dper = Div(a.per > 0 ? a.per : 1);
    // Narrow pieces waste the memory's width: where whole rows allow wider ones, the pairs are exchanged through LDS instead (fp16 8 x 2048 tokens, 20
    // heads of 96, 17 pairs: forward 130 -> 65 us, with gradients 361 -> 165; heads of 128, 21 pairs: 123 -> 63, 369 -> 167).
    int v = piece(dtype, a.D, a.pairs, mask);
    const int whole = piece(dtype, a.D, 0, mask);
    a.exchange = whole > v;
    if (a.exchange) v = whole;
    a.pitch = a.exchange ? a.pairs + a.pairs / 16 + 1 : a.pairs;
    a.units = pa_div_up(a.D, 2 * v);
    a.lpr = 1;
    while (a.lpr < a.units && a.lpr < 64) a.lpr <<= 1;
    a.tb = turn_tokens(a.tokens, a.side[0].heads + a.side[1].heads, a.lpr, bwd);
    return v;
}

size_t lds_of(const NormArgs &a) { return ((size_t)2 * a.tb * a.pitch + (a.exchange ? (256 / a.lpr) * (a.D + a.D / 16 + 1) : 0)) * 4; }

}  // namespace

PA_API int pa_qk_norm_rotary(int dtype, int b, int n, int h, int hk, int d, const void *q, long qb, long qn, long qh, const void *k, long kb, long kn, long kh,
                             const void *qw, const void *kw, int w_f32, const void *pos, int ptype, long pb, const float *freq, int axes, int per, float eps,
                             int interleaved, void *q_out, void *k_out, pa_stream_t stream)
{
    int rc = norm_check("pa_qk_norm_rotary", dtype, b, n, h, hk, d, axes, per, ptype, eps, pos, freq);
    if (rc != PA_OK) return rc;
    if (b == 0 || n == 0) return PA_OK;
    PA_REQUIRE((h == 0 || (q && q_out)) && (hk == 0 || (k && k_out)), "pa_qk_norm_rotary: null tensor");
    NormArgs a = {};
    a.side[0] = {q, nullptr, qw, q_out, qb, qn, qh, 0, 0, 0, h, Div()};
    a.side[1] = {k, nullptr, kw, k_out, kb, kn, kh, 0, 0, 0, hk, Div()};
    a.pos = pos; a.freq = freq; a.pb = pb;
    a.N = n; a.D = d; a.axes = axes; a.per = per; a.interleaved = interleaved; a.wtype = w_f32; a.ptype = ptype; a.eps = eps;
    const int es = dtype == F32 ? 4 : 2;
    const int v = norm_plan(a, dtype, b, false, alignment_of(es, {q, k, q_out, k_out}, {qb, qn, qh, kb, kn, kh, d}));
    const long turns = (a.tokens + a.tb - 1) / a.tb, groups = turns < MAXTURNS ? turns : MAXTURNS;
    const size_t lds = lds_of(a);
    hipStream_t st = (hipStream_t)stream;
    if (dtype == F32) launch_norm<float, false>(a, v, dim3((unsigned)groups), lds, st);
    else if (dtype == F16) launch_norm<_Float16, false>(a, v, dim3((unsigned)groups), lds, st);
    else launch_norm<__bf16, false>(a, v, dim3((unsigned)groups), lds, st);
    PA_CHECK_LAUNCH("pa_qk_norm_rotary");
    return PA_OK;
}

PA_API long pa_qk_norm_rotary_backward_scratch_floats(int b, int n, int d) { return b <= 0 || n <= 0 || d <= 0 ? 0 : ((long)b * n < MAXGROUPS ? (long)b * n : MAXGROUPS) * 2 * d; }

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
    a.side[0] = {q, gq, qw, dq, qb, qn, qh, gqb, gqn, gqh, h, Div()};
    a.side[1] = {k, gk, kw, dk, kb, kn, kh, gkb, gkn, gkh, hk, Div()};
    a.pos = pos; a.freq = freq; a.pb = pb;
    a.N = n; a.D = d; a.axes = axes; a.per = per; a.interleaved = interleaved; a.wtype = w_f32; a.ptype = ptype; a.eps = eps;
    a.part = dqw || dkw ? scratch : nullptr;
    const int es = dtype == F32 ? 4 : 2;
    const int v = norm_plan(a, dtype, b, true, alignment_of(es, {q, k, gq, gk, dq, dk}, {qb, qn, qh, kb, kn, kh, gqb, gqn, gqh, gkb, gkn, gkh, d}));
    const int groups = groups_of(a.tokens, a.tb);
    size_t lds = lds_of(a);
    if (lds < (size_t)2 * d * 4) lds = (size_t)2 * d * 4;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == F32) launch_norm<float, true>(a, v, dim3(groups), lds, st);
    else if (dtype == F16) launch_norm<_Float16, true>(a, v, dim3(groups), lds, st);
    else launch_norm<__bf16, true>(a, v, dim3(groups), lds, st);
    if (a.part) hipLaunchKernelGGL(weight_kernel, dim3(pa_div_up(2 * d, 16)), dim3(1024), 0, st, a.part, groups, d, dqw, dkw);
    PA_CHECK_LAUNCH("pa_qk_norm_rotary_backward");
    return PA_OK;
}
