// urnn_norm.hip -- the norms around a block in one pass, forward and backward.  Per row of D channels:
//   p  = act(g) * (y * ry) * w,   ry = 1 / sqrt(mean(y^2) + eps)        the norm after the block and its gate
//   r' = r + s * p                                                      the residual with its scale
//   n  = r' * rr * v,             rr = 1 / sqrt(mean(r'^2) + eps)       the norm before the next block
// without w there is no first norm (ry = 1), without g, r or s that factor or term is left out.
// Backward, with t = dn v, hat = r' rr, yh = y ry:
//   dr = dr' + rr (t - hat mean(t hat)),  dp = s dr,  q = dp act(g) w,  dy = ry (q - yh mean(q yh)),  dg = dp yh w act'(g),
//   dv = sum_rows dn hat,  dw = sum_rows dp act(g) yh,  ds = sum_rows dr p.
//
// Memory-bound.  A row lives in the registers of NT threads, EPT values each, so that everything is read once and both means are
// taken on the way: NT = 16 (D <= 128), 64 (<= 512), 128, 256, 512, 1024, eight values to a thread (sixteen beyond 8192 channels;
// sixteen at half the threads: 8192 x 4096 77 us against 70, fewer waves wait for memory).  The backward reads y, g, r again instead
// of r' and the forward's statistics: r' was rounded on its way out, and it is as many bytes.  Its column sums stay in registers over
// all rows of a block and are folded in a fixed order.  8192 x 4096 bf16: 70 us, 4.8 TB/s.
//
// Widths that no 16 bytes divide take the same accesses at the element's alignment; a row's last group is its last V elements moved
// down in registers, so that no branch makes one load wait for another.  12 345 x 1001 fp32 50 us, with the backward 126, 5.1 TB/s (element
// by element 139); 8192 x 2001 bf16 43 us, with the backward 120 (element by element 80 and 298; with a branch at the last group 59
// and 143; x 2000 35 and 107).
#include "urnn_seq.h"

enum { ACT_NONE = 0, ACT_SIGMOID = 1, ACT_SILU = 2 };

template <int NT>
__device__ __forceinline__ void row_sum2(float &a, float &b, float (*red)[2])
{
    float v[2] = {a, b};
    if (NT == 16) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            v[i] += dpp_move<0xB1>(v[i]);
            v[i] += dpp_move<0x4E>(v[i]);
            v[i] += dpp_move<0x141>(v[i]);
            v[i] += dpp_move<0x140>(v[i]);
        }
    } else {
        wave_sum_n<2>(v);
        if (NT > 64) {                               // red: this reduction's own pair of every wave; the caller's next ones use others
            if ((threadIdx.x & 63) == 0) { red[threadIdx.x >> 6][0] = v[0]; red[threadIdx.x >> 6][1] = v[1]; }
            __syncthreads();
            const int first = threadIdx.x / NT * (NT / 64);
            v[0] = v[1] = 0.0f;
#pragma unroll
            for (int w = 0; w < NT / 64; ++w) { v[0] += red[first + w][0]; v[1] += red[first + w][1]; }
        }
    }
    a = v[0];
    b = v[1];
}

// act(g) and act'(g)
__device__ __forceinline__ void gate_of(int act, float g, float &a, float &da)
{
    if (act == ACT_NONE) { a = g; da = 1.0f; return; }
    const float s = sigmoid_f(g);
    if (act == ACT_SIGMOID) { a = s; da = s * (1.0f - s); return; }
    a = g * s;
    da = s * fmaf(g, 1.0f - s, 1.0f);
}

// Values of a thread: EPT / V groups of V adjacent channels, NT V apart.
template <typename T>
__device__ __forceinline__ const T *row_at(const void *base, const SeqStride &s, long row, unsigned inner)
{
    const unsigned r = (unsigned)row;                // fewer than 2^28 rows
    return reinterpret_cast<const T *>(base) + (long)(r / inner) * s.b + (long)(r % inner) * s.t;
}
// WIDE: rows start on 16 bytes and hold whole groups; otherwise a row holds one group at least (or V is 1).
template <typename T, int V, int NT, int EPT, bool WIDE>
__device__ __forceinline__ void row_load(const T *row, int ln, int D, float (&v)[EPT])
{
#pragma unroll
    for (int c = 0; c < EPT / V; ++c) {
        const int d = (c * NT + ln) * V;
        Pack<T, V> t = {};
        if constexpr (!WIDE) t = load_tail<T, V>(row, d, D);
        else if (d < D) t = *reinterpret_cast<const Pack<T, V> *>(row + d);
#pragma unroll
        for (int i = 0; i < V; ++i) v[c * V + i] = to_f(t.v[i]);
    }
}
template <typename T, int V, int NT, int EPT, bool WIDE>
__device__ __forceinline__ void row_store(T *row, int ln, int D, const float (&v)[EPT])
{
#pragma unroll
    for (int c = 0; c < EPT / V; ++c) {
        const int d = (c * NT + ln) * V;
        Pack<T, V> t;
#pragma unroll
        for (int i = 0; i < V; ++i) t.v[i] = from_f<T>(v[c * V + i]);
        if constexpr (!WIDE) store_tail<T, V>(row, t, d, D);
        else if (d < D) stream_store(row + d, t);
    }
}
// A parameter (fp32): in groups of at most four
template <int V, int NT, int EPT, bool WIDE>
__device__ __forceinline__ void par_load(const float *w, int ln, int D, float fill, float (&v)[EPT])
{
    constexpr int W = V % 4 == 0 ? 4 : 1;
#pragma unroll
    for (int c = 0; c < EPT / V; ++c)
#pragma unroll
        for (int k = 0; k < V; k += W) {
            const int d = (c * NT + ln) * V + k;
            Pack<float, W> t;
#pragma unroll
            for (int i = 0; i < W; ++i) t.v[i] = fill;
            if constexpr (!WIDE) {
                if (w) t = load_tail<float, W>(w, d, D);
            } else if (w && d < D) t = *reinterpret_cast<const Pack<float, W> *>(w + d);
#pragma unroll
            for (int i = 0; i < W; ++i) v[c * V + k + i] = t.v[i];
        }
}

template <int V, int NT, int EPT, bool WIDE>
__device__ __forceinline__ void par_store(float *w, int ln, int D, const float (&v)[EPT])
{
    constexpr int W = V % 4 == 0 ? 4 : 1;
#pragma unroll
    for (int c = 0; c < EPT / V; ++c)
#pragma unroll
        for (int k = 0; k < V; k += W) {
            const int d = (c * NT + ln) * V + k;
            Pack<float, W> t;
#pragma unroll
            for (int i = 0; i < W; ++i) t.v[i] = v[c * V + k + i];
            if constexpr (!WIDE) store_tail<float, W>(w, t, d, D);
            else if (d < D) *reinterpret_cast<Pack<float, W> *>(w + d) = t;
        }
}

template <typename T, int V, int NT, int EPT, bool WIDE>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void norm_kernel(const NormParams p)
{
    __shared__ float red[2][NT < 256 ? 4 : NT / 64][2];
    constexpr int RB = NT < 256 ? 256 / NT : 1;
    const int ln = threadIdx.x % NT, D = p.dim;
    const long row0 = (long)blockIdx.x * RB + threadIdx.x / NT;
    const bool ok = row0 < p.rows;
    const long row = ok ? row0 : 0;
    const float inv = 1.0f / (float)D;
    float y[EPT], r[EPT], w[EPT], s[EPT], v[EPT];
    row_load<T, V, NT, EPT, WIDE>(row_at<T>(p.y, p.sy, row, p.inner), ln, D, y);
#pragma unroll
    for (int i = 0; i < EPT; ++i) r[i] = 0.0f;
    if (p.residual) row_load<T, V, NT, EPT, WIDE>(row_at<T>(p.residual, p.sr, row, p.inner), ln, D, r);
    float g[EPT];
    if (p.gate) row_load<T, V, NT, EPT, WIDE>(row_at<T>(p.gate, p.sg, row, p.inner), ln, D, g);
    par_load<V, NT, EPT, WIDE>(p.post_w, ln, D, 1.0f, w);
    par_load<V, NT, EPT, WIDE>(p.scale, ln, D, 1.0f, s);
    par_load<V, NT, EPT, WIDE>(p.pre_w, ln, D, 0.0f, v);
    float ss = 0.0f, none = 0.0f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) ss = fmaf(y[i], y[i], ss);
    row_sum2<NT>(ss, none, red[0]);
    const float ry = p.post_w ? __builtin_amdgcn_rsqf(fmaf(ss, inv, p.eps)) : 1.0f;
    ss = 0.0f;
#pragma unroll
    for (int i = 0; i < EPT; ++i) {
        float q = y[i] * ry * w[i];
        if (p.gate) {
            float a, da;
            gate_of(p.act, g[i], a, da);
            q *= a;
        }
        r[i] = fmaf(s[i], q, r[i]);
        ss = fmaf(r[i], r[i], ss);
    }
    row_sum2<NT>(ss, none, red[1]);
    const float rr = __builtin_amdgcn_rsqf(fmaf(ss, inv, p.eps));
    if (!ok) return;
    if (p.res_out) row_store<T, V, NT, EPT, WIDE>(reinterpret_cast<T *>(p.res_out) + row * D, ln, D, r);
#pragma unroll
    for (int i = 0; i < EPT; ++i) r[i] *= rr * v[i];
    row_store<T, V, NT, EPT, WIDE>(reinterpret_cast<T *>(p.normed) + row * D, ln, D, r);
}

template <typename T, int V, int NT, int EPT, bool WIDE>
__global__ __launch_bounds__(NT < 256 ? 256 : NT) void norm_backward_kernel(const NormParams p)
{
    __shared__ float red[3][NT < 256 ? 4 : NT / 64][2];
    constexpr int RB = NT < 256 ? 256 / NT : 1;
    __shared__ float fold[RB > 1 ? 256 * EPT : 1];
    const int ln = threadIdx.x % NT, rg = threadIdx.x / NT, D = p.dim;
    const float inv = 1.0f / (float)D;
    float w[EPT], s[EPT], v[EPT], cv[EPT] = {}, cw[EPT] = {}, cs[EPT] = {};
    par_load<V, NT, EPT, WIDE>(p.post_w, ln, D, 1.0f, w);
    par_load<V, NT, EPT, WIDE>(p.scale, ln, D, 1.0f, s);
    par_load<V, NT, EPT, WIDE>(p.pre_w, ln, D, 0.0f, v);
    for (long base = (long)blockIdx.x * RB; base < p.rows; base += (long)gridDim.x * RB) {
        const long row0 = base + rg;
        const bool ok = row0 < p.rows;
        const long row = ok ? row0 : base;
        float y[EPT], r[EPT], g[EPT], dn[EPT], dr[EPT], a[EPT], da[EPT];
        row_load<T, V, NT, EPT, WIDE>(row_at<T>(p.y, p.sy, row, p.inner), ln, D, y);
#pragma unroll
        for (int i = 0; i < EPT; ++i) { r[i] = dn[i] = dr[i] = 0.0f; a[i] = 1.0f; da[i] = 0.0f; }
        if (p.residual) row_load<T, V, NT, EPT, WIDE>(row_at<T>(p.residual, p.sr, row, p.inner), ln, D, r);
        if (p.gate) row_load<T, V, NT, EPT, WIDE>(row_at<T>(p.gate, p.sg, row, p.inner), ln, D, g);
        if (p.dnormed) row_load<T, V, NT, EPT, WIDE>(row_at<T>(p.dnormed, p.sdn, row, p.inner), ln, D, dn);
        if (p.dres) row_load<T, V, NT, EPT, WIDE>(row_at<T>(p.dres, p.sdr, row, p.inner), ln, D, dr);
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < EPT; ++i) s1 = fmaf(y[i], y[i], s1);
        row_sum2<NT>(s1, s2, red[0]);
        const float ry = p.post_w ? __builtin_amdgcn_rsqf(fmaf(s1, inv, p.eps)) : 1.0f;
        s1 = s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            if (p.gate) gate_of(p.act, g[i], a[i], da[i]);
            y[i] *= ry;                                          // yh
            g[i] = a[i] * y[i];                                  // act(g) yh; p = g w
            r[i] = fmaf(s[i] * w[i], g[i], r[i]);                // r'
            s1 = fmaf(r[i], r[i], s1);
            s2 = fmaf(dn[i] * v[i], r[i], s2);
        }
        row_sum2<NT>(s1, s2, red[1]);
        const float rr = __builtin_amdgcn_rsqf(fmaf(s1, inv, p.eps)), m1 = s2 * inv * rr;
        s1 = s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < EPT; ++i) {
            const float hat = r[i] * rr;
            dr[i] += rr * fmaf(-hat, m1, dn[i] * v[i]);
            if (ok) {
                cv[i] = fmaf(dn[i], hat, cv[i]);
                cw[i] = fmaf(dr[i] * s[i], g[i], cw[i]);
                cs[i] = fmaf(dr[i], g[i] * w[i], cs[i]);
            }
            const float dpw = dr[i] * s[i] * w[i];
            r[i] = dpw * a[i];                                   // q
            da[i] *= dpw * y[i];                                 // dg
            s2 = fmaf(r[i], y[i], s2);
        }
        row_sum2<NT>(s1, s2, red[2]);
        const float m2 = p.post_w ? s2 * inv : 0.0f;
        if (ok) {
            if (p.dresidual) row_store<T, V, NT, EPT, WIDE>(reinterpret_cast<T *>(p.dresidual) + row * D, ln, D, dr);
            if (p.dgate) row_store<T, V, NT, EPT, WIDE>(reinterpret_cast<T *>(p.dgate) + row * D, ln, D, da);
#pragma unroll
            for (int i = 0; i < EPT; ++i) r[i] = ry * fmaf(-y[i], m2, r[i]);
            row_store<T, V, NT, EPT, WIDE>(reinterpret_cast<T *>(p.dy) + row * D, ln, D, r);
        }
    }
    auto put = [&](int which, const float (&c)[EPT]) {
        float *out = p.partial + ((long)blockIdx.x * 3 + which) * D;
        if (RB == 1) {
            par_store<V, NT, EPT, WIDE>(out, ln, D, c);
        } else {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < EPT; ++i) fold[(rg * EPT + i) * NT + ln] = c[i];
            __syncthreads();
            for (int k = threadIdx.x; k < NT * EPT; k += 256) {
                float t = 0.0f;
#pragma unroll
                for (int l = 0; l < RB; ++l) t += fold[l * NT * EPT + k];
                const int i = k / NT, d = ((i / V) * NT + k % NT) * V + i % V;
                if (d < D) out[d] = t;
            }
        }
    };
    put(0, cv);
    put(1, cw);
    put(2, cs);
}

// 16 columns and 64 lanes of parts to a block, eight loads of a lane in flight: the sums are short and there are few of them.
struct SumOut { float *p[3]; long end[3]; };
__global__ __launch_bounds__(1024) void sum_parts_kernel(const float *__restrict__ src, int parts, long n, SumOut out, int accumulate)
{
    __shared__ double s[64][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4;
    const long i = (long)blockIdx.x * 16 + c;
    double a = 0.0;
    if (i < n) {
        int t = r;
        for (; t + 7 * 64 < parts; t += 8 * 64) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = src[(long)(t + 64 * k) * n + i];
#pragma unroll
            for (int k = 0; k < 8; ++k) a += (double)v[k];
        }
        for (; t < parts; t += 64) a += (double)src[(long)t * n + i];
    }
    s[r][c] = a;
    for (int w = 32; w >= 1; w >>= 1) {
        __syncthreads();
        if (r < w) s[r][c] += s[r + w][c];
    }
    if (r || i >= n) return;
    const int k = i < out.end[0] ? 0 : i < out.end[1] ? 1 : 2;
    if (!out.p[k]) return;
    float *o = out.p[k] + (i - (k ? out.end[k - 1] : 0));
    *o = (accumulate ? *o : 0.0f) + (float)s[0][c];
}
hipError_t urnn_launch_sum_parts(const float *src, int parts, const long (&n)[3], float *const (&out)[3], int accumulate, hipStream_t st)
{
    const long all = n[0] + n[1] + n[2];
    const SumOut o = {{out[0], out[1], out[2]}, {n[0], n[0] + n[1], all}};
    sum_parts_kernel<<<dim3((unsigned)((all + 15) / 16)), 1024, 0, st>>>(src, parts, all, o, accumulate);
    return hipGetLastError();
}

static int row_threads(int D) { return D <= 128 ? 16 : D <= 512 ? 64 : D <= 1024 ? 128 : D <= 2048 ? 256 : D <= 4096 ? 512 : 1024; }
double urnn_norm_threads(long rows, int D)
{
    const int nt = row_threads(D), rb = nt < 256 ? 256 / nt : 1;
    return (double)((rows - 1) / rb + 1) * (nt * rb);
}
int urnn_norm_parts(long rows, int D)
{
    const int nt = row_threads(D), rb = nt < 256 ? 256 / nt : 1;
    const long blocks = (rows + rb - 1) / rb, most = nt <= 256 ? 768 : 256;      // resident: three blocks of 256, one of 512 or 1024
    const long turns = (blocks + most - 1) / most;                // the same number of turns for every block
    return (int)((blocks + turns - 1) / turns);
}

template <typename T, int V, int NT, int EPT, bool WIDE>
static hipError_t launch_norm(const NormParams &p, bool backward, hipStream_t st)
{
    constexpr int threads = NT < 256 ? 256 : NT, RB = NT < 256 ? 256 / NT : 1;
    if (backward) norm_backward_kernel<T, V, NT, EPT, WIDE><<<dim3((unsigned)p.parts), threads, 0, st>>>(p);
    else norm_kernel<T, V, NT, EPT, WIDE><<<dim3((unsigned)((p.rows + RB - 1) / RB)), threads, 0, st>>>(p);
    return hipGetLastError();
}
template <typename T, int V, bool WIDE>
static hipError_t by_width(const NormParams &p, bool backward, hipStream_t st)
{
    const int D = p.dim;
    if (!WIDE && D < V) return launch_norm<T, 1, 16, 8, true>(p, backward, st);
    if (D <= 128) return launch_norm<T, V, 16, 8, WIDE>(p, backward, st);
    if (D <= 512) return launch_norm<T, V, 64, 8, WIDE>(p, backward, st);
    if (D <= 1024) return launch_norm<T, V, 128, 8, WIDE>(p, backward, st);
    if (D <= 2048) return launch_norm<T, V, 256, 8, WIDE>(p, backward, st);
    if (D <= 4096) return launch_norm<T, V, 512, 8, WIDE>(p, backward, st);
    if (D <= 8192) return launch_norm<T, V, 1024, 8, WIDE>(p, backward, st);
    return launch_norm<T, V, 1024, 16, WIDE>(p, backward, st);
}
static hipError_t by_type(const NormParams &p, int dtype, bool wide, bool backward, hipStream_t st)
{
    if (dtype == URNN_F32) return wide ? by_width<float, 4, true>(p, backward, st) : by_width<float, 4, false>(p, backward, st);
    if (dtype == URNN_BF16) return wide ? by_width<bf16_t, 8, true>(p, backward, st) : by_width<bf16_t, 8, false>(p, backward, st);
    return wide ? by_width<f16_t, 8, true>(p, backward, st) : by_width<f16_t, 8, false>(p, backward, st);
}

hipError_t urnn_launch_norm(const NormParams &p, int dtype, bool wide, hipStream_t st) { return by_type(p, dtype, wide, false, st); }
hipError_t urnn_launch_norm_backward(const NormParams &p, int dtype, bool wide, float *dpre, float *dpost, float *dscale, int accumulate, hipStream_t st)
{
    hipError_t e = by_type(p, dtype, wide, true, st);
    float *const outs[3] = {dpre, dpost, dscale};
    const long sizes[3] = {p.dim, p.dim, p.dim};
    if (e == hipSuccess) e = urnn_launch_sum_parts(p.partial, p.parts, sizes, outs, accumulate, st);
    return e;
}
