// urnn_conv_seq.hip -- short causal depthwise convolution along time, forward, single token and backward:
//   p[t] = bias + sum_k w[k] line[t + k],   line = [state (K - 1 inputs before the first) | x],   y = p or p sigmoid(p)
// The carried state is the last K - 1 entries of the line.  Backward, with dp = dy act'(p):
//   dline[j] = sum_k w[k] dp[j - k]  (+ the gradient of the carried state),   dw[k] = sum_t dp[t] line[t + k],   dbias = sum_t dp[t].
//
// Memory-bound: one read of x, one write of y.  A thread holds V adjacent channels (16 bytes) and walks T tokens with the last
// K - 1 inputs in registers, so that an input is read once but for the K - 1 rows before a chunk; threads of a wave are adjacent in
// the channels.  V = 1 where rows are not 16-byte aligned.  2 x 4096 x 4096 bf16: 26.4 us, 5.1 TB/s, what a copy of those bytes
// takes; 6 x 1531 x 1001 fp32 (no row aligned, padded): 12.6 us, with the backward and its sums 44 to 48 us from box to
// box, about 3 TB/s.
#include "urnn_seq.h"

#include <type_traits>

template <typename T, int V>
__device__ __forceinline__ void load_v(const T *src, float (&v)[V])
{
    const Pack<T, V> t = *reinterpret_cast<const Pack<T, V> *>(src);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f(t.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_v(T *dst, const float (&v)[V])
{
    Pack<T, V> t;
#pragma unroll
    for (int i = 0; i < V; ++i) t.v[i] = from_f<T>(v[i]);
    stream_store(dst, t);
}

// The same for the backward's groups, at rows of any alignment.
template <typename T, int V>
__device__ __forceinline__ void load_l(const T *src, float (&v)[V])
{
    const Pack<T, V> t = load_any<T, V>(src);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = to_f(t.v[i]);
}
template <typename T, int V>
__device__ __forceinline__ void store_l(T *dst, const float (&v)[V])
{
    Pack<T, V> t;
#pragma unroll
    for (int i = 0; i < V; ++i) t.v[i] = from_f<T>(v[i]);
    store_any<T, V>(dst, t);
}

// The taps of V channels: w[k] belongs to line[t + k].  The weights of V adjacent channels are V K adjacent floats.
template <int V, int K>
__device__ __forceinline__ void load_taps(const ConvSeqParams &p, int d, float (&w)[K][V], float (&bias)[V])
{
    constexpr int W = V % 4 == 0 ? 4 : 1;
#pragma unroll
    for (int i = 0; i < V * K; i += W) {
        const Pack<float, W> t = *reinterpret_cast<const Pack<float, W> *>(p.weight + (long)d * K + i);
#pragma unroll
        for (int j = 0; j < W; ++j) w[(i + j) % K][(i + j) / K] = t.v[j];
    }
#pragma unroll
    for (int i = 0; i < V; i += W) {
        Pack<float, W> t = {};
        if (p.bias) t = *reinterpret_cast<const Pack<float, W> *>(p.bias + d + i);
#pragma unroll
        for (int j = 0; j < W; ++j) bias[i + j] = t.v[j];
    }
}

template <typename T, int V, int K>
__global__ __launch_bounds__(256) void conv_seq_kernel(const ConvSeqParams p)
{
    constexpr int U = 4;
    const unsigned nv = p.dim / V, item = blockIdx.x * 256u + threadIdx.x, row = item / nv;     // fewer than 2^32 items: launch_conv
    if (row >= (unsigned)p.batch * p.chunks) return;
    const int d = (int)(item % nv) * V, chunk = (int)(row % p.chunks), b = (int)(row / p.chunks);
    const int len = seq_len(p.lengths, b, p.L);
    const long t0 = (long)chunk * p.T, tend = t0 + p.T < p.L ? t0 + p.T : p.L, te = tend < len ? tend : len;
    const T *x = reinterpret_cast<const T *>(p.x) + b * p.sx.b + d;
    const T *state = p.state ? reinterpret_cast<const T *>(p.state) + (long)b * (K - 1) * p.dim + d : nullptr;
    T *y = reinterpret_cast<T *>(p.y) + (long)b * p.L * p.dim + d;
    float w[K][V], bias[V], win[K][V];                           // the newest input is win[K - 1]
    load_taps<V, K>(p, d, w, bias);
    auto line = [&](long j, float (&v)[V]) {                     // entry j of the line counted from x[0]: j < 0 is the state
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = 0.0f;
        if (j >= 0) load_v<T, V>(x + j * p.sx.t, v);
        else if (state && j >= -(K - 1)) load_v<T, V>(state + (j + K - 1) * p.dim, v);
    };
    if (t0 < te) {
#pragma unroll
        for (int k = 1; k < K; ++k) line(t0 - K + k, win[k]);
    }
    for (long t = t0; t < te; t += U) {
        float in[U][V];
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (t + j < te) load_v<T, V>(x + (t + j) * p.sx.t, in[j]);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            if (t + j >= te) break;
            float o[V];
#pragma unroll
            for (int i = 0; i < V; ++i) {
#pragma unroll
                for (int k = 0; k < K - 1; ++k) win[k][i] = win[k + 1][i];
                win[K - 1][i] = in[j][i];
                float a = bias[i];
#pragma unroll
                for (int k = 0; k < K; ++k) a = fmaf(w[k][i], win[k][i], a);
                o[i] = p.silu ? silu_f(a) : a;
            }
            store_v<T, V>(y + (t + j) * p.dim, o);
        }
    }
    float zero[V] = {};
    for (long t = te > t0 ? te : t0; t < tend; ++t) store_v<T, V>(y + t * p.dim, zero);
    if (p.state_out && chunk == 0) {
        T *so = reinterpret_cast<T *>(p.state_out) + (long)b * (K - 1) * p.dim + d;
        for (int i = 0; i < K - 1; ++i) {
            float v[V];
            line((long)len - (K - 1) + i, v);
            store_v<T, V>(so + (long)i * p.dim, v);
        }
    }
}

// One token.  state_out may be state: a thread reads its K - 1 entries before it writes them.
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void conv_seq_step_kernel(const ConvSeqParams p)
{
    const unsigned nv = p.dim / V, item = blockIdx.x * 256u + threadIdx.x;
    const int d = (int)(item % nv) * V, b = (int)(item / nv);
    if (b >= p.batch) return;
    const long base = (long)b * (K - 1) * p.dim + d;
    const T *state = reinterpret_cast<const T *>(p.state) + base;
    T *so = reinterpret_cast<T *>(p.state_out) + base;
    float w[K][V], bias[V], win[K][V];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) load_v<T, V>(state + (long)k * p.dim, win[k]);
    load_v<T, V>(reinterpret_cast<const T *>(p.x) + b * p.sx.b + d, win[K - 1]);
    load_taps<V, K>(p, d, w, bias);
    float o[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float a = bias[i];
#pragma unroll
        for (int k = 0; k < K; ++k) a = fmaf(w[k][i], win[k][i], a);
        o[i] = p.silu ? silu_f(a) : a;
    }
#pragma unroll
    for (int k = 1; k < K; ++k) store_v<T, V>(so + (long)(k - 1) * p.dim, win[k]);
    store_v<T, V>(reinterpret_cast<T *>(p.y) + (long)b * p.dim + d, o);
}

// Backward.  A block is XB channel vectors by YB token lanes; token lane y of part r walks the chunks r YB + y, + parts YB, ... of the
// B sequences, T tokens each.  For token t of a chunk it needs dp[t .. t + K - 1] and so the inputs from t - K + 1 on: the window
// runs K - 1 tokens ahead of the token whose dx is complete.  Its sums for dw and dbias stay in registers over all its chunks;
// lanes are added in LDS, parts by urnn_launch_sum_parts: no atomics, the same bits every time.
template <typename T, int V, int K>
__global__ __launch_bounds__(256) void conv_seq_backward_kernel(const ConvSeqParams p, int xb)
{
    __shared__ float s_sum[256 * V];
    const int nv = (p.dim + V - 1) / V, yb = 256 / xb, xi = threadIdx.x % xb, yi = threadIdx.x / xb;
    const int cbs = (nv + xb - 1) / xb, cb = blockIdx.x % cbs, part = blockIdx.x / cbs;
    const int cv = cb * xb + xi;
    const bool ok = cv < nv;
    auto channel = [&](int c) { return c * V < p.dim - V ? c * V : p.dim - V; };     // the last group repeats channels of the one before it, bit for bit
    const int d = ok ? channel(cv) : 0;
    float w[K][V], bias[V], dw[K][V] = {}, db[V] = {};
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = p.bias ? p.bias[d + i] : 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) w[k][i] = p.weight[(long)(d + i) * K + k];
    }
    const long all = (long)p.batch * p.chunks;
    for (long c = (long)part * yb + yi; ok && c < all; c += (long)p.parts * yb) {
        const int b = (int)(c / p.chunks);
        const int len = seq_len(p.lengths, b, p.L);
        const long t0 = c % p.chunks * p.T, tend = t0 + p.T < p.L ? t0 + p.T : p.L, te = tend < len ? tend : len;
        const bool first = t0 == 0;
        const T *x = reinterpret_cast<const T *>(p.x) + b * p.sx.b + d, *dy = reinterpret_cast<const T *>(p.dout) + b * p.so.b + d;
        const T *state = p.state ? reinterpret_cast<const T *>(p.state) + (long)b * (K - 1) * p.dim + d : nullptr;
        const T *dso = p.dstate_out ? reinterpret_cast<const T *>(p.dstate_out) + (long)b * (K - 1) * p.dim + d : nullptr;
        T *dx = reinterpret_cast<T *>(p.dx) + (long)b * p.L * p.dim + d;
        T *dst = p.dstate ? reinterpret_cast<T *>(p.dstate) + (long)b * (K - 1) * p.dim + d : nullptr;
        auto line = [&](long j, float (&v)[V]) {
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = 0.0f;
            if (j >= 0) {
                if (j < len) load_l<T, V>(x + j * p.sx.t, v);
            } else if (state && j >= -(K - 1)) load_l<T, V>(state + (j + K - 1) * p.dim, v);
        };
        // dp and the line's window of token s: win[k] = line entry s - K + 1 + k
        float win[K][V], dp[K][V];                             // dp[k]: token s - K + 1 + k
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) dp[k][i] = 0.0f;
        if (t0 < te || first) {
#pragma unroll
            for (int k = 1; k < K; ++k) line(t0 - K + k, win[k]);
            // s: the token whose dp is formed; j = s - K + 1: the line entry whose gradient is complete then
            const long send = te + K - 1;
            constexpr int U = 4;                                 // tokens of x and dy in flight
            float ahead[U][V], dahead[U][V];
            for (long s0 = t0; s0 < send; s0 += U) {
#pragma unroll
                for (int a = 0; a < U; ++a) {
#pragma unroll
                    for (int i = 0; i < V; ++i) ahead[a][i] = dahead[a][i] = 0.0f;
                    if (s0 + a < len && s0 + a < send) {
                        load_l<T, V>(x + (s0 + a) * p.sx.t, ahead[a]);
                        load_l<T, V>(dy + (s0 + a) * p.so.t, dahead[a]);
                    }
                }
#pragma unroll
                for (int a = 0; a < U; ++a) {
                    const long s = s0 + a;
                    if (s >= send) break;
                    float (&in)[V] = ahead[a], (&dyv)[V] = dahead[a];
                    const bool live = s < len, own = s < te;         // tokens behind the chunk count for dx, not for the sums
#pragma unroll
                    for (int i = 0; i < V; ++i) {
#pragma unroll
                        for (int k = 0; k < K - 1; ++k) { win[k][i] = win[k + 1][i]; dp[k][i] = dp[k + 1][i]; }
                        win[K - 1][i] = in[i];
                        float g = 0.0f;
                        if (live) {
                            g = dyv[i];
                            if (p.silu) {
                                float a = bias[i];
#pragma unroll
                                for (int k = 0; k < K; ++k) a = fmaf(w[k][i], win[k][i], a);
                                const float sg = sigmoid_f(a);
                                g *= sg * fmaf(a, 1.0f - sg, 1.0f);
                            }
                        }
                        dp[K - 1][i] = g;
                        if (own) {
                            db[i] += g;
#pragma unroll
                            for (int k = 0; k < K; ++k) dw[k][i] = fmaf(g, win[k][i], dw[k][i]);
                        }
                    }
                    // dline[j] = sum_k w[k] dp[token j + (K - 1) - k], tokens j .. j + K - 1: dp[0 .. K - 1] of tokens s - K + 1 ..
                    const long j = s - (K - 1);
                    if (j >= te || (j < t0 && !first)) continue;
                    float o[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float a = 0.0f;
#pragma unroll
                        for (int k = 0; k < K; ++k) a = fmaf(w[k][i], dp[K - 1 - k][i], a);
                        o[i] = a;
                    }
                    if (dso && j >= (long)len - (K - 1)) {
                        float v[V];
                        load_l<T, V>(dso + (j - ((long)len - (K - 1))) * p.dim, v);
#pragma unroll
                        for (int i = 0; i < V; ++i) o[i] += v[i];
                    }
                    if (j >= 0) store_l<T, V>(dx + j * p.dim, o);
                    else if (dst) store_l<T, V>(dst + (j + K - 1) * p.dim, o);
                }
            }
        }
        float zero[V] = {};
        for (long t = te > t0 ? te : t0; t < tend; ++t) store_l<T, V>(dx + t * p.dim, zero);
    }
    // fold the token lanes, K taps and the bias one after the other
    for (int k = 0; k <= K; ++k) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float v = db[i];
#pragma unroll
            for (int kk = 0; kk < K; ++kk) v = kk == k ? dw[kk][i] : v;
            s_sum[(yi * V + i) * xb + xi] = v;
        }
        __syncthreads();
        for (int r = threadIdx.x; r < xb * V; r += 256) {
            float a = 0.0f;
            for (int l = 0; l < yb; ++l) a += s_sum[l * V * xb + r];
            const int i = r / xb, c = cb * xb + r % xb;
            if (c < nv) p.partial[(long)part * (K + 1) * p.dim + (k < K ? (channel(c) + i) * K + k : K * p.dim + channel(c) + i)] = a;
        }
    }
}

// Work split of the backward: a block takes XB groups of BV channels, parts x 256 / XB token lanes share the chunks.  1024 blocks: four to a
// compute unit; twice as many lose 3 % at 6 x 1531 x 1001 (more partial sums, no more bytes in flight).  Two channels to a thread: the
// window, the sums and what is in flight are 11 values of each, and four or eight channels leave too few waves to wait for memory.  With
// the forward, 2 x 4096 x 2000 bf16 60 us with two, 80 with four, 110 with eight; x 2001 77 us, 99 with one.
enum { BV = 2 };
static int conv_xb(int nv) { int xb = 8; while (xb < 64 && xb < nv) xb <<= 1; return xb; }
static int conv_parts(int B, int L, int D, int cover)
{
    const int cbs = (D + cover - 1) / cover;
    long parts = (1024 + cbs - 1) / cbs;
    const long most = ((long)B * ((L + 7) / 8) + 3) / 4;         // four token lanes of eight tokens at least
    if (parts > most) parts = most;
    return parts < 1 ? 1 : (int)parts;
}
int urnn_conv_seq_parts(int B, int L, int D) { return conv_parts(B, L, D, 64 * BV); }

template <typename T, int V, int K>
static hipError_t launch_conv_backward(ConvSeqParams p, hipStream_t st)
{
    const int nv = (p.dim + V - 1) / V;
    const int xb = conv_xb(nv), cbs = (nv + xb - 1) / xb;
    p.parts = urnn_conv_seq_parts(p.batch, p.L, p.dim);
    const long lanes = (long)p.parts * (256 / xb);
    long T_ = ((long)p.batch * p.L + lanes - 1) / lanes;     // about one chunk per lane, 8 .. 64 tokens
    T_ = T_ < 8 ? 8 : T_ > 64 ? 64 : T_;
    if (T_ > p.L) T_ = p.L;
    p.T = (int)T_;
    p.chunks = (p.L + p.T - 1) / p.T;
    conv_seq_backward_kernel<T, V, K><<<dim3((unsigned)(cbs * p.parts)), 256, 0, st>>>(p, xb);
    return hipGetLastError();
}

template <typename T, int V, int K>
static hipError_t launch_conv(ConvSeqParams p, int what, hipStream_t st)
{
    const int nv = p.dim / V;
    if (what == 1) {
        const long items = (long)p.batch * nv;
        conv_seq_step_kernel<T, V, K><<<dim3((unsigned)((items + 255) / 256)), 256, 0, st>>>(p);
        return hipGetLastError();
    }
    // Tokens of a thread: 32, so that the K - 1 rows before a chunk are a tenth of its reads, and fewer (4 at least) until there are
    // 131 072 threads, two waves to a SIMD, where the latency of a walk counts more than the rows read twice.
    p.T = 32;
    while ((long)p.batch * nv * ((p.L + p.T - 1) / p.T) > 0xf0000000l) p.T <<= 1;      // items are counted in 32 bits
    while (p.T > 4 && (long)p.batch * nv * ((p.L + p.T - 1) / p.T) < (1 << 17)) p.T >>= 1;
    p.chunks = (p.L + p.T - 1) / p.T;
    const long items = (long)p.batch * p.chunks * nv;
    conv_seq_kernel<T, V, K><<<dim3((unsigned)((items + 255) / 256)), 256, 0, st>>>(p);
    return hipGetLastError();
}

template <typename T, int V>
static hipError_t by_taps(const ConvSeqParams &p, int what, hipStream_t st)
{
    return p.K == 2 ? launch_conv<T, V, 2>(p, what, st) : p.K == 3 ? launch_conv<T, V, 3>(p, what, st) : launch_conv<T, V, 4>(p, what, st);
}
static hipError_t by_type(const ConvSeqParams &p, int dtype, bool wide, int what, hipStream_t st)
{
    if (dtype == URNN_F32) return wide ? by_taps<float, 4>(p, what, st) : by_taps<float, 1>(p, what, st);
    if (dtype == URNN_BF16) return wide ? by_taps<bf16_t, 8>(p, what, st) : by_taps<bf16_t, 1>(p, what, st);
    return wide ? by_taps<f16_t, 8>(p, what, st) : by_taps<f16_t, 1>(p, what, st);
}

template <typename T, int V>
static hipError_t backward_by_taps(const ConvSeqParams &p, hipStream_t st)
{
    return p.K == 2 ? launch_conv_backward<T, V, 2>(p, st) : p.K == 3 ? launch_conv_backward<T, V, 3>(p, st) : launch_conv_backward<T, V, 4>(p, st);
}

hipError_t urnn_launch_conv_seq(ConvSeqParams p, int dtype, bool wide, hipStream_t st) { return by_type(p, dtype, wide, 0, st); }
hipError_t urnn_launch_conv_seq_step(const ConvSeqParams &p, int dtype, bool wide, hipStream_t st) { return by_type(p, dtype, wide, 1, st); }
hipError_t urnn_launch_conv_seq_backward(const ConvSeqParams &p, int dtype, float *dweight, float *dbias, int accumulate, hipStream_t st)
{
    auto go = [&](auto v) {
        constexpr int V = decltype(v)::value;
        return dtype == URNN_F32 ? backward_by_taps<float, V>(p, st) : dtype == URNN_BF16 ? backward_by_taps<bf16_t, V>(p, st) : backward_by_taps<f16_t, V>(p, st);
    };
    const hipError_t e = p.dim >= BV ? go(std::integral_constant<int, BV>()) : go(std::integral_constant<int, 1>());
    if (e != hipSuccess) return e;
    const long sizes[3] = {(long)p.dim * p.K, p.dim, 0};
    float *const outs[3] = {dweight, dbias, nullptr};
    return urnn_launch_sum_parts(p.partial, urnn_conv_seq_parts(p.batch, p.L, p.dim), sizes, outs, accumulate, st);
}
