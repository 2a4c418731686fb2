// urnn_seq.h -- shared pieces of the sequence operators (short causal convolution, selective state space scan, norms around a block):
// element types, the activations, parameter blocks and launchers.
#pragma once
#include "urnn_common.h"
#include "urnn_kernels.h"

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// One rounding to nearest even from fp32; everything between a load and a store is fp32.
template <typename T> __device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }

// V consecutive elements as one access (V * sizeof(T) <= 16 bytes, naturally aligned).
template <typename T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// A store past the L2's lines: what a kernel writes here is read again by another launch at the earliest, and a line that stays dirty
// in one XCD's L2 is written out before that launch starts anyway.  Measured: the single-token scan of 256 sequences of 4096 channels 43 -> 30 us, the
// convolution of 8192 tokens of 4096 channels 34 -> 26 us, the norms 72 -> 70 us; the backward's and the scan's narrower stores do not
// gain, and loads through the same hint lose it all again.
template <typename T, int V>
__device__ __forceinline__ void stream_store(T *dst, const Pack<T, V> &t)
{
    if constexpr (sizeof(t) == 16) __builtin_nontemporal_store(__builtin_bit_cast(u32x4, t), reinterpret_cast<u32x4 *>(dst));
    else *reinterpret_cast<Pack<T, V> *>(dst) = t;
}

#define URNN_LOG2E 1.44269504088896340736f
#define URNN_LN2 0.69314718055994530942f

// exp(x) as 2^(x log2 e): v_exp_f32, relative error about 2^-23 + |x| 2^-24.
__device__ __forceinline__ float exp_fast(float x) { return __builtin_amdgcn_exp2f(x * URNN_LOG2E); }
__device__ __forceinline__ float sigmoid_f(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_fast(-x)); }
__device__ __forceinline__ float silu_f(float x) { return x * sigmoid_f(x); }

// The scan's A for decays as powers of two.  The product of a finite A beyond 2.36e38 leaves float32: it is held at the largest float, so that
// a step of 0 keeps the state (0 inf would be NaN).  An A that is infinite itself stays so.
__device__ __forceinline__ float a_log2(float A)
{
    const float a = A * URNN_LOG2E;
    return fabsf(A) <= __FLT_MAX__ ? fminf(fmaxf(a, -__FLT_MAX__), __FLT_MAX__) : a;
}

// softplus(x) = max(x, 0) + log1p(e), e = exp(-|x|) in (0, 1].  log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3: the series
// 2 s (1 + s^2/3 + s^4/5 + ...) to s^12/13 leaves 1.4e-8 of the value, and keeps full relative accuracy where e is tiny (a step of
// exp(x) for x << 0), which log(1 + e) loses.
__device__ __forceinline__ float softplus_f(float x)
{
    const float e = exp_fast(-fabsf(x));
    const float s = e * __builtin_amdgcn_rcpf(2.0f + e), q = s * s;
    float p = 1.0f / 13.0f;
    p = fmaf(p, q, 1.0f / 11.0f);
    p = fmaf(p, q, 1.0f / 9.0f);
    p = fmaf(p, q, 1.0f / 7.0f);
    p = fmaf(p, q, 1.0f / 5.0f);
    p = fmaf(p, q, 1.0f / 3.0f);
    p = fmaf(p, q, 1.0f);
    return fmaxf(x, 0.0f) + 2.0f * s * p;
}

// A lane's value through a DPP pattern that has a source for every lane (no value for others to keep: it folds into the addition).
template <int CTRL>
__device__ __forceinline__ float dpp_all(float v)
{
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
// Sum over the four lanes of a quad, returned to all of them.
__device__ __forceinline__ float quad_sum(float v)
{
    v += dpp_all<0xB1>(v);
    v += dpp_all<0x4E>(v);
    return v;
}

// V elements at the element's own alignment: one access of V * sizeof(T) bytes all the same (global memory takes any alignment).
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_any(const T *src)
{
    Pack<T, V> t;
    __builtin_memcpy(&t, src, sizeof(t));
    return t;
}
template <typename T, int V>
__device__ __forceinline__ void store_any(T *dst, const Pack<T, V> &t)
{
    typedef unsigned any4 __attribute__((ext_vector_type(4), aligned(2)));
    if constexpr (sizeof(t) == 16) __builtin_nontemporal_store(__builtin_bit_cast(any4, t), reinterpret_cast<any4 *>(dst));
    else __builtin_memcpy(dst, &t, sizeof(t));
}
// Group d .. d + V - 1 of a row of D >= V elements, those from D on as zeros: the row's last V elements, moved down (16 bytes; no branch,
// which would make every load wait for the one before it).
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_tail(const T *row, int d, int D)
{
    static_assert(sizeof(T) * V == 16, "two 64-bit halves");
    struct Halves { unsigned long long lo, hi; };
    const int at = d + V <= D ? d : D - V, out = d - at;         // elements to drop, V or more: all
    Halves h = __builtin_bit_cast(Halves, load_any<T, V>(row + at));
    const int bits = (out & (V - 1)) * 8 * (int)sizeof(T), sh = bits & 63;
    const unsigned long long down = sh ? (h.lo >> sh) | (h.hi << (64 - sh)) : h.lo, hi = h.hi >> sh;
    h.lo = out >= V ? 0 : bits >= 64 ? hi : down;
    h.hi = out >= V || bits >= 64 ? 0 : hi;
    return __builtin_bit_cast(Pack<T, V>, h);
}
// ... stored element by element where it is not whole
template <typename T, int V>
__device__ __forceinline__ void store_tail(T *row, const Pack<T, V> &t, int d, int D)
{
    if (d + V <= D) store_any<T, V>(row + d, t);
    else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (d + i < D) row[d + i] = t.v[i];
    }
}

// Tokens of sequence b that count: lengths clamped to [0, L], so that no length can reach outside the tensors.
__device__ __forceinline__ int seq_len(const int *lengths, int b, int L)
{
    if (!lengths) return L;
    const int n = lengths[b];
    return n < 0 ? 0 : (n > L ? L : n);
}

// A (B, L, C) tensor: element strides of batch and token, the channels are adjacent.
struct SeqStride { long b, t; };

enum { URNN_SEQ_MAX_STATES = 64, URNN_SEQ_MAX_TAPS = 4, URNN_SEQ_MAX_NORM = 16384 };

// A quad's share of a row of N states: lane q holds states q E .. q E + E - 1, those beyond N as zeros.  vec: the row's W-wide
// accesses are aligned and inside or outside as a whole (states_vec).
template <int E>
__device__ __forceinline__ void load_states(const float *row, int q, int N, bool vec, float (&v)[E])
{
    constexpr int W = E < 4 ? E : 4;
#pragma unroll
    for (int e = 0; e < E; e += W) {
        const int n = q * E + e;
        if (vec) {                                   // N % W == 0: a group of W states is inside or outside as a whole
            Pack<float, W> t = {};
            if (n < N) t = *reinterpret_cast<const Pack<float, W> *>(row + n);
#pragma unroll
            for (int i = 0; i < W; ++i) v[e + i] = t.v[i];
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i) v[e + i] = n + i < N ? row[n + i] : 0.0f;
        }
    }
}

template <int E, bool STREAM = false>
__device__ __forceinline__ void store_states(float *row, int q, int N, bool vec, const float (&v)[E])
{
    constexpr int W = E < 4 ? E : 4;
#pragma unroll
    for (int e = 0; e < E; e += W) {
        const int n = q * E + e;
        if (vec) {
            Pack<float, W> t;
#pragma unroll
            for (int i = 0; i < W; ++i) t.v[i] = v[e + i];
            if (n < N) {
                if constexpr (STREAM) stream_store(row + n, t);
                else *reinterpret_cast<Pack<float, W> *>(row + n) = t;
            }
        } else {
#pragma unroll
            for (int i = 0; i < W; ++i)
                if (n + i < N) row[n + i] = v[e + i];
        }
    }
}

__device__ __forceinline__ bool states_vec(const void *a, int N, int W)
{
    return N % W == 0 && (reinterpret_cast<uintptr_t>(a) & (W * sizeof(float) - 1)) == 0;
}

// ---- selective scan --------------------------------------------------------------------------------------------------
struct ScanParams {
    const void *u, *delta, *B, *C, *z, *dout;        // (B,L,D), B / C (B,L,G,N)
    SeqStride su, sd, sB, sC, sz, so;
    const float *A, *D, *bias;                       // (D,N), (D) or NULL, (D) or NULL
    const float *state;                              // (B,D,N) or NULL
    const int *lengths;                              // (B) or NULL
    void *y;                                         // (B,L,D) contiguous
    float *state_out;                                // (B,D,N) or NULL
    float *keep;                                     // checkpoints [B][ceil(L/URNN_SCAN_CK)][D][NP], or NULL
    float *sum;                                      // chunk summaries: sum of the steps [B][chunks][D] ...
    float *S;                                        // ... and the state of a chunk that starts from zero [B][chunks][D][NP]
    int batch, L, dim, N, G, chunks, CL, softplus;
    // backward
    int slots, pieces, waves;                        // blocks along the batch; summaries of a chunk; waves of a block
    int wide;                                        // all (B,L,D) rows start on 16 bytes
    const float *dstate_out;                         // (B,D,N) or NULL
    void *du, *ddelta, *dz;                          // (B,L,D) contiguous
    float *dstate;                                   // (B,D,N) or NULL
    void *dB, *dC;                                   // (B,L,G,N) contiguous
    int direct;                                      // a group is one block: dB and dC leave the main pass as they are
    float *dBp, *dCp;                                // per channel block: [blocks of a group][B][L][G][N]
    float *dAp;                                      // per (batch slot, chunk): [parts][D N | D | D], sums for dA, dD, ddelta_bias
};

#define URNN_SCAN_CB 64     // channels of a forward wave
enum { SCAN_STATES = 0, SCAN_FULL = 1, SCAN_BACK = 2, SCAN_STEP = 3 };

// Tokens between two checkpoints of the state: what the backward holds in registers of decays and states at a time, 2 CK NP / 4 (x 2
// channels up to 16 states).
__host__ __device__ static constexpr int urnn_scan_ck(int np) { return np == 64 ? 4 : 8; }
__host__ __device__ static constexpr int urnn_scan_ed(int np) { return np <= 16 ? 2 : 1; }    // channels of a backward lane

static inline int urnn_scan_np(int N) { return N <= 4 ? 4 : N <= 8 ? 8 : N <= 16 ? 16 : N <= 32 ? 32 : 64; }

// Channels of a thread in the backward's elementwise work: a segment's tokens by a wave's channels over 64 lanes.
__host__ __device__ static constexpr int urnn_scan_v(int np) { return urnn_scan_ck(np) * 16 * urnn_scan_ed(np) / 64; }
// Waves of a backward block: at most four, as many as the channels of a group divide into evenly (96 channels are three, not four).
__host__ __device__ static inline int urnn_scan_waves(int Dg, int np)
{
    const int cw = 16 * urnn_scan_ed(np), w = (Dg + cw - 1) / cw, blocks = (w + 3) / 4;
    return (w + blocks - 1) / blocks;
}
// Place of channel c among the w channels of a backward wave, in the record of checkpoints: the wave's lane for channels V i .. V i + V - 1
// spreads them over its LDS rows so that neighbours of a row are V channels apart, and reads a row's states side by side.
__host__ __device__ static inline int keep_rank(int c, int w, int V) { return w % V == 0 ? c % V * (w / V) + c / V : c; }

hipError_t urnn_launch_scan(const ScanParams &p, int dtype, hipStream_t st);
hipError_t urnn_launch_scan_back_summaries(const ScanParams &p, int dtype, hipStream_t st);
hipError_t urnn_launch_scan_step(const ScanParams &p, int dtype, hipStream_t st);
int urnn_scan_chunks(int B, int L, int D, int *CL);
hipError_t urnn_launch_scan_backward(const ScanParams &p, int dtype, float *dA, float *dD, float *dbias, int accumulate, hipStream_t st);
int urnn_scan_backward_chunks(int B, int L, int D, int G, int N, int *CL, int *slots, int *pieces);

// ---- short causal convolution ----------------------------------------------------------------------------------------
struct ConvSeqParams {
    const void *x, *dout;                            // (B,L,D)
    SeqStride sx, so;
    const float *weight, *bias;                      // (D,K), (D) or NULL
    const void *state;                               // (B,K-1,D) contiguous or NULL: the inputs before the first, oldest first
    const int *lengths;
    void *y, *state_out;                             // (B,L,D), (B,K-1,D) or NULL
    int batch, L, dim, K, silu;
    int T, chunks;                                   // tokens of a thread's chunk, chunks of a sequence
    // backward
    const void *dstate_out;                          // (B,K-1,D) or NULL
    void *dx, *dstate;                               // (B,L,D), (B,K-1,D) or NULL
    float *partial;                                  // [parts][dim K | dim]: sums of a block's tokens for weight and bias
    int parts;
};

hipError_t urnn_launch_conv_seq(ConvSeqParams p, int dtype, bool wide, hipStream_t st);
hipError_t urnn_launch_conv_seq_step(const ConvSeqParams &p, int dtype, bool wide, hipStream_t st);
hipError_t urnn_launch_conv_seq_backward(const ConvSeqParams &p, int dtype, float *dweight, float *dbias, int accumulate, hipStream_t st);
int urnn_conv_seq_parts(int B, int L, int D);

// ---- norms around a block ----------------------------------------------------------------------------------------------
struct NormParams {
    const void *y, *gate, *residual, *dnormed, *dres; // (M,D) rows; gate, residual, dnormed, dres may be NULL
    SeqStride sy, sg, sr, sdn, sdr;                  // row r is at (r / inner) b + (r % inner) t
    unsigned inner;
    const float *pre_w, *post_w, *scale;             // (D); post_w / scale may be NULL
    void *normed, *res_out;                          // (M,D) contiguous
    void *dy, *dgate, *dresidual;                    // (M,D) contiguous; dgate / dresidual may be NULL
    float *partial;                                  // [parts][3][D]: dpre_w, dpost_w, dscale
    long rows;
    int dim, act, parts;
    float eps;
};

hipError_t urnn_launch_norm(const NormParams &p, int dtype, bool wide, hipStream_t st);
hipError_t urnn_launch_norm_backward(const NormParams &p, int dtype, bool wide, float *dpre, float *dpost, float *dscale, int accumulate, hipStream_t st);
int urnn_norm_parts(long rows, int D);
double urnn_norm_threads(long rows, int D);          // of a forward launch

// src [parts][n[0] + n[1] + n[2]] -> out[k] (+)= the sums over parts of its columns; out[k] may be NULL.  In double, in a fixed order.
hipError_t urnn_launch_sum_parts(const float *src, int parts, const long (&n)[3], float *const (&out)[3], int accumulate, hipStream_t st);
