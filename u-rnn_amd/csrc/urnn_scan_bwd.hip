// urnn_scan_bwd.hip -- selective state space scan, backward.  With d_t = dout_t silu(z_t), a_t[n] = exp(step_t A[n]) and, from the last
// token to the first, the gradient of the state
//   k_t[n] = C_t[n] d_t + a_(t+1)[n] k_(t+1)[n]        (behind the last token: dstate_out)
// per channel and state
//   dC_t[n] = sum_channels d_t h_t[n]                  dB_t[n] = sum_channels k_t[n] step_t u_t
//           = sum_channels d_t a_t h_(t-1)[n] + B_t[n] sum_channels d_t step_t u_t       (C . h likewise: h_t itself is not formed again)
//   w = k_t[n] a_t[n] h_(t-1)[n]                       dA[n] = sum_tokens w step_t
//   du_t = step_t sum_n k_t B_t + D d_t                dstep_t = sum_n w A + u_t sum_n k_t B_t,   ddelta_t = dstep_t softplus'(raw_t)
//   dz_t = dout_t (sum_n C_t h_t + D u_t) silu'(z_t)   dD = sum d_t u_t
//
// The states are needed from the last to the first.  The forward left one every CK tokens; from there CK tokens are run forward again,
// with a_t and a_t h_(t-1) of the half that is walked next in registers, and then walked backward: no division by a decay, and the
// exponentials of one half twice (both halves' values would not leave room for two waves).  A quad holds a channel's states, E = N / 4 to a
// lane; a lane holds ED = 2 channels (one from 32 states on), so that the two sums of different kind cost little: over the states, two
// DPP adds per channel and sum; over the channels (dB, dC), first in the lane, then by halving over the wave -- v_permlane32_swap and
// v_permlane16_swap move two values and add them in one go -- and by two DPP adds: about two issue slots per state.  Blocks of one to four
// waves, as the channels of a group divide into waves of 16 ED, add their waves' sums through LDS; where a group takes several blocks they
// leave partial rows in fp32, which a last kernel adds in a fixed order: no atomics.
//
// Few sequences: the time axis is cut into chunks as in the forward; a first pass leaves what a chunk hands to the left when nothing
// comes from its right (k' = a_first (..)), and the sum of its steps; a short kernel carries it over the chunks.
//
// What bounds it is first the issue of the vector unit: 4 x 2048 x 2048 of 16 states bf16 280 us with the unit busy in 77 % of the cycles, of
// 493 us for a whole training step.  26.4 vector instructions per state of 64 channels, where the formulas above have 13.6 operations: 9.2
// fma, 6.1 products, 3.4 sums, 2.0 exponentials (one half's twice, and the elementwise work's), 5.6 lane swaps, selects, conversions and
// moves.  The rest are two waves to a SIMD that wait for each other's LDS rows and for chains.  15 625 sequences of 12 tokens and 96 channels
// of 8 states fp32: 277 to 285 us, the unit busy 46 %, 1.3 TB/s; blocks of three waves leave one SIMD in four without work there.
#include "urnn_seq.h"

#include <type_traits>

// Sum v[i] over the 16 quads of the wave (lanes with equal lane & 3).  2 E values; result r[m] (m < max(1, E / 2)) holds, in row rho of
// 16 lanes, value 4 m + {0, 2, 1, 3}[rho] (E = 1: value rho / 2).
__device__ __forceinline__ float add_swapped32(float a, float b)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float add_swapped16(float a, float b)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// Sum over G adjacent lanes (G = 8 or 16, aligned), returned to all of them.
template <int G>
__device__ __forceinline__ float group_sum(float v)
{
    v = quad_sum(v);
    v += dpp_all<0x141>(v);                          // row_half_mirror
    if (G == 16) v += dpp_all<0x140>(v);             // row_mirror
    return v;
}
template <int E>
__device__ __forceinline__ void channel_sums(const float (&v)[2 * E], float (&r)[E < 2 ? 1 : E / 2])
{
    float s[E];
#pragma unroll
    for (int i = 0; i < E; ++i) s[i] = add_swapped32(v[2 * i], v[2 * i + 1]);
    if (E == 1) r[0] = add_swapped16(s[0], s[0]);
#pragma unroll
    for (int m = 0; m < E / 2; ++m) r[m] = add_swapped16(s[2 * m], s[2 * m + 1]);
#pragma unroll
    for (int m = 0; m < (E < 2 ? 1 : E / 2); ++m) {
        r[m] += dpp_all<0x128>(r[m]);                // row_ror:8
        r[m] += dpp_all<0x124>(r[m]);                // row_ror:4
    }
}

// S[c] (chunk c's own) -> what chunk c - 1 receives from its right: K[c - 1] = exp(A sum[c]) K[c] + S[c], K[last] = dstate_out.
template <int NP>
__global__ __launch_bounds__(256) void scan_back_carry_kernel(const float *__restrict__ A, const float *__restrict__ sum, float *S,
                                                              const float *__restrict__ dstate_out, int dim, int N, int chunks, long count)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    const long b = i / ((long)dim * NP), r = i % ((long)dim * NP);
    const int d = (int)(r / NP), n = (int)(r % NP);
    const float A2 = n < N ? a_log2(A[(long)d * N + n]) : 0.0f;
    float *s = S + b * chunks * dim * NP + r;
    const float *w = sum + b * chunks * dim + d;
    float k = dstate_out && n < N ? dstate_out[(b * dim + d) * N + n] : 0.0f;
    constexpr int U = 16;
    for (int c0 = chunks - 1; c0 >= 1; c0 -= U) {
        float sv[U], wv[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const int c = c0 - j >= 1 ? c0 - j : 1;
            sv[j] = s[(long)c * dim * NP];
            wv[j] = w[(long)c * dim];
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (c0 - j >= 1) {
                k = wv[j] == 0.0f || k == 0.0f ? k + sv[j] : fmaf(__builtin_amdgcn_exp2f(wv[j] * A2), k, sv[j]);
                s[(long)(c0 - j) * dim * NP] = k;
            }
    }
}

// V adjacent channels of a token as they lie in memory: they wait in registers for a whole tile, two 16-bit values to a register.
template <typename T, int V> struct Raw {
    static constexpr int WORDS = V * sizeof(T) < 4 ? 1 : V * sizeof(T) / 4;
    unsigned w[WORDS];
    __device__ __forceinline__ float get(int i) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return to_f(__builtin_bit_cast(T, (unsigned short)(w[i / 2] >> (16 * (i & 1)))));
    }
    // channels from `valid` on as zeros; WIDE: rows start on 16 bytes and all V are there
    template <bool WIDE> __device__ __forceinline__ void load(const void *from, int valid)
    {
        const T *src = reinterpret_cast<const T *>(from);
        if constexpr (WIDE && V * sizeof(T) >= 4) {
            constexpr int W = WORDS < 4 ? WORDS : 4;
#pragma unroll
            for (int k = 0; k < WORDS; k += W) {
                const Pack<unsigned, W> t = *reinterpret_cast<const Pack<unsigned, W> *>(reinterpret_cast<const unsigned *>(src) + k);
#pragma unroll
                for (int i = 0; i < W; ++i) w[k + i] = t.v[i];
            }
        } else {
#pragma unroll
            for (int k = 0; k < WORDS; ++k) w[k] = 0;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < valid) {
                    if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(src[i]);
                    else w[i / 2] |= (unsigned)__builtin_bit_cast(unsigned short, src[i]) << (16 * (i & 1));
                }
        }
    }
};
template <typename T, int V, bool WIDE>
__device__ __forceinline__ void store_channels(void *to, int valid, const float (&v)[V])
{
    T *dst = reinterpret_cast<T *>(to);
    constexpr int W = V * sizeof(T) < 16 ? V : 16 / sizeof(T);
    if constexpr (WIDE) {
#pragma unroll
        for (int k = 0; k < V; k += W) {
            Pack<T, W> t;
#pragma unroll
            for (int i = 0; i < W; ++i) t.v[i] = from_f<T>(v[k + i]);
            *reinterpret_cast<Pack<T, W> *>(dst + k) = t;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < valid) dst[i] = from_f<T>(v[i]);
    }
}

// A wave's LDS is its own: its operations are done in order, this keeps the compiler's in order as well.
__device__ __forceinline__ void wave_fence()
{
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

template <typename T, int NP, bool WIDE>
__global__ __launch_bounds__(256, NP <= 8 ? 3 : 2) void scan_backward_kernel(const ScanParams p)
{
    constexpr int E = NP / 4, W = E < 4 ? E : 4, ED = urnn_scan_ed(NP), CK = urnn_scan_ck(NP), CW = 16 * ED;
    constexpr int HT = CK / 2;                                   // tokens whose decays and states are in registers at a time
    constexpr int V = urnn_scan_v(NP), CG = CW / V, RB = CK * NP < 64 ? 1 : CK * NP / 64;
    static_assert(CG * CK == 64, "a wave's lanes are the tokens of a segment by groups of V channels");
    __shared__ alignas(16) Pack<float, 4> s_io[4][CK * CW];      // in: (step, step u, d, -); out: (sum w A log2 e, sum k B, sum C h, step)
    __shared__ alignas(16) float s_row[4][2][CK * NP];           // B, C
    __shared__ float s_bc[2][4][CK][2 * NP];                     // [turn][wave][token][sum k step u | sum d a h]
    __shared__ float s_ds[2][4][CK];                             // [turn][wave][token] sum over channels d step u
    __shared__ float s_cb[4][CK];                                // C . B of a token
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), q = lane & 3;
    const int CB = p.waves * CW, Dg = p.dim / p.G, cbs = (Dg + CB - 1) / CB;
    const int cb = blockIdx.x % (cbs * p.G), g = cb / cbs, c0 = g * Dg + (cb % cbs) * CB, cend = (g + 1) * Dg;
    const int chunk = blockIdx.x / (cbs * p.G) % p.chunks, slot = blockIdx.x / (cbs * p.G) / p.chunks;
    const int segs = (p.L + CK - 1) / CK;
    const int w0 = c0 + wave * CW;                               // the wave's first channel
    const int width = cend - w0 < CW ? (cend > w0 ? cend - w0 : 0) : CW;
    const bool sp = p.softplus != 0;
    Pack<float, 4> *const io = s_io[wave];
    float *const rowB = s_row[wave][0], *const rowC = s_row[wave][1];

    // elementwise: token lt of a segment, channels w0 + V lg ..  Channel V lg + i has its slot at i CG + lg of the token's row, so that
    // the threads of a token write side by side.
    const int lg = lane % CG, lt = lane / CG;
    const int evalid = width - V * lg;                           // channels there, of V
    const bool eok = evalid > 0;
    const int ech = eok ? w0 + V * lg : c0;
    // the lane's bias and skip, and its sums for their gradients: in LDS, where they cost no registers in between
    typedef Pack<float, V> Chan;
    __shared__ alignas(16) Chan s_par[4][2][CG], s_sum[4][2][64];
    Chan *const par = &s_par[wave][0][lg], *const acc = &s_sum[wave][0][lane];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        par[0].v[i] = p.bias && i < evalid ? p.bias[ech + i] : 0.0f;         // the same from all tokens' lanes
        par[CG].v[i] = p.D && i < evalid ? p.D[ech + i] : 0.0f;
        acc[0].v[i] = acc[64].v[i] = 0.0f;
    }
    wave_fence();
    const bool gated = p.z != nullptr;
    // Addresses: a uniform pointer to a segment's first token, and the lane's byte offset from there in 32 bits (the host checks that
    // CK tokens are within 4 GB).
    constexpr long TS = sizeof(T);
    const unsigned cho = ech * (unsigned)TS, ou = lt * (unsigned)(p.su.t * TS) + cho, od = lt * (unsigned)(p.sd.t * TS) + cho;
    const unsigned oo = lt * (unsigned)(p.so.t * TS) + cho, oz = gated ? lt * (unsigned)(p.sz.t * TS) + cho : 0;
    const unsigned oy = lt * (unsigned)(p.dim * TS) + cho;
    const int rn = lane % NP, rt = lane / NP;                    // rows of B, C: values lane + 64 i, token rt + 64 / NP i, state rn
    const bool rok = rn < p.N && rt < CK;
    const unsigned oB = (rok ? rt : 0) * (unsigned)(p.sB.t * TS) + (rok ? rn : 0) * (unsigned)TS, oC = (rok ? rt : 0) * (unsigned)(p.sC.t * TS) + (rok ? rn : 0) * (unsigned)TS;
    // scan: slots sc[k] of a row, states q E ..
    int sc[ED], sch[ED], srank[ED];
    bool sok[ED];
    float A2[ED][E], dA[ED][E];
#pragma unroll
    for (int k = 0; k < ED; ++k) {
        sc[k] = 16 * k + (lane >> 2);
        const int c = sc[k] % CG * V + sc[k] / CG;               // the slot's channel
        sok[k] = c < width;
        sch[k] = sok[k] ? w0 + c : c0;
        srank[k] = sok[k] ? w0 + keep_rank(c, width, V) : c0;
        load_states<E>(p.A + (long)sch[k] * p.N, q, p.N, states_vec(p.A, p.N, W), A2[k]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            A2[k][e] = sok[k] ? a_log2(A2[k][e]) : 0.0f;                     // not a product with 0: A may be -inf
            A2[k][e] = A2[k][e] < -3.0e38f ? -3.0e38f : A2[k][e];            // 0 * A2 stays 0: a step of 0 keeps the state
            dA[k][e] = 0.0f;
        }
    }

    const long tb = (long)chunk * p.CL, tfull = tb + p.CL < p.L ? tb + p.CL : p.L;
    auto end_of = [&](int b) -> long {                           // behind the last token of sequence b in this chunk; tb: none
        const int len = __builtin_amdgcn_readfirstlane(seq_len(p.lengths, b, p.L));
        return tfull < len ? tfull : (len > tb ? len : tb);
    };
    // what is fetched ahead: a segment's inputs and the state before it
    Raw<T, V> ru = {}, rd = {}, rz = {}, ro = {};
    T rB[RB] = {}, rC[RB] = {};
    float ck[ED][E] = {};
    const char *qu, *qd, *qz, *qo, *qB, *qC;                     // the segment to fetch next
    const float *qk = nullptr;
    int qn = 0;                                                  // its tokens
    auto fetch = [&]() {
        if (eok && lt < qn) {
            ru.template load<WIDE>(qu + ou, evalid);
            rd.template load<WIDE>(qd + od, evalid);
            ro.template load<WIDE>(qo + oo, evalid);
            if (gated) rz.template load<WIDE>(qz + oz, evalid);
        }
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            rB[i] = rC[i] = T(0.0f);
            if (rok && rt + 64 / NP * i < qn) {
                rB[i] = *reinterpret_cast<const T *>(qB + 64 / NP * i * p.sB.t * TS + oB);
                rC[i] = *reinterpret_cast<const T *>(qC + 64 / NP * i * p.sC.t * TS + oC);
            }
        }
        qn = CK;                                                 // the ones before are whole
        qu -= CK * p.su.t * TS;
        qd -= CK * p.sd.t * TS;
        qo -= CK * p.so.t * TS;
        qz -= CK * p.sz.t * TS;
        qB -= CK * p.sB.t * TS;
        qC -= CK * p.sC.t * TS;
    };
    auto fetch_states = [&]() {
#pragma unroll
        for (int k = 0; k < ED; ++k)
            if (sok[k]) load_states<E>(qk + (long)srank[k] * NP, q, NP, true, ck[k]);
        qk -= (long)p.dim * NP;
    };
    // the last segment of the next sequence that has one
    auto fetch_sequence = [&](int b) {
        for (; b < p.batch; b += p.slots) {
            const long te = end_of(b);
            if (te > tb) {
                const long t0 = tb + (te - 1 - tb) / CK * CK;
                qn = (int)(te - t0);
                qu = reinterpret_cast<const char *>(p.u) + (b * p.su.b + t0 * p.su.t) * TS;
                qd = reinterpret_cast<const char *>(p.delta) + (b * p.sd.b + t0 * p.sd.t) * TS;
                qo = reinterpret_cast<const char *>(p.dout) + (b * p.so.b + t0 * p.so.t) * TS;
                qz = gated ? reinterpret_cast<const char *>(p.z) + (b * p.sz.b + t0 * p.sz.t) * TS : qu;
                qB = reinterpret_cast<const char *>(p.B) + (b * p.sB.b + t0 * p.sB.t + (long)g * p.N) * TS;
                qC = reinterpret_cast<const char *>(p.C) + (b * p.sC.b + t0 * p.sC.t + (long)g * p.N) * TS;
                qk = p.keep + ((long)b * segs + t0 / CK) * p.dim * NP;
                fetch();
                return;
            }
        }
        qk = nullptr;                                            // no further segment
    };
    fetch_sequence(slot);
    if (qk) fetch_states();
    int turn = 0;

    for (int b = slot; b < p.batch; b += p.slots) {
        const long te = end_of(b);
        // rows of dB and dC: this channel block's partial ones, or the results where the group is one block
        const long prow = p.direct ? (long)b * p.L : ((long)(cb % cbs) * p.batch + b) * p.L;
        auto put_bc = [&](int which, long t, int n, float v) {
            const long at = ((prow + t) * p.G + g) * p.N + n;
            if (p.direct) reinterpret_cast<T *>(which ? p.dC : p.dB)[at] = from_f<T>(v);
            else (which ? p.dCp : p.dBp)[at] = v;
        };
        float carry[ED][E];
#pragma unroll
        for (int k = 0; k < ED; ++k) {
#pragma unroll
            for (int e = 0; e < E; ++e) carry[k][e] = 0.0f;
            if (sok[k]) {
                if (chunk + 1 < p.chunks) {
                    load_states<E>(p.S + (((long)b * p.chunks + chunk + 1) * p.pieces * p.dim + sch[k]) * NP, q, NP, true, carry[k]);
                } else if (p.dstate_out) {
                    load_states<E>(p.dstate_out + ((long)b * p.dim + sch[k]) * p.N, q, p.N, states_vec(p.dstate_out, p.N, W), carry[k]);
                }
            }
        }
        for (long t0 = tb + (te - 1 - tb) / CK * CK; t0 >= tb && t0 < te; t0 -= CK, turn ^= 1) {
            const int nt = te - t0 < CK ? (int)(te - t0) : CK;
            const Raw<T, V> cu = ru, cd = rd, cz = rz, co = ro;
            const bool here = eok && lt < nt;                    // tokens behind the sequence: steps of zero, which change nothing
            const Chan bias = par[0];
            float ds = 0.0f, dot = 0.0f;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float raw = cd.get(i) + bias.v[i], s = softplus_f(raw), step = here ? (sp ? s : raw) : 0.0f;
                const float d = here ? co.get(i) * (gated ? silu_f(cz.get(i)) : 1.0f) : 0.0f, su = here ? step * cu.get(i) : 0.0f;
                io[lt * CW + i * CG + lg] = {{step, su, d, 0.0f}};
                ds = fmaf(d, su, ds);
            }
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                if (lane + 64 * i < CK * NP) {
                    rowB[lane + 64 * i] = to_f(rB[i]);
                    rowC[lane + 64 * i] = to_f(rC[i]);
                }
            }
            wave_fence();
#pragma unroll
            for (int n = 0; n < NP / CG; ++n) dot = fmaf(rowB[lt * NP + n * CG + lg], rowC[lt * NP + n * CG + lg], dot);
            if (NP < CG) dot = lg < NP ? rowB[lt * NP + lg] * rowC[lt * NP + lg] : 0.0f;
            ds = group_sum<CG>(ds);
            dot = group_sum<CG>(dot);
            s_ds[turn][wave][lt] = ds;                           // the same from all lanes of a token
            s_cb[wave][lt] = dot;
            if (t0 - CK >= tb) fetch();
            else fetch_sequence(b + p.slots);

            float a[HT][ED][E], ah[HT][ED][E], h[ED][E];
            auto forward = [&](int j0) {                         // HT tokens from j0 on: h, and what the way back needs of them
#pragma unroll
                for (int j = 0; j < HT; ++j) {
                    float Bv[E];
#pragma unroll
                    for (int e = 0; e < E; e += W) {
                        const Pack<float, W> v = *reinterpret_cast<const Pack<float, W> *>(rowB + (j0 + j) * NP + q * E + e);
#pragma unroll
                        for (int i = 0; i < W; ++i) Bv[e + i] = v.v[i];
                    }
#pragma unroll
                    for (int k = 0; k < ED; ++k) {
                        const Pack<float, 2> in = *reinterpret_cast<const Pack<float, 2> *>(io + (j0 + j) * CW + sc[k]);
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            a[j][k][e] = __builtin_amdgcn_exp2f(in.v[0] * A2[k][e]);
                            ah[j][k][e] = a[j][k][e] * h[k][e];
                            h[k][e] = fmaf(in.v[1], Bv[e], ah[j][k][e]);
                        }
                    }
                }
            };
            auto from_checkpoint = [&]() {
#pragma unroll
                for (int k = 0; k < ED; ++k)
#pragma unroll
                    for (int e = 0; e < E; ++e) h[k][e] = ck[k][e];
            };
            auto backward = [&](int j0) {
#pragma unroll
                for (int j = HT - 1; j >= 0; --j) {
                    float Bv[E], Cv[E], v[2 * E] = {};           // v: dB's terms, then dC's
#pragma unroll
                    for (int e = 0; e < E; e += W) {
                        const Pack<float, W> vb = *reinterpret_cast<const Pack<float, W> *>(rowB + (j0 + j) * NP + q * E + e);
                        const Pack<float, W> vc = *reinterpret_cast<const Pack<float, W> *>(rowC + (j0 + j) * NP + q * E + e);
#pragma unroll
                        for (int i = 0; i < W; ++i) { Bv[e + i] = vb.v[i]; Cv[e + i] = vc.v[i]; }
                    }
#pragma unroll
                    for (int k = 0; k < ED; ++k) {
                        const Pack<float, 4> in = io[(j0 + j) * CW + sc[k]];
                        float SW = 0.0f, SG = 0.0f, SY = 0.0f;
#pragma unroll
                        for (int e = 0; e < E; ++e) {
                            const float kk = fmaf(Cv[e], in.v[2], carry[k][e]), w = kk * ah[j][k][e];
                            SW = fmaf(w, A2[k][e], SW);
                            SG = fmaf(kk, Bv[e], SG);
                            SY = fmaf(Cv[e], ah[j][k][e], SY);   // h = a h + step u B: the second term's sums are common to
                            dA[k][e] = fmaf(w, in.v[0], dA[k][e]);       // all states (C . B) and to all channels (d step u)
                            v[e] = fmaf(kk, in.v[1], v[e]);
                            v[E + e] = fmaf(ah[j][k][e], in.v[2], v[E + e]);
                            carry[k][e] = a[j][k][e] * kk;
                        }
                        SW = quad_sum(SW);
                        SG = quad_sum(SG);
                        SY = quad_sum(SY);
                        io[(j0 + j) * CW + sc[k]] = {{SW, SG, SY, in.v[0]}};       // the same from all four lanes
                    }
                    float r[E < 2 ? 1 : E / 2];
                    channel_sums<E>(v, r);
                    float *o = s_bc[turn][wave][j0 + j];
                    const int rho = lane >> 4, qr = (lane >> 2) & 3;
                    if (E == 1) {
                        o[(lane >> 5) * NP + q] = r[0];          // every quad of a row has its sums: all of them write
                    } else {
                        const int in4 = ((rho & 1) << 1) | (rho >> 1);
                        constexpr int M = E / 2 < 4 ? E / 2 : 4;
#pragma unroll
                        for (int m0 = 0; m0 < E / 2; m0 += M) {
                            float val = r[m0];
#pragma unroll
                            for (int m = 1; m < M; ++m) val = (qr & (M - 1)) == m ? r[m0 + m] : val;
                            const int idx = 4 * (m0 + (qr & (M - 1))) + in4;     // value: dB of state q E + idx, or dC from E on
                            o[(idx / E) * NP + q * E + idx % E] = val;
                        }
                    }
                }
            };
            from_checkpoint();
            if (nt > HT) {
                forward(0);
                forward(HT);
                backward(HT);
                from_checkpoint();
            }
            forward(0);
            if (qk) fetch_states();
            backward(0);
            wave_fence();
            if (here) {
                float odz[V], odd[V], odu[V];
                const Chan bias = par[0], skip = par[CG];
                const float cb_t = s_cb[wave][lt];
                Chan dD = acc[0], db = acc[64];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const Pack<float, 4> r = io[lt * CW + i * CG + lg];
                    const float raw = cd.get(i) + bias.v[i], uf = cu.get(i), of = co.get(i);
                    float d = of;
                    if (gated) {
                        const float zf = cz.get(i), sg = sigmoid_f(zf);
                        d = of * zf * sg;
                        odz[i] = of * fmaf(fmaf(r.v[3], cb_t, skip.v[i]), uf, r.v[2]) * sg * fmaf(zf, 1.0f - sg, 1.0f);
                    }
                    const float dstep = fmaf(r.v[0], URNN_LN2, r.v[1] * uf), dd = dstep * (sp ? sigmoid_f(raw) : 1.0f);
                    odd[i] = dd;
                    odu[i] = fmaf(r.v[1], r.v[3], d * skip.v[i]);
                    dD.v[i] = fmaf(d, uf, dD.v[i]);
                    db.v[i] += dd;
                }
                acc[0] = dD;
                acc[64] = db;
                const long at = ((long)b * p.L + t0) * p.dim * TS;
                store_channels<T, V, WIDE>(reinterpret_cast<char *>(p.ddelta) + at + oy, evalid, odd);
                store_channels<T, V, WIDE>(reinterpret_cast<char *>(p.du) + at + oy, evalid, odu);
                if (gated) store_channels<T, V, WIDE>(reinterpret_cast<char *>(p.dz) + at + oy, evalid, odz);
            }
            __syncthreads();                                     // the four waves' sums are there; the next segment's go to the other turn
            for (int k = tid; k < nt * 2 * NP; k += 64 * p.waves) {
                const int t = k / (2 * NP), w = k % (2 * NP), n = w % NP;
                float sum, ds;
                if (p.waves == 4) {
                    sum = (s_bc[turn][0][t][w] + s_bc[turn][1][t][w]) + (s_bc[turn][2][t][w] + s_bc[turn][3][t][w]);
                    ds = (s_ds[turn][0][t] + s_ds[turn][1][t]) + (s_ds[turn][2][t] + s_ds[turn][3][t]);
                } else {
                    sum = s_bc[turn][0][t][w];
                    ds = s_ds[turn][0][t];
                    for (int l = 1; l < p.waves; ++l) { sum += s_bc[turn][l][t][w]; ds += s_ds[turn][l][t]; }
                }
                if (w >= NP) sum = fmaf(rowB[t * NP + n], ds, sum);
                if (n < p.N) put_bc(w / NP, t0 + t, n, sum);
            }
            wave_fence();                                        // the wave's rows are read: the next segment's may be written
        }
        const float none[V] = {};
        for (long t = te; t < tfull; t += CK) {                  // rows behind the sequence are zeros
            const long at = ((long)b * p.L + t) * p.dim * TS;
            if (eok && t + lt < tfull) {
                store_channels<T, V, WIDE>(reinterpret_cast<char *>(p.ddelta) + at + oy, evalid, none);
                store_channels<T, V, WIDE>(reinterpret_cast<char *>(p.du) + at + oy, evalid, none);
                if (gated) store_channels<T, V, WIDE>(reinterpret_cast<char *>(p.dz) + at + oy, evalid, none);
            }
        }
        for (long k = te * NP + tid; k < tfull * NP; k += 64 * p.waves) {
            const int n = (int)(k % NP);
            if (n < p.N) {
                put_bc(0, k / NP, n, 0.0f);
                put_bc(1, k / NP, n, 0.0f);
            }
        }
        if (p.dstate && chunk == 0) {
#pragma unroll
            for (int k = 0; k < ED; ++k)
                if (sok[k]) store_states<E>(p.dstate + ((long)b * p.dim + sch[k]) * p.N, q, p.N, states_vec(p.dstate, p.N, W), carry[k]);
        }
    }
    float *sums = p.dAp + ((long)slot * p.chunks + chunk) * p.dim * (p.N + 2);      // this part's dA, dD, ddelta_bias
#pragma unroll
    for (int k = 0; k < ED; ++k)
        if (sok[k]) store_states<E>(sums + (long)sch[k] * p.N, q, p.N, states_vec(sums, p.N, W), dA[k]);
    wave_fence();
#pragma unroll
    for (int i = 0; i < V; ++i) io[lt * CW + i * CG + lg] = {{acc[0].v[i], acc[64].v[i], 0.0f, 0.0f}};
    wave_fence();
    if (lane < CW) {
        float x = 0.0f, y = 0.0f;
        for (int t = 0; t < CK; ++t) { x += io[t * CW + lane].v[0]; y += io[t * CW + lane].v[1]; }
        const int c = lane % CG * V + lane / CG;
        if (c < width) {
            sums[(long)p.dim * p.N + w0 + c] = x;
            sums[(long)p.dim * (p.N + 1) + w0 + c] = y;
        }
    }
}

// dB, dC (B,L,G,N) = sum over the channel blocks of a group, rounded once.
template <typename T>
__global__ __launch_bounds__(256) void scan_fold_rows_kernel(const float *__restrict__ dBp, const float *__restrict__ dCp, int blocks, long n, T *dB, T *dC)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    float x = 0.0f, y = 0.0f;
    for (int k = 0; k < blocks; ++k) { x += dBp[k * n + i]; y += dCp[k * n + i]; }
    dB[i] = from_f<T>(x);
    dC[i] = from_f<T>(y);
}

// Chunks of the time axis, blocks along the batch, and the pieces that a chunk's summary is made of (the summaries are waves of 64
// channels, which a block of the main pass has four of: they need more chunks to fill the chip).
int urnn_scan_backward_chunks(int B, int L, int D, int G, int N, int *CL, int *slots, int *pieces)
{
    const int np = urnn_scan_np(N), CB = urnn_scan_waves(D / G, np) * 16 * urnn_scan_ed(np);      // channels of a block
    const long cbs = (long)G * ((D / G + CB - 1) / CB), blocks = (long)B * cbs;
    long want = blocks >= 512 ? 1 : (512 + blocks - 1) / blocks;
    const long most = (L + 63) / 64;
    if (want > most) want = most;
    if (want < 1) want = 1;
    long cl = (L + want - 1) / want;
    cl = (cl + 63) / 64 * 64;
    *CL = (int)cl;
    const int chunks = (int)((L + cl - 1) / cl);
    int m = 1;
    while (m < 8 && cl % (32 * m) == 0 && cl / (2 * m) >= 64 && blocks * chunks * m < 2048) m *= 2;
    *pieces = m;
    // several sequences to a block once there are as many blocks as fit the chip at a time, three to a compute unit up to 8 states and two
    // beyond: the parameters' sums then stay in registers over the sequences.  15 625 short sequences: 768 blocks 277 us, 1024, of
    // which 256 wait for the others, 341.
    const long fit = np <= 8 ? 768 : 512;
    long s = fit / (cbs * chunks);
    if (s < 1) s = 1;
    if (s > B) s = B;
    *slots = (int)s;
    return chunks;
}

template <typename T, int NP>
static hipError_t launch_backward(const ScanParams &p, float *dA, float *dD, float *dbias, int accumulate, hipStream_t st)
{
    const int Dg = p.dim / p.G, CB = urnn_scan_waves(Dg, NP) * 16 * urnn_scan_ed(NP), gcbs = (Dg + CB - 1) / CB;
    if (p.chunks > 1) {
        ScanParams ps = p;
        ps.chunks = p.chunks * p.pieces;
        ps.CL = p.CL / p.pieces;
        const hipError_t e = urnn_launch_scan_back_summaries(ps, sizeof(T) == 4 ? URNN_F32 : std::is_same<T, bf16_t>::value ? URNN_BF16 : URNN_F16, st);
        if (e != hipSuccess) return e;
        const long count = (long)p.batch * p.dim * NP;
        scan_back_carry_kernel<NP><<<dim3((unsigned)((count + 255) / 256)), 256, 0, st>>>(p.A, p.sum, p.S, p.dstate_out, p.dim, p.N, ps.chunks, count);
    }
    const dim3 grid((unsigned)(gcbs * p.G * p.chunks * p.slots));
    if (p.wide) scan_backward_kernel<T, NP, true><<<grid, 64 * p.waves, 0, st>>>(p);
    else scan_backward_kernel<T, NP, false><<<grid, 64 * p.waves, 0, st>>>(p);
    const long n = (long)p.batch * p.L * p.G * p.N;
    if (!p.direct) scan_fold_rows_kernel<T><<<dim3((unsigned)((n + 255) / 256)), 256, 0, st>>>(p.dBp, p.dCp, gcbs, n, reinterpret_cast<T *>(p.dB), reinterpret_cast<T *>(p.dC));
    hipError_t e = hipGetLastError();
    float *const outs[3] = {dA, dD, dbias};
    const long sizes[3] = {(long)p.dim * p.N, p.dim, p.dim};
    if (e == hipSuccess) e = urnn_launch_sum_parts(p.dAp, p.slots * p.chunks, sizes, outs, accumulate, st);
    return e;
}

template <typename T>
static hipError_t by_states(const ScanParams &p, float *dA, float *dD, float *dbias, int accumulate, hipStream_t st)
{
    switch (urnn_scan_np(p.N)) {
    case 4: return launch_backward<T, 4>(p, dA, dD, dbias, accumulate, st);
    case 8: return launch_backward<T, 8>(p, dA, dD, dbias, accumulate, st);
    case 16: return launch_backward<T, 16>(p, dA, dD, dbias, accumulate, st);
    case 32: return launch_backward<T, 32>(p, dA, dD, dbias, accumulate, st);
    default: return launch_backward<T, 64>(p, dA, dD, dbias, accumulate, st);
    }
}

hipError_t urnn_launch_scan_backward(const ScanParams &p, int dtype, float *dA, float *dD, float *dbias, int accumulate, hipStream_t st)
{
    return dtype == URNN_F32 ? by_states<float>(p, dA, dD, dbias, accumulate, st)
         : dtype == URNN_BF16 ? by_states<bf16_t>(p, dA, dD, dbias, accumulate, st) : by_states<f16_t>(p, dA, dD, dbias, accumulate, st);
}
