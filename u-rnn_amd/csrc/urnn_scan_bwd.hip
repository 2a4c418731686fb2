// urnn_scan_bwd.hip -- selective state space scan, backward.  With d_t = dout_t silu(z_t), a_t[n] = exp(step_t A[n]) and, from the last
// token to the first, the gradient of the state
//   k_t[n] = C_t[n] d_t + a_(t+1)[n] k_(t+1)[n]        (behind the last token: dstate_out)
// per channel and state
//   dC_t[n] = sum_channels d_t h_t[n]                  dB_t[n] = sum_channels k_t[n] step_t u_t
//   w = k_t[n] a_t[n] h_(t-1)[n]                       dA[n] = sum_tokens w step_t
//   du_t = step_t sum_n k_t B_t + D d_t                dstep_t = sum_n w A + u_t sum_n k_t B_t,   ddelta_t = dstep_t softplus'(raw_t)
//   dz_t = dout_t (sum_n C_t h_t + D u_t) silu'(z_t)   dD = sum d_t u_t
//
// The states are needed from the last to the first.  The forward left one every CK tokens; from there CK tokens are run forward again,
// with a_t and a_t h_(t-1) of all of them in registers (2 CK E values per channel), and then walked backward: no division by a decay, and
// every exponential once.  A quad holds a channel's states as in the forward; a lane holds ED = 2 channels, so that the two sums of
// different kind cost little: over the states, two DPP adds per channel and sum; over the channels (dB, dC), first in the lane, then by
// halving over the wave -- v_permlane32_swap and v_permlane16_swap move two values and add them in one go -- and by two DPP adds:
// about two issue slots per state against ~17 for the rest.  Blocks leave their sums over 64 ED channels as partial rows in fp32, which a
// last kernel adds in a fixed order: no atomics.
//
// Few sequences: the time axis is cut into chunks as in the forward; a first pass leaves what a chunk hands to the left when nothing
// comes from its right (k' = a_first (..)), and the sum of its steps; a short kernel carries it over the chunks.
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
        r[m] += dpp_move<0x128>(r[m]);               // row_ror:8
        r[m] += dpp_move<0x124>(r[m]);               // row_ror:4
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
    const float A2 = n < N ? A[(long)d * N + n] * URNN_LOG2E : 0.0f;
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
                k = wv[j] == 0.0f ? k + sv[j] : fmaf(__builtin_amdgcn_exp2f(wv[j] * A2), k, sv[j]);
                s[(long)(c0 - j) * dim * NP] = k;
            }
    }
}

// V adjacent channels of a token as they lie in memory: they wait in registers for a whole tile, two 16-bit values to a register.
template <typename T, int V> struct Raw {
    unsigned w[V * sizeof(T) / 4];
    __device__ __forceinline__ float get(int i) const
    {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return to_f(__builtin_bit_cast(T, (unsigned short)(w[i / 2] >> (16 * (i & 1)))));
    }
    // channels from `valid` on as zeros; wide: rows start on 16 bytes and all V are there
    __device__ __forceinline__ void load(const T *src, int valid, bool wide)
    {
        if (wide) {
            constexpr int W = V * sizeof(T) / 4 < 4 ? V * sizeof(T) / 4 : 4;
#pragma unroll
            for (int k = 0; k < (int)(V * sizeof(T) / 4); k += W) {
                const Pack<unsigned, W> t = *reinterpret_cast<const Pack<unsigned, W> *>(reinterpret_cast<const unsigned *>(src) + k);
#pragma unroll
                for (int i = 0; i < W; ++i) w[k + i] = t.v[i];
            }
        } else {
#pragma unroll
            for (int k = 0; k < (int)(V * sizeof(T) / 4); ++k) w[k] = 0;
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < valid) {
                    if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(src[i]);
                    else w[i / 2] |= (unsigned)__builtin_bit_cast(unsigned short, src[i]) << (16 * (i & 1));
                }
        }
    }
};
template <typename T, int V>
__device__ __forceinline__ void store_channels(T *dst, int valid, bool wide, const float (&v)[V])
{
    constexpr int W = V * sizeof(T) < 16 ? V : 16 / sizeof(T);
    if (wide) {
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

template <typename T, int NP>
__global__ __launch_bounds__(256, 2) void scan_backward_kernel(const ScanParams p)
{
    constexpr int E = NP / 4, W = E < 4 ? E : 4, ED = urnn_scan_ed(NP), CK = urnn_scan_ck(NP), CB = 64 * ED, TT = urnn_scan_tt(NP);
    constexpr int V = urnn_scan_v(NP), CG = CB / V, RB = TT * NP / 256 < 1 ? 1 : TT * NP / 256;
    __shared__ alignas(16) Pack<float, 4> s_io[TT * CB];         // in: (step, step u, d, -); out: (sum w A log2 e, sum k B, sum C h, step)
    __shared__ alignas(16) float s_B[TT * NP], s_C[TT * NP];
    __shared__ float s_bc[4 * TT * 2 * NP];                      // [wave][token][dB | dC]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, q = lane & 3;
    const int Dg = p.dim / p.G, cbs = (Dg + CB - 1) / CB;
    const int cb = blockIdx.x % (cbs * p.G), g = cb / cbs, c0 = g * Dg + (cb % cbs) * CB, cend = (g + 1) * Dg;
    const int chunk = blockIdx.x / (cbs * p.G) % p.chunks, slot = blockIdx.x / (cbs * p.G) / p.chunks;
    const long segs = (p.L + CK - 1) / CK;
    const int width = cend - c0 < CB ? cend - c0 : CB;
    const bool sp = p.softplus != 0;

    // elementwise: token lt of a tile, channels c0 + V lg ..  Channel V lg + i has its slot at i CG + lg of the token's row, so that the
    // threads of a token write side by side.
    const int lg = tid % CG, lt = tid / CG;
    const int evalid = width - V * lg;                           // channels there, of V
    const bool eok = evalid > 0, ewide = p.wide && evalid >= V;
    const int ech = c0 + (eok ? V * lg : 0);
    float bias[V], skip[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        bias[i] = p.bias && i < evalid ? p.bias[ech + i] : 0.0f;
        skip[i] = p.D && i < evalid ? p.D[ech + i] : 0.0f;
    }
    // scan: slots sc[k] of a row, states q E ..
    int sc[ED], sch[ED], srank[ED];
    bool sok[ED];
    float A2[ED][E], dA[ED][E];
#pragma unroll
    for (int k = 0; k < ED; ++k) {
        sc[k] = wave * 16 * ED + 16 * k + (lane >> 2);
        const int c = sc[k] % CG * V + sc[k] / CG;               // the slot's channel
        sok[k] = c < width;
        sch[k] = c0 + (sok[k] ? c : 0);
        srank[k] = c0 + keep_rank(sok[k] ? c : 0, width, V);
        load_states<E>(p.A + (long)sch[k] * p.N, q, p.N, states_vec(p.A, p.N, W), A2[k]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            A2[k][e] *= sok[k] ? URNN_LOG2E : 0.0f;
            A2[k][e] = A2[k][e] < -3.0e38f ? -3.0e38f : A2[k][e];            // 0 * A2 stays 0: a step of 0 keeps the state
            dA[k][e] = 0.0f;
        }
    }
    float dD[V] = {}, dbias[V] = {};

    for (int b = slot; b < p.batch; b += p.slots) {
        const int len = __builtin_amdgcn_readfirstlane(seq_len(p.lengths, b, p.L));
        const long tb = (long)chunk * p.CL, tfull = tb + p.CL < p.L ? tb + p.CL : p.L, te = tfull < len ? tfull : len;
        const T *u = reinterpret_cast<const T *>(p.u) + b * p.su.b + ech, *dl = reinterpret_cast<const T *>(p.delta) + b * p.sd.b + ech;
        const T *z = p.z ? reinterpret_cast<const T *>(p.z) + b * p.sz.b + ech : nullptr, *dout = reinterpret_cast<const T *>(p.dout) + b * p.so.b + ech;
        const T *Bp = reinterpret_cast<const T *>(p.B) + b * p.sB.b + (long)g * p.N, *Cp = reinterpret_cast<const T *>(p.C) + b * p.sC.b + (long)g * p.N;
        const long base = (long)b * p.L * p.dim + ech;
        T *du = reinterpret_cast<T *>(p.du) + base, *ddl = reinterpret_cast<T *>(p.ddelta) + base, *dz = reinterpret_cast<T *>(p.dz) + base;
        // partial rows of this channel block: [cb in group][b][t][g][n]
        const long prow = ((long)(cb % cbs) * p.batch + b) * p.L;
        float *dBp = p.dBp + (prow * p.G + g) * p.N, *dCp = p.dCp + (prow * p.G + g) * p.N;
        const long pt = (long)p.G * p.N;

        float carry[ED][E], ck[ED][E];
#pragma unroll
        for (int k = 0; k < ED; ++k) {
#pragma unroll
            for (int e = 0; e < E; ++e) carry[k][e] = ck[k][e] = 0.0f;
            if (sok[k]) {
                if (chunk + 1 < p.chunks) {
                    const float *s = p.S + (((long)b * p.chunks + chunk + 1) * p.pieces * p.dim + sch[k]) * NP + q * E;
#pragma unroll
                    for (int e = 0; e < E; ++e) carry[k][e] = s[e];
                } else if (p.dstate_out) {
                    load_states<E>(p.dstate_out + ((long)b * p.dim + sch[k]) * p.N, q, p.N, states_vec(p.dstate_out, p.N, W), carry[k]);
                }
            }
        }
        auto load_ck = [&](long seg) {
#pragma unroll
            for (int k = 0; k < ED; ++k)
                if (sok[k]) load_states<E>(p.keep + (((long)b * segs + seg) * p.dim + srank[k]) * NP, q, NP, true, ck[k]);
        };
        Raw<T, V> ru = {}, rd = {}, rz = {}, ro = {};
        T rB[RB] = {}, rC[RB] = {};
        auto fetch = [&](long t0) {
            const long t = t0 + lt;
            if (eok && t < te) {
                ru.load(u + t * p.su.t, evalid, ewide);
                rd.load(dl + t * p.sd.t, evalid, ewide);
                ro.load(dout + t * p.so.t, evalid, ewide);
                if (z) rz.load(z + t * p.sz.t, evalid, ewide);
            }
#pragma unroll
            for (int i = 0; i < RB; ++i) {
                const int k = tid + 256 * i, n = k % NP;
                const long tr = t0 + k / NP;
                rB[i] = rC[i] = T(0.0f);
                if (k < TT * NP && n < p.N && tr < te) {
                    rB[i] = Bp[tr * p.sB.t + n];
                    rC[i] = Cp[tr * p.sC.t + n];
                }
            }
        };
        if (tb < te) {
            long t0 = tb + (te - 1 - tb) / TT * TT;
            load_ck((te - 1) / CK);
            fetch(t0);
            for (; t0 >= tb; t0 -= TT) {
                const int nt = te - t0 < TT ? (int)(te - t0) : TT;
                const Raw<T, V> cu = ru, cd = rd, cz = rz, co = ro;
                const bool here = eok && lt < nt;                // tokens behind the sequence: steps of zero, which change nothing
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float raw = cd.get(i) + bias[i], s = softplus_f(raw), step = here ? (sp ? s : raw) : 0.0f;
                    const float d = co.get(i) * (z ? silu_f(cz.get(i)) : 1.0f);
                    s_io[lt * CB + i * CG + lg] = {{step, here ? step * cu.get(i) : 0.0f, here ? d : 0.0f, 0.0f}};
                }
#pragma unroll
                for (int i = 0; i < RB; ++i) {
                    const int k = tid + 256 * i;
                    if (k < TT * NP) { s_B[k] = to_f(rB[i]); s_C[k] = to_f(rC[i]); }
                }
                __syncthreads();
                if (t0 - TT >= tb) fetch(t0 - TT);

                for (int s0 = (nt - 1) / CK * CK; s0 >= 0; s0 -= CK) {
                    float a[CK][ED][E], ah[CK][ED][E], h[ED][E];
#pragma unroll
                    for (int k = 0; k < ED; ++k)
#pragma unroll
                        for (int e = 0; e < E; ++e) h[k][e] = ck[k][e];
                    if (t0 + s0 > tb) load_ck((t0 + s0) / CK - 1);
#pragma unroll
                    for (int j = 0; j < CK; ++j) {
                        {
                            const int t = s0 + j;
                            float Bv[E];
#pragma unroll
                            for (int e = 0; e < E; e += W) {
                                const Pack<float, W> v = *reinterpret_cast<const Pack<float, W> *>(s_B + t * NP + q * E + e);
#pragma unroll
                                for (int i = 0; i < W; ++i) Bv[e + i] = v.v[i];
                            }
#pragma unroll
                            for (int k = 0; k < ED; ++k) {
                                const Pack<float, 2> in = *reinterpret_cast<const Pack<float, 2> *>(s_io + t * CB + sc[k]);
#pragma unroll
                                for (int e = 0; e < E; ++e) {
                                    a[j][k][e] = __builtin_amdgcn_exp2f(in.v[0] * A2[k][e]);
                                    ah[j][k][e] = a[j][k][e] * h[k][e];
                                    h[k][e] = fmaf(in.v[1], Bv[e], ah[j][k][e]);
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int j = CK - 1; j >= 0; --j) {
                        {
                            const int t = s0 + j;
                            float Bv[E], Cv[E], v[2 * E] = {};               // v: dB's terms, then dC's
#pragma unroll
                            for (int e = 0; e < E; e += W) {
                                const Pack<float, W> vb = *reinterpret_cast<const Pack<float, W> *>(s_B + t * NP + q * E + e);
                                const Pack<float, W> vc = *reinterpret_cast<const Pack<float, W> *>(s_C + t * NP + q * E + e);
#pragma unroll
                                for (int i = 0; i < W; ++i) { Bv[e + i] = vb.v[i]; Cv[e + i] = vc.v[i]; }
                            }
#pragma unroll
                            for (int k = 0; k < ED; ++k) {
                                const Pack<float, 4> in = s_io[t * CB + sc[k]];
                                float SW = 0.0f, SG = 0.0f, SY = 0.0f;
#pragma unroll
                                for (int e = 0; e < E; ++e) {
                                    const float kk = fmaf(Cv[e], in.v[2], carry[k][e]), hj = fmaf(in.v[1], Bv[e], ah[j][k][e]), w = kk * ah[j][k][e];
                                    SW = fmaf(w, A2[k][e], SW);
                                    SG = fmaf(kk, Bv[e], SG);
                                    SY = fmaf(Cv[e], hj, SY);
                                    dA[k][e] = fmaf(w, in.v[0], dA[k][e]);
                                    v[e] = fmaf(kk, in.v[1], v[e]);
                                    v[E + e] = fmaf(hj, in.v[2], v[E + e]);
                                    carry[k][e] = a[j][k][e] * kk;
                                }
                                SW = quad_sum(SW);
                                SG = quad_sum(SG);
                                SY = quad_sum(SY);
                                if (q == 0) s_io[t * CB + sc[k]] = {{SW, SG, SY, in.v[0]}};
                            }
                            float r[E < 2 ? 1 : E / 2];
                            channel_sums<E>(v, r);
                            float *o = s_bc + (wave * TT + t) * 2 * NP;
                            const int rho = lane >> 4, qr = (lane >> 2) & 3;
                            if (E == 1) {
                                if ((lane & 31) < 4) o[(lane >> 5) * NP + q] = r[0];
                            } else {
                                const int in4 = ((rho & 1) << 1) | (rho >> 1);
#pragma unroll
                                for (int m0 = 0; m0 < E / 2; m0 += 4) {
                                    float val = r[m0];
#pragma unroll
                                    for (int m = m0 + 1; m < m0 + 4 && m < E / 2; ++m) val = qr == m - m0 ? r[m] : val;
                                    const int idx = 4 * (m0 + qr) + in4;       // value: dB of state q E + idx, or dC from E on
                                    if (m0 + qr < E / 2) o[(idx / E) * NP + q * E + idx % E] = val;
                                }
                            }
                        }
                    }
                }
                __syncthreads();
                if (eok && lt < nt) {
                    float odz[V], odd[V], odu[V];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const Pack<float, 4> r = s_io[lt * CB + i * CG + lg];
                        const float raw = cd.get(i) + bias[i], uf = cu.get(i), of = co.get(i);
                        float d = of;
                        if (z) {
                            const float zf = cz.get(i), sg = sigmoid_f(zf);
                            d = of * zf * sg;
                            odz[i] = of * fmaf(skip[i], uf, r.v[2]) * sg * fmaf(zf, 1.0f - sg, 1.0f);
                        }
                        const float dstep = fmaf(r.v[0], URNN_LN2, r.v[1] * uf), dd = dstep * (sp ? sigmoid_f(raw) : 1.0f);
                        odd[i] = dd;
                        odu[i] = fmaf(r.v[1], r.v[3], d * skip[i]);
                        dD[i] = fmaf(d, uf, dD[i]);
                        dbias[i] += dd;
                    }
                    const long at = (t0 + lt) * p.dim;
                    store_channels<T, V>(ddl + at, evalid, ewide, odd);
                    store_channels<T, V>(du + at, evalid, ewide, odu);
                    if (z) store_channels<T, V>(dz + at, evalid, ewide, odz);
                }
                for (int k = tid; k < nt * 2 * NP; k += 256) {
                    const int t = k / (2 * NP), w = k % (2 * NP), n = w % NP;
                    if (n < p.N) {
                        float s = 0.0f;
#pragma unroll
                        for (int l = 0; l < 4; ++l) s += s_bc[(l * TT + t) * 2 * NP + w];
                        (w < NP ? dBp : dCp)[(t0 + t) * pt + n] = s;
                    }
                }
            }
        }
        const long z0 = te > tb ? te : tb;                       // rows behind the sequence are zeros
        const float none[V] = {};
        for (long t = z0 + lt; eok && t < tfull; t += TT) {
            store_channels<T, V>(du + t * p.dim, evalid, ewide, none);
            store_channels<T, V>(ddl + t * p.dim, evalid, ewide, none);
            if (z) store_channels<T, V>(dz + t * p.dim, evalid, ewide, none);
        }
        for (long k = z0 * NP + tid; k < tfull * NP; k += 256) {
            const long t = k / NP;
            const int n = (int)(k % NP);
            if (n < p.N) dBp[t * pt + n] = dCp[t * pt + n] = 0.0f;
        }
        if (p.dstate && chunk == 0) {
#pragma unroll
            for (int k = 0; k < ED; ++k)
                if (sok[k]) store_states<E>(p.dstate + ((long)b * p.dim + sch[k]) * p.N, q, p.N, states_vec(p.dstate, p.N, W), carry[k]);
        }
        __syncthreads();                                         // the next sequence's tile overwrites s_io, s_B, s_C and s_bc
    }
    float *sums = p.dAp + ((long)slot * p.chunks + chunk) * p.dim * (p.N + 2);      // this part's dA, dD, ddelta_bias
#pragma unroll
    for (int k = 0; k < ED; ++k)
        if (sok[k]) store_states<E>(sums + (long)sch[k] * p.N, q, p.N, states_vec(sums, p.N, W), dA[k]);
#pragma unroll
    for (int i = 0; i < V; ++i) s_io[lt * CB + i * CG + lg] = {{dD[i], dbias[i], 0.0f, 0.0f}};
    __syncthreads();
    if (tid < CB) {
        float x = 0.0f, y = 0.0f;
        for (int t = 0; t < TT; ++t) { x += s_io[t * CB + tid].v[0]; y += s_io[t * CB + tid].v[1]; }
        const int c = tid % CG * V + tid / CG;
        if (c < width) {
            sums[(long)p.dim * p.N + c0 + c] = x;
            sums[(long)p.dim * (p.N + 1) + c0 + c] = y;
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
int urnn_scan_backward_chunks(int B, int L, int D, int N, int *CL, int *slots, int *pieces)
{
    const int CB = 64 * urnn_scan_ed(urnn_scan_np(N));
    const long cbs = (D + CB - 1) / CB, blocks = (long)B * cbs;
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
    long s = B;                                                  // several sequences to a block once there are enough blocks
    while (s > 1 && s * cbs * chunks > 1024) s = (s + 1) / 2;
    *slots = (int)s;
    return chunks;
}

template <typename T, int NP>
static hipError_t launch_backward(const ScanParams &p, float *dA, float *dD, float *dbias, void *dB, void *dC, int accumulate, hipStream_t st)
{
    const int Dg = p.dim / p.G, CB = 64 * urnn_scan_ed(NP), gcbs = (Dg + CB - 1) / CB;
    if (p.chunks > 1) {
        ScanParams ps = p;
        ps.chunks = p.chunks * p.pieces;
        ps.CL = p.CL / p.pieces;
        const hipError_t e = urnn_launch_scan_back_summaries(ps, sizeof(T) == 4 ? URNN_F32 : std::is_same<T, bf16_t>::value ? URNN_BF16 : URNN_F16, st);
        if (e != hipSuccess) return e;
        const long count = (long)p.batch * p.dim * NP;
        scan_back_carry_kernel<NP><<<dim3((unsigned)((count + 255) / 256)), 256, 0, st>>>(p.A, p.sum, p.S, p.dstate_out, p.dim, p.N, ps.chunks, count);
    }
    scan_backward_kernel<T, NP><<<dim3((unsigned)(gcbs * p.G * p.chunks * p.slots)), 256, 0, st>>>(p);
    const long n = (long)p.batch * p.L * p.G * p.N;
    scan_fold_rows_kernel<T><<<dim3((unsigned)((n + 255) / 256)), 256, 0, st>>>(p.dBp, p.dCp, gcbs, n, reinterpret_cast<T *>(dB), reinterpret_cast<T *>(dC));
    hipError_t e = hipGetLastError();
    float *const outs[3] = {dA, dD, dbias};
    const long sizes[3] = {(long)p.dim * p.N, p.dim, p.dim};
    if (e == hipSuccess) e = urnn_launch_sum_parts(p.dAp, p.slots * p.chunks, sizes, outs, accumulate, st);
    return e;
}

template <typename T>
static hipError_t by_states(const ScanParams &p, float *dA, float *dD, float *dbias, void *dB, void *dC, int accumulate, hipStream_t st)
{
    switch (urnn_scan_np(p.N)) {
    case 4: return launch_backward<T, 4>(p, dA, dD, dbias, dB, dC, accumulate, st);
    case 8: return launch_backward<T, 8>(p, dA, dD, dbias, dB, dC, accumulate, st);
    case 16: return launch_backward<T, 16>(p, dA, dD, dbias, dB, dC, accumulate, st);
    case 32: return launch_backward<T, 32>(p, dA, dD, dbias, dB, dC, accumulate, st);
    default: return launch_backward<T, 64>(p, dA, dD, dbias, dB, dC, accumulate, st);
    }
}

hipError_t urnn_launch_scan_backward(const ScanParams &p, int dtype, float *dA, float *dD, float *dbias, void *dB, void *dC, int accumulate, hipStream_t st)
{
    return dtype == URNN_F32 ? by_states<float>(p, dA, dD, dbias, dB, dC, accumulate, st)
         : dtype == URNN_BF16 ? by_states<bf16_t>(p, dA, dD, dbias, dB, dC, accumulate, st) : by_states<f16_t>(p, dA, dD, dbias, dB, dC, accumulate, st);
}
