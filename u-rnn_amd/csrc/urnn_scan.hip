// urnn_scan.hip -- selective state space scan, forward:
//   step_t = softplus(delta_t + bias)                      (or delta_t + bias)
//   h_t[n] = exp(step_t A[n]) h_(t-1)[n] + step_t u_t B_t[n]
//   y_t    = (sum_n C_t[n] h_t[n] + D u_t) * silu(z_t)
// per channel; B and C are shared by the channels of a group.
//
// Mapping.  A channel's NP (padded) states lie on the four lanes of a quad, E = NP / 4 in each lane's registers, so that the state
// never leaves them along the whole sequence; a wave holds 16 channels, a block of four waves 64.  Tokens pass in tiles of 32: the
// block turns a tile's inputs into fp32 (step, step * u) pairs and fp32 rows of B and C in LDS with whole-line loads (64 channels of
// a token are adjacent), then every wave walks the tile's tokens: per token one 8-byte and 2 E 4-byte LDS reads per lane, and per
// state one exponential (quarter rate) and four fp32 operations.  y is summed over the quad with two DPP adds, and gate, skip and
// store are done for the whole tile again.  The inputs of the next tile are in flight while a tile is walked.
//
// Few long sequences do not fill the chip with B * D / 64 blocks: the time axis is cut into chunks (urnn_scan_chunks).  The recurrence
// is linear, h_end = P h_begin + S with S the state of a chunk that starts from zero and P = exp(A * sum of its steps): one pass
// leaves (S, sum of steps) of every chunk, a short kernel carries the states over the chunks, and the full pass starts each chunk
// from its true state.  The first pass costs all exponentials once more (7 of the full pass's ~11 issue slots per state).
#include "urnn_seq.h"

enum { SCAN_STATES = 0, SCAN_FULL = 1 };

template <typename T, int NP, int MODE>
__global__ __launch_bounds__(256) void scan_kernel(const ScanParams p)
{
    constexpr int E = NP / 4, W = E < 4 ? E : 4, TT = 32, CK = urnn_scan_ck(NP), CB = URNN_SCAN_CB, R = TT * CB / 256, RB = TT * NP / 256 < 1 ? 1 : TT * NP / 256;
    __shared__ alignas(16) Pack<float, 2> s_in[TT * CB];         // (step, step * u)
    __shared__ alignas(16) float s_B[TT * NP];
    __shared__ alignas(16) float s_C[MODE == SCAN_FULL ? TT * NP : 4];
    __shared__ float s_y[MODE == SCAN_FULL ? TT * CB : 1];
    const int tid = threadIdx.x, lane = tid & 63, q = lane & 3;
    const int Dg = p.dim / p.G, cbs = (Dg + CB - 1) / CB;
    const int cb = blockIdx.x % (cbs * p.G), g = cb / cbs, c0 = g * Dg + (cb % cbs) * CB, cend = (g + 1) * Dg;
    const int walked = MODE == SCAN_STATES ? p.chunks - 1 : p.chunks;           // nothing reads the last chunk's summary
    const int chunk = blockIdx.x / (cbs * p.G) % walked, b = blockIdx.x / (cbs * p.G) / walked;
    const int len = seq_len(p.lengths, b, p.L);
    const long tb = (long)chunk * p.CL, tfull = tb + p.CL < p.L ? tb + p.CL : p.L;
    const long te = tfull < len ? tfull : len;
    const T *u = reinterpret_cast<const T *>(p.u) + b * p.su.b, *dl = reinterpret_cast<const T *>(p.delta) + b * p.sd.b;
    const T *z = p.z ? reinterpret_cast<const T *>(p.z) + b * p.sz.b : nullptr;
    const T *Bp = reinterpret_cast<const T *>(p.B) + b * p.sB.b + (long)g * p.N, *Cp = reinterpret_cast<const T *>(p.C) + b * p.sC.b + (long)g * p.N;
    T *y = reinterpret_cast<T *>(p.y) + (long)b * p.L * p.dim;

    // the elementwise role: channel lc of the block, tokens lt + 4 i of a tile
    const int lc = tid & 63, lt = tid >> 6, ech = c0 + lc;
    const bool eok = ech < cend;
    const float bias = p.bias && eok ? p.bias[ech] : 0.0f, skip = p.D && eok ? p.D[ech] : 0.0f;
    // the scan role: channel sch, states q E .. q E + E - 1
    const int sc = tid >> 2, sch = c0 + sc;
    const bool sok = sch < cend;
    const int rch = sok ? sch : c0;
    const bool vA = states_vec(p.A, p.N, W);
    float A2[E], h[E];
    load_states<E>(p.A + (long)rch * p.N, q, p.N, vA, A2);
#pragma unroll
    for (int e = 0; e < E; ++e) { A2[e] *= URNN_LOG2E; h[e] = 0.0f; }
    if (MODE == SCAN_FULL && chunk > 0) {
        const float *s = p.S + (((long)b * p.chunks + chunk - 1) * p.dim + rch) * NP + q * E;
#pragma unroll
        for (int e = 0; e < E; ++e) h[e] = s[e];
    } else if (p.state && chunk == 0) {
        load_states<E>(p.state + ((long)b * p.dim + rch) * p.N, q, p.N, states_vec(p.state, p.N, W), h);
    }
    float total = 0.0f;                                          // STATES: this thread's share of the chunk's sum of steps

    T ru[R] = {}, rd[R] = {}, rz[R] = {}, rB[RB] = {}, rC[RB] = {};
    auto fetch = [&](long t0) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const long t = t0 + lt + 4 * i;
            if (eok && t < te) {
                ru[i] = u[t * p.su.t + ech];
                rd[i] = dl[t * p.sd.t + ech];
                if (MODE == SCAN_FULL && z) rz[i] = z[t * p.sz.t + ech];
            }
        }
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            const int k = tid + 256 * i, n = k % NP;
            const long t = t0 + k / NP;
            rB[i] = rC[i] = T(0.0f);
            if (k < TT * NP && n < p.N && t < te) {
                rB[i] = Bp[t * p.sB.t + n];
                if (MODE == SCAN_FULL) rC[i] = Cp[t * p.sC.t + n];
            }
        }
    };
    if (tb < te) fetch(tb);
    for (long t0 = tb; t0 < te; t0 += TT) {
        const int nt = te - t0 < TT ? (int)(te - t0) : TT;
        T cu[R], cz[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float raw = to_f(rd[i]) + bias, step = p.softplus ? softplus_f(raw) : raw, uf = to_f(ru[i]);
            s_in[(lt + 4 * i) * CB + lc] = {{step, step * uf}};
            if (MODE == SCAN_STATES && lt + 4 * i < nt) total += step;
            cu[i] = ru[i];
            cz[i] = rz[i];
        }
#pragma unroll
        for (int i = 0; i < RB; ++i) {
            const int k = tid + 256 * i;
            if (k < TT * NP) {
                s_B[k] = to_f(rB[i]);
                if (MODE == SCAN_FULL) s_C[k] = to_f(rC[i]);
            }
        }
        __syncthreads();
        if (t0 + TT < te) fetch(t0 + TT);
        auto token = [&](int t) -> float {
            const Pack<float, 2> in = s_in[t * CB + sc];
            float y0 = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e += W) {
                const Pack<float, W> Bv = *reinterpret_cast<const Pack<float, W> *>(s_B + t * NP + q * E + e);
                Pack<float, W> Cv;
                if (MODE == SCAN_FULL) Cv = *reinterpret_cast<const Pack<float, W> *>(s_C + t * NP + q * E + e);
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    h[e + i] = fmaf(__builtin_amdgcn_exp2f(in.v[0] * A2[e + i]), h[e + i], in.v[1] * Bv.v[i]);
                    if (MODE == SCAN_FULL) y0 = fmaf(Cv.v[i], h[e + i], y0);
                }
            }
            return y0;
        };
        auto checkpoint = [&](int t) {                           // the state before token t0 + t, t a multiple of CK
            if (MODE == SCAN_FULL && p.keep && sok) {
                const long seg = (t0 + t) / CK, segs = (p.L + CK - 1) / CK;
                float *k = p.keep + (((long)b * segs + seg) * p.dim + sch) * NP + q * E;
#pragma unroll
                for (int e = 0; e < E; e += W) {
                    Pack<float, W> v;
#pragma unroll
                    for (int i = 0; i < W; ++i) v.v[i] = h[e + i];
                    *reinterpret_cast<Pack<float, W> *>(k + e) = v;
                }
            }
        };
        int t = 0;
        for (; t + 4 <= nt; t += 4) {
            if (t % CK == 0) checkpoint(t);
            float mine = 0.0f;                                   // lane q of the quad keeps token t + q
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float yj = token(t + j);
                if (MODE == SCAN_FULL) {
                    yj = quad_sum(yj);
                    mine = q == j ? yj : mine;
                }
            }
            if (MODE == SCAN_FULL) s_y[(t + q) * CB + sc] = mine;
        }
        for (; t < nt; ++t) {
            if (t % CK == 0) checkpoint(t);
            const float yj = token(t);
            if (MODE == SCAN_FULL) {
                const float s = quad_sum(yj);
                if (q == 0) s_y[t * CB + sc] = s;
            }
        }
        __syncthreads();
        if (MODE == SCAN_FULL && eok) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int tt = lt + 4 * i;
                if (tt < nt) {
                    float v = fmaf(skip, to_f(cu[i]), s_y[tt * CB + lc]);
                    if (z) v *= silu_f(to_f(cz[i]));
                    y[(t0 + tt) * p.dim + ech] = from_f<T>(v);
                }
            }
        }
    }
    if (MODE == SCAN_FULL) {
        const long z0 = te > tb ? te : tb;                       // rows behind the sequence are zeros
        if (eok)
            for (long t = z0 + lt; t < tfull; t += 4) y[t * p.dim + ech] = from_f<T>(0.0f);
        const int last = len > 0 ? (len - 1) / p.CL : 0;         // the chunk that holds the sequence's last token
        if (p.state_out && sok && chunk == last)
            store_states<E>(p.state_out + ((long)b * p.dim + sch) * p.N, q, p.N, states_vec(p.state_out, p.N, W), h);
    } else {
        __syncthreads();
        s_in[tid].v[0] = total;
        __syncthreads();
        if (tid < CB && eok) {
            float t = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) t += s_in[tid + CB * i].v[0];
            p.sum[((long)b * p.chunks + chunk) * p.dim + ech] = t;
        }
        if (sok) {
            float *s = p.S + (((long)b * p.chunks + chunk) * p.dim + sch) * NP + q * E;
#pragma unroll
            for (int e = 0; e < E; ++e) s[e] = h[e];
        }
    }
}

// S[c] (a chunk's end state from a zero start; chunk 0 from the given state) -> the end state itself:
// H[c] = exp(A sum[c]) H[c - 1] + S[c].  One thread per (b, d, n); the loads do not depend on the chain.  A chunk without tokens
// (sum 0) passes the state on as it is, also where A is infinite.
template <int NP>
__global__ __launch_bounds__(256) void scan_carry_kernel(const float *__restrict__ A, const float *__restrict__ sum, float *S, int dim, int N, int chunks, long count)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    const long b = i / ((long)dim * NP), r = i % ((long)dim * NP);
    const int d = (int)(r / NP), n = (int)(r % NP);
    const float A2 = n < N ? A[(long)d * N + n] * URNN_LOG2E : 0.0f;
    float *s = S + b * chunks * dim * NP + r;
    const float *w = sum + b * chunks * dim + d;
    float h = s[0];
    constexpr int U = 8;
    for (int c0 = 1; c0 < chunks; c0 += U) {
        float sv[U], wv[U];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            const int c = c0 + k < chunks ? c0 + k : chunks - 1;
            sv[k] = s[(long)c * dim * NP];
            wv[k] = w[(long)c * dim];
        }
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (c0 + k < chunks) {
                h = wv[k] == 0.0f ? h + sv[k] : fmaf(__builtin_amdgcn_exp2f(wv[k] * A2), h, sv[k]);
                s[(long)(c0 + k) * dim * NP] = h;
            }
    }
}

int urnn_scan_chunks(int B, int L, int D, int *CL)
{
    const long blocks = (long)B * ((D + URNN_SCAN_CB - 1) / URNN_SCAN_CB);
    long want = blocks >= 512 ? 1 : (1024 + blocks - 1) / blocks;
    const long most = (L + 63) / 64;
    if (want > most) want = most;
    if (want < 1) want = 1;
    long cl = (L + want - 1) / want;
    cl = (cl + 31) / 32 * 32;
    if (cl < 32) cl = 32;
    *CL = (int)cl;
    const int chunks = (int)((L + cl - 1) / cl);
    return chunks < 1 ? 1 : chunks;
}

template <typename T, int NP>
static hipError_t launch_scan(const ScanParams &p, hipStream_t st)
{
    const int Dg = p.dim / p.G, cbs = p.G * ((Dg + URNN_SCAN_CB - 1) / URNN_SCAN_CB);
    if (p.chunks > 1) {
        scan_kernel<T, NP, SCAN_STATES><<<dim3((unsigned)(cbs * (p.chunks - 1) * p.batch)), 256, 0, st>>>(p);
        const long count = (long)p.batch * p.dim * NP;
        scan_carry_kernel<NP><<<dim3((unsigned)((count + 255) / 256)), 256, 0, st>>>(p.A, p.sum, p.S, p.dim, p.N, p.chunks, count);
    }
    scan_kernel<T, NP, SCAN_FULL><<<dim3((unsigned)(cbs * p.chunks * p.batch)), 256, 0, st>>>(p);
    return hipGetLastError();
}

// One token: state and inputs are read once, the new state and y written once.  A quad per channel again, no LDS.  state_out may be
// state: every thread reads its own states before it writes them.
template <typename T, int NP>
__global__ __launch_bounds__(256) void scan_step_kernel(const ScanParams p)
{
    constexpr int E = NP / 4, W = E < 4 ? E : 4;
    const long item = (long)blockIdx.x * 64 + (threadIdx.x >> 2);
    const int q = threadIdx.x & 3;
    if (item >= (long)p.batch * p.dim) return;
    const int b = (int)(item / p.dim), d = (int)(item % p.dim), g = d / (p.dim / p.G);
    float h[E], A2[E], Bv[E], Cv[E];
    load_states<E>(p.state + item * p.N, q, p.N, states_vec(p.state, p.N, W), h);
    load_states<E>(p.A + (long)d * p.N, q, p.N, states_vec(p.A, p.N, W), A2);
    const T *Bp = reinterpret_cast<const T *>(p.B) + b * p.sB.b + (long)g * p.N, *Cp = reinterpret_cast<const T *>(p.C) + b * p.sC.b + (long)g * p.N;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const int n = q * E + e;
        Bv[e] = n < p.N ? to_f(Bp[n]) : 0.0f;
        Cv[e] = n < p.N ? to_f(Cp[n]) : 0.0f;
    }
    const float u = to_f(reinterpret_cast<const T *>(p.u)[b * p.su.b + d]);
    const float raw = to_f(reinterpret_cast<const T *>(p.delta)[b * p.sd.b + d]) + (p.bias ? p.bias[d] : 0.0f);
    const float zf = p.z ? to_f(reinterpret_cast<const T *>(p.z)[b * p.sz.b + d]) : 0.0f;
    const float skip = p.D ? p.D[d] : 0.0f;
    const float step = p.softplus ? softplus_f(raw) : raw, su = step * u;
    float y = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        h[e] = fmaf(exp_fast(step * A2[e]), h[e], su * Bv[e]);
        y = fmaf(Cv[e], h[e], y);
    }
    y = fmaf(skip, u, quad_sum(y));
    if (p.z) y *= silu_f(zf);
    store_states<E>(p.state_out + item * p.N, q, p.N, states_vec(p.state_out, p.N, W), h);
    if (q == 0) reinterpret_cast<T *>(p.y)[item] = from_f<T>(y);
}

template <typename T, int NP>
static hipError_t launch_step(const ScanParams &p, hipStream_t st)
{
    const long items = (long)p.batch * p.dim;
    scan_step_kernel<T, NP><<<dim3((unsigned)((items + 63) / 64)), 256, 0, st>>>(p);
    return hipGetLastError();
}

template <typename T>
static hipError_t by_states(const ScanParams &p, bool step, hipStream_t st)
{
    switch (urnn_scan_np(p.N)) {
    case 4: return step ? launch_step<T, 4>(p, st) : launch_scan<T, 4>(p, st);
    case 8: return step ? launch_step<T, 8>(p, st) : launch_scan<T, 8>(p, st);
    case 16: return step ? launch_step<T, 16>(p, st) : launch_scan<T, 16>(p, st);
    case 32: return step ? launch_step<T, 32>(p, st) : launch_scan<T, 32>(p, st);
    default: return step ? launch_step<T, 64>(p, st) : launch_scan<T, 64>(p, st);
    }
}

static hipError_t by_type(const ScanParams &p, int dtype, bool step, hipStream_t st)
{
    return dtype == URNN_F32 ? by_states<float>(p, step, st) : dtype == URNN_BF16 ? by_states<bf16_t>(p, step, st) : by_states<f16_t>(p, step, st);
}

hipError_t urnn_launch_scan(const ScanParams &p, int dtype, hipStream_t st) { return by_type(p, dtype, false, st); }
hipError_t urnn_launch_scan_step(const ScanParams &p, int dtype, hipStream_t st) { return by_type(p, dtype, true, st); }
