// urnn_scan.hip -- selective state space scan, forward and single token:
//   step_t = softplus(delta_t + bias)                      (or delta_t + bias)
//   h_t[n] = exp(step_t A[n]) h_(t-1)[n] + step_t u_t B_t[n]
//   y_t    = (sum_n C_t[n] h_t[n] + D u_t) * silu(z_t)
// per channel; B and C are shared by the channels of a group.
//
// Mapping.  A lane is a channel: all of its states stay in registers along the sequence, the sum over states needs no other lane, and
// the elementwise work (softplus, gate, conversions) is done once.  A wave is 64 adjacent channels of one sequence -- whole 128-byte
// lines of a 16-bit row per access -- and a block of its own, so that nothing waits for another wave.  The rows of B of a group of
// tokens (GT: eight, four from 32 states on) lie across the lanes, a state to a lane; the outer product with the lanes' inputs,
// B_t[n] (step u), is added to the decayed states by v_mfma_f32_4x4x1 (fp32 as the vector unit's; four states of 64 channels in 8 cycles
// of the otherwise idle matrix pipe), which broadcasts four values of the row; C's rows are read from LDS, the same address in all lanes.
// The inputs of the next group are in flight meanwhile.  (With a quad to a channel, as in the backward, all four lanes repeat the
// elementwise part or pass it on through LDS: the full pass over 32 768 x 2048 took 417 us then and 359 with a lane, at that step.)
//
// What bounds it is the vector unit: per state one exponential (measured: the time of 1.6 to 2 fp32 operations) and three fp32
// operations, per token and channel about 45 more: 119 issue slots at 16 states, 35e12 lane-slots/s of the chip (by the counters 114
// instructions, 20 of them exponentials or reciprocals).  4 x 2048 x 2048 bf16: 92 us of 56 us of slots, the vector unit busy in 63 % of
// the cycles (waves at two to a SIMD wait for their loads and for the chain of a state from token to token), 1.5 TB/s; 32 768 x 2048
// 460 us with both passes, busy 84 and 89 %, of 226 us of slots for one.
//
// Few long sequences do not fill the chip with B * D / 64 waves: the time axis is cut into chunks (urnn_scan_chunks).  The recurrence
// is linear, h_end = P h_begin + S with S the state of a chunk that starts from zero and P = exp(A * sum of its steps): one pass
// leaves (S, sum of steps) of every chunk, a short kernel carries the states over the chunks, and the full pass starts each chunk
// from its true state.  The first pass costs the exponentials once more (32 768 x 2048: 222 us next to the full pass's 285).  The same
// kernel, run from the last token to the first, gives the backward its chunk summaries.
#include "urnn_seq.h"

#include <type_traits>
#include <utility>

// h[k] = (decayed h[k]) + outer product of x (one per lane) with the row's values 4 k .. 4 k + 3: v_mfma_f32_4x4x1, sixteen blocks of four
// states by four lanes.  The rows of the tokens lie across the lanes of v, NP values after one another; the instruction broadcasts
// four of them, of token J, to all blocks.
template <int J, int K, int NP, int RV>
__device__ __forceinline__ void add_outer(const float (&v)[RV], float x, f32x4 (&h)[NP / 4])
{
    if constexpr (K < NP / 4) {
        constexpr int at = J * NP + 4 * K;
        h[K] = __builtin_amdgcn_mfma_f32_4x4x1f32(v[at / 64], x, h[K], 4, at % 64 / 4, 0);
        add_outer<J, K + 1, NP, RV>(v, x, h);
    }
}

// f(0), f(1), ... f(G - 1), the first `left` of them (left >= G: without a test)
template <bool ALL, typename F, int... I>
__device__ __forceinline__ void tokens(F &f, int left, std::integer_sequence<int, I...>)
{
    ((ALL || I < left ? f(std::integral_constant<int, I>()) : void()), ...);
}

template <typename T, int NP, int MODE>
__global__ __launch_bounds__(64, 2) void scan_kernel(const ScanParams p)
{
    constexpr int CK = urnn_scan_ck(NP), CB = URNN_SCAN_CB, GT = NP <= 16 ? 8 : 4, RV = GT * NP < 64 ? 1 : GT * NP / 64, TPV = 64 / NP;
    constexpr bool FULL = MODE == SCAN_FULL, BACK = MODE == SCAN_BACK;
    __shared__ alignas(16) float s_C[FULL ? GT * NP : 4];
    const int lane = threadIdx.x;
    const int Dg = p.dim / p.G, cbs = (Dg + CB - 1) / CB;
    const int cb = blockIdx.x % (cbs * p.G), g = cb / cbs, c0 = g * Dg + (cb % cbs) * CB, cend = (g + 1) * Dg;
    const int walked = FULL ? p.chunks : p.chunks - 1;           // nothing reads the summary of the last chunk (BACK: the first)
    const int rest = blockIdx.x / (cbs * p.G), chunk = (BACK ? 1 : 0) + rest % walked, b = rest / walked;
    const int len = __builtin_amdgcn_readfirstlane(seq_len(p.lengths, b, p.L));
    const long tb = (long)chunk * p.CL, tfull = tb + p.CL < p.L ? tb + p.CL : p.L, te = tfull < len ? tfull : len;
    const int n = te > tb ? (int)(te - tb) : 0;                  // tokens to walk; token i is first + dir i
    const long first = BACK ? te - 1 : tb, dir = BACK ? -1 : 1;
    // Lanes beyond the group repeat its block's first channel, bit for bit: what they store is what that lane stores.
    const int ch = c0 + lane < cend ? c0 + lane : c0;
    // Every stream is a uniform running pointer, to the next token to fetch, and the lane's byte offset in a row.  The rows of B and C of
    // GT tokens come as RV values to a lane: value lane + 64 r is state (lane + 64 r) % NP of token (lane + 64 r) / NP.
    const bool gated = MODE != SCAN_STATES && p.z != nullptr;
    const unsigned chb = ch * (unsigned)sizeof(T);
    const int rn = lane % NP, rt = lane / NP;
    const bool okr = rn < p.N && rt < GT;
    const long ut = (BACK ? -p.so.t : p.su.t) * (long)sizeof(T), dt = dir * p.sd.t * (long)sizeof(T), zt = gated ? dir * p.sz.t * (long)sizeof(T) : dt;
    const long Bt = p.sB.t * (long)sizeof(T), Ct = dir * p.sC.t * (long)sizeof(T), yt = (long)p.dim * sizeof(T);
    const char *pu = reinterpret_cast<const char *>(BACK ? p.dout : p.u) + (BACK ? b * p.so.b + first * p.so.t : b * p.su.b + first * p.su.t) * (long)sizeof(T);
    const char *pd = reinterpret_cast<const char *>(p.delta) + (b * p.sd.b + first * p.sd.t) * (long)sizeof(T);
    const char *pz = gated ? reinterpret_cast<const char *>(p.z) + (b * p.sz.b + first * p.sz.t) * (long)sizeof(T) : pd;
    const char *pB = reinterpret_cast<const char *>(p.B) + (b * p.sB.b + first * p.sB.t + (long)g * p.N) * (long)sizeof(T);
    const char *pC = reinterpret_cast<const char *>(p.C) + (b * p.sC.b + first * p.sC.t + (long)g * p.N) * (long)sizeof(T);
    char *py = reinterpret_cast<char *>(p.y) + ((long)b * p.L + tb) * p.dim * (long)sizeof(T);
    const float bias = p.bias ? p.bias[ch] : 0.0f, skip = p.D ? p.D[ch] : 0.0f;
    const bool sp = p.softplus != 0;

    float A2[NP], h0[NP];
    f32x4 h[NP / 4];
    load_states<NP>(p.A + (long)ch * p.N, 0, p.N, states_vec(p.A, p.N, 4), A2);
#pragma unroll
    for (int k = 0; k < NP; ++k) { A2[k] = a_log2(A2[k]); h0[k] = 0.0f; }
    if (FULL && chunk > 0) load_states<NP>(p.S + (((long)b * p.chunks + chunk - 1) * p.dim + ch) * NP, 0, NP, true, h0);
    else if (!BACK && p.state && chunk == 0) load_states<NP>(p.state + ((long)b * p.dim + ch) * p.N, 0, p.N, states_vec(p.state, p.N, 4), h0);
#pragma unroll
    for (int k = 0; k < NP; ++k) h[k / 4][k % 4] = h0[k];
    float total = 0.0f;                                          // summaries: the chunk's sum of steps

    const long offr = (okr ? rn : 0) * (long)sizeof(T), offB = (okr ? rt : 0) * Bt + offr, offC = (okr ? rt : 0) * Ct + offr;
    T fu[GT], fd[GT], fz[GT], fB[RV], fC[RV];
    auto fetch_tokens = [&](int left) {                          // the next min(GT, left) tokens; the last again where there are fewer
        if (left >= GT) {
#pragma unroll
            for (int r = 0; r < RV; ++r) {
                if (!BACK) fB[r] = *reinterpret_cast<const T *>(pB + r * TPV * Bt + offB);
                if (MODE != SCAN_STATES) fC[r] = *reinterpret_cast<const T *>(pC + r * TPV * Ct + offC);
            }
            pB += GT * Bt;
            pC += GT * Ct;
#pragma unroll
            for (int j = 0; j < GT; ++j) {
                fu[j] = *reinterpret_cast<const T *>(pu + chb);
                fd[j] = *reinterpret_cast<const T *>(pd + chb);
                if (MODE != SCAN_STATES) fz[j] = *reinterpret_cast<const T *>(pz + chb);
                pu += ut;
                pd += dt;
                pz += zt;
            }
        } else {
#pragma unroll
            for (int r = 0; r < RV; ++r) {
                const int t = okr ? r * TPV + rt : 0, k = t < left ? t : left - 1;
                if (!BACK) fB[r] = *reinterpret_cast<const T *>(pB + k * Bt + offr);
                if (MODE != SCAN_STATES) fC[r] = *reinterpret_cast<const T *>(pC + k * Ct + offr);
            }
#pragma unroll
            for (int j = 0; j < GT; ++j) {
                const long k = j < left ? j : left - 1;
                fu[j] = *reinterpret_cast<const T *>(pu + k * ut + chb);
                fd[j] = *reinterpret_cast<const T *>(pd + k * dt + chb);
                if (MODE != SCAN_STATES) fz[j] = *reinterpret_cast<const T *>(pz + k * zt + chb);
            }
        }
    };
    if (n > 0) fetch_tokens(n);
    for (int i = 0; i < n; i += GT) {
        float st[GT], in[GT], gate[GT], uf[GT], row[RV];         // row: B's; BACK: C's
#pragma unroll
        for (int r = 0; r < RV; ++r) {
            row[r] = okr ? to_f(BACK ? fC[r] : fB[r]) : 0.0f;
            if (FULL && rt < GT) s_C[lane + 64 * r] = okr ? to_f(fC[r]) : 0.0f;
        }
        if (FULL) __syncthreads();                               // one wave: orders the rows' writes before their reads
#pragma unroll
        for (int j = 0; j < GT; ++j) {
            const float raw = to_f(fd[j]) + bias, s = softplus_f(raw);
            st[j] = sp ? s : raw;
            uf[j] = to_f(fu[j]);
            const float sl = MODE == SCAN_STATES ? 1.0f : silu_f(to_f(fz[j]));
            gate[j] = gated ? sl : 1.0f;
            in[j] = uf[j] * (BACK ? gate[j] : st[j]);            // step u, or d
        }
        if (i + GT < n) fetch_tokens(n - (i + GT));
        auto checkpoint = [&](int j) {                           // the state before token tb + i + j
            const int blk = 16 * urnn_scan_ed(NP), cl = ch - g * Dg, cbeg = cl / blk * blk, w = Dg - cbeg < blk ? Dg - cbeg : blk;
            const long seg = (tb + i + j) / CK, segs = (p.L + CK - 1) / CK;
            f32x4 *k = reinterpret_cast<f32x4 *>(p.keep + (((long)b * segs + seg) * p.dim + g * Dg + cbeg + keep_rank(cl - cbeg, w, urnn_scan_v(NP))) * NP);
#pragma unroll
            for (int e = 0; e < NP / 4; ++e) k[e] = h[e];
        };
        auto token = [&](auto jc) {
            constexpr int j = decltype(jc)::value;
            if (FULL && j % (CK < GT ? CK : GT) == 0 && (i + j) % CK == 0 && p.keep) checkpoint(j);
            if (BACK) add_outer<j, 0, NP, RV>(row, in[j], h);        // h <- a (h + C d), otherwise h <- a h + B (step u)
#pragma unroll
            for (int k = 0; k < NP; ++k) h[k / 4][k % 4] *= __builtin_amdgcn_exp2f(st[j] * A2[k]);
            if (!BACK) add_outer<j, 0, NP, RV>(row, in[j], h);
            if (FULL) {
                float y0 = 0.0f, y1 = 0.0f;
#pragma unroll
                for (int k = 0; k < NP / 4; ++k) {
                    const f32x4 c = *reinterpret_cast<const f32x4 *>(s_C + j * NP + 4 * k);
                    y0 = fmaf(c[0], h[k][0], y0);
                    y1 = fmaf(c[1], h[k][1], y1);
                    y0 = fmaf(c[2], h[k][2], y0);
                    y1 = fmaf(c[3], h[k][3], y1);
                }
                const float v = fmaf(skip, uf[j], y0 + y1) * gate[j];
                *reinterpret_cast<T *>(py + chb) = from_f<T>(v);
                py += yt;
            } else {
                total += st[j];
            }
        };
        if (i + GT <= n) tokens<true>(token, GT, std::make_integer_sequence<int, GT>());
        else tokens<false>(token, n - i, std::make_integer_sequence<int, GT>());
    }
#pragma unroll
    for (int k = 0; k < NP; ++k) h0[k] = h[k / 4][k % 4];
    if (FULL) {
        for (long t = tb + n; t < tfull; ++t, py += yt) *reinterpret_cast<T *>(py + chb) = from_f<T>(0.0f);      // rows behind the sequence are zeros
        const int last = len > 0 ? (len - 1) / p.CL : 0;         // the chunk that holds the sequence's last token
        if (p.state_out && chunk == last)
            store_states<NP>(p.state_out + ((long)b * p.dim + ch) * p.N, 0, p.N, states_vec(p.state_out, p.N, 4), h0);
    } else {
        p.sum[((long)b * p.chunks + chunk) * p.dim + ch] = total;
        store_states<NP>(p.S + (((long)b * p.chunks + chunk) * p.dim + ch) * NP, 0, NP, true, h0);
    }
}

// S[c] (a chunk's end state from a zero start; chunk 0 from the given state) -> the end state itself:
// H[c] = exp(A sum[c]) H[c - 1] + S[c].  One thread per (b, d, n); the loads do not depend on the chain.  A chunk without tokens
// (sum 0) passes the state on as it is, also where A is infinite; a state of zero stays out of it, also where A is positive and the
// product of a chunk's decays overflows.
template <int NP>
__global__ __launch_bounds__(256) void scan_carry_kernel(const float *__restrict__ A, const float *__restrict__ sum, float *S, int dim, int N, int chunks, long count)
{
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= count) return;
    const long b = i / ((long)dim * NP), r = i % ((long)dim * NP);
    const int d = (int)(r / NP), n = (int)(r % NP);
    const float A2 = n < N ? a_log2(A[(long)d * N + n]) : 0.0f;
    float *s = S + b * chunks * dim * NP + r;
    const float *w = sum + b * chunks * dim + d;
    float h = s[0];
    constexpr int U = 16;
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
                h = wv[k] == 0.0f || h == 0.0f ? h + sv[k] : fmaf(__builtin_amdgcn_exp2f(wv[k] * A2), h, sv[k]);
                s[(long)(c0 + k) * dim * NP] = h;
            }
    }
}

// A launch's blocks: the chunks of a sequence, then the next sequence.  (The sequences of a chunk first, so that a padded batch's empty
// chunks come last: 7 x 1021 x 1000 63 against 67 us, but 2 x 19 166 x 1032 359 against 333 and 12 x 3000 x 1500 277 against 257.)
//
// Chunks of the time axis: one from 640 waves on, below that as many as give 9216 waves (three turns of the three that each of the 1024
// SIMDs holds), but none shorter than 32 tokens.  The border, sequences of 2048 tokens bf16 cut and in one chunk: 128 waves 145 and 659 us,
// 320 301 and 680, 608 530 and 684, 640 572 and 684, 896 778 and 696 -- the two meet near 800, so that between 640 and there one chunk
// loses up to a sixth.  Waves are counted as of one group: several narrow groups launch more of them than the rule knows of.
// The number, measured with 3000 waves of 64 tokens at least and with 9216 of 32: 32 768 tokens of 2048 channels 483 and 462 us (12 288:
// 476), seven sequences of up to 1021 tokens of 1000 channels 72 and 67; a training step of 4 x 2048 x 2048, whose forward takes the same
// chunks, loses by it: 482 and 495.
int urnn_scan_chunks(int B, int L, int D, int *CL)
{
    const long waves = (long)B * ((D + URNN_SCAN_CB - 1) / URNN_SCAN_CB);
    long want = waves >= 640 ? 1 : (9216 + waves - 1) / waves;
    const long most = (L + 31) / 32;
    if (want > most) want = most;
    if (want < 1) want = 1;
    long cl = (L + want - 1) / want;
    cl = (cl + 15) / 16 * 16;
    *CL = (int)cl;
    return (int)((L + cl - 1) / cl);
}

template <typename T, int NP, int MODE>
static void launch_pass(const ScanParams &p, hipStream_t st)
{
    const int Dg = p.dim / p.G, cbs = p.G * ((Dg + URNN_SCAN_CB - 1) / URNN_SCAN_CB);
    const int walked = MODE == SCAN_FULL ? p.chunks : p.chunks - 1;
    scan_kernel<T, NP, MODE><<<dim3((unsigned)(cbs * walked * p.batch)), 64, 0, st>>>(p);
}

template <typename T, int NP>
static hipError_t launch_scan(const ScanParams &p, hipStream_t st)
{
    if (p.chunks > 1) {
        launch_pass<T, NP, SCAN_STATES>(p, st);
        const long count = (long)p.batch * p.dim * NP;
        scan_carry_kernel<NP><<<dim3((unsigned)((count + 255) / 256)), 256, 0, st>>>(p.A, p.sum, p.S, p.dim, p.N, p.chunks, count);
    }
    launch_pass<T, NP, SCAN_FULL>(p, st);
    return hipGetLastError();
}

// One token: state and inputs are read once, the new state and y written once.  A quad per channel, no LDS; a thread takes the same
// channel of R sequences, so that their loads are in flight together and A, bias and skip are read once for them.  state_out may be
// state: every thread reads its own states before it writes them.  Memory-bound: 256 x 4096 channels of 16 states 29.6 us, 4.8 TB/s;
// one sequence of 192 channels 3 us, and 13 for the call.
template <typename T, int E>
__device__ __forceinline__ void load_row(const T *row, int q, int N, bool vec, float (&v)[E])
{
    constexpr int W = E < 4 ? E : 4;
    if (vec) {
#pragma unroll
        for (int e = 0; e < E; e += W) {
            Pack<T, W> t = {};
            if (q * E + e < N) t = *reinterpret_cast<const Pack<T, W> *>(row + q * E + e);
#pragma unroll
            for (int i = 0; i < W; ++i) v[e + i] = to_f(t.v[i]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = q * E + e < N ? to_f(row[q * E + e]) : 0.0f;
    }
}

template <typename T, int NP, int R>
__global__ __launch_bounds__(256) void scan_step_kernel(const ScanParams p)
{
    constexpr int E = NP / 4, W = E < 4 ? E : 4;
    const unsigned item = blockIdx.x * 64u + (threadIdx.x >> 2), d = item % p.dim;
    const int q = threadIdx.x & 3, b0 = (int)(item / p.dim) * R, g = d / (p.dim / p.G);
    if (b0 >= p.batch) return;
    const bool vs = states_vec(p.state, p.N, W), vo = states_vec(p.state_out, p.N, W);
    const bool vB = ((reinterpret_cast<uintptr_t>(p.B) | (p.sB.b | p.N) * sizeof(T)) & (W * sizeof(T) - 1)) == 0;
    const bool vC = ((reinterpret_cast<uintptr_t>(p.C) | (p.sC.b | p.N) * sizeof(T)) & (W * sizeof(T) - 1)) == 0;
    float h[R][E], Bv[R][E], Cv[R][E], A2[E], u[R], dl[R], zf[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const long b = b0 + r < p.batch ? b0 + r : b0;
        load_states<E>(p.state + (b * p.dim + d) * p.N, q, p.N, vs, h[r]);
        load_row<T, E>(reinterpret_cast<const T *>(p.B) + b * p.sB.b + (long)g * p.N, q, p.N, vB, Bv[r]);
        load_row<T, E>(reinterpret_cast<const T *>(p.C) + b * p.sC.b + (long)g * p.N, q, p.N, vC, Cv[r]);
        u[r] = to_f(reinterpret_cast<const T *>(p.u)[b * p.su.b + d]);
        dl[r] = to_f(reinterpret_cast<const T *>(p.delta)[b * p.sd.b + d]);
        zf[r] = p.z ? to_f(reinterpret_cast<const T *>(p.z)[b * p.sz.b + d]) : 0.0f;
    }
    load_states<E>(p.A + (long)d * p.N, q, p.N, states_vec(p.A, p.N, W), A2);
    const float bias = p.bias ? p.bias[d] : 0.0f, skip = p.D ? p.D[d] : 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (b0 + r >= p.batch) break;
        const long b = b0 + r;
        const float raw = dl[r] + bias, step = p.softplus ? softplus_f(raw) : raw, su = step * u[r];
        float y = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            h[r][e] = fmaf(exp_fast(step * A2[e]), h[r][e], su * Bv[r][e]);
            y = fmaf(Cv[r][e], h[r][e], y);
        }
        y = fmaf(skip, u[r], quad_sum(y));
        if (p.z) y *= silu_f(zf[r]);
        store_states<E, true>(p.state_out + (b * p.dim + d) * p.N, q, p.N, vo, h[r]);
        if (q == 0) reinterpret_cast<T *>(p.y)[b * p.dim + d] = from_f<T>(y);
    }
}

template <typename T, int NP, int R>
static hipError_t launch_step_rows(const ScanParams &p, hipStream_t st)
{
    const long items = (long)((p.batch + R - 1) / R) * p.dim;
    scan_step_kernel<T, NP, R><<<dim3((unsigned)((items + 63) / 64)), 256, 0, st>>>(p);
    return hipGetLastError();
}
// Four sequences to a thread once the threads still fill the chip (2048 blocks of 256): 256 x 4096 44 us with one, 33 with four; fewer
// blocks would leave compute units idle, which a single sequence's call at 192 channels cannot afford.
template <typename T, int NP>
static hipError_t launch_step(const ScanParams &p, hipStream_t st)
{
    if constexpr (NP <= 16)
        if ((long)p.batch * p.dim >= 4l * 64 * 2048) return launch_step_rows<T, NP, 4>(p, st);
    return launch_step_rows<T, NP, 1>(p, st);
}

template <typename T>
static hipError_t by_states(const ScanParams &p, int what, hipStream_t st)
{
    auto go = [&](auto np) {
        constexpr int NP = decltype(np)::value;
        if (what == SCAN_STEP) return launch_step<T, NP>(p, st);
        if (what == SCAN_BACK) { launch_pass<T, NP, SCAN_BACK>(p, st); return hipGetLastError(); }
        return launch_scan<T, NP>(p, st);
    };
    switch (urnn_scan_np(p.N)) {
    case 4: return go(std::integral_constant<int, 4>());
    case 8: return go(std::integral_constant<int, 8>());
    case 16: return go(std::integral_constant<int, 16>());
    case 32: return go(std::integral_constant<int, 32>());
    default: return go(std::integral_constant<int, 64>());
    }
}

static hipError_t by_type(const ScanParams &p, int dtype, int what, hipStream_t st)
{
    return dtype == URNN_F32 ? by_states<float>(p, what, st) : dtype == URNN_BF16 ? by_states<bf16_t>(p, what, st) : by_states<f16_t>(p, what, st);
}

hipError_t urnn_launch_scan(const ScanParams &p, int dtype, hipStream_t st) { return by_type(p, dtype, SCAN_FULL, st); }
hipError_t urnn_launch_scan_step(const ScanParams &p, int dtype, hipStream_t st) { return by_type(p, dtype, SCAN_STEP, st); }
hipError_t urnn_launch_scan_back_summaries(const ScanParams &p, int dtype, hipStream_t st) { return by_type(p, dtype, SCAN_BACK, st); }
