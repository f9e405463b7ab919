// Selective state space scan, backward.  The forward's mathematics and the names: ssm_util.h.
//
// With S the state in front of a block, dS the gradient of the state behind it (both from ssm_states_kernel), per head:
//   G1[t,s] = C_t . B_s,  G2[t,s] = dy_t . x_s,  L[t,s] = exp(a_t - a_s) for s <= t, else 0
//   dx_s = dt_s (sum_t G1 L dy_t + e_s dS B_s) + D dy_s,                     e_s = exp(a_T - a_s)
//   dB_s = sum_t W[t,s] C_t + dt_s e_s dS^T x_s,   dC_t = sum_s W[t,s] B_s + exp(a_t) S^T dy_t,     W = G2 L dt_s
//   R_t = sum_{s<t} Q dt_s + C_t . exp(a_t) S^T dy_t,   K_s = sum_{t>=s} Q[t,s] + B_s . e_s dS^T x_s,   Q = G1 G2 L
//   d(a step)_t = sum_{u>=t} (R_u - dt_u (K_u - Q[u,u])) + exp(a_T) <S, dS> + sum_s dt_s B_s . e_s dS^T x_s
//   d(dt')_t = A d(a step)_t + K_t,   dA = sum_t dt_t d(a step)_t,   dD = sum_t G2[t,t]
// (the diagonal cancels in R - dt K and is left out of both, so that strong decays do not lose the gradient of A in it).
//
// A workgroup owns one block and the heads of one group (or a share of them, where blocks and groups alone are too few): G1 stays in its registers,
// the T x T sums W and the gradients of B and C are added up over the heads there, so dB and dC cost two products per block instead of two per
// head, and no partial sums in memory.  Operands that are f32 by nature are used as three bf16 pieces where an f32 result depends on them (S and dS:
// R, K -> dA, ddt_bias); W and G1 L, which only end in bf16 outputs, are rounded once, and dS in dx takes its first piece.
#include "ssm_util.h"

namespace dc {
namespace {

template <typename T, int NP>
struct BwdLds {
    static constexpr int PIECES = sizeof(T) == 4 ? 1 : PIECES_F32;
    T b[TB * pitch<T>(NP)], c[TB * pitch<T>(NP)], x[TB * pitch<T>(PT)], y[TB * pitch<T>(PT)], s[PIECES][PT * pitch<T>(NP)], m[TB * pitch<T>(TB)];
    Steps st;
    float R[TB], diag[TB], KI[TB], col[16][TB], dot[4], trace[4];
};

// A head's S or dS tile on its way to LDS, as f32 or as three bf16 pieces (the slots' rows are padded to whole vectors).
template <typename T, int NP>
struct StateTile {
    Tile<float, NP, 4> v;
    __device__ __forceinline__ void load(const SsmArgs& a, const float* buf, int64_t slot, int h, int p0, int P) {
        v.load(buf + ((slot * a.H + h) * a.P + p0) * a.NS, a.NS, P, a.NS);
    }
    __device__ __forceinline__ void store(T (*lds)[PT * pitch<T>(NP)], int P, int NS) const {
        if constexpr (sizeof(T) == 4) {
            v.store(lds[0], pitch<T>(NP), P, NS);
        } else {
            typedef bf16_t four __attribute__((ext_vector_type(4)));
#pragma unroll
            for (int k = 0; k < v.N; ++k) {
                const int idx = k * 256 + threadIdx.x, at = idx / v.PER_ROW * pitch<T>(NP) + idx % v.PER_ROW * 4;
                four out[PIECES_F32];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    bf16_t p[PIECES_F32];
                    split_bf16(idx / v.PER_ROW < P && idx % v.PER_ROW * 4 < NS ? v.v[k][e] : 0.f, p);
#pragma unroll
                    for (int pc = 0; pc < PIECES_F32; ++pc) out[pc][e] = p[pc];
                }
#pragma unroll
                for (int pc = 0; pc < PIECES_F32; ++pc) *reinterpret_cast<four*>(lds[pc] + at) = out[pc];
            }
        }
    }
    __device__ __forceinline__ float dot(const StateTile& o, int P, int NS) const {
        float s = 0.f;
#pragma unroll
        for (int k = 0; k < v.N; ++k) {
            const int idx = k * 256 + threadIdx.x;
            if (idx / v.PER_ROW < P && idx % v.PER_ROW * 4 < NS)
#pragma unroll
                for (int e = 0; e < 4; ++e) s = fmaf(v.v[k][e], o.v.v[k][e], s);
        }
        return s;
    }
};

template <typename T, int NP, int V>
__global__ void __launch_bounds__(256) ssm_bwd_kernel(SsmArgs a) {
    typedef Mat<T> M;
    constexpr int LX = pitch<T>(PT), LN = pitch<T>(NP), LM = pitch<T>(TB), NK = NP / M::KS, NC = NP / 16;
    constexpr int PIECES = BwdLds<T, NP>::PIECES;
    extern __shared__ __attribute__((aligned(16))) char lds_raw[];
    BwdLds<T, NP>& L = *reinterpret_cast<BwdLds<T, NP>*>(lds_raw);
    const int slot = blockIdx.x, grp = blockIdx.y, share = blockIdx.z, Hg = a.H / a.G;
    if (slot >= a.base[a.n_seq]) return;
    const int b = a.map[slot], blk = slot - a.base[b];
    const SeqRange q = seq_range(a.seq_off, a.seq_len, b, a.rows, a.max_len);
    const int64_t row0 = q.off + (int64_t)blk * TB;
    const int rows = min(TB, q.len - blk * TB);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, i = lane & 15, g = lane >> 4, N = a.N;
    {
        Tile<T, NP, V> tb, tc;
        tb.load(static_cast<const T*>(a.B) + row0 * a.ldb + (int64_t)grp * N, a.ldb, rows, N);
        tc.load(static_cast<const T*>(a.C) + row0 * a.ldc + (int64_t)grp * N, a.ldc, rows, N);
        tb.store(L.b, LN, rows, N);
        tc.store(L.c, LN, rows, N);
    }
    __syncthreads();
    // this wave's rows: r0 + 4 g + r, of t as of s
    const int r0 = 16 * wave;
    f32x4 G1[TB / 16], W[TB / 16], dB[NC], dC[NC];
#pragma unroll
    for (int c = 0; c < TB / 16; ++c) {
        G1[c] = f32x4{};
        W[c] = f32x4{};
        if (c <= wave) {
#pragma unroll
            for (int k = 0; k < NK; ++k)
                G1[c] = M::mma(M::row(L.c + r0 * LN + k * M::KS, LN, i, g), M::row(L.b + 16 * c * LN + k * M::KS, LN, i, g), G1[c]);
        }
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) { dB[c] = f32x4{}; dC[c] = f32x4{}; }
    const int kbegin = r0 / M::KS * M::KS, kend = (r0 + 16 + M::KS - 1) / M::KS * M::KS;      // rows t >= s, columns s <= t, in whole steps
    const int h_first = grp * Hg + share * Hg / a.hsplit, h_last = grp * Hg + (share + 1) * Hg / a.hsplit;
    for (int h = h_first; h < h_last; ++h) {
        const float A = a.A[h], bias = a.dt_bias ? a.dt_bias[h] : 0.f, D = a.D ? a.D[h] : 0.f;
        float raw = 0.f;
        if (wave == 0) {
            raw = lane < rows ? (float)static_cast<const T*>(a.dt)[(row0 + lane) * a.lddt + h] : 0.f;
            make_steps<false>(L.st, a, raw, lane < rows, A, bias, lane);
        }
        float dot = 0.f, trace = 0.f, R[4] = {}, KI[4] = {}, diag[4] = {}, col[TB / 16] = {};   // sums over this lane's columns
        for (int pt = 0; pt < a.ptiles; ++pt) {
            const int p0 = pt * PT, P = min(a.P - p0, PT);
            Tile<T, PT, V> tx, ty;
            StateTile<T, NP> ts, td;
            tx.load(static_cast<const T*>(a.x) + row0 * a.ldx + (int64_t)h * a.P + p0, a.ldx, rows, P);
            ty.load(static_cast<const T*>(a.dy) + row0 * a.lddy + (int64_t)h * a.P + p0, a.lddy, rows, P);
            ts.load(a, a.S, slot, h, p0, P);
            td.load(a, a.dS, slot, h, p0, P);
            tx.store(L.x, LX, rows, P);
            ty.store(L.y, LX, rows, P);
            ts.store(L.s, P, a.NS);
            dot += ts.dot(td, P, a.NS);
            __syncthreads();
            // the rows with each other
#pragma unroll
            for (int c = 0; c < TB / 16; ++c) {
                f32x4 m = {};
                if (c <= wave) {
                    f32x4 G2 = {};
#pragma unroll
                    for (int k = 0; k < PT / M::KS; ++k)
                        G2 = M::mma(M::row(L.y + r0 * LX + k * M::KS, LX, i, g), M::row(L.x + 16 * c * LX + k * M::KS, LX, i, g), G2);
                    const int s = 16 * c + i;
                    const float hs = L.st.hi[s], ls = L.st.lo[s], ds = L.st.dt[s];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int t = r0 + 4 * g + r;
                        const float l = s <= t ? __expf(gap(L.st, t, hs, ls)) : 0.f, gl = s <= t ? G2[r] * l : 0.f;
                        m[r] = s <= t ? G1[c][r] * l : 0.f;
                        const float qv = s <= t ? G1[c][r] * gl : 0.f;
                        W[c][r] = fmaf(gl, ds, W[c][r]);
                        if (s < t) {
                            col[c] += qv;
                            R[r] = fmaf(qv, ds, R[r]);
                        } else if (s == t) {
                            diag[r] += qv;
                            trace += G2[r];
                        }
                    }
                }
                if (pt == 0) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) L.m[(r0 + 4 * g + r) * LM + 16 * c + i] = (T)m[r];
                }
            }
            // dC_t += exp(a_t) S^T dy_t
            float e[4];
            {
                f32x4 acc[NC];
#pragma unroll
                for (int c = 0; c < NC; ++c) acc[c] = f32x4{};
#pragma unroll
                for (int k = 0; k < PT / M::KS; ++k) {
                    const typename M::frag f = M::row(L.y + r0 * LX + k * M::KS, LX, i, g);
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int pc = PIECES - 1; pc >= 0; --pc) acc[c] = M::mma(f, M::col(L.s[pc] + k * M::KS * LN + 16 * c, LN, i, g), acc[c]);
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) e[r] = __expf(L.st.hi[r0 + 4 * g + r]);
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float v = e[r] * acc[c][r];
                        dC[c][r] += v;
                        R[r] = fmaf(v, (float)L.c[(r0 + 4 * g + r) * LN + 16 * c + i], R[r]);
                    }
            }
            __syncthreads();
            td.store(L.s, P, a.NS);
            __syncthreads();
            // dB_s += dt_s e_s dS^T x_s
            float ds[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int s = r0 + 4 * g + r;
                ds[r] = L.st.dt[s];
                e[r] = __expf(gap(L.st, TB - 1, L.st.hi[s], L.st.lo[s]));
            }
            {
                f32x4 acc[NC];
#pragma unroll
                for (int c = 0; c < NC; ++c) acc[c] = f32x4{};
#pragma unroll
                for (int k = 0; k < PT / M::KS; ++k) {
                    const typename M::frag f = M::row(L.x + r0 * LX + k * M::KS, LX, i, g);
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int pc = PIECES - 1; pc >= 0; --pc) acc[c] = M::mma(f, M::col(L.s[pc] + k * M::KS * LN + 16 * c, LN, i, g), acc[c]);
                }
#pragma unroll
                for (int c = 0; c < NC; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float v = e[r] * acc[c][r];
                        dB[c][r] = fmaf(ds[r], v, dB[c][r]);
                        KI[r] = fmaf(v, (float)L.b[(r0 + 4 * g + r) * LN + 16 * c + i], KI[r]);
                    }
            }
            // dx_s = dt_s (e_s dS B_s + sum_t G1 L dy_t) + D dy_s
            {
                f32x4 acc[PT / 16];
#pragma unroll
                for (int c = 0; c < PT / 16; ++c) acc[c] = f32x4{};
#pragma unroll
                for (int k = 0; k < NK; ++k) {
                    const typename M::frag f = M::row(L.b + r0 * LN + k * M::KS, LN, i, g);
#pragma unroll
                    for (int c = 0; c < PT / 16; ++c) acc[c] = M::mma(f, M::row(L.s[0] + 16 * c * LN + k * M::KS, LN, i, g), acc[c]);
                }
#pragma unroll
                for (int c = 0; c < PT / 16; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[c][r] *= e[r];
                for (int k = kbegin; k < TB; k += M::KS) {
                    const typename M::frag f = M::col(L.m + k * LM + r0, LM, i, g);
#pragma unroll
                    for (int c = 0; c < PT / 16; ++c) acc[c] = M::mma(f, M::col(L.y + k * LX + 16 * c, LX, i, g), acc[c]);
                }
                // out through this wave's rows of x, which nobody else reads any more
                T* out = L.x + r0 * LX;
#pragma unroll
                for (int c = 0; c < PT / 16; ++c)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        out[(4 * g + r) * LX + 16 * c + i] = (T)fmaf(ds[r], acc[c][r], D * (float)L.y[(r0 + 4 * g + r) * LX + 16 * c + i]);
                typedef T vec_t __attribute__((ext_vector_type(V)));
                constexpr int PER_ROW = PT / V;
                T* dx = static_cast<T*>(a.dx) + (row0 + r0) * a.lddx + (int64_t)h * a.P + p0;
#pragma unroll
                for (int k = 0; k < 16 * PER_ROW / 64; ++k) {
                    const int idx = k * 64 + lane, r = idx / PER_ROW, c = idx % PER_ROW * V;
                    if (r0 + r < rows && c < P) *reinterpret_cast<vec_t*>(dx + r * a.lddx + c) = *reinterpret_cast<const vec_t*>(out + r * LX + c);
                }
            }
            if (pt + 1 == a.ptiles) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float sR = sum16(R[r]), sK = sum16(KI[r]), sd = sum16(diag[r]);
                    if (i == 0) { L.R[r0 + 4 * g + r] = sR; L.KI[r0 + 4 * g + r] = sK; L.diag[r0 + 4 * g + r] = sd; }
                }
#pragma unroll
                for (int c = 0; c < TB / 16; ++c) L.col[4 * wave + g][16 * c + i] = col[c];
                dot = wave_sum(dot);
                trace = wave_sum(trace);
                if (lane == 0) { L.dot[wave] = dot; L.trace[wave] = trace; }
            }
            __syncthreads();
        }
        if (wave == 0) {                                     // lane = row
            float K = L.KI[lane];
#pragma unroll
            for (int k = 0; k < 16; ++k) K += L.col[k][lane];
            const float d = L.st.dt[lane];
            // exp(a_T) <S, dS> + sum_s dt_s KI_s reach every row of the block: they stand behind its last one
            const double behind = (double)__expf(L.st.total) * (double)((L.dot[0] + L.dot[1]) + (L.dot[2] + L.dot[3])) + wave_sum((double)(d * L.KI[lane]));
            const double da = (double)L.R[lane] - (double)(d * K);
            const double pre = wave_prefix(da, lane), all = __shfl(pre, 63, 64);
            const float suffix = (float)(all - pre + da + behind);
            float ddt = fmaf(A, suffix, K + L.diag[lane]);
            if (a.softplus) ddt *= 1.f / (1.f + expf(-(raw + bias)));
            if (lane >= rows) ddt = 0.f;
            if (lane < rows) static_cast<T*>(a.ddt)[(row0 + lane) * a.ldddt + h] = (T)ddt;
            const float sA = wave_sum(d * suffix), sb = wave_sum(ddt);
            if (lane == 0) {
                float* p = a.part + ((int64_t)slot * a.H + h) * 3;
                p[0] = sA;
                p[1] = (L.trace[0] + L.trace[1]) + (L.trace[2] + L.trace[3]);
                p[2] = sb;
            }
        }
    }
    // dC_t += sum_s W[t,s] B_s, dB_s += sum_t W[t,s] C_t
    // (no wave reads m between here and the barrier; wave 0's last rows of R, K, .. are not touched any more)
#pragma unroll
    for (int c = 0; c < TB / 16; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) L.m[(r0 + 4 * g + r) * LM + 16 * c + i] = (T)W[c][r];
    __syncthreads();
    for (int k = 0; k < kend; k += M::KS) {
        const typename M::frag f = M::row(L.m + r0 * LM + k, LM, i, g);
#pragma unroll
        for (int c = 0; c < NC; ++c) dC[c] = M::mma(f, M::col(L.b + k * LN + 16 * c, LN, i, g), dC[c]);
    }
    for (int k = kbegin; k < TB; k += M::KS) {
        const typename M::frag f = M::col(L.m + k * LM + r0, LM, i, g);
#pragma unroll
        for (int c = 0; c < NC; ++c) dB[c] = M::mma(f, M::col(L.c + k * LN + 16 * c, LN, i, g), dB[c]);
    }
    if (a.hsplit > 1) {
        float* p = a.part_bc + (((int64_t)share * a.rows + row0) * a.G + grp) * 2 * N;
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = r0 + 4 * g + r, n = 16 * c + i;
                if (t < rows && n < N) {
                    float* o = p + (int64_t)t * a.G * 2 * N + n;
                    o[0] = dB[c][r];
                    o[N] = dC[c][r];
                }
            }
        return;
    }
    typedef T vec_t __attribute__((ext_vector_type(V)));
    constexpr int PER_ROW = NP / V;
    T* const out = L.s[0] + r0 * LN;                          // this wave's rows; S and dS are used up
#pragma unroll
    for (int w = 0; w < 2; ++w) {
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) out[(4 * g + r) * LN + 16 * c + i] = (T)(w ? dC[c][r] : dB[c][r]);
        const int64_t ld = w ? a.lddc : a.lddb;
        T* const p = static_cast<T*>(w ? a.dC : a.dB) + (row0 + r0) * ld + (int64_t)grp * N;
#pragma unroll
        for (int k = 0; k < 16 * PER_ROW / 64; ++k) {
            const int idx = k * 64 + lane, r = idx / PER_ROW, c = idx % PER_ROW * V;
            if (r0 + r < rows && c < N) *reinterpret_cast<vec_t*>(p + r * ld + c) = *reinterpret_cast<const vec_t*>(out + r * LN + c);
        }
    }
}

// The first slot of each sequence (its blocks have consecutive ones) and the sequence of each slot.  One workgroup.  Slots are counted to `cap`:
// sequences that overlap, which the rows do not allow for, are cut there.
__global__ void __launch_bounds__(1024) ssm_slots_kernel(SsmArgs a) {
    __shared__ int64_t sums[16], carry;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid == 0) carry = 0;
    __syncthreads();
    for (int b0 = 0; b0 < a.n_seq; b0 += 1024) {
        const int b = b0 + tid;
        int64_t n = 0;
        if (b < a.n_seq) n = blocks_of(seq_range(a.seq_off, a.seq_len, b, a.rows, a.max_len).len);
        int64_t v = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t u = __shfl_up((long long)v, o, 64);
            if (lane >= o) v += u;
        }
        if (lane == 63) sums[wave] = v;
        __syncthreads();
        int64_t before = carry;
        for (int w = 0; w < wave; ++w) before += sums[w];
        const int end = (int)min(before + v, (int64_t)a.cap), begin = (int)min(before + v - n, (int64_t)a.cap);
        if (b < a.n_seq) {
            a.base[b + 1] = end;
            for (int k = begin; k < end; ++k) a.map[k] = b;
        }
        __syncthreads();
        if (tid == 1023) carry = min(before + v, (int64_t)a.cap);
        __syncthreads();
    }
    if (tid == 0) a.base[0] = 0;
}

// The heads' shares of dB and dC.  A workgroup per slot and group.
template <typename T>
__global__ void __launch_bounds__(256) ssm_bc_kernel(SsmArgs a) {
    const int slot = blockIdx.x, grp = blockIdx.y, N = a.N;
    if (slot >= a.base[a.n_seq]) return;
    const int b = a.map[slot], blk = slot - a.base[b];
    const SeqRange q = seq_range(a.seq_off, a.seq_len, b, a.rows, a.max_len);
    const int64_t row0 = q.off + (int64_t)blk * TB;
    const int rows = min(TB, q.len - blk * TB);
    for (int e = threadIdx.x; e < rows * 2 * N; e += 256) {
        const int r = e / (2 * N), n = e % (2 * N);
        float s = 0.f;
        for (int k = 0; k < a.hsplit; ++k) s += a.part_bc[(((int64_t)k * a.rows + row0 + r) * a.G + grp) * 2 * N + n];
        if (n < N) static_cast<T*>(a.dB)[(row0 + r) * a.lddb + (int64_t)grp * N + n] = (T)s;
        else static_cast<T*>(a.dC)[(row0 + r) * a.lddc + (int64_t)grp * N + n - N] = (T)s;
    }
}

// dA, dD, ddt_bias of one head: the slots' sums, in f64 and always in the same order.
__global__ void __launch_bounds__(256) ssm_params_kernel(SsmArgs a) {
    const int h = blockIdx.x, n = a.base[a.n_seq];
    double s[3] = {};
#pragma unroll 4
    for (int k = threadIdx.x; k < n; k += 256) {
        const float* p = a.part + ((int64_t)k * a.H + h) * 3;
#pragma unroll
        for (int j = 0; j < 3; ++j) s[j] += (double)p[j];
    }
    __shared__ double red[3][4];
#pragma unroll
    for (int j = 0; j < 3; ++j) {
        s[j] = wave_sum(s[j]);
        if ((threadIdx.x & 63) == 0) red[j][threadIdx.x >> 6] = s[j];
    }
    __syncthreads();
    if (threadIdx.x < 3) {
        float* out = threadIdx.x == 0 ? a.dA : threadIdx.x == 1 ? a.dD : a.ddt_bias;
        const double* v = red[threadIdx.x];
        if (out) out[h] = (float)((v[0] + v[1]) + (v[2] + v[3]));
    }
}

template <typename T, int NP, int V>
int launch_bwd(const SsmArgs& a, hipStream_t s) {
    constexpr size_t bytes = sizeof(BwdLds<T, NP>);
    static_assert(bytes <= 160 * 1024, "LDS of a workgroup");
    if (bytes > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(ssm_bwd_kernel<T, NP, V>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != hipSuccess) { set_error("dc_ssm_scan_bwd: LDS", (int)e); return (int)e; }
    }
    hipLaunchKernelGGL((ssm_bwd_kernel<T, NP, V>), dim3(a.cap, a.G, a.hsplit), dim3(256), bytes, s, a);
    return launch_check("dc_ssm_scan_bwd");
}
template <typename T, int V>
int launch_bwd_n(const SsmArgs& a, hipStream_t s) {
    return a.N <= 32 ? launch_bwd<T, 32, V>(a, s) : a.N <= 64 ? launch_bwd<T, 64, V>(a, s) : launch_bwd<T, 128, V>(a, s);
}

bool bwd_vec(const SsmArgs& a, int type) {
    const int V = type ? 8 : 4;
    uintptr_t p = 0;
    for (const void* t : {a.x, a.B, a.C, a.dy, (const void*)a.dx, (const void*)a.dB, (const void*)a.dC, (const void*)a.h0, (const void*)a.dhT, (const void*)a.dh0}) p |= reinterpret_cast<uintptr_t>(t);
    return a.P % V == 0 && a.N % V == 0 && a.ldx % V == 0 && a.ldb % V == 0 && a.ldc % V == 0 && a.lddy % V == 0 && a.lddx % V == 0 && a.lddb % V == 0 &&
           a.lddc % V == 0 && (p & 15) == 0;
}

constexpr int64_t BWD_WORKGROUPS = 512;

// Everything that depends on the sizes alone; returns the scratch's bytes and, with a pointer, places its parts.
int64_t bwd_plan(SsmArgs& a, char* scratch) {
    ssm_segments(a, BWD_WORKGROUPS / 2);                     // both directions run in one launch
    const int64_t cap = a.rows / TB + a.n_seq, blocks = (int64_t)a.n_seq * blocks_of(a.max_len);
    a.cap = (int)cap;
    a.NS = (a.N + 7) / 8 * 8;
    const int64_t have = (blocks < cap ? blocks : cap) * a.G;
    int64_t split = have > 0 ? BWD_WORKGROUPS / have : 1;
    if (split > a.H / a.G) split = a.H / a.G;
    a.hsplit = split < 1 ? 1 : (int)split;
    int64_t at = 0;
    auto take = [&](int64_t bytes) {
        char* p = scratch ? scratch + at : nullptr;
        at += (bytes + 255) / 256 * 256;
        return p;
    };
    a.base = reinterpret_cast<int32_t*>(take(4 * ((int64_t)a.n_seq + 1)));
    a.map = reinterpret_cast<int32_t*>(take(4 * cap));
    a.part = reinterpret_cast<float*>(take(12 * cap * a.H));
    a.S = reinterpret_cast<float*>(take(4 * cap * a.H * a.P * a.NS));
    a.dS = reinterpret_cast<float*>(take(4 * cap * a.H * a.P * a.NS));
    if (a.nseg > 1) {
        const int64_t n = (int64_t)a.n_seq * a.nseg * a.H;
        a.seg_state = reinterpret_cast<float*>(take(4 * n * a.P * a.N));
        a.seg_dstate = reinterpret_cast<float*>(take(4 * n * a.P * a.N));
        a.seg_a = reinterpret_cast<float*>(take(4 * n));
    }
    if (a.hsplit > 1) a.part_bc = reinterpret_cast<float*>(take(8 * a.hsplit * a.rows * a.G * a.N));
    return at;
}

}  // namespace

int64_t ssm_scan_bwd_scratch(int64_t rows, int n_seq, int max_len, int H, int P, int G, int N) {
    if (rows < 0 || n_seq < 0 || max_len < 0 || H < 1 || G < 1 || H % G || P < 1 || N < 1) return 0;
    SsmArgs a = {};
    a.rows = rows; a.n_seq = n_seq; a.max_len = max_len; a.H = H; a.P = P; a.G = G; a.N = N;
    return bwd_plan(a, nullptr);
}

int ssm_scan_bwd(SsmArgs a, int type, void* scratch, int64_t scratch_bytes, hipStream_t s) {
    if (int rc = ssm_check("dc_ssm_scan_bwd", a, type)) return rc;
    if (a.rows / TB + a.n_seq > 0x7fffffff || a.G > 65535) { set_error("dc_ssm_scan_bwd", 1103); return 1103; }
    if (!a.dA || (a.rows && (!a.dy || !a.dx || !a.ddt || !a.dB || !a.dC))) { set_error("dc_ssm_scan_bwd", 1104); return 1104; }
    if (!scratch || (reinterpret_cast<uintptr_t>(scratch) & 15) || scratch_bytes < bwd_plan(a, static_cast<char*>(scratch))) {
        set_error("dc_ssm_scan_bwd: scratch", 1105);
        return 1105;
    }
    if (work_items(a) > 0x7fffffff) { set_error("dc_ssm_scan_bwd", 1103); return 1103; }
    const bool vec = bwd_vec(a, type);
    hipLaunchKernelGGL(ssm_slots_kernel, dim3(1), dim3(1024), 0, s, a);
    if (int rc = launch_check("dc_ssm_scan_bwd")) return rc;
    if (a.n_seq) {
        if (a.nseg > 1) {
            if (int rc = ssm_states(a, type, vec, true, true, s)) return rc;
            if (int rc = ssm_join_segments(a, true, s)) return rc;
        }
        if (int rc = ssm_states(a, type, vec, true, false, s)) return rc;
        int rc;
        if (type == 0) rc = vec ? launch_bwd_n<float, 4>(a, s) : launch_bwd_n<float, 1>(a, s);
        else rc = vec ? launch_bwd_n<bf16_t, 8>(a, s) : launch_bwd_n<bf16_t, 1>(a, s);
        if (rc) return rc;
        if (a.hsplit > 1) {
            if (type == 0) hipLaunchKernelGGL(ssm_bc_kernel<float>, dim3(a.cap, a.G), dim3(256), 0, s, a);
            else hipLaunchKernelGGL(ssm_bc_kernel<bf16_t>, dim3(a.cap, a.G), dim3(256), 0, s, a);
            if (int rc2 = launch_check("dc_ssm_scan_bwd")) return rc2;
        }
    }
    hipLaunchKernelGGL(ssm_params_kernel, dim3(a.H), dim3(256), 0, s, a);
    return launch_check("dc_ssm_scan_bwd");
}

}  // namespace dc
