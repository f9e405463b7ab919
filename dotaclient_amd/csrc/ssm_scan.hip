// Selective state space scan over packed sequences, forward, and the single step.  The mathematics: ssm_util.h.
//
// Prompts: a workgroup of four waves walks the blocks of one sequence (or of one segment of it), one head and up to 64 of its columns p, sixteen a wave.
// The state stays in the accumulators from the first block to the last, x, B, C are read once and y is written once.  Per block:
//   M[t][s] = exp(a_t - a_s) (C_t . B_s) dt_s, the ten 16 x 16 tiles with s <= t shared out evenly over the waves, through LDS;
//   y^T = x^T M^T + exp(a_t) S C^T + D x^T and the new state for each wave's own columns, so that no wave waits for another one's part of S.
// Where the sequences, heads and columns give too few workgroups (few, long sequences) the sequences are cut into segments: a first kernel computes what
// each segment adds to a zero state, a second one runs along the segments, and the scan starts each segment from there.
#include "ssm_util.h"

namespace dc {
namespace {

template <typename T, int NP>
struct FwdLds {
    T x[TB * pitch<T>(PT)], b[TB * pitch<T>(NP)], c[TB * pitch<T>(NP)], m[TB * pitch<T>(TB)];
    Steps st[2];
};

// The twelve 16 x 16 tiles (row tile, column tile) of M that products with it read: ten with s <= t, and two zero ones that complete
// the 32-column steps of row tiles 0 and 2.  Wave w takes w, w + 4, w + 8.
__device__ __forceinline__ int tile_row(int u) { return (0x203323213210ull >> (4 * u)) & 15; }
__device__ __forceinline__ int tile_col(int u) { return (0x310102103210ull >> (4 * u)) & 15; }

template <typename T, int NP, int V>
__global__ void __launch_bounds__(256) ssm_fwd_kernel(SsmArgs a) {
    typedef Mat<T> M;
    constexpr int LX = pitch<T>(PT), LN = pitch<T>(NP), LM = pitch<T>(TB), NK = NP / M::KS;
    extern __shared__ __attribute__((aligned(16))) char lds_raw[];
    FwdLds<T, NP>& L = *reinterpret_cast<FwdLds<T, NP>*>(lds_raw);
    int unit, h, pbase;
    if (!work_item(a, unit, h, pbase)) return;
    const int b = unit / a.nseg, seg = unit % a.nseg, grp = h / (a.H / a.G);
    const SeqRange q = seq_range(a.seq_off, a.seq_len, b, a.rows, a.max_len);
    const int nb = blocks_of(q.len), first = seg * a.seg_blocks;
    if (first >= nb && seg > 0) return;
    const int last = min(nb, first + a.seg_blocks);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4, p0 = 16 * wave;
    const int P = min(a.P - pbase, PT), N = a.N;
    const int64_t state_at = ((int64_t)b * a.H + h) * a.P * N + (int64_t)pbase * N;
    f32x4 S[NP / 16];
    const float* init = a.nseg > 1 ? a.seg_state + ((int64_t)unit * a.H + h) * a.P * N + (int64_t)pbase * N : a.h0 ? a.h0 + state_at : nullptr;
    load_state<NP, V>(S, init, N, p0, P, N, i, g);
    const float A = a.A[h], bias = a.dt_bias ? a.dt_bias[h] : 0.f, D = a.D ? a.D[h] : 0.f;
    const T* xp = static_cast<const T*>(a.x) + q.off * a.ldx + (int64_t)h * a.P + pbase;
    const T* bp = static_cast<const T*>(a.B) + q.off * a.ldb + (int64_t)grp * N;
    const T* cp = static_cast<const T*>(a.C) + q.off * a.ldc + (int64_t)grp * N;
    const T* dp = static_cast<const T*>(a.dt) + q.off * a.lddt + h;
    T* yp = static_cast<T*>(a.y) + q.off * a.ldy + (int64_t)h * a.P + pbase;
    Tile<T, PT, V> tx;
    Tile<T, NP, V> tb, tc;
    auto fetch = [&](int blk) {
        const int64_t t0 = (int64_t)blk * TB;
        const int rows = min(TB, q.len - (int)t0);
        tx.load(xp + t0 * a.ldx, a.ldx, rows, P);
        tb.load(bp + t0 * a.ldb, a.ldb, rows, N);
        tc.load(cp + t0 * a.ldc, a.ldc, rows, N);
    };
    // step sizes: wave 3 makes those of the next block from what it loaded one block before
    auto fetch_dt = [&](int blk) { return dp[min((int64_t)blk * TB + lane, (int64_t)q.len - 1) * a.lddt]; };
    T raw = (T)0.f;
    if (first < last) {
        if (wave == 3) raw = fetch_dt(first);
        fetch(first);
        if (wave == 3) {
            make_steps<false>(L.st[first & 1], a, (float)raw, first * TB + lane < q.len, A, bias, lane);
            raw = fetch_dt(first + 1);
        }
    }
    for (int blk = first; blk < last; ++blk) {
        const int64_t t0 = (int64_t)blk * TB;
        const int rows = min(TB, q.len - (int)t0);
        const Steps& st = L.st[blk & 1];
        tx.store(L.x, LX, rows, P);
        tb.store(L.b, LN, rows, N);
        tc.store(L.c, LN, rows, N);
        __syncthreads();
        if (blk + 1 < last) fetch(blk + 1);
        // M, as (C B^T)^T: lane i owns row t, four neighbouring s of it
#pragma unroll
        for (int u = 0; u < 3; ++u) {
            const int jt = tile_row(wave + 4 * u), js = tile_col(wave + 4 * u);
            if (16 * jt >= rows) continue;
            f32x4 m = {};
            if (js <= jt) {
#pragma unroll
                for (int k = 0; k < NK; ++k)
                    m = M::mma(M::row(L.b + 16 * js * LN + k * M::KS, LN, i, g), M::row(L.c + 16 * jt * LN + k * M::KS, LN, i, g), m);
                const int t = 16 * jt + i, s = 16 * js + 4 * g;
                const float ht = st.hi[t], lt = st.lo[t];
                const f32x4 hs = *reinterpret_cast<const f32x4*>(st.hi + s), ls = *reinterpret_cast<const f32x4*>(st.lo + s),
                            ds = *reinterpret_cast<const f32x4*>(st.dt + s);
#pragma unroll
                for (int r = 0; r < 4; ++r) m[r] = s + r <= t ? m[r] * (__expf((ht - hs[r]) + (lt - ls[r])) * ds[r]) : 0.f;
            }
            *reinterpret_cast<typename Four<T>::vec*>(L.m + (16 * jt + i) * LM + 16 * js + 4 * g) = four<T>(m);
        }
        if (wave == 3 && blk + 1 < last) {
            make_steps<false>(L.st[(blk + 1) & 1], a, (float)raw, t0 + TB + lane < q.len, A, bias, lane);
            raw = fetch_dt(blk + 2);
        }
        __syncthreads();
        f32x4 y[TB / 16];
#pragma unroll
        for (int jt = 0; jt < TB / 16; ++jt) {
            y[jt] = f32x4{};
            if (16 * jt >= rows) continue;
            // S is rounded once to bf16 there, like M: both only end in y
#pragma unroll
            for (int k = 0; k < NK; ++k) {
                typename M::frag sf;
                if constexpr (sizeof(T) == 4) {
                    sf = S[k];
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) sf[e] = (T)S[2 * k + (e >> 2)][e & 3];
                }
                y[jt] = M::mma(sf, M::row(L.c + 16 * jt * LN + k * M::KS, LN, i, g), y[jt]);
            }
            y[jt] *= __expf(st.hi[16 * jt + i]);
        }
#pragma unroll
        for (int k = 0; k < TB; k += M::KS) {
            if (k >= rows) continue;
            const typename M::frag xf = M::col(L.x + k * LX + p0, LX, i, g);
#pragma unroll
            for (int jt = k / 16; jt < TB / 16; ++jt)
                if (16 * jt < rows) y[jt] = M::mma(xf, M::row(L.m + 16 * jt * LM + k, LM, i, g), y[jt]);
        }
#pragma unroll
        for (int jt = 0; jt < TB / 16; ++jt) {
            const int t = 16 * jt + i, p = p0 + 4 * g;
            if (t >= rows || p >= P) continue;
            const typename Four<T>::vec xv = *reinterpret_cast<const typename Four<T>::vec*>(L.x + t * LX + p);
#pragma unroll
            for (int r = 0; r < 4; ++r) y[jt][r] = fmaf(D, (float)xv[r], y[jt][r]);
            T* out = yp + (t0 + t) * a.ldy + p;
            const typename Four<T>::vec o = four<T>(y[jt]);
            if (V > 1) {
                *reinterpret_cast<typename Four<T>::vec*>(out) = o;
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (p + r < P) out[r] = o[r];
            }
        }
        const float et = __expf(st.total);
#pragma unroll
        for (int c = 0; c < NP / 16; ++c) S[c] *= et;
        state_update<T, NP>(S, L.x, LX, L.b, LN, st.w, p0, rows, i, g);
        __syncthreads();
    }
    if (last == nb && a.hT) store_state<NP, V>(S, a.hT + state_at, N, p0, P, N, i, g);
}

template <typename T, int NP>
struct StateLds {
    T x[TB * pitch<T>(PT)], b[TB * pitch<T>(NP)];
    Steps st[2];
};

// The states alone.  Forward (blockIdx.y = 0): x, B from h0; reverse (1): dy, C from dhT, the blocks from the last to the first.
// FINAL: the segments' own sums from zero and the sum of their dt A, for ssm_join_segments.  Else: from the segment's start, the state in front of
// (reverse: the gradient of the state behind) every block to its slot, for the backward kernel.
template <typename T, int NP, int V, bool REV, bool FINAL>
__device__ __forceinline__ void states(const SsmArgs& a, StateLds<T, NP>& L) {
    constexpr int LX = pitch<T>(PT), LN = pitch<T>(NP);
    int unit, h, pbase;
    if (!work_item(a, unit, h, pbase)) return;
    const int b = unit / a.nseg, seg = unit % a.nseg, grp = h / (a.H / a.G);
    const SeqRange q = seq_range(a.seq_off, a.seq_len, b, a.rows, a.max_len);
    int nb = blocks_of(q.len), slot = 0;
    if constexpr (!FINAL) {
        slot = a.base[b];
        nb = min(nb, a.base[b + 1] - slot);
    }
    const int first = seg * a.seg_blocks, last = min(nb, first + a.seg_blocks);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i = lane & 15, g = lane >> 4, p0 = 16 * wave;
    const int P = min(a.P - pbase, PT), N = a.N;
    const int64_t seg_at = ((int64_t)unit * a.H + h) * a.P * N + (int64_t)pbase * N, state_at = ((int64_t)b * a.H + h) * a.P * N + (int64_t)pbase * N;
    float* const seg_state = REV ? a.seg_dstate : a.seg_state;
    const float* const user = REV ? a.dhT : a.h0;
    f32x4 S[NP / 16];
    load_state<NP, V>(S, FINAL ? nullptr : a.nseg > 1 ? seg_state + seg_at : user ? user + state_at : nullptr, N, p0, P, N, i, g);
    const float A = a.A[h], bias = a.dt_bias ? a.dt_bias[h] : 0.f;
    const T* xp = static_cast<const T*>(REV ? a.dy : a.x);
    const T* bp = static_cast<const T*>(REV ? a.C : a.B);
    const int64_t ldx = REV ? a.lddy : a.ldx, ldb = REV ? a.ldc : a.ldb;
    xp += q.off * ldx + (int64_t)h * a.P + pbase;
    bp += q.off * ldb + (int64_t)grp * N;
    const T* dp = static_cast<const T*>(a.dt) + q.off * a.lddt + h;
    Tile<T, PT, V> tx;
    Tile<T, NP, V> tb;
    double sum = 0.0;
    auto fetch = [&](int blk) {
        const int64_t t0 = (int64_t)blk * TB;
        const int rows = min(TB, q.len - (int)t0);
        tx.load(xp + t0 * ldx, ldx, rows, P);
        tb.load(bp + t0 * ldb, ldb, rows, N);
    };
    auto fetch_dt = [&](int blk) { return dp[max((int64_t)0, min((int64_t)blk * TB + lane, (int64_t)q.len - 1)) * a.lddt]; };
    auto block = [&](int j) { return REV ? last - 1 - j : first + j; };
    T raw = (T)0.f;
    if (first < last) {
        if (wave == 3) raw = fetch_dt(block(0));
        fetch(block(0));
        if (wave == 3) {
            make_steps<REV>(L.st[0], a, (float)raw, block(0) * TB + lane < q.len, A, bias, lane);
            raw = fetch_dt(block(1));
        }
    }
    for (int j = 0; j < last - first; ++j) {
        const int blk = block(j);
        const int rows = min(TB, q.len - blk * TB);
        const Steps& st = L.st[j & 1];
        const bool more = j + 1 < last - first;
        tx.store(L.x, LX, rows, P);
        tb.store(L.b, LN, rows, N);
        __syncthreads();
        if (more) fetch(block(j + 1));
        if constexpr (!FINAL) store_state<NP, 4>(S, (REV ? a.dS : a.S) + (((int64_t)(slot + blk) * a.H + h) * a.P + pbase) * a.NS, a.NS, p0, P, a.NS, i, g);
        const float et = __expf(st.total);
        sum += (double)st.total;
#pragma unroll
        for (int c = 0; c < NP / 16; ++c) S[c] *= et;
        state_update<T, NP>(S, L.x, LX, L.b, LN, st.w, p0, rows, i, g);
        if (wave == 3 && more) {
            make_steps<REV>(L.st[(j + 1) & 1], a, (float)raw, block(j + 1) * TB + lane < q.len, A, bias, lane);
            raw = fetch_dt(block(j + 2));
        }
        __syncthreads();
    }
    if constexpr (FINAL) {
        store_state<NP, V>(S, seg_state + seg_at, N, p0, P, N, i, g);
        if (!REV && pbase == 0 && threadIdx.x == 0) a.seg_a[(int64_t)unit * a.H + h] = (float)sum;
    } else if (REV) {
        if (first == 0 && a.dh0) store_state<NP, V>(S, a.dh0 + state_at, N, p0, P, N, i, g);
    }
}

template <typename T, int NP, int V, bool FINAL>
__global__ void __launch_bounds__(256) ssm_states_kernel(SsmArgs a) {
    __shared__ __attribute__((aligned(16))) StateLds<T, NP> L;
    if (blockIdx.y == 0) states<T, NP, V, false, FINAL>(a, L);
    else states<T, NP, V, true, FINAL>(a, L);
}

// In place: what each segment adds -> the state in front of it (blockIdx.y = 1: the gradient of the state behind it, from the last segment on).
__global__ void __launch_bounds__(256) ssm_join_kernel(SsmArgs a) {
    const int PN = a.P * a.N;
    const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, n = (int64_t)a.H * PN;
    if (e >= (int64_t)a.n_seq * n) return;
    const int b = (int)(e / n), h = (int)(e % n / PN);
    const bool rev = blockIdx.y == 1;
    const float* user = rev ? a.dhT : a.h0;
    float* buf = (rev ? a.seg_dstate : a.seg_state) + (int64_t)b * a.nseg * n + e % n;
    const float* dec = a.seg_a + (int64_t)b * a.nseg * a.H + h;
    float S = user ? user[e] : 0.f;
#pragma unroll 8
    for (int j = 0; j < a.nseg; ++j) {
        const int seg = rev ? a.nseg - 1 - j : j;
        const float add = buf[seg * n], d = dec[(int64_t)seg * a.H];
        buf[seg * n] = S;
        S = fmaf(__expf(d), S, add);
    }
}

// One row per sequence.  Sixteen lanes own a row p of the state, a workgroup sixteen rows of one sequence and head.
template <typename T, int V>
__global__ void __launch_bounds__(256) ssm_step_kernel(SsmArgs a) {
    const int ptiles = (a.P + 15) / 16;
    const int64_t blk = blockIdx.x;
    const int b = (int)(blk / ((int64_t)a.H * ptiles)), h = (int)(blk / ptiles % a.H), p = (int)(blk % ptiles) * 16 + (threadIdx.x >> 4), i = threadIdx.x & 15;
    if (p >= a.P) return;                                   // whole rows of sixteen lanes
    const int grp = h / (a.H / a.G);
    float d = (float)static_cast<const T*>(a.dt)[b * a.lddt + h] + (a.dt_bias ? a.dt_bias[h] : 0.f);
    if (a.softplus) d = softplus_f(d);
    const float x = (float)static_cast<const T*>(a.x)[b * a.ldx + (int64_t)h * a.P + p], e = __expf(d * a.A[h]), dx = d * x;
    const T* B = static_cast<const T*>(a.B) + b * a.ldb + (int64_t)grp * a.N;
    const T* C = static_cast<const T*>(a.C) + b * a.ldc + (int64_t)grp * a.N;
    const int64_t at = (((int64_t)b * a.H + h) * a.P + p) * a.N;
    float y = 0.f;
    for (int n = i * V; n < a.N; n += 16 * V) {
        float s[V], bv[V], cv[V];
        if (a.h0) load_vec<float, V>(a.h0 + at + n, s);
        load_vec<T, V>(B + n, bv);
        load_vec<T, V>(C + n, cv);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            s[k] = a.h0 ? fmaf(s[k], e, dx * bv[k]) : dx * bv[k];
            y = fmaf(s[k], cv[k], y);
        }
        store_vec<float, V>(a.hT + at + n, s);
    }
    y = sum16(y);
    if (i == 0) static_cast<T*>(a.y)[b * a.ldy + (int64_t)h * a.P + p] = (T)(y + (a.D ? a.D[h] : 0.f) * x);
}

template <typename T, int NP, int V>
int launch_fwd(const SsmArgs& a, hipStream_t s) {
    constexpr size_t bytes = sizeof(FwdLds<T, NP>);
    static_assert(bytes <= 160 * 1024, "LDS of a workgroup");
    if (bytes > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(ssm_fwd_kernel<T, NP, V>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        if (e != hipSuccess) { set_error("dc_ssm_scan_fwd: LDS", (int)e); return (int)e; }
    }
    hipLaunchKernelGGL((ssm_fwd_kernel<T, NP, V>), dim3((unsigned)work_items(a)), dim3(256), bytes, s, a);
    return launch_check("dc_ssm_scan_fwd");
}
template <typename T, int V>
int launch_fwd_n(const SsmArgs& a, hipStream_t s) {
    return a.N <= 32 ? launch_fwd<T, 32, V>(a, s) : a.N <= 64 ? launch_fwd<T, 64, V>(a, s) : launch_fwd<T, 128, V>(a, s);
}

template <typename T, int NP, int V>
int launch_states(const SsmArgs& a, bool both, bool final_only, hipStream_t s) {
    const dim3 grid((unsigned)work_items(a), both ? 2 : 1);
    if (final_only) hipLaunchKernelGGL((ssm_states_kernel<T, NP, V, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((ssm_states_kernel<T, NP, V, false>), grid, dim3(256), 0, s, a);
    return launch_check("ssm_states");
}
template <typename T, int V>
int launch_states_n(const SsmArgs& a, bool both, bool final_only, hipStream_t s) {
    return a.N <= 32 ? launch_states<T, 32, V>(a, both, final_only, s) : a.N <= 64 ? launch_states<T, 64, V>(a, both, final_only, s)
                                                                                   : launch_states<T, 128, V>(a, both, final_only, s);
}

}  // namespace

int ssm_states(const SsmArgs& a, int type, bool vec, bool both, bool final_only, hipStream_t s) {
    if (type == 0) return vec ? launch_states_n<float, 4>(a, both, final_only, s) : launch_states_n<float, 1>(a, both, final_only, s);
    return vec ? launch_states_n<bf16_t, 8>(a, both, final_only, s) : launch_states_n<bf16_t, 1>(a, both, final_only, s);
}

int ssm_join_segments(const SsmArgs& a, bool both, hipStream_t s) {
    const int64_t n = (int64_t)a.n_seq * a.H * a.P * a.N;
    hipLaunchKernelGGL(ssm_join_kernel, dim3((unsigned)((n + 255) / 256), both ? 2 : 1), dim3(256), 0, s, a);
    return launch_check("ssm_join");
}

int ssm_check(const char* what, const SsmArgs& a, int type) {
    if (type != 0 && type != 1) { set_error(what, 1101); return 1101; }
    if (a.H < 1 || a.G < 1 || a.H % a.G || a.H > 4096 || a.P < 1 || a.P > 256 || a.N < 1 || a.N > 128) { set_error(what, 1102); return 1102; }
    if (a.rows < 0 || a.n_seq < 0 || a.max_len < 0 || (int64_t)a.n_seq * a.H * ((a.P + 15) / 16) > 0x3fffffff) { set_error(what, 1103); return 1103; }
    if (!a.A || (a.rows && (!a.x || !a.dt || !a.B || !a.C))) { set_error(what, 1104); return 1104; }
    return 0;
}

// Segments: none while the sequences, heads and column tiles alone give a workgroup to every CU or the sequences are short.
void ssm_segments(SsmArgs& a, int64_t workgroups) {
    const int blocks = blocks_of(a.max_len);
    a.ptiles = (a.P + PT - 1) / PT;
    const int64_t have = (int64_t)a.n_seq * a.H * a.ptiles;
    int64_t nseg = have > 0 ? workgroups / have : 1;
    if (nseg > blocks / 2) nseg = blocks / 2;
    if (nseg < 2) nseg = 1;
    a.seg_blocks = nseg > 1 ? (int)((blocks + nseg - 1) / nseg) : (blocks > 0 ? blocks : 1);
    a.nseg = nseg > 1 ? (blocks + a.seg_blocks - 1) / a.seg_blocks : 1;
}

static bool scan_vec(const SsmArgs& a, int type) {
    const int V = type ? 8 : 4;
    const uintptr_t p = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.B) | reinterpret_cast<uintptr_t>(a.C) | reinterpret_cast<uintptr_t>(a.y) |
                        reinterpret_cast<uintptr_t>(a.h0) | reinterpret_cast<uintptr_t>(a.hT);
    return a.P % V == 0 && a.N % V == 0 && a.ldx % V == 0 && a.ldb % V == 0 && a.ldc % V == 0 && a.ldy % V == 0 && (p & 15) == 0;
}

constexpr int64_t FWD_WORKGROUPS = 1024;

int64_t ssm_scan_scratch(int n_seq, int max_len, int H, int P, int N) {
    SsmArgs a = {};
    a.n_seq = n_seq; a.max_len = max_len; a.H = H; a.P = P; a.N = N;
    ssm_segments(a, FWD_WORKGROUPS);
    return a.nseg == 1 ? 0 : (int64_t)n_seq * a.nseg * H * ((int64_t)P * N + 1) * (int64_t)sizeof(float);
}

int ssm_scan_fwd(SsmArgs a, int type, void* scratch, int64_t scratch_bytes, hipStream_t s) {
    if (int rc = ssm_check("dc_ssm_scan_fwd", a, type)) return rc;
    if (a.n_seq == 0) return 0;
    if (!a.y && a.rows) { set_error("dc_ssm_scan_fwd", 1104); return 1104; }
    ssm_segments(a, FWD_WORKGROUPS);
    if (work_items(a) > 0x7fffffff) { set_error("dc_ssm_scan_fwd", 1103); return 1103; }
    const bool vec = scan_vec(a, type);
    if (a.nseg > 1) {
        if (!scratch || scratch_bytes < ssm_scan_scratch(a.n_seq, a.max_len, a.H, a.P, a.N)) { set_error("dc_ssm_scan_fwd: scratch", 1105); return 1105; }
        a.seg_state = static_cast<float*>(scratch);
        a.seg_a = a.seg_state + (int64_t)a.n_seq * a.nseg * a.H * a.P * a.N;
        if (int rc = ssm_states(a, type, vec, false, true, s)) return rc;
        if (int rc = ssm_join_segments(a, false, s)) return rc;
    }
    if (type == 0) return vec ? launch_fwd_n<float, 4>(a, s) : launch_fwd_n<float, 1>(a, s);
    return vec ? launch_fwd_n<bf16_t, 8>(a, s) : launch_fwd_n<bf16_t, 1>(a, s);
}

int ssm_step(SsmArgs a, int type, hipStream_t s) {
    a.rows = a.n_seq;
    if (int rc = ssm_check("dc_ssm_step", a, type)) return rc;
    if (a.n_seq == 0) return 0;
    if (!a.y || !a.hT) { set_error("dc_ssm_step", 1104); return 1104; }
    const uintptr_t p = reinterpret_cast<uintptr_t>(a.h0) | reinterpret_cast<uintptr_t>(a.hT), q = reinterpret_cast<uintptr_t>(a.B) | reinterpret_cast<uintptr_t>(a.C);
    const bool vec = a.N % 4 == 0 && a.ldb % 4 == 0 && a.ldc % 4 == 0 && (p & 15) == 0 && (q & (type ? 7 : 15)) == 0;
    const dim3 grid((unsigned)((int64_t)a.n_seq * a.H * ((a.P + 15) / 16)));
    if (type == 0) {
        if (vec) hipLaunchKernelGGL((ssm_step_kernel<float, 4>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((ssm_step_kernel<float, 1>), grid, dim3(256), 0, s, a);
    } else {
        if (vec) hipLaunchKernelGGL((ssm_step_kernel<bf16_t, 4>), grid, dim3(256), 0, s, a);
        else hipLaunchKernelGGL((ssm_step_kernel<bf16_t, 1>), grid, dim3(256), 0, s, a);
    }
    return launch_check("dc_ssm_step");
}

}  // namespace dc
