// Backward of the packed attention.  With P = exp2(c S - lse) recomputed from the forward's row statistics:
//     dV = P^T dO,  dP = dO V^T,  dS = P o (dP - delta),  delta = rowsum(dO o O),  dQ = scale dS K,  dK = scale dS^T Q
// Two kernels without atomics, each owning what it sums, so the result does not depend on timing: one workgroup per 128 keys
// walks over the queries of all heads of its group (dK, dV), one per 128 queries walks over the keys (dQ).  That costs seven
// products a tile pair instead of five; the two that are repeated are what the order of an atomic sum would otherwise cost.
#include "attn_tile.h"
#include "attention.h"

namespace attn {

constexpr int BM = 128, BN = 64;

// delta[head][row] = sum over d of go * o, 16 lanes a row
template <typename T>
__global__ __launch_bounds__(256) void attention_delta_kernel(const T* __restrict__ go, const T* __restrict__ o, float* __restrict__ delta,
                                                              int64_t rows, int total_q, int heads, int dim)
{
    constexpr int N = Vec16<T>::N;
    const int64_t row = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    if (row >= rows) return;
    float sum = 0.f;
    for (int d = (threadIdx.x % 16) * N; d < dim; d += 16 * N) {
        float a[N], b[N];
        load_floats<T, N>(go + row * dim + d, a);
        load_floats<T, N>(o + row * dim + d, b);
#pragma unroll
        for (int i = 0; i < N; ++i) sum = fmaf(a[i], b[i], sum);
    }
#pragma unroll
    for (int s = 8; s > 0; s >>= 1) sum += __shfl_xor(sum, s, 64);
    if (threadIdx.x % 16 == 0) delta[(row % heads) * total_q + row / heads] = sum;
}

// dK, dV: a lane pair is a key, its K and V fragments and both gradients stay in registers; tiles of 64 queries (Q, dO, lse,
// delta) go through LDS, each read by rows (scores, dP) and by columns (the two gradients).
template <typename T, int DPAD>
__global__ __launch_bounds__(256, sizeof(T) == 2 && DPAD < 128 ? 2 : 1) void attention_dkdv_kernel(Params p)
{
    typedef Tile<T, DPAD, BN> Tl;
    typedef typename Elem<T>::Frag Frag;
    typedef float f4 __attribute__((ext_vector_type(4)));
    constexpr int STATS = 2 * BN * 4, BUF = 2 * Tl::BYTES + STATS;
    extern __shared__ __attribute__((aligned(16))) char lds[];            // [2 buffers][Q tile, dO tile, lse, delta]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int slots = num_slots(p.nseq, p.total_k, BM);
    const Work w = work_of(blockIdx.x, slots, p.heads_k, 1);
    if (w.slot < 0) return;
    const int s = __builtin_amdgcn_readfirstlane(find_seq(p.cu_k, p.nseq, p.total_k, w.slot, BM, lane));
    const Seq sq = seq_of(p, s);
    const int row0 = (w.slot - (sq.k0 / BM + s)) * BM;                    // first key within the sequence
    if (row0 >= sq.kcap) return;
    const int kw0 = row0 + wave * 32, ki = kw0 + (lane & 31), shift = sq.lk - sq.lq;

    Frag kf[DPAD / 16], vf[DPAD / 16];
    load_row_frags<T, DPAD>(kf, (const T*)p.k + (int64_t)(sq.k0 + ki) * p.k_tok + (int64_t)w.kvh * p.k_head, ki < sq.lk, p.dim, lane);
    load_row_frags<T, DPAD>(vf, (const T*)p.v + (int64_t)(sq.k0 + ki) * p.v_tok + (int64_t)w.kvh * p.v_head, ki < sq.lk, p.dim, lane);

    // query tiles that see any of the workgroup's keys
    const int first = p.causal ? max(0, row0 - shift) / BN : 0;
    const int ntiles = row0 < sq.lk ? max(0, (sq.lq + BN - 1) / BN - first) : 0, steps = ntiles * p.group;

    Filler<T, DPAD, BN, 4> fq, fo;
    fq.init(p.q_tok, p.dim, wave, lane);
    fo.init((int64_t)p.heads_q * p.dim, p.dim, wave, lane);
    auto fill = [&](int it) {
        const int head = w.kvh * p.group + it / ntiles, r = (first + it % ntiles) * BN, left = sq.lq - r;
        const int64_t row = sq.q0 + r;
        char* buf = lds + (it & 1) * BUF;
        fq.issue((const T*)p.q + row * p.q_tok + (int64_t)head * p.q_head, left, buf);
        fo.issue((const T*)p.go + (row * p.heads_q + head) * p.dim, left, buf + Tl::BYTES);
        if (wave < 2) {
            const float* src = (wave ? p.delta : p.lse) + (int64_t)head * p.total_q + row;
            const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(src), 0, (left < BN ? left : BN) * 4, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (LDS_PTR void*)(buf + 2 * Tl::BYTES + wave * BN * 4), 4, lane * 4, 0, 0, 0);
        }
    };
    const int rbase = Tl::row_base(lane), cbase = Tl::col_base(lane);
    f32x16 dk[DPAD / 32], dv[DPAD / 32];
#pragma unroll
    for (int b = 0; b < DPAD / 32; ++b) dk[b] = dv[b] = f32x16{};
    if (steps) fill(0);
    for (int it = 0; it < steps; ++it) {
        wait_loads<0>();
        barrier();
        if (it + 1 < steps) fill(it + 1);
        const int q0 = (first + it % ntiles) * BN;
        const char *qt = lds + (it & 1) * BUF, *ot = qt + Tl::BYTES;
        const float *lse = reinterpret_cast<const float*>(ot + Tl::BYTES), *delta = lse + BN;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const int qb = q0 + b * 32;
            if (kw0 >= sq.lk || (p.causal && kw0 > qb + 31 + shift)) continue;       // nothing to see for this wave
            f32x16 sc = f32x16{}, dp = f32x16{};
#pragma unroll
            for (int d = 0; d < DPAD / 16; ++d) sc = Elem<T>::mma(Tl::row(qt, rbase, b, d), kf[d], sc);
#pragma unroll
            for (int d = 0; d < DPAD / 16; ++d) dp = Elem<T>::mma(Tl::row(ot, rbase, b, d), vf[d], dp);
            const bool edge = p.causal && kw0 + 31 > qb + shift;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f4 ls = *reinterpret_cast<const f4*>(lse + b * 32 + r * 8 + half * 4);
                const f4 de = *reinterpret_cast<const f4*>(delta + b * 32 + r * 8 + half * 4);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float pr = __builtin_amdgcn_exp2f(fmaf(sc[r * 4 + i], p.scale_log2, -ls[i]));
                    const float ds = pr * (dp[r * 4 + i] - de[i]);
                    const bool hidden = edge && ki > qb + r * 8 + half * 4 + i + shift;
                    sc[r * 4 + i] = hidden ? 0.f : pr;
                    dp[r * 4 + i] = hidden ? 0.f : ds;
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const Frag pf = frag_of<T>(sc, k), df = frag_of<T>(dp, k);
#pragma unroll
                for (int c = 0; c < DPAD / 32; ++c) {
                    dv[c] = Elem<T>::mma(Tl::col(ot, cbase, c, b * 2 + k), pf, dv[c]);
                    dk[c] = Elem<T>::mma(Tl::col(qt, cbase, c, b * 2 + k), df, dk[c]);
                }
            }
        }
    }
    if (ki >= sq.kcap) return;
    const bool live = ki < sq.lk;                     // rows of the slot behind its keys get zeros
    const int64_t at = ((int64_t)(sq.k0 + ki) * p.heads_k + w.kvh) * p.dim;
#pragma unroll
    for (int c = 0; c < DPAD / 32; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = c * 32 + r * 8 + half * 4;
            if (d >= p.dim) continue;
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { a[i] = live ? dk[c][r * 4 + i] * p.scale : 0.f; b[i] = live ? dv[c][r * 4 + i] : 0.f; }
            store4((T*)p.dk + at + d, a[0], a[1], a[2], a[3]);
            store4((T*)p.dv + at + d, b[0], b[1], b[2], b[3]);
        }
}

// dQ: as the forward, with dO beside Q in registers and K read by columns, too
template <typename T, int DPAD>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void attention_dq_kernel(Params p)
{
    typedef Tile<T, DPAD, BN> Tl;
    typedef typename Elem<T>::Frag Frag;
    extern __shared__ __attribute__((aligned(16))) char lds[];            // [2 buffers][K tile, V tile]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int slots = num_slots(p.nseq, p.total_q, BM);
    const Work w = work_of(blockIdx.x, slots, p.heads_k, p.group);
    if (w.slot < 0) return;
    const int s = __builtin_amdgcn_readfirstlane(find_seq(p.cu_q, p.nseq, p.total_q, w.slot, BM, lane));
    const Seq sq = seq_of(p, s);
    const int row0 = (w.slot - (sq.q0 / BM + s)) * BM;
    if (row0 >= sq.lq) return;
    const int head = w.kvh * p.group + w.g, shift = sq.lk - sq.lq;
    const int qi = row0 + wave * 32 + (lane & 31);
    const bool present = qi < sq.lq;
    const int64_t orow = ((int64_t)(sq.q0 + qi) * p.heads_q + head) * p.dim;

    Frag qf[DPAD / 16], of[DPAD / 16];
    load_row_frags<T, DPAD>(qf, (const T*)p.q + (int64_t)(sq.q0 + qi) * p.q_tok + (int64_t)head * p.q_head, present, p.dim, lane);
    load_row_frags<T, DPAD>(of, (const T*)p.go + orow, present, p.dim, lane);
    const float lse = present ? p.lse[(int64_t)head * p.total_q + sq.q0 + qi] : INFINITY;
    const float delta = present ? p.delta[(int64_t)head * p.total_q + sq.q0 + qi] : 0.f;

    const int see = p.causal ? min(sq.lk, qi + 1 + shift) : sq.lk;
    const int see_first = p.causal ? min(sq.lk, row0 + wave * 32 + 1 + shift) : sq.lk;
    const int see_wave = p.causal ? min(sq.lk, row0 + wave * 32 + 32 + shift) : sq.lk;
    const int see_block = p.causal ? min(sq.lk, min(row0 + BM, sq.lq) + shift) : sq.lk;
    const int tiles = see_block > 0 ? (see_block + BN - 1) / BN : 0;

    Filler<T, DPAD, BN, 4> fk, fv;
    fk.init(p.k_tok, p.dim, wave, lane);
    fv.init(p.v_tok, p.dim, wave, lane);
    const T* kbase = (const T*)p.k + (int64_t)sq.k0 * p.k_tok + (int64_t)w.kvh * p.k_head;
    const T* vbase = (const T*)p.v + (int64_t)sq.k0 * p.v_tok + (int64_t)w.kvh * p.v_head;
    auto fill = [&](int t) {
        char* buf = lds + (t & 1) * 2 * Tl::BYTES;
        fk.issue(kbase + (int64_t)t * BN * p.k_tok, sq.lk - t * BN, buf);
        fv.issue(vbase + (int64_t)t * BN * p.v_tok, sq.lk - t * BN, buf + Tl::BYTES);
    };
    const int rbase = Tl::row_base(lane), cbase = Tl::col_base(lane);
    f32x16 acc[DPAD / 32];
#pragma unroll
    for (int b = 0; b < DPAD / 32; ++b) acc[b] = f32x16{};
    if (tiles) fill(0);
    for (int t = 0; t < tiles; ++t) {
        wait_loads<0>();
        barrier();
        if (t + 1 < tiles) fill(t + 1);
        const int key0 = t * BN;
        if (key0 >= see_wave) continue;
        const char *kt = lds + (t & 1) * 2 * Tl::BYTES, *vt = kt + Tl::BYTES;
        const bool edge = key0 + BN > see_first;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            f32x16 sc = f32x16{}, dp = f32x16{};
#pragma unroll
            for (int d = 0; d < DPAD / 16; ++d) sc = Elem<T>::mma(Tl::row(kt, rbase, b, d), qf[d], sc);
#pragma unroll
            for (int d = 0; d < DPAD / 16; ++d) dp = Elem<T>::mma(Tl::row(vt, rbase, b, d), of[d], dp);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float pr = __builtin_amdgcn_exp2f(fmaf(sc[i], p.scale_log2, -lse));
                const float ds = pr * (dp[i] - delta);
                dp[i] = edge && key0 + b * 32 + (i / 4) * 8 + half * 4 + i % 4 >= see ? 0.f : ds;
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const Frag df = frag_of<T>(dp, k);
#pragma unroll
                for (int c = 0; c < DPAD / 32; ++c) acc[c] = Elem<T>::mma(Tl::col(kt, cbase, c, b * 2 + k), df, acc[c]);
            }
        }
    }
    if (!present) return;
    T* out = (T*)p.dq + orow;
#pragma unroll
    for (int c = 0; c < DPAD / 32; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = c * 32 + r * 8 + half * 4;
            if (d < p.dim) store4(out + d, acc[c][r * 4] * p.scale, acc[c][r * 4 + 1] * p.scale, acc[c][r * 4 + 2] * p.scale, acc[c][r * 4 + 3] * p.scale);
        }
}

// Instantiated by name: this compiler's host pass leaves the stubs of the implicit instantiations out.
#define SEMPYR_BWD_KERNELS(T, D) template __global__ void attention_dkdv_kernel<T, D>(Params); template __global__ void attention_dq_kernel<T, D>(Params);
SEMPYR_BWD_KERNELS(float, 32) SEMPYR_BWD_KERNELS(float, 64) SEMPYR_BWD_KERNELS(float, 128)
SEMPYR_BWD_KERNELS(f16, 32) SEMPYR_BWD_KERNELS(f16, 64) SEMPYR_BWD_KERNELS(f16, 128)
SEMPYR_BWD_KERNELS(bf16, 32) SEMPYR_BWD_KERNELS(bf16, 64) SEMPYR_BWD_KERNELS(bf16, 128)
#undef SEMPYR_BWD_KERNELS

template <typename T, int DPAD>
static int launch_bwd_d(const Params& p, hipStream_t st) {
    const int64_t bk = work_blocks(num_slots(p.nseq, p.total_k, BM), p.heads_k, 1);
    const int64_t bq = work_blocks(num_slots(p.nseq, p.total_q, BM), p.heads_k, p.group);
    if (bk > 0x7FFFFFFF || bq > 0x7FFFFFFF) SEMPYR_FAIL("attention_bwd: too many tiles");
    const int tile = Tile<T, DPAD, BN>::BYTES, lds_kv = 4 * tile + 4 * BN * 4, lds_q = 4 * tile;
    if (p.total_k > 0) {
        if (int rc = allow_lds((const void*)attention_dkdv_kernel<T, DPAD>, lds_kv)) return rc;
        attention_dkdv_kernel<T, DPAD><<<(unsigned)bk, 256, lds_kv, st>>>(p);
        SEMPYR_CHECK_LAUNCH();
    }
    if (p.total_q > 0) {
        if (int rc = allow_lds((const void*)attention_dq_kernel<T, DPAD>, lds_q)) return rc;
        attention_dq_kernel<T, DPAD><<<(unsigned)bq, 256, lds_q, st>>>(p);
        SEMPYR_CHECK_LAUNCH();
    }
    return 0;
}

template <typename T>
static int launch_bwd_t(const Params& p, float* delta, hipStream_t st) {
    const int64_t rows = (int64_t)p.total_q * p.heads_q;
    if (rows > 0) {
        if (rows > 0x7FFFFFFFll * 16) SEMPYR_FAIL("attention_bwd: too many rows");
        attention_delta_kernel<T><<<(unsigned)((rows + 15) / 16), 256, 0, st>>>((const T*)p.go, (const T*)p.o, delta, rows, p.total_q, p.heads_q, p.dim);
        SEMPYR_CHECK_LAUNCH();
    }
    if (p.dim <= 32) return launch_bwd_d<T, 32>(p, st);
    if (p.dim <= 64) return launch_bwd_d<T, 64>(p, st);
    return launch_bwd_d<T, 128>(p, st);
}

int launch_bwd(int dtype, const Params& p, float* delta, hipStream_t st) {
    if (dtype == SEMPYR_F32) return launch_bwd_t<float>(p, delta, st);
    if (dtype == SEMPYR_F16) return launch_bwd_t<f16>(p, delta, st);
    return launch_bwd_t<bf16>(p, delta, st);
}

}  // namespace attn
