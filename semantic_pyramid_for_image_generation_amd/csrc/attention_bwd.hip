// Backward of the packed attention.  With P recomputed from the forward's row statistics (see Stats):
//     dV = P^T dO,  dP = dO V^T,  dS = P o (dP - delta),  delta = rowsum(dO o O),  dQ = scale dS K,  dK = scale dS^T Q
// Two kernels without atomics, each owning what it sums, so the result does not depend on timing: one workgroup per 32 or 64
// keys walks over the queries of all heads of its group (dK, dV), one per 128 queries walks over the keys (delta, dQ; it runs
// first).  That costs seven
// products a tile pair instead of five; the two that are repeated are what the order of an atomic sum would otherwise cost.
#include "attn_tile.h"
#include "attention.h"

namespace attn {

// dK, dV of 32 KB keys.  The steps of a workgroup -- tiles of 32 queries of every head of the group -- are dealt to its four
// waves; a wave streams its tiles (Q, dO, row statistics) through an LDS ring of its own, so there is no barrier in the loop, and
// reads each by rows (scores, dP) and by columns (the two gradients).  K and V fragments and both gradients of all the keys
// stay in registers: with KB = 2 every fragment that is read from LDS feeds two products (one for each 32 keys), which halves
// the LDS traffic that would otherwise bound the loop.  At the end the waves' sums are joined in LDS in wave order.
template <typename T, int DPAD> struct KeyTile {
    typedef Tile<T, DPAD, 32> Tl;
    static constexpr int KB = sizeof(T) == 4 && DPAD <= 64 ? 2 : 1, KEYS = 32 * KB;
    static constexpr int WAVES = sizeof(T) * DPAD > 256 ? 2 : 4;        // two where four rings would not fit the LDS
    static constexpr int BUF = 2 * Tl::BYTES + (Stats<T>::N + 1) * 256, PAD = DPAD + 4;
    static constexpr int STAGES = 2, LOADS = 2 * Tl::LOADS + 1 + Stats<T>::N;
    static constexpr int RINGS = WAVES * STAGES * BUF, JOIN = WAVES * KEYS * PAD * 4, LDS = RINGS > JOIN ? RINGS : JOIN;
};

template <typename T, int DPAD>
__global__ __launch_bounds__(256, sizeof(T) * DPAD <= 128 ? 2 : 1) void attention_dkdv_kernel(Params p)
{
    typedef KeyTile<T, DPAD> Kt;
    typedef Tile<T, DPAD, 32> Tl;
    typedef typename Elem<T>::Frag Frag;
    typedef float f4 __attribute__((ext_vector_type(4)));
    constexpr int KB = Kt::KB, KEYS = Kt::KEYS, WAVES = Kt::WAVES;
    extern __shared__ __attribute__((aligned(16))) char lds[];            // [wave][2 buffers][Q tile, dO tile, delta, statistics]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Work w = work_of(blockIdx.x, p.heads_k, 1);
    const Where where = locate<true>(p, w.number, KEYS, lane);
    if (!where.ok) return;
    const Seq sq = where.sq;
    const int row0 = where.row, shift = sq.lk - sq.lq;                    // first key within the sequence

    Frag kf[KB][DPAD / 16], vf[KB][DPAD / 16];
    f32x16 dk[KB][DPAD / 32], dv[KB][DPAD / 32];
#pragma unroll
    for (int n = 0; n < KB; ++n) {
        const int ki = row0 + n * 32 + (lane & 31);
        load_row_frags<T, DPAD>(kf[n], (const T*)p.k + (int64_t)(sq.k0 + ki) * p.k_tok + (int64_t)w.kvh * p.k_head, ki < sq.lk, p.dim, lane);
        load_row_frags<T, DPAD>(vf[n], (const T*)p.v + (int64_t)(sq.k0 + ki) * p.v_tok + (int64_t)w.kvh * p.v_head, ki < sq.lk, p.dim, lane);
#pragma unroll
        for (int c = 0; c < DPAD / 32; ++c) dk[n][c] = dv[n][c] = f32x16{};
    }

    // query tiles that see any of the keys
    const int first = p.causal ? max(0, row0 - shift) / 32 : 0;
    const int ntiles = row0 < sq.lk ? max(0, (sq.lq + 31) / 32 - first) : 0;
    Filler<T, DPAD, 32, 1> fq, fo;
    fq.init(p.q_tok, p.dim, 0, lane);
    fo.init((int64_t)p.heads_q * p.dim, p.dim, 0, lane);
    char* ring = lds + wave * Kt::STAGES * Kt::BUF;
    // a wave's steps: head g of the group and tile t of it, counted from the sequence's end: workgroups of one sequence start on
    // the same tiles whatever their diagonal, and find them in L2
    struct Step { int g, t; };
    auto advance = [&](Step s) {
        s.t += WAVES;
        while (s.t >= ntiles) { s.t -= ntiles; ++s.g; }
        return s;
    };
    auto fill = [&](Step s, int b) {                  // behind the last step: zeros, so that the loop's waits stay the same
        const bool more = s.g < p.group;
        const int r = (first + ntiles - 1 - s.t) * 32, head = w.kvh * p.group + (more ? s.g : 0), left = more ? sq.lq - r : 0;
        const int64_t row = sq.q0 + r;
        char* buf = ring + b * Kt::BUF;
        fq.issue((const T*)p.q + row * p.q_tok + (int64_t)head * p.q_head, left, buf);
        fo.issue((const T*)p.go + (row * p.heads_q + head) * p.dim, left, buf + Tl::BYTES);
        // 64 floats each: statistics of rows behind the tile are fetched, too, and not used; those behind the sequence become
        // 0 (their Q and dO are zeros)
        const int64_t at = (int64_t)head * p.total_q + row;
        const int bytes = (left < 64 ? left : 64) * 4;
#pragma unroll
        for (int u = 0; u <= Stats<T>::N; ++u) {
            const float* src = (u == 0 ? p.delta : p.stats + (u - 1) * (int64_t)p.heads_q * p.total_q) + at;
            const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(src), 0, bytes, 0x00020000);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (LDS_PTR void*)(buf + 2 * Tl::BYTES + u * 256), 4, lane * 4, 0, 0, 0);
        }
    };
    const int rbase = Tl::row_base(lane), cbase = Tl::col_base(lane);
    Step cur = {0, wave - WAVES}, next = cur;
    if (ntiles > 0) {
        next = cur = advance(cur);
#pragma unroll
        for (int u = 0; u < Kt::STAGES - 1; ++u) { fill(next, u); next = advance(next); }
    }
    int b = 0;
    for (; ntiles > 0 && cur.g < p.group; cur = advance(cur), b = b + 1 == Kt::STAGES ? 0 : b + 1) {
        wait_lds();                                   // the buffer filled next was read in the step before
        fill(next, b == 0 ? Kt::STAGES - 1 : b - 1);
        next = advance(next);
        wait_loads<(Kt::STAGES - 1) * Kt::LOADS>();
        const int qb = (first + ntiles - 1 - cur.t) * 32;
        const char *qt = ring + b * Kt::BUF, *ot = qt + Tl::BYTES;
        const float *delta = reinterpret_cast<const float*>(ot + Tl::BYTES), *ref = delta + 64, *inv = ref + 64;
        f32x16 sc[KB], dp[KB];
#pragma unroll
        for (int n = 0; n < KB; ++n) sc[n] = dp[n] = f32x16{};
#pragma unroll
        for (int d = 0; d < DPAD / 16; ++d) {
            const Frag f = Tl::row(qt, rbase, 0, d);
#pragma unroll
            for (int n = 0; n < KB; ++n) sc[n] = Elem<T>::mma(f, kf[n][d], sc[n]);
        }
#pragma unroll
        for (int d = 0; d < DPAD / 16; ++d) {
            const Frag f = Tl::row(ot, rbase, 0, d);
#pragma unroll
            for (int n = 0; n < KB; ++n) dp[n] = Elem<T>::mma(f, vf[n][d], dp[n]);
        }
        const bool edge = p.causal && row0 + KEYS - 1 > qb + shift;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const f4 rf = *reinterpret_cast<const f4*>(ref + r * 8 + half * 4), de = *reinterpret_cast<const f4*>(delta + r * 8 + half * 4);
            f4 iv;
            if constexpr (Stats<T>::N == 2) iv = *reinterpret_cast<const f4*>(inv + r * 8 + half * 4);
#pragma unroll
            for (int n = 0; n < KB; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float pr = score_exp<T>(sc[n][r * 4 + i], p.scale_log2, rf[i]);
                    if constexpr (Stats<T>::N == 2) pr *= iv[i];
                    sc[n][r * 4 + i] = pr;
                    dp[n][r * 4 + i] = pr * (dp[n][r * 4 + i] - de[i]);
                }
        }
        if (edge) {
#pragma unroll
            for (int n = 0; n < KB; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (row0 + n * 32 + (lane & 31) > qb + (i / 4) * 8 + half * 4 + i % 4 + shift) sc[n][i] = dp[n][i] = 0.f;
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int c = 0; c < DPAD / 32; ++c) {
                    const Frag fo_ = Tl::col(ot, cbase, c, k), fq_ = Tl::col(qt, cbase, c, k);
#pragma unroll
                    for (int n = 0; n < KB; ++n) {
                        dv[n][c] = Elem<T>::mma(fo_, frag_of<T>(sc[n], k), dv[n][c]);
                        dk[n][c] = Elem<T>::mma(fq_, frag_of<T>(dp[n], k), dk[n][c]);
                    }
                }
        } else {
            Frag x[2][DPAD / 32];
            Tl::template cols<0>(x, ot, cbase);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int n = 0; n < KB; ++n) {
                    const Frag pf = frag_of<T>(sc[n], k);
#pragma unroll
                    for (int c = 0; c < DPAD / 32; ++c) dv[n][c] = Elem<T>::mma(x[k][c], pf, dv[n][c]);
                }
            Tl::template cols<0>(x, qt, cbase);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int n = 0; n < KB; ++n) {
                    const Frag df = frag_of<T>(dp[n], k);
#pragma unroll
                    for (int c = 0; c < DPAD / 32; ++c) dk[n][c] = Elem<T>::mma(x[k][c], df, dk[n][c]);
                }
        }
    }

    // join: [wave][key][dim] fp32 in LDS, dV first, then dK
    wait_loads<0>();
    float* joined = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        barrier();                                    // the rings are done with, or the sums of dV have been read
#pragma unroll
        for (int n = 0; n < KB; ++n)
#pragma unroll
            for (int c = 0; c < DPAD / 32; ++c)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const f32x16& a = which ? dk[n][c] : dv[n][c];
                    *reinterpret_cast<f4*>(joined + (wave * KEYS + n * 32 + (lane & 31)) * Kt::PAD + c * 32 + r * 8 + half * 4) =
                        f4{a[r * 4], a[r * 4 + 1], a[r * 4 + 2], a[r * 4 + 3]};
                }
        __syncthreads();
        const float f = which ? p.scale : 1.f;
        for (int e = threadIdx.x; e < KEYS * (DPAD / 4); e += 64 * WAVES) {
            const int key = e / (DPAD / 4), d = e % (DPAD / 4) * 4, ki = row0 + key;
            if (ki >= sq.kcap || d >= p.dim) continue;
            f4 v = {0.f, 0.f, 0.f, 0.f};
            if (ki < sq.lk)                           // rows of the slot behind its keys get zeros
#pragma unroll
                for (int u = 0; u < WAVES; ++u) v += *reinterpret_cast<const f4*>(joined + (u * KEYS + key) * Kt::PAD + d);
            store4((T*)(which ? p.dk : p.dv) + ((int64_t)(sq.k0 + ki) * p.heads_k + w.kvh) * p.dim + d, v[0] * f, v[1] * f, v[2] * f, v[3] * f);
        }
    }
}

// delta and dQ: as the forward, with dO beside Q in registers and K read by columns, too.
template <typename T, int DPAD>
__global__ __launch_bounds__(256, sizeof(T) * DPAD <= 256 ? 2 : 1) void attention_dq_kernel(Params p)
{
    typedef Tile<T, DPAD, BN> Tl;
    typedef typename Elem<T>::Frag Frag;
    constexpr int STAGES = stages_of<T, DPAD>();
    extern __shared__ __attribute__((aligned(16))) char lds[];            // [buffer][K tile, V tile]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const Work w = work_of(blockIdx.x, p.heads_k, p.group);
    const Where at = locate<false>(p, w.number, BM, lane);
    if (!at.ok) return;
    const Seq sq = at.sq;
    const int row0 = at.row;
    const int head = w.kvh * p.group + w.g, shift = sq.lk - sq.lq;
    const int qi = row0 + wave * 32 + (lane & 31);
    const bool present = qi < sq.lq;
    const int64_t orow = ((int64_t)(sq.q0 + qi) * p.heads_q + head) * p.dim;

    Frag qf[DPAD / 16], of[DPAD / 16];
    load_row_frags<T, DPAD>(qf, (const T*)p.q + (int64_t)(sq.q0 + qi) * p.q_tok + (int64_t)head * p.q_head, present, p.dim, lane);
    load_row_frags<T, DPAD>(of, (const T*)p.go + orow, present, p.dim, lane);
    const int64_t stat = (int64_t)head * p.total_q + sq.q0 + qi;
    const float ref = present ? p.stats[stat] : INFINITY;
    // delta = rowsum(dO o O), kept for the other kernel.  For 16-bit types O is taken with what its rounding left (o_low): an
    // error of delta is common to a row, dQ would carry the rounding of O (2^-9 for bf16) in full.
    float delta = 0.f;
    {
        Frag x[DPAD / 16];
        load_row_frags<T, DPAD>(x, (const T*)p.o + orow, present, p.dim, lane);
#pragma unroll
        for (int d = 0; d < DPAD / 16; ++d)
#pragma unroll
            for (int i = 0; i < 8; ++i) delta = fmaf((float)x[d][i], (float)of[d][i], delta);
        if (sizeof(T) == 2 && p.o_low) {
            load_row_frags<T, DPAD>(x, (const T*)p.o_low + orow, present, p.dim, lane);
#pragma unroll
            for (int d = 0; d < DPAD / 16; ++d)
#pragma unroll
                for (int i = 0; i < 8; ++i) delta = fmaf((float)x[d][i], (float)of[d][i], delta);
        }
        delta = half_sum(delta);
        if (present && half == 0) p.delta[stat] = delta;
    }

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
    auto fill = [&](int t, int b) {                   // behind the last tile: zeros, so that the loop's waits stay the same
        char* buf = lds + b * 2 * Tl::BYTES;
        const int left = t < tiles ? sq.lk - t * BN : 0, at = t < tiles ? t * BN : 0;
        fk.issue(kbase + (int64_t)at * p.k_tok, left, buf);
        fv.issue(vbase + (int64_t)at * p.v_tok, left, buf + Tl::BYTES);
    };
    const int rbase = Tl::row_base(lane), cbase = Tl::col_base(lane);
    f32x16 acc[DPAD / 32];
#pragma unroll
    for (int b = 0; b < DPAD / 32; ++b) acc[b] = f32x16{};
    if (tiles) {
#pragma unroll
        for (int u = 0; u < STAGES - 1; ++u) fill(u, u);
    }
    int b = 0;
    for (int t = 0; t < tiles; ++t, b = b + 1 == STAGES ? 0 : b + 1) {
        wait_loads<(STAGES - 2) * 2 * Filler<T, DPAD, BN, 4>::N>();
        barrier();                                   // tile t is complete, nobody reads the buffer of tile t - 1 any more
        fill(t + STAGES - 1, b == 0 ? STAGES - 1 : b - 1);
        const int key0 = t * BN;
        if (key0 >= see_wave) continue;
        const char *kt = lds + b * 2 * Tl::BYTES, *vt = kt + Tl::BYTES;
        const bool edge = key0 + BN > see_first;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            f32x16 sc = f32x16{}, dp = f32x16{};
#pragma unroll
            for (int d = 0; d < DPAD / 16; ++d) sc = Elem<T>::mma(Tl::row(kt, rbase, n, d), qf[d], sc);
#pragma unroll
            for (int d = 0; d < DPAD / 16; ++d) dp = Elem<T>::mma(Tl::row(vt, rbase, n, d), of[d], dp);
#pragma unroll
            for (int i = 0; i < 16; ++i)
                dp[i] = score_exp<T>(sc[i], p.scale_log2, ref) * (dp[i] - delta);
            if (edge) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key0 + n * 32 + (i / 4) * 8 + half * 4 + i % 4 >= see) dp[i] = 0.f;
            }
            if constexpr (sizeof(T) == 4) {
                // 32 keys are summed by themselves first, see the forward
#pragma unroll
                for (int c = 0; c < DPAD / 32; ++c) {
                    f32x16 part = f32x16{};
#pragma unroll
                    for (int k = 0; k < 2; ++k) part = Elem<T>::mma(Tl::col(kt, cbase, c, n * 2 + k), frag_of<T>(dp, k), part);
                    acc[c] += part;
                }
            } else {
                Frag x[2][DPAD / 32];
                n == 0 ? Tl::template cols<0>(x, kt, cbase) : Tl::template cols<2>(x, kt, cbase);
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const Frag df = frag_of<T>(dp, k);
#pragma unroll
                    for (int c = 0; c < DPAD / 32; ++c) acc[c] = Elem<T>::mma(x[k][c], df, acc[c]);
                }
            }
        }
    }
    wait_loads<0>();
    if (!present) return;
    float f = p.scale;
    if (sizeof(T) == 4) f *= p.stats[(int64_t)p.heads_q * p.total_q + stat];
    T* out = (T*)p.dq + orow;
#pragma unroll
    for (int c = 0; c < DPAD / 32; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = c * 32 + r * 8 + half * 4;
            if (d < p.dim) store4(out + d, acc[c][r * 4] * f, acc[c][r * 4 + 1] * f, acc[c][r * 4 + 2] * f, acc[c][r * 4 + 3] * f);
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
    typedef KeyTile<T, DPAD> Kt;
    const int64_t bk = work_blocks(num_tiles(p.nseq, p.total_k, Kt::KEYS), p.heads_k, 1);
    const int64_t bq = work_blocks(num_tiles(p.nseq, p.total_q, BM), p.heads_k, p.group);
    if (bk > 0x7FFFFFFF || bq > 0x7FFFFFFF) SEMPYR_FAIL("attention_bwd: too many tiles");
    const int lds_q = stages_of<T, DPAD>() * 2 * Tile<T, DPAD, BN>::BYTES;
    if (p.total_q > 0) {
        if (int rc = allow_lds((const void*)attention_dq_kernel<T, DPAD>, lds_q)) return rc;
        attention_dq_kernel<T, DPAD><<<(unsigned)bq, 256, lds_q, st>>>(p);
        SEMPYR_CHECK_LAUNCH();
    }
    if (p.total_k > 0) {
        if (int rc = allow_lds((const void*)attention_dkdv_kernel<T, DPAD>, Kt::LDS)) return rc;
        attention_dkdv_kernel<T, DPAD><<<(unsigned)bk, 64 * Kt::WAVES, Kt::LDS, st>>>(p);
        SEMPYR_CHECK_LAUNCH();
    }
    return 0;
}

template <typename T>
static int launch_bwd_t(const Params& p, hipStream_t st) {
    if (p.dim <= 32) return launch_bwd_d<T, 32>(p, st);
    if (p.dim <= 64) return launch_bwd_d<T, 64>(p, st);
    return launch_bwd_d<T, 128>(p, st);
}

int launch_bwd(int dtype, const Params& p, hipStream_t st) {
    if (dtype == SEMPYR_F32) return launch_bwd_t<float>(p, st);
    if (dtype == SEMPYR_F16) return launch_bwd_t<f16>(p, st);
    return launch_bwd_t<bf16>(p, st);
}

}  // namespace attn
