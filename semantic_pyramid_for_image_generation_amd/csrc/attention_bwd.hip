// Backward of the packed attention.  With P recomputed from the forward's row statistics (see Stats):
//     dV = P^T dO,  dP = dO V^T,  dS = P o (dP - delta),  delta = rowsum(dO o O),  dQ = scale dS K,  dK = scale dS^T Q
// Two kernels without atomics, each owning what it sums, so the result does not depend on timing: one workgroup per 32 or 64
// keys walks over the queries of all heads of its group (dK, dV), one per 128 queries walks over the keys (delta, dQ; it runs
// first).  That costs seven
// products a tile pair instead of five; the two that are repeated are what the order of an atomic sum would otherwise cost.
#include "attn_tile.h"
#include "attention.h"

namespace attn {

// dK, dV of 32 SHARE keys: a lane pair is a key, its K and V fragments and both gradients stay in registers.  The steps of a
// workgroup -- tiles of 32 queries of every head of the group -- are dealt to GROUPS groups of SHARE waves, which divides the
// longest workgroup's walk.  The waves of a group hold different keys and share its tiles (Q, dO, row statistics), each of
// which is read by rows (scores, dP) and by columns (the two gradients).  At the end the groups' sums are joined in LDS.
// 16-bit types: a ring for every wave, no barrier in the loop (packed batch of 16 196 tokens, 16/4 heads of 64, causal, bf16:
// 213 to 227 us, in pairs 260: there the longest walk counts).  fp32: pairs, whose rings leave room for two waves a SIMD (16 x 1024
// tokens, 2 heads of 64: 156 to 160 us, alone 170; MFMA 75 % busy).
template <typename T, int DPAD> struct KeyTile {
    typedef Tile<T, DPAD, 32> Tl;
    static constexpr int SHARE = sizeof(T) == 4 ? 2 : 1, GROUPS = 4 / SHARE, KEYS = 32 * SHARE, STAGES = 2;
    static constexpr int BUF = 2 * Tl::BYTES + (Stats<T>::N + 1) * 256, PAD = DPAD + 4;
    static constexpr int RINGS = GROUPS * STAGES * BUF, JOIN = GROUPS * KEYS * PAD * 4, LDS = RINGS > JOIN ? RINGS : JOIN;
    static constexpr int WAVES_SIMD = DPAD <= 64 ? 2 : 1;               // by registers: heads of 128 need more than 256
};

// REST: see rest_of().
template <typename T, int DPAD, bool REST>
__global__ __launch_bounds__(256, (KeyTile<T, DPAD>::WAVES_SIMD)) WAVES_PER_SIMD((KeyTile<T, DPAD>::WAVES_SIMD)) void attention_dkdv_kernel(Params p)
{
    typedef KeyTile<T, DPAD> Kt;
    typedef Tile<T, DPAD, 32> Tl;
    typedef typename Elem<T>::Frag Frag;
    typedef float f4 __attribute__((ext_vector_type(4)));
    constexpr int KEYS = Kt::KEYS, STAGES = Kt::STAGES, SHARE = Kt::SHARE, GROUPS = Kt::GROUPS;
    extern __shared__ __attribute__((aligned(16))) char lds[];            // [group][buffer][Q tile, dO tile, delta, statistics]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    const int group = wave / SHARE, member = wave % SHARE;
    const Work w = work_of(blockIdx.x, p.heads_k, 1);
    const Where where = locate<true>(p, w.number, KEYS, lane);
    if (!where.ok) return;
    const Seq sq = where.sq;
    const int row0 = where.row, shift = sq.lk - sq.lq;                    // first key within the sequence
    const int kw0 = row0 + member * 32, ki = kw0 + (lane & 31);

    Frag kf[DPAD / 16], vf[DPAD / 16];
    load_row_frags<T, DPAD>(kf, (const T*)p.k + (int64_t)(sq.k0 + ki) * p.k_tok + (int64_t)w.kvh * p.k_head, ki < sq.lk, p.dim, lane);
    load_row_frags<T, DPAD>(vf, (const T*)p.v + (int64_t)(sq.k0 + ki) * p.v_tok + (int64_t)w.kvh * p.v_head, ki < sq.lk, p.dim, lane);
    settle(kf);
    settle(vf);
    f32x16 dk[DPAD / 32], dv[DPAD / 32];
#pragma unroll
    for (int c = 0; c < DPAD / 32; ++c) dk[c] = dv[c] = f32x16{};
    ColumnScale scale;

    // query tiles that see any of the keys; a group's steps: head g and tile t of it, counted from the
    // sequence's end
    const int first = p.causal ? max(0, row0 - shift) / 32 : 0;
    const int ntiles = row0 < sq.lk ? max(0, (sq.lq + 31) / 32 - first) : 0;
    struct Step { int g, t; };
    auto advance = [&](Step s, int by) {
        s.t += by;
        while (s.t >= ntiles) { s.t -= ntiles; ++s.g; }
        return s;
    };
    Filler<T, DPAD, 32, SHARE> fq, fo;
    fq.init(p.q_tok, p.dim, member, lane);
    fo.init((int64_t)p.heads_q * p.dim, p.dim, member, lane);
    char* ring = lds + group * STAGES * Kt::BUF;
    auto fill = [&](Step s, int b) {                  // behind the last step: zeros, so that the loop's waits stay the same
        const bool more = s.g < p.group;
        const int r = (first + ntiles - 1 - s.t) * 32, head = w.kvh * p.group + (more ? s.g : 0), left = more ? sq.lq - r : 0;
        const int64_t row = sq.q0 + r;
        char* buf = ring + b * Kt::BUF;
        fq.issue((const T*)p.q + row * p.q_tok + (int64_t)head * p.q_head, left, buf);
        fo.issue((const T*)p.go + (row * p.heads_q + head) * p.dim, left, buf + Tl::BYTES);
        // 64 floats each (by every wave of the group, the same values): those behind the tile are not used, those behind the
        // sequence become 0 (their Q and dO are zeros)
        const int64_t at = (int64_t)head * p.total_q + row;
        const int bytes = (left < 64 ? left : 64) * 4;
#pragma unroll
        for (int u = 0; u <= Stats<T>::N; ++u) {
            const float* src = (u == 0 ? p.delta : p.stats + (u - 1) * (int64_t)p.heads_q * p.total_q) + at;
            dma4(buffer_desc(src, bytes), lane * 4, buf + 2 * Tl::BYTES + u * 256);
        }
    };
    constexpr int LOADS = 2 * Filler<T, DPAD, 32, SHARE>::N + 1 + Stats<T>::N;
    const int rbase = Tl::row_base(lane), cbase = Tl::col_base(lane);
    // Steps of this group; waves that share barriers take as many rounds as the first group, on zeros at the end.  Nothing is
    // skipped inside the loop (keys behind the sequence, tiles above the diagonal): with a way around the products the compiler
    // copies the sums at every turn, 15 % of the time for heads of 128.
    const int rounds = (ntiles * p.group + GROUPS - 1 - (SHARE > 1 ? 0 : group)) / GROUPS;
    Step cur = {0, 0}, next = cur;
    if (rounds > 0) {
        next = cur = advance(cur, group);
#pragma unroll
        for (int u = 0; u < STAGES - 1; ++u) { fill(next, u); next = advance(next, GROUPS); }
    }
    int b = 0;
    for (int round = 0; round < rounds; ++round, cur = advance(cur, GROUPS), b = b + 1 == STAGES ? 0 : b + 1) {
        wait_loads<(STAGES - 2) * LOADS>();
        if constexpr (SHARE > 1) barrier();           // this round's tiles are complete, nobody reads the last round's any more
        else wait_lds();
        fill(next, b == 0 ? STAGES - 1 : b - 1);
        next = advance(next, GROUPS);
        const int qb = (first + ntiles - 1 - cur.t) * 32;
        const char *qt = ring + b * Kt::BUF, *ot = qt + Tl::BYTES;
        const float *delta = reinterpret_cast<const float*>(ot + Tl::BYTES), *ref = delta + 64, *inv = ref + 64;
        f32x16 sc = f32x16{}, dp = f32x16{};
        pipelined<Frag, DPAD / 8, BATCH<T>>([&](int i) { return Tl::row(i < DPAD / 16 ? qt : ot, rbase, 0, i % (DPAD / 16)); }, [&](int i, Frag f) {
            if (i < DPAD / 16) sc = Elem<T>::mma(f, kf[i], sc);
            else dp = Elem<T>::mma(f, vf[i - DPAD / 16], dp);
        });
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const f4 rf = *reinterpret_cast<const f4*>(ref + r * 8 + half * 4), de = *reinterpret_cast<const f4*>(delta + r * 8 + half * 4);
            f4 iv;
            if constexpr (Stats<T>::N == 2) iv = *reinterpret_cast<const f4*>(inv + r * 8 + half * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float pr = score_exp<T>(sc[r * 4 + i], p.scale_log2, rf[i]);
                if constexpr (Stats<T>::N == 2) pr *= iv[i];
                sc[r * 4 + i] = pr;
                dp[r * 4 + i] = pr * (dp[r * 4 + i] - de[i]);
            }
        }
        if (p.causal && kw0 + 31 > qb + shift) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (ki > qb + (i / 4) * 8 + half * 4 + i % 4 + shift) sc[i] = dp[i] = 0.f;
        }
        if constexpr (NARROW<T>) {
            scale.fit(dp, ki < sq.lk, [&](float x) {
#pragma unroll
                for (int c = 0; c < DPAD / 32; ++c)
#pragma unroll
                    for (int i = 0; i < 16; ++i) dk[c][i] *= x;
            });
#pragma unroll
            for (int i = 0; i < 16; ++i) dp[i] *= scale.f;
        }
        if constexpr (sizeof(T) == 4) {
            // A tile's 32 queries are summed by themselves first, see the forward (16 x 1024 tokens, 2 heads of 64: 154 -> 156 us; 8192
            // tokens, 8/1 heads of 128, causal: 8.6 -> 9.4 ms).  The empty assembly keeps the compiler from putting the additions off,
            // which takes more registers than there are.
            f32x16 part;
            pipelined<Frag, DPAD / 8, BATCH<T>>([&](int i) { return Tl::col(i / 2 % 2 ? qt : ot, cbase, i / 4, i % 2); }, [&](int i, Frag f) {
                const int k = i % 2, which = i / 2 % 2;
                f32x16& sum = which ? dk[i / 4] : dv[i / 4];
                if (k == 0) part = f32x16{};
                part = Elem<T>::mma(f, frag_of<T>(which ? dp : sc, k), part);
                if (k == 1) {
                    sum += part;
                    asm volatile("" : "+v"(sum));
                }
            });
        } else {
            Frag pf, df, pr, dr;
            pipelined<Frag, DPAD / 8, BATCH<T>>([&](int i) { return Tl::col(i % 2 ? qt : ot, cbase, i / 2 % (DPAD / 32), i / 2 / (DPAD / 32)); },
                                                [&](int i, Frag f) {
                const int c = i / 2 % (DPAD / 32), k = i / 2 / (DPAD / 32);
                if (c == 0 && i % 2 == 0) {
                    pf = frag_of<T>(sc, k);
                    df = frag_of<T>(dp, k);
                    if constexpr (REST) { pr = rest_of<T>(sc, pf, k); dr = rest_of<T>(dp, df, k); }
                }
                if (i % 2) dk[c] = Elem<T>::mma(f, df, dk[c]);
                else dv[c] = Elem<T>::mma(f, pf, dv[c]);
                if constexpr (REST) {
                    if (i % 2) dk[c] = Elem<T>::mma(f, dr, dk[c]);
                    else dv[c] = Elem<T>::mma(f, pr, dv[c]);
                }
            });
        }
    }

    // join: [group][key][dim] fp32 in LDS, dV first, then dK
    wait_loads<0>();
    float* joined = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        barrier();                                    // the rings are done with, or the sums of dV have been read
#pragma unroll
        for (int c = 0; c < DPAD / 32; ++c)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const f32x16& a = which ? dk[c] : dv[c];
                f4 v = {a[r * 4], a[r * 4 + 1], a[r * 4 + 2], a[r * 4 + 3]};
                if (NARROW<T> && which) v *= ldexpf(1.f, -P_BITS<T> - scale.bits);          // the groups' powers differ
                *reinterpret_cast<f4*>(joined + (wave * 32 + (lane & 31)) * Kt::PAD + c * 32 + r * 8 + half * 4) = v;
            }
        __syncthreads();
        const float f = which ? p.scale : ldexpf(1.f, -P_BITS<T>);
        for (int e = threadIdx.x; e < KEYS * (DPAD / 4); e += 256) {
            const int key = e / (DPAD / 4), d = e % (DPAD / 4) * 4, row = row0 + key;
            if (row >= sq.kcap || d >= p.dim) continue;
            f4 v = {0.f, 0.f, 0.f, 0.f};
            if (row < sq.lk)                          // rows of the slot behind its keys get zeros
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) v += *reinterpret_cast<const f4*>(joined + (g * KEYS + key) * Kt::PAD + d);
            store4((T*)(which ? p.dk : p.dv) + ((int64_t)(sq.k0 + row) * p.heads_k + w.kvh) * p.dim + d, v[0] * f, v[1] * f, v[2] * f, v[3] * f);
        }
    }
}

// delta and dQ (packed batch of 16 196 tokens, 16/4 heads of 64, causal, bf16: 133 to 141 us; 16 x 1024 tokens, 2 heads of 64, fp32: 123,
// MFMA 70 % busy): as the forward, with dO beside Q in registers and K read by columns, too.
template <typename T, int DPAD, bool REST>
__global__ __launch_bounds__(256, sizeof(T) * DPAD <= 256 ? 2 : 1) WAVES_PER_SIMD((sizeof(T) * DPAD <= 256 ? 2 : 1)) void attention_dq_kernel(Params p)
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

    settle(qf);
    settle(of);
    asm volatile("" ::"v"(ref), "v"(delta));
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
    ColumnScale scale;
    if (tiles) {
#pragma unroll
        for (int u = 0; u < STAGES - 1; ++u) fill(u, u);
    }
    int b = 0;
    auto turn = [&](int t) {
        wait_loads<(STAGES - 2) * 2 * Filler<T, DPAD, BN, 4>::N>();
        barrier();                                   // tile t is complete, nobody reads the buffer of tile t - 1 any more
        fill(t + STAGES - 1, b == 0 ? STAGES - 1 : b - 1);
    };
    // Tiles above the diagonal for all of this wave's queries come last and only need its part of the ring.  (A branch around
    // the products would make the compiler copy the sums at every turn.)
    const int mine = min(tiles, (max(see_wave, 0) + BN - 1) / BN);
    int t = 0;
    for (; t < mine; ++t, b = b + 1 == STAGES ? 0 : b + 1) {
        turn(t);
        const int key0 = t * BN;
        const char *kt = lds + b * 2 * Tl::BYTES, *vt = kt + Tl::BYTES;
        const bool edge = key0 + BN > see_first;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            f32x16 sc = f32x16{}, dp = f32x16{};
            pipelined<Frag, DPAD / 8, BATCH<T>>([&](int i) { return Tl::row(i % 2 ? vt : kt, rbase, n, i / 2); }, [&](int i, Frag f) {
                if (i % 2) dp = Elem<T>::mma(f, of[i / 2], dp);
                else sc = Elem<T>::mma(f, qf[i / 2], sc);
            });
#pragma unroll
            for (int i = 0; i < 16; ++i)
                dp[i] = score_exp<T>(sc[i], p.scale_log2, ref) * (dp[i] - delta);
            if (edge) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key0 + n * 32 + (i / 4) * 8 + half * 4 + i % 4 >= see) dp[i] = 0.f;
            }
            if constexpr (NARROW<T>) {
                scale.fit(dp, true, [&](float x) {
#pragma unroll
                    for (int c = 0; c < DPAD / 32; ++c)
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[c][i] *= x;
                });
#pragma unroll
                for (int i = 0; i < 16; ++i) dp[i] *= scale.f;
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
                Frag df, dr;
                pipelined<Frag, DPAD / 16, BATCH<T>>([&](int i) { return Tl::col(kt, cbase, i % (DPAD / 32), n * 2 + i / (DPAD / 32)); }, [&](int i, Frag f) {
                    const int c = i % (DPAD / 32);
                    if (c == 0) {
                        df = frag_of<T>(dp, i / (DPAD / 32));
                        if constexpr (REST) dr = rest_of<T>(dp, df, i / (DPAD / 32));
                    }
                    acc[c] = Elem<T>::mma(f, df, acc[c]);
                    if constexpr (REST) acc[c] = Elem<T>::mma(f, dr, acc[c]);
                });
            }
        }
    }
    for (; t < tiles; ++t, b = b + 1 == STAGES ? 0 : b + 1) turn(t);
    wait_loads<0>();
    if (!present) return;
    float f = p.scale;
    if (sizeof(T) == 4) f *= p.stats[(int64_t)p.heads_q * p.total_q + stat];
    if (NARROW<T>) f = ldexpf(f, -P_BITS<T> - scale.bits);
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
#define SEMPYR_BWD_KERNELS(T, D, R) \
    template __global__ void attention_dkdv_kernel<T, D, R>(Params); template __global__ void attention_dq_kernel<T, D, R>(Params);
#define SEMPYR_BWD_DIMS(T, R) SEMPYR_BWD_KERNELS(T, 32, R) SEMPYR_BWD_KERNELS(T, 64, R) SEMPYR_BWD_KERNELS(T, 128, R)
SEMPYR_BWD_DIMS(float, false)
SEMPYR_BWD_DIMS(f16, false)
SEMPYR_BWD_DIMS(f16, true)
SEMPYR_BWD_DIMS(bf16, false)
SEMPYR_BWD_DIMS(bf16, true)
#undef SEMPYR_BWD_DIMS
#undef SEMPYR_BWD_KERNELS

template <typename T, int DPAD, bool REST>
static int launch_bwd_d(const Params& p, hipStream_t st) {
    typedef KeyTile<T, DPAD> Kt;
    const int64_t bk = work_blocks(num_tiles(p.nseq, p.total_k, Kt::KEYS), p.heads_k, 1);
    const int64_t bq = work_blocks(num_tiles(p.nseq, p.total_q, BM), p.heads_k, p.group);
    if (!grid_fits(bk, 256) || !grid_fits(bq, 256)) SEMPYR_FAIL("attention_bwd: too many tiles");
    const int lds_q = stages_of<T, DPAD>() * 2 * Tile<T, DPAD, BN>::BYTES;
    if (p.total_q > 0) {
        if (int rc = allow_lds((const void*)attention_dq_kernel<T, DPAD, REST>, lds_q)) return rc;
        attention_dq_kernel<T, DPAD, REST><<<(unsigned)bq, 256, lds_q, st>>>(p);
        SEMPYR_CHECK_LAUNCH();
    }
    if (p.total_k > 0) {
        if (int rc = allow_lds((const void*)attention_dkdv_kernel<T, DPAD, REST>, Kt::LDS)) return rc;
        attention_dkdv_kernel<T, DPAD, REST><<<(unsigned)bk, 256, Kt::LDS, st>>>(p);
        SEMPYR_CHECK_LAUNCH();
    }
    return 0;
}

template <typename T, bool REST>
static int launch_bwd_t(const Params& p, hipStream_t st) {
    if (p.dim <= 32) return launch_bwd_d<T, 32, REST>(p, st);
    if (p.dim <= 64) return launch_bwd_d<T, 64, REST>(p, st);
    return launch_bwd_d<T, 128, REST>(p, st);
}

int launch_bwd(int dtype, const Params& p, hipStream_t st) {
    // Rounding P and dS to 16 bits adds as much error as the results' own rounding.  Over many keys that evens out at 1.4
    // times the latter; a few short sequences can come out worse, and there -- less than a workgroup of 32 keys a CU, waiting
    // for memory and launches anyway -- the rest is multiplied, too.
    const bool rest = (int64_t)p.total_k * p.heads_k <= 8192;
    if (dtype == SEMPYR_F32) return launch_bwd_t<float, false>(p, st);
    if (dtype == SEMPYR_F16) return rest ? launch_bwd_t<f16, true>(p, st) : launch_bwd_t<f16, false>(p, st);
    return rest ? launch_bwd_t<bf16, true>(p, st) : launch_bwd_t<bf16, false>(p, st);
}

}  // namespace attn
