// Forward of the packed attention: O = softmax(scale Q K^T + mask) V in one pass over the keys with a running maximum and sum.
//
// A workgroup owns 128 queries of one head, a wave 32 of them (a query = a lane pair, see attn_tile.h).  Per tile of 64 keys:
//     S^T = K Q^T, P = exp2(c S - c m), l += sum P, O^T += V^T P
// with c = scale log2(e) and a reference m that follows the maximum in steps (l and O^T are rescaled when it moves).  Queries
// and the output accumulator stay in registers; K and V tiles come through a ring in LDS, the next tiles' DMA runs under the
// current tile's products.
//
// 16384 tokens, 16/2 heads of 128, causal, fp16: 1.12 to 1.19 ms, 980 to 924 TFLOP/s, 88 to 83 % of an 8192^3 library product's.  Bound
// by the matrix and the vector pipe in turn -- counters: MFMA busy in 50 % of the cycles, the vector pipe in 57 %, LDS waits 4 % of
// the waves' time, no bank conflicts -- at a clock that the load takes down to 1.8 GHz.  fp32 (16 x 1024 tokens, 2 heads of 64, 89
// to 91 us): MFMA 62 % busy, one wave a SIMD.
#include "attn_tile.h"
#include "attention.h"

namespace attn {

// waves a SIMD holds, by registers
template <typename T, int DPAD> constexpr int fwd_waves() { return sizeof(T) * DPAD <= 128 ? 3 : sizeof(T) * DPAD <= 256 ? 2 : 1; }

template <typename T, int DPAD>
__global__ __launch_bounds__(256, (fwd_waves<T, DPAD>())) WAVES_PER_SIMD((fwd_waves<T, DPAD>())) void attention_fwd_kernel(Params p)
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
    const int row0 = at.row;                                          // within the sequence
    const int head = w.kvh * p.group + w.g, shift = sq.lk - sq.lq;
    const int qi = row0 + wave * 32 + (lane & 31);
    const bool present = qi < sq.lq;

    Frag qf[DPAD / 16];
    load_row_frags<T, DPAD>(qf, (const T*)p.q + (int64_t)(sq.q0 + qi) * p.q_tok + (int64_t)head * p.q_head, present, p.dim, lane);

    settle(qf);

    // keys this lane's query sees, those the wave's first and the workgroup's last query see
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
    float m = -INFINITY, base = 0.f, l = 0.f;            // reference, see REF_SLACK; its form for the exponential; sum
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
        f32x16 sc[2] = {f32x16{}, f32x16{}};
        pipelined<Frag, DPAD / 8, BATCH<T>>([&](int i) { return Tl::row(kt, rbase, i % 2, i / 2); },
                                         [&](int i, Frag f) { sc[i % 2] = Elem<T>::mma(f, qf[i / 2], sc[i % 2]); });
        if (key0 + BN > see_first) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key0 + b * 32 + (i / 4) * 8 + half * 4 + i % 4 >= see) sc[b][i] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[b][i]);
        mx = half_max(mx);
        float factor = 1.f;
        if (__any((mx - m) * p.scale_log2 > REF_SLACK<T>)) {                // (never for NaN; a row without a key: -inf > slack)
            const float top = fmaxf(m, mx), moved = score_ref<T>(top, p.scale_log2);
            const float alpha = score_move<T>(m, top, p.scale_log2);
            m = top;
            base = moved;
            l *= alpha;
            factor = alpha;
        }
        // (multiplied always: under the branch the compiler copies the sums on the other way, 6 % of the time)
#pragma unroll
        for (int b = 0; b < DPAD / 32; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[b][i] *= factor;
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                sc[b][i] = score_exp<T>(sc[b][i], p.scale_log2, base);
                sum += sc[b][i];
            }
        l += sum;
        if constexpr (sizeof(T) == 4) {
            // a tile's products are summed by themselves first: a chain over all keys would lose bits with its length
#pragma unroll
            for (int b = 0; b < DPAD / 32; ++b) {
                f32x16 part = f32x16{};
#pragma unroll
                for (int k = 0; k < 4; ++k) part = Elem<T>::mma(Tl::col(vt, cbase, b, k), frag_of<T>(sc[k / 2], k % 2), part);
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[b][i] += part[i];
            }
        } else {
            Frag pf;
            pipelined<Frag, DPAD / 8, BATCH<T>>([&](int i) { return Tl::col(vt, cbase, i % (DPAD / 32), i / (DPAD / 32)); }, [&](int i, Frag f) {
                const int k = i / (DPAD / 32), b = i % (DPAD / 32);
                if (b == 0) pf = frag_of<T>(sc[k / 2], k % 2);
                acc[b] = Elem<T>::mma(f, pf, acc[b]);
            });
        }
    }
    for (; t < tiles; ++t, b = b + 1 == STAGES ? 0 : b + 1) turn(t);
    wait_loads<0>();
    if (p.causal && !finite_in_wave(acc, present)) {
#pragma unroll
        for (int b = 0; b < DPAD / 32; ++b) acc[b] = f32x16{};
        sum_seen<T, DPAD>(acc, qf, kbase, vbase, p, 0, min(sq.lk, max(see_wave, 0)), see, base, lane);
    }
    l = half_sum(l);                                 // each lane half has summed its own keys
    if (!present) return;
    const float inv = l == 0.f ? 0.f : 1.f / l;      // no key: zeros
    const int64_t out = ((int64_t)(sq.q0 + qi) * p.heads_q + head) * p.dim;
#pragma unroll
    for (int b = 0; b < DPAD / 32; ++b)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int d = b * 32 + r * 8 + half * 4;
            if (d < p.dim) store_out<T>(p, out + d, acc[b][r * 4] * inv, acc[b][r * 4 + 1] * inv, acc[b][r * 4 + 2] * inv, acc[b][r * 4 + 3] * inv);
        }
    if (p.stats && half == 0) Stats<T>::store(p, (int64_t)head * p.total_q + sq.q0 + qi, m, l);
}

template <typename T, int DPAD>
static int launch_fwd_d(const Params& p, hipStream_t st) {
    const int64_t blocks = work_blocks(num_tiles(p.nseq, p.total_q, BM), p.heads_k, p.group);
    if (!grid_fits(blocks, 256)) SEMPYR_FAIL("attention_fwd: too many tiles");
    const int bytes = stages_of<T, DPAD>() * 2 * Tile<T, DPAD, BN>::BYTES;
    if (int rc = allow_lds((const void*)attention_fwd_kernel<T, DPAD>, bytes)) return rc;
    attention_fwd_kernel<T, DPAD><<<(unsigned)blocks, 256, bytes, st>>>(p);
    SEMPYR_CHECK_LAUNCH();
    return 0;
}

int launch_fwd(int dtype, const Params& p, hipStream_t st) {
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        if (p.dim <= 32) return launch_fwd_d<T, 32>(p, st);
        if (p.dim <= 64) return launch_fwd_d<T, 64>(p, st);
        return launch_fwd_d<T, 128>(p, st);
    });
}

}  // namespace attn
