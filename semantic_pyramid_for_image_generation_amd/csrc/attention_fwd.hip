// Forward of the packed attention: O = softmax(scale Q K^T + mask) V in one pass over the keys with a running maximum and sum.
//
// A workgroup owns 128 queries of one head, a wave 32 of them (a query = a lane pair, see attn_tile.h).  Per tile of 64 keys:
//     S^T = K Q^T, running maximum m, P = exp2(c S - c m), l += sum P, O^T = O^T exp2(c (m_old - m)) + V^T P
// with c = scale log2(e).  Queries and the output accumulator stay in registers; K and V tiles are double-buffered in LDS, the
// next tile's DMA runs under the current tile's products.
#include "attn_tile.h"
#include "attention.h"

namespace attn {

constexpr int BM = 128, BN = 64;

template <typename T, int DPAD>
__global__ __launch_bounds__(256, 2) void attention_fwd_kernel(Params p)
{
    typedef Tile<T, DPAD, BN> Tl;
    typedef typename Elem<T>::Frag Frag;
    extern __shared__ __attribute__((aligned(16))) char lds[];            // [2 buffers][K tile, V tile]
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
    auto fill = [&](int t) {
        char* buf = lds + (t & 1) * 2 * Tl::BYTES;
        fk.issue(kbase + (int64_t)t * BN * p.k_tok, sq.lk - t * BN, buf);
        fv.issue(vbase + (int64_t)t * BN * p.v_tok, sq.lk - t * BN, buf + Tl::BYTES);
    };
    const int rbase = Tl::row_base(lane), cbase = Tl::col_base(lane);

    f32x16 acc[DPAD / 32];
#pragma unroll
    for (int b = 0; b < DPAD / 32; ++b) acc[b] = f32x16{};
    float m = -INFINITY, l = 0.f;
    if (tiles) fill(0);
    for (int t = 0; t < tiles; ++t) {
        wait_loads<0>();
        barrier();                                   // tile t is complete, nobody reads the other buffer any more
        if (t + 1 < tiles) fill(t + 1);
        const int key0 = t * BN;
        if (key0 >= see_wave) continue;              // above the diagonal for all of this wave's queries
        const char *kt = lds + (t & 1) * 2 * Tl::BYTES, *vt = kt + Tl::BYTES;
        f32x16 sc[2] = {f32x16{}, f32x16{}};
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int d = 0; d < DPAD / 16; ++d) sc[b] = Elem<T>::mma(Tl::row(kt, rbase, b, d), qf[d], sc[b]);
        if (key0 + BN > see_first) {
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (key0 + b * 32 + (i / 4) * 8 + half * 4 + i % 4 >= see) sc[b][i] = -INFINITY;
        }
        float mx = m;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[b][i]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float base = score_ref<T>(mx, p.scale_log2);                  // 0 for a row that has seen no key yet
        const float alpha = score_exp<T>(m, p.scale_log2, base);
        m = mx;
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                sc[b][i] = score_exp<T>(sc[b][i], p.scale_log2, base);
                sum += sc[b][i];
            }
        l = l * alpha + sum;
        if constexpr (sizeof(T) == 4) {
            // a tile's products are summed by themselves first: a chain over all keys would lose bits with its length
#pragma unroll
            for (int b = 0; b < DPAD / 32; ++b) {
                f32x16 part = f32x16{};
#pragma unroll
                for (int k = 0; k < 4; ++k) part = Elem<T>::mma(Tl::col(vt, cbase, b, k), frag_of<T>(sc[k / 2], k % 2), part);
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[b][i] = fmaf(acc[b][i], alpha, part[i]);
            }
        } else {
#pragma unroll
            for (int b = 0; b < DPAD / 32; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[b][i] *= alpha;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const Frag pf = frag_of<T>(sc[k / 2], k % 2);
#pragma unroll
                for (int b = 0; b < DPAD / 32; ++b) acc[b] = Elem<T>::mma(Tl::col(vt, cbase, b, k), pf, acc[b]);
            }
        }
    }
    l += __shfl_xor(l, 32, 64);                      // each lane half has summed its own keys
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
    if (blocks > 0x7FFFFFFF) SEMPYR_FAIL("attention_fwd: too many tiles");
    const int bytes = 4 * Tile<T, DPAD, BN>::BYTES;
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
