// Forward of the packed attention where there are few rows: single new tokens against long caches, small maps.
//
// The queries of a group's heads are packed into the 32 columns of a tile (row r = query r / heads, head r % heads), so K and V
// are read once for the whole group, and the keys are split twice: over `splits` workgroups and, tile by tile of 32, over the
// waves of a workgroup.  A wave streams its tiles through an LDS ring of its own (no barrier in the loop, one tile in flight
// while one is used) and keeps a running maximum and sum; the waves' results are joined in LDS, those of the workgroups by a
// second kernel from fp32 partial sums.  Bound by reading K and V; the matrix pipe has most of its columns idle for a single
// token and time to spare: it also takes what rounding the probabilities to 16 bits leaves (no difference in time).
#include "attn_tile.h"
#include "attention.h"

namespace attn {

constexpr int BK = 32;

// Two waves a workgroup: 64 KiB of rings for 16-bit heads of 128, so a second workgroup's start and end (search, first tiles,
// join) overlap this one's stream.  Eight requests' tokens against up to 32768 keys, 32/8 heads of 128, bf16 (549 MB): 2 waves
// and 1024 workgroups 120 us (4.6 TB/s), 4 and 512 119, 2 and 2048 127, 4 and 2048 175.
template <typename T, int DPAD> struct Split {
    typedef Tile<T, DPAD, BK> Tl;
    static constexpr int WAVES = 2;
    static constexpr int RING = 4 * Tl::BYTES, PAD = DPAD + 4;       // ring: two buffers of a K and a V tile
    static constexpr int STATS = WAVES * 32 * 2 * 4, LDS = WAVES * RING + STATS;
    static_assert(WAVES * 32 * PAD * 4 <= WAVES * RING, "the joined results reuse the rings");
};

template <typename T, int DPAD>
__global__ __launch_bounds__(128, 1) void attention_split_kernel(Params p, SplitPlan plan, float* __restrict__ part_o,
                                                                  float* __restrict__ part_ml)
{
    typedef Split<T, DPAD> Sp;
    typedef Tile<T, DPAD, BK> Tl;
    typedef typename Elem<T>::Frag Frag;
    typedef float f4 __attribute__((ext_vector_type(4)));
    constexpr int WAVES = Sp::WAVES, THREADS = 64 * WAVES;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
    int idx = blockIdx.x;
    const int chunk = idx % plan.head_chunks; idx /= plan.head_chunks;
    const int kvh = idx % p.heads_k; idx /= p.heads_k;
    const int split = idx % plan.splits, number = idx / plan.splits;
    const int QT = plan.queries;                     // queries of a tile
    const Where at = locate<false>(p, number, QT, lane);
    if (!at.ok) return;
    const Seq sq = at.sq;
    const int row0 = at.row;
    const int shift = sq.lk - sq.lq, col = lane & 31;
    // column -> query and head
    auto query_of = [&](int c) { return row0 + c / plan.heads; };
    auto head_of = [&](int c) { return chunk * plan.heads + c % plan.heads; };
    auto present_of = [&](int c) { return c < QT * plan.heads && query_of(c) < sq.lq && head_of(c) < p.group; };
    const int qi = query_of(col);
    const bool present = present_of(col);

    Frag qf[DPAD / 16];
    load_row_frags<T, DPAD>(qf, (const T*)p.q + (int64_t)(sq.q0 + qi) * p.q_tok + (int64_t)(kvh * p.group + head_of(col)) * p.q_head,
                            present, p.dim, lane);

    settle(qf);

    const int last = min(row0 + QT, sq.lq);          // queries of the tile end here
    const int see = p.causal ? min(sq.lk, qi + 1 + shift) : sq.lk;
    const int see_first = p.causal ? min(sq.lk, row0 + 1 + shift) : sq.lk;
    const int see_block = p.causal ? min(sq.lk, last + shift) : sq.lk;
    const int tiles = see_block > 0 ? (see_block + BK - 1) / BK : 0;
    const int per = (tiles + plan.splits - 1) / plan.splits;
    const int t0 = split * per + wave, t1 = min(tiles, (split + 1) * per);

    Filler<T, DPAD, BK, 1> fk, fv;
    fk.init(p.k_tok, p.dim, 0, lane);
    fv.init(p.v_tok, p.dim, 0, lane);
    const T* kbase = (const T*)p.k + (int64_t)sq.k0 * p.k_tok + (int64_t)kvh * p.k_head;
    const T* vbase = (const T*)p.v + (int64_t)sq.k0 * p.v_tok + (int64_t)kvh * p.v_head;
    char* ring = lds + wave * Sp::RING;
    auto fill = [&](int t, int b) {
        char* buf = ring + b * 2 * Tl::BYTES;
        fk.issue(kbase + (int64_t)t * BK * p.k_tok, sq.lk - t * BK, buf);
        fv.issue(vbase + (int64_t)t * BK * p.v_tok, sq.lk - t * BK, buf + Tl::BYTES);
    };
    const int rbase = Tl::row_base(lane), cbase = Tl::col_base(lane);
    f32x16 acc[DPAD / 32];
#pragma unroll
    for (int b = 0; b < DPAD / 32; ++b) acc[b] = f32x16{};
    float m = -INFINITY, base = 0.f, l = 0.f;
    if (t0 < t1) fill(t0, 0);
    int b = 0;
    for (int t = t0; t < t1; t += WAVES, b ^= 1) {
        if (t + WAVES < t1) {
            wait_lds();                              // nothing still reads the buffer that is filled now
            fill(t + WAVES, b ^ 1);
            wait_loads<2 * Tl::LOADS>();             // this tile is complete, the next one is in flight
        } else {
            wait_loads<0>();
        }
        const char *kt = ring + b * 2 * Tl::BYTES, *vt = kt + Tl::BYTES;
        f32x16 sc = f32x16{};
#pragma unroll
        for (int d = 0; d < DPAD / 16; ++d) sc = Elem<T>::mma(Tl::row(kt, rbase, 0, d), qf[d], sc);
        const int key0 = t * BK;
        if (key0 + BK > see_first) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (key0 + (i / 4) * 8 + half * 4 + i % 4 >= see) sc[i] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[i]);
        mx = half_max(mx);
        if (__any((mx - m) * p.scale_log2 > REF_SLACK<T>)) {
            const float top = fmaxf(m, mx), moved = score_ref<T>(top, p.scale_log2);
            const float alpha = score_move<T>(m, top, p.scale_log2);
            m = top;
            base = moved;
            l *= alpha;
#pragma unroll
            for (int c = 0; c < DPAD / 32; ++c)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[c][i] *= alpha;
        }
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            sc[i] = score_exp<T>(sc[i], p.scale_log2, base);
            sum += sc[i];
        }
        l += sum;
        if constexpr (sizeof(T) == 4) {
            // a tile's products are summed by themselves first, see attention_fwd.hip
#pragma unroll
            for (int c = 0; c < DPAD / 32; ++c) {
                f32x16 part = f32x16{};
#pragma unroll
                for (int k = 0; k < 2; ++k) part = Elem<T>::mma(Tl::col(vt, cbase, c, k), frag_of<T>(sc, k), part);
                acc[c] += part;
            }
        } else {
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const Frag pf = frag_of<T>(sc, k), pr = rest_of<T>(sc, pf, k);
#pragma unroll
                for (int c = 0; c < DPAD / 32; ++c) {
                    const Frag f = Tl::col(vt, cbase, c, k);
                    acc[c] = Elem<T>::mma(f, pf, acc[c]);
                    acc[c] = Elem<T>::mma(f, pr, acc[c]);
                }
            }
        }
    }
    if (p.causal && !finite_in_wave(acc, present)) {
#pragma unroll
        for (int c = 0; c < DPAD / 32; ++c) acc[c] = f32x16{};
        for (int t = t0; t < t1; t += WAVES) sum_seen<T, DPAD>(acc, qf, kbase, vbase, p, t * BK, min(sq.lk, (t + 1) * BK), see, base, lane);
    }
    l = half_sum(l);

    // join the waves: [wave][column][dim] in LDS, every thread then owns four elements of a column
    wait_lds();
    barrier();
    float* joined = reinterpret_cast<float*>(lds);
    float* stats = reinterpret_cast<float*>(lds + WAVES * Sp::RING);      // [wave][column]{m, l}
#pragma unroll
    for (int c = 0; c < DPAD / 32; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            *reinterpret_cast<f4*>(joined + (wave * 32 + col) * Sp::PAD + c * 32 + r * 8 + half * 4) =
                f4{acc[c][r * 4], acc[c][r * 4 + 1], acc[c][r * 4 + 2], acc[c][r * 4 + 3]};
    if (half == 0) {
        stats[(wave * 32 + col) * 2] = m;
        stats[(wave * 32 + col) * 2 + 1] = l;
    }
    __syncthreads();
    constexpr int PER_COL = THREADS / 32;            // threads of a column
    const int c = threadIdx.x / PER_COL;
    if (!present_of(c)) return;
    float top = -INFINITY, f[WAVES], total = 0.f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, stats[(w * 32 + c) * 2]);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const float mw = stats[(w * 32 + c) * 2];
        f[w] = score_move<T>(mw, top, p.scale_log2);
        total += f[w] * stats[(w * 32 + c) * 2 + 1];
    }
    const int head = kvh * p.group + head_of(c);
    const int64_t token = sq.q0 + query_of(c), row = token * p.heads_q + head, rows = (int64_t)p.total_q * p.heads_q;
    const bool whole = plan.splits == 1;
    const float inv = !whole ? 1.f : total == 0.f ? 0.f : 1.f / total;
    for (int d = (threadIdx.x % PER_COL) * 4; d < p.dim; d += PER_COL * 4) {
        f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < WAVES; ++w) v += f[w] * *reinterpret_cast<const f4*>(joined + (w * 32 + c) * Sp::PAD + d);
        v *= inv;
        if (whole) store_out<T>(p, row * p.dim + d, v[0], v[1], v[2], v[3]);
        else if (total != 0.f) *reinterpret_cast<f4*>(part_o + (split * rows + row) * p.dim + d) = v;
    }
    if (threadIdx.x % PER_COL == 0) {
        if (!whole) {
            part_ml[(split * rows + row) * 2] = top;
            part_ml[(split * rows + row) * 2 + 1] = total;
        } else if (p.stats) {
            Stats<T>::store(p, (int64_t)head * p.total_q + token, top, total);
        }
    }
}

// Joins the partial results of `splits` workgroups: a workgroup a row, 32 lanes hold the row's elements, the eight groups of 32
// lanes take every eighth split (the loads of a thread are independent), a sum over the groups in order ends it.
template <typename T>
__global__ __launch_bounds__(256) void attention_join_kernel(Params p, int splits, const float* __restrict__ part_o,
                                                             const float* __restrict__ part_ml)
{
    typedef float f4 __attribute__((ext_vector_type(4)));
    typedef float f2 __attribute__((ext_vector_type(2)));
    __shared__ f4 sums[8][32];
    __shared__ float totals[8];
    const int64_t rows = (int64_t)p.total_q * p.heads_q, row = blockIdx.x;
    const int lane = threadIdx.x % 32, group = threadIdx.x / 32, d = lane * 4;
    const f2* ml = reinterpret_cast<const f2*>(part_ml);
    float top = -INFINITY;
    for (int s = lane; s < splits; s += 32) top = fmaxf(top, ml[s * rows + row][0]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    float total = 0.f;
    f4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = group; s < splits; s += 8) {
        const f2 x = ml[s * rows + row];
        if (x[1] == 0.f) continue;                   // no key in this split; its partial sums were not written
        const float f = score_move<T>(x[0], top, p.scale_log2);
        total += f * x[1];
        if (d < p.dim) v += f * *reinterpret_cast<const f4*>(part_o + (s * rows + row) * p.dim + d);
    }
    sums[group][lane] = v;
    if (lane == 0) totals[group] = total;
    __syncthreads();
    if (group) return;
#pragma unroll
    for (int g = 1; g < 8; ++g) { v += sums[g][lane]; total += totals[g]; }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    if (d < p.dim) store_out<T>(p, row * p.dim + d, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    if (p.stats && lane == 0) Stats<T>::store(p, (row % p.heads_q) * p.total_q + row / p.heads_q, top, total);
}

// A tile of the one-pass kernel holds 128 queries of one head; where those tiles cannot occupy the 256 CUs, the rows are
// packed and the keys split instead.
SplitPlan plan_split(const Params& p) {
    SplitPlan s = {};
    const int64_t tiles = ((int64_t)p.total_q / 128 + p.nseq) * p.heads_q;
    s.head_chunks = (p.group + 31) / 32;
    s.heads = (p.group + s.head_chunks - 1) / s.head_chunks;
    s.queries = 32 / s.heads;
    const bool few_queries = (int64_t)p.total_q <= (int64_t)s.queries * p.nseq;        // a tile a sequence holds them on average
    if (p.total_q == 0 || (tiles > 256 && !few_queries)) return s;
    const int64_t packed = ((int64_t)(p.total_q + s.queries - 1) / s.queries + (p.nseq > 1 ? p.nseq : 0) / 2) * p.heads_k * s.head_chunks;
    const int64_t keys = p.nseq > 0 ? p.total_k / p.nseq : 0, most = (keys + 2 * BK - 1) / (2 * BK);      // a tile a wave
    int64_t n = (1024 + packed - 1) / packed;
    n = n < most ? n : most;
    s.splits = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
    return s;
}

template <typename T, int DPAD>
static int launch_split_d(const Params& p, const SplitPlan& plan, float* ws, hipStream_t st) {
    typedef Split<T, DPAD> Sp;
    const int64_t rows = (int64_t)p.total_q * p.heads_q;
    const int64_t blocks = (int64_t)num_tiles(p.nseq, p.total_q, plan.queries) * plan.splits * p.heads_k * plan.head_chunks;
    if (!grid_fits(blocks, 64 * Sp::WAVES) || (plan.splits > 1 && !grid_fits(rows, 256))) SEMPYR_FAIL("attention_fwd: too many tiles");
    float* ml = ws ? ws + plan.splits * rows * p.dim : nullptr;
    if (int rc = allow_lds((const void*)attention_split_kernel<T, DPAD>, Sp::LDS)) return rc;
    attention_split_kernel<T, DPAD><<<(unsigned)blocks, 64 * Sp::WAVES, Sp::LDS, st>>>(p, plan, ws, ml);
    SEMPYR_CHECK_LAUNCH();
    if (plan.splits > 1) {
        attention_join_kernel<T><<<(unsigned)rows, 256, 0, st>>>(p, plan.splits, ws, ml);
        SEMPYR_CHECK_LAUNCH();
    }
    return 0;
}

// Instantiated by name, see attention_bwd.hip.
#define SEMPYR_SPLIT_KERNELS(T) template __global__ void attention_join_kernel<T>(Params, int, const float*, const float*); \
    template __global__ void attention_split_kernel<T, 32>(Params, SplitPlan, float*, float*); \
    template __global__ void attention_split_kernel<T, 64>(Params, SplitPlan, float*, float*); \
    template __global__ void attention_split_kernel<T, 128>(Params, SplitPlan, float*, float*);
SEMPYR_SPLIT_KERNELS(float)
SEMPYR_SPLIT_KERNELS(f16)
SEMPYR_SPLIT_KERNELS(bf16)
#undef SEMPYR_SPLIT_KERNELS

int launch_split(int dtype, const Params& p, const SplitPlan& plan, float* ws, hipStream_t st) {
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        if (p.dim <= 32) return launch_split_d<T, 32>(p, plan, ws, st);
        if (p.dim <= 64) return launch_split_d<T, 64>(p, plan, ws, st);
        return launch_split_d<T, 128>(p, plan, ws, st);
    });
}

}  // namespace attn
