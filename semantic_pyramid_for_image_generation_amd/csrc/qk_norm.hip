// Norms of queries and keys for each head with the rotary position in the same pass, forward and backward.
//
//   xhat = x * r, r = (mean(x^2) + eps)^(-1/2) over a head's `dim` elements;  h = xhat * w;  y = R(positions) h
//   R turns pair j = (a, b) by the angle positions[axis(j)] * freq(j):  (a c - b s, a s + b c)
//   backward: g' = R^T g;  dw = sum over tokens and heads of g' * xhat;  dx = r (g' w - xhat mean(g' w xhat))
// Without weights the norm is left out: y = R x, dx = R^T g.
//
// Angles: positions are integers, so an angle in turns is position * (freq / 2 pi) modulo 1.  The host stores freq / 2 pi as a
// 64-bit fraction; the product wraps modulo 2^64, which IS the reduction modulo one turn, exact for every int32 position (error
// 2^-64 of a turn a step).  The nearest quarter turn is split off in integers, the rest (at most 1/8 turn, rounded once to 24
// bits) goes through the Taylor polynomials of sine and cosine (next terms below 2e-9 on +-pi/4).
//
// Bound by memory: x is read once and y written once (and g, dx).  A group of lanes owns a row (token, head); a lane holds P
// pairs, that is two 16-byte vectors, in such a way that both halves of every pair lie in the same lane, in either pair
// order -- the rotation needs no exchange, the norm log2(lanes) shuffles.  A group walks over a slice of the token's heads with the
// sines and cosines of its pairs in registers.  32768 tokens, 32 + 8 heads of 128, bf16, forward: 671 MB in 138 us (4.9 TB/s,
// 94 % of a copy's rate); 16196 tokens, 16 + 4 heads of 96, fp16 (124 and 187 MB): forward 32 us, backward 51 + 4 us.
#include "tokens.h"

namespace {

struct RopeParams {
    const void* x[2];              // queries, keys (element strides below)
    const void* g[2];              // backward: gradients of the outputs (contiguous)
    void* y[2];                    // forward: outputs; backward: gradients of x (contiguous)
    const void* w[2];              // norm weights, or both null
    int64_t xs_tok[2], xs_head[2];
    const int32_t* positions;
    const uint64_t* freqs;
    float* partials;               // backward: [blocks][2][dim]
    int64_t tokens;
    int heads[2], dim, pairs, axes, section_end[4], interleaved;
    int slice, slices;             // heads a group walks over, slices a token has
    int lanes;                     // lanes of a group, for the kernels that do not know them at compile time
    float eps, inv_dim;
};

__device__ __forceinline__ void sin_cos_turns(uint64_t turns, float& s, float& c) {
    const int32_t t = (int32_t)(turns >> 32);                       // turns * 2^32, signed: [-1/2, 1/2)
    const uint32_t quarter = ((uint32_t)t + 0x20000000u) >> 30;     // nearest multiple of a quarter turn
    const int32_t rest = t - (int32_t)(quarter << 30);              // [-2^29, 2^29): at most an eighth of a turn
    const float a = (float)rest * (float)(6.283185307179586 / 4294967296.0), a2 = a * a;
    const float sn = fmaf(a * a2, fmaf(a2, fmaf(a2, fmaf(a2, 1.f / 362880, -1.f / 5040), 1.f / 120), -1.f / 6), a);
    const float cs = fmaf(a2, fmaf(a2, fmaf(a2, fmaf(a2, fmaf(a2, -1.f / 3628800, 1.f / 40320), -1.f / 720), 1.f / 24), -0.5f), 1.f);
    const float u = (quarter & 1) ? cs : sn, v = (quarter & 1) ? sn : cs;
    s = (quarter & 2) ? -u : u;
    c = ((quarter + 1) & 2) ? -v : v;
}

// The 2 * P elements of a lane: a[i], b[i] are the halves of pair p0 + i.
template <typename T, int P, bool VEC>
struct RowIo {
    int off_a, off_b, p0, dim, pairs;
    bool inter, active;

    __device__ RowIo(const RopeParams& q, int lane) {
        dim = q.dim; pairs = q.pairs; inter = q.interleaved != 0;
        p0 = lane * P;
        active = p0 < dim / 2;
        // behind the rotated part the rest of the head is seen as pairs, too, turned by nothing
        if (inter) { off_a = 2 * p0; off_b = 2 * p0 + P; }
        else if (p0 < pairs) { off_a = p0; off_b = p0 + pairs; }
        else { off_a = pairs + p0; off_b = dim / 2 + p0; }
    }
    __device__ __forceinline__ int elem(int i, int half) const {
        const int p = p0 + i;
        if (inter) return 2 * p + half;
        if (p < pairs) return p + half * pairs;
        return half ? dim / 2 + p : pairs + p;
    }
    __device__ __forceinline__ void load(const T* __restrict__ row, float* a, float* b) const {
        if (VEC) {
            float u[P], v[P];
            if (active) { load_floats<T, P>(row + off_a, u); load_floats<T, P>(row + off_b, v); }
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float ia = 2 * i < P ? u[(2 * i) % P] : v[(2 * i) % P], ib = 2 * i + 1 < P ? u[(2 * i + 1) % P] : v[(2 * i + 1) % P];
                a[i] = !active ? 0.f : inter ? ia : u[i];
                b[i] = !active ? 0.f : inter ? ib : v[i];
            }
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const bool in = p0 + i < dim / 2;
                a[i] = in ? (float)row[elem(i, 0)] : 0.f;
                b[i] = in ? (float)row[elem(i, 1)] : 0.f;
            }
        }
    }
    __device__ __forceinline__ void store(T* __restrict__ row, const float* a, const float* b) const {
        if (VEC) {
            if (!active) return;
            float u[P], v[P];
#pragma unroll
            for (int i = 0; i < P; ++i) {
                u[i] = !inter ? a[i] : (i & 1) ? b[i / 2] : a[i / 2];
                v[i] = !inter ? b[i] : (i & 1) ? b[(P + i) / 2] : a[(P + i) / 2];
            }
            store_floats<T, P>(row + off_a, u);
            store_floats<T, P>(row + off_b, v);
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (p0 + i < dim / 2) { row[elem(i, 0)] = (T)a[i]; row[elem(i, 1)] = (T)b[i]; }
        }
    }
};

template <int P>
__device__ __forceinline__ void lane_angles(const RopeParams& q, int p0, int64_t token, float* s, float* c) {
    const int32_t* pos = q.positions + token * q.axes;
    int64_t at[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) at[k] = k < q.axes ? (int64_t)pos[k] : 0;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int p = p0 + i;
        if (p < q.pairs) {
            const int64_t x = p < q.section_end[0] ? at[0] : p < q.section_end[1] ? at[1] : p < q.section_end[2] ? at[2] : at[3];
            sin_cos_turns(q.freqs[p] * (uint64_t)x, s[i], c[i]);
        } else {
            s[i] = 0.f; c[i] = 1.f;
        }
    }
}

// Groups of `LANES` lanes, a power of two; LANES 0: of any number, `lanes`, where that fits more groups into a wave (six lanes
// for heads of 96 in 16 bits: ten groups instead of eight).  The lanes behind the last whole group have none.
template <int LANES>
struct Group {
    int lanes, per_wave, lane, number;                 // number: within the workgroup
    bool whole;

    __device__ explicit Group(const RopeParams& q) {
        const int at = threadIdx.x & 63;
        lanes = LANES ? LANES : q.lanes;
        per_wave = 64 / lanes;
        lane = at % lanes;
        number = (threadIdx.x >> 6) * per_wave + at / lanes;
        whole = at < per_wave * lanes;
    }
    __device__ __forceinline__ float sum(float v) const {
        if (LANES) {
#pragma unroll
            for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
            return v;
        }
        // pairwise into lane 0: at distance o the lanes below o are complete sums of what lies o, 2 o, .. behind them
        const int at = threadIdx.x & 63;
        for (int o = lanes > 32 ? 32 : lanes > 16 ? 16 : lanes > 8 ? 8 : lanes > 4 ? 4 : 2; o > 0; o >>= 1) {
            const float t = __shfl(v, at + o, 64);
            v += lane + o < lanes ? t : 0.f;
        }
        return __shfl(v, at - lane, 64);
    }
};

template <typename T, int P, int LANES, bool VEC>
__global__ __launch_bounds__(256) void qk_norm_rope_kernel(RopeParams q)
{
    const Group<LANES> group(q);
    const int64_t item = (int64_t)blockIdx.x * 4 * group.per_wave + group.number;
    const int64_t token = item / q.slices;
    if (!group.whole || token >= q.tokens) return;     // whole groups leave: the shuffles below stay inside a group
    const RowIo<T, P, VEC> io(q, group.lane);
    float s[P], c[P];
    lane_angles<P>(q, io.p0, token, s, c);
    const bool norm = q.w[0] != nullptr;
    const int total = q.heads[0] + q.heads[1], h0 = (int)(item - token * q.slices) * q.slice;
    const int h1 = h0 + q.slice < total ? h0 + q.slice : total;
    for (int h = h0; h < h1; ++h) {
        const int part = h >= q.heads[0], head = part ? h - q.heads[0] : h;
        float a[P], b[P];
        io.load((const T*)q.x[part] + token * q.xs_tok[part] + head * q.xs_head[part], a, b);
        if (norm) {
            float wa[P], wb[P], sum = 0.f;
            io.load((const T*)q.w[part], wa, wb);
#pragma unroll
            for (int i = 0; i < P; ++i) sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
            const float r = 1.f / sqrtf(fmaf(group.sum(sum), q.inv_dim, q.eps));
#pragma unroll
            for (int i = 0; i < P; ++i) { a[i] *= r * wa[i]; b[i] *= r * wb[i]; }
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float u = a[i] * c[i] - b[i] * s[i];
            b[i] = a[i] * s[i] + b[i] * c[i];
            a[i] = u;
        }
        io.store((T*)q.y[part] + (token * q.heads[part] + head) * q.dim, a, b);
    }
}

// Backward.  A fixed number of workgroups walks over the rows (x and g are read together, dx is written); a lane adds up its
// elements of dw in registers, a workgroup writes one row of partial sums, weight_grad_kernel adds those in block order: the
// result does not depend on timing.
template <typename T, int P, int LANES, bool VEC>
__global__ __launch_bounds__(256) void qk_norm_rope_bwd_kernel(RopeParams q)
{
    extern __shared__ float sh[];                      // [4 waves][2][dim]; LANES 0: [groups][2][dim]
    const Group<LANES> group(q);
    const int groups = 4 * group.per_wave;
    const RowIo<T, P, VEC> io(q, group.lane);
    const bool norm = q.w[0] != nullptr;
    const int total = q.heads[0] + q.heads[1];
    float ga[2][P], gb[2][P];
#pragma unroll
    for (int i = 0; i < P; ++i) ga[0][i] = ga[1][i] = gb[0][i] = gb[1][i] = 0.f;
    for (int64_t item = (int64_t)blockIdx.x * groups + group.number; group.whole && item < q.tokens * q.slices;
         item += (int64_t)gridDim.x * groups) {
        const int64_t token = item / q.slices;
        float s[P], c[P];
        lane_angles<P>(q, io.p0, token, s, c);
        const int h0 = (int)(item - token * q.slices) * q.slice, h1 = h0 + q.slice < total ? h0 + q.slice : total;
        for (int h = h0; h < h1; ++h) {
            const int part = h >= q.heads[0], head = part ? h - q.heads[0] : h;
            const int64_t row = (token * q.heads[part] + head) * q.dim;
            float u[P], v[P];
            io.load((const T*)q.g[part] + row, u, v);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float t = u[i] * c[i] + v[i] * s[i];
                v[i] = v[i] * c[i] - u[i] * s[i];
                u[i] = t;
            }
            if (norm) {
                float a[P], b[P], wa[P], wb[P], sum = 0.f, dot = 0.f;
                io.load((const T*)q.x[part] + token * q.xs_tok[part] + head * q.xs_head[part], a, b);
                io.load((const T*)q.w[part], wa, wb);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    sum = fmaf(a[i], a[i], fmaf(b[i], b[i], sum));
                    dot = fmaf(u[i] * wa[i], a[i], fmaf(v[i] * wb[i], b[i], dot));
                }
                const float r = 1.f / sqrtf(fmaf(group.sum(sum), q.inv_dim, q.eps));
                const float m = group.sum(dot) * q.inv_dim * r;          // mean(g' w xhat)
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const float xa = a[i] * r, xb = b[i] * r;
                    if (part) { ga[1][i] = fmaf(u[i], xa, ga[1][i]); gb[1][i] = fmaf(v[i], xb, gb[1][i]); }
                    else { ga[0][i] = fmaf(u[i], xa, ga[0][i]); gb[0][i] = fmaf(v[i], xb, gb[0][i]); }
                    u[i] = r * (u[i] * wa[i] - xa * m);
                    v[i] = r * (v[i] * wb[i] - xb * m);
                }
            }
            io.store((T*)q.y[part] + row, u, v);
        }
    }
    if (!norm) return;
    // what is added up next: a wave's sums, or every group's by itself
    const int row = LANES ? threadIdx.x >> 6 : group.number, rows = LANES ? 4 : groups;
#pragma unroll
    for (int part = 0; part < 2; ++part)
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float u = ga[part][i], v = gb[part][i];
            if (LANES) {
#pragma unroll
                for (int o = LANES; o < 64; o <<= 1) { u += __shfl_xor(u, o, 64); v += __shfl_xor(v, o, 64); }
            }
            if (group.whole && (!LANES || (threadIdx.x & 63) < LANES) && io.p0 + i < q.dim / 2) {
                sh[(row * 2 + part) * q.dim + io.elem(i, 0)] = u;
                sh[(row * 2 + part) * q.dim + io.elem(i, 1)] = v;
            }
        }
    __syncthreads();
    for (int e = threadIdx.x; e < 2 * q.dim; e += 256) {
        const int part = e / q.dim, d = e - part * q.dim;
        float t = 0.f;
        for (int k = 0; k < rows; ++k) t += sh[(k * 2 + part) * q.dim + d];
        q.partials[(int64_t)blockIdx.x * 2 * q.dim + e] = t;
    }
}

// dw[part][d] = sum over blocks of partials[block][part][d]: 8 columns a workgroup, 128 threads a column, fixed order.
template <typename T>
__global__ __launch_bounds__(1024) void weight_grad_kernel(const float* __restrict__ partials, int blocks, int dim, T* __restrict__ dwq,
                                                           T* __restrict__ dwk)
{
    const int c = threadIdx.x % 8, col = blockIdx.x * 8 + c, row0 = threadIdx.x / 8;
    float t = 0.f;
    if (col < 2 * dim) {
#pragma unroll 8
        for (int r = row0; r < blocks; r += 128) t += partials[(int64_t)r * 2 * dim + col];
    }
    __shared__ float sh[128][9];
    sh[row0][c] = t;
    __syncthreads();
#pragma unroll
    for (int half = 64; half > 0; half /= 2) {
        if (row0 < half) sh[row0][c] += sh[row0 + half][c];
        __syncthreads();
    }
    if (row0 == 0 && col < 2 * dim) (col < dim ? dwq : dwk)[col < dim ? col : col - dim] = (T)sh[0][c];
}

// Backward: three workgroups a CU (16-bit types: what the registers allow at once; a fourth would wait for the others' end), one
// row of partial sums each.  Heads a group walks over at most: short slices spread the walks over the fixed number of
// groups (16196 tokens, 16 + 4 heads of 96, fp16, backward: slices of 8 and 1024 workgroups 57 us, 8 and 768 52, 4 and 768 50);
// forward: 32768 tokens, 32 + 8 heads of 128: 8 139 us, 4 143.
constexpr int MAX_BLOCKS = 768, FWD_SLICE = 8, BWD_SLICE = 4;

int check_desc(const sempyr_rope_desc* d, const char* who) {
    if (!d) SEMPYR_FAIL("%s: null descriptor", who);
    if (!dtype_ok(d->dtype)) SEMPYR_FAIL("%s: unknown element type %d", who, d->dtype);
    if (d->dim < 2 || d->dim > 512 || d->dim % 2) SEMPYR_FAIL("%s: head dim must be even and at most 512, got %d", who, d->dim);
    if (d->heads_q < 1 || d->heads_k < 1 || d->heads_q > 4096 || d->heads_k > 4096) SEMPYR_FAIL("%s: %d / %d heads", who, d->heads_q, d->heads_k);
    if (d->axes < 1 || d->axes > 4) SEMPYR_FAIL("%s: 1 to 4 position axes, got %d", who, d->axes);
    int sum = 0;
    for (int k = 0; k < d->axes; ++k) {
        if (d->sections[k] < 0) SEMPYR_FAIL("%s: negative section", who);
        sum += d->sections[k];
        if (sum > d->dim / 2) SEMPYR_FAIL("%s: the sections hold more than dim / 2 = %d pairs", who, d->dim / 2);
    }
    if (sum < 1) SEMPYR_FAIL("%s: no pair to rotate", who);
    if (d->tokens < 0 || d->tokens > (int64_t)1 << 31) SEMPYR_FAIL("%s: %lld tokens", who, (long long)d->tokens);
    if (!(d->eps >= 0.f)) SEMPYR_FAIL("%s: eps must not be negative", who);
    return 0;
}

// lanes of a group (exact: the kernels with LANES 0), workgroups for one item (a slice of a token's heads) a group
struct Launch { int lanes; bool vec, exact; int64_t blocks; };

// Vector form where every row and both halves of a lane's pairs start on 16 bytes; element-wise loads otherwise (unaligned
// views, rotated parts that are no multiple of a vector).
Launch prepare(const sempyr_rope_desc* d, RopeParams& q, const void* const* ptrs, int nptrs, int most) {
    Launch l;
    const int sz = dtype_size(d->dtype), n = 16 / sz;
    q.tokens = d->tokens; q.heads[0] = d->heads_q; q.heads[1] = d->heads_k;
    q.dim = d->dim; q.axes = d->axes; q.interleaved = d->interleaved; q.eps = d->eps; q.inv_dim = 1.f / d->dim;
    q.pairs = 0;
    for (int k = 0; k < 4; ++k) { q.pairs += k < d->axes ? d->sections[k] : 0; q.section_end[k] = q.pairs; }
    q.xs_tok[0] = d->q_stride_token; q.xs_tok[1] = d->k_stride_token;
    q.xs_head[0] = d->q_stride_head; q.xs_head[1] = d->k_stride_head;
    l.vec = (d->dim / 2) % n == 0 && (d->interleaved || q.pairs % n == 0);
    for (int k = 0; k < 2; ++k) l.vec = l.vec && q.xs_tok[k] * sz % 16 == 0 && q.xs_head[k] * sz % 16 == 0;
    for (int k = 0; k < nptrs; ++k) l.vec = l.vec && aligned16(ptrs[k]);
    const int need = (d->dim / 2 + n - 1) / n;
    l.lanes = 1;
    while (l.lanes < need) l.lanes *= 2;
    l.exact = l.vec && 64 / need > 64 / l.lanes;
    if (l.exact) l.lanes = need;
    q.lanes = l.lanes;
    // A group walks over several heads to share the sines and cosines, as long as enough groups are left to fill the chip
    // (256 CUs x 8 waves).
    const int total = d->heads_q + d->heads_k;
    q.slice = 1;
    while (q.slice < most && q.slice < total && d->tokens * ceil_div(total, q.slice * 2) * l.lanes >= 64ll * 2048) q.slice *= 2;
    q.slices = ceil_div(total, q.slice);
    q.slice = ceil_div(total, q.slices);               // 20 heads in 7, 7 and 6, not 8, 8 and 4
    const int groups = 4 * (64 / l.lanes);
    l.blocks = (d->tokens * q.slices + groups - 1) / groups;
    return l;
}

template <typename T, bool BWD>
int launch(const RopeParams& q, const Launch& l, unsigned blocks, hipStream_t st) {
    constexpr int P = Vec16<T>::N;
    auto go = [&](auto lanes) {
        constexpr int LANES = decltype(lanes)::value;
        // (exact groups: dim = 2 P lanes, at most 256 lanes: 32 KiB)
        const size_t lds = BWD ? (LANES ? 4 : 4 * (64 / l.lanes)) * 2 * (size_t)q.dim * sizeof(float) : 0;
        auto run = [&](auto vec) {
            constexpr bool VEC = decltype(vec)::value;
            if constexpr (BWD) qk_norm_rope_bwd_kernel<T, P, LANES, VEC><<<blocks, 256, lds, st>>>(q);
            else qk_norm_rope_kernel<T, P, LANES, VEC><<<blocks, 256, 0, st>>>(q);
        };
        if constexpr (LANES == 0) run(std::true_type());
        else if (l.vec) run(std::true_type());
        else run(std::false_type());
        SEMPYR_CHECK_LAUNCH();
        return 0;
    };
    if (l.exact) return go(std::integral_constant<int, 0>());
    switch (l.lanes) {
        case 1: return go(std::integral_constant<int, 1>());
        case 2: return go(std::integral_constant<int, 2>());
        case 4: return go(std::integral_constant<int, 4>());
        case 8: return go(std::integral_constant<int, 8>());
        case 16: return go(std::integral_constant<int, 16>());
        case 32: return go(std::integral_constant<int, 32>());
        default: return go(std::integral_constant<int, 64>());
    }
}

}  // namespace

extern "C" int sempyr_qk_norm_rope_fwd(const sempyr_rope_desc* d, const void* xq, const void* xk, const int32_t* positions,
                                       const uint64_t* freqs, const void* wq, const void* wk, void* yq, void* yk, void* stream)
{
    if (int rc = check_desc(d, "qk_norm_rope_fwd")) return rc;
    if (d->tokens == 0) return 0;
    if (!xq || !xk || !positions || !freqs || !yq || !yk) SEMPYR_FAIL("qk_norm_rope_fwd: null pointer");
    if (!wq != !wk) SEMPYR_FAIL("qk_norm_rope_fwd: norm weights of both or of neither");
    RopeParams q = {};
    q.x[0] = xq; q.x[1] = xk; q.y[0] = yq; q.y[1] = yk; q.w[0] = wq; q.w[1] = wk;
    q.positions = positions; q.freqs = freqs;
    const void* ptrs[] = {xq, xk, yq, yk, wq, wk};
    const Launch l = prepare(d, q, ptrs, 6, FWD_SLICE);
    const int64_t blocks = l.blocks;
    if (!grid_fits(blocks, 256)) SEMPYR_FAIL("qk_norm_rope_fwd: too many rows");
    const hipStream_t st = (hipStream_t)stream;
    HbmScope scope("qk_norm_rope_kernel", 2.0 * d->tokens * (d->heads_q + d->heads_k) * d->dim * dtype_size(d->dtype), st);
    return with_dtype(d->dtype, [&](auto t) { return launch<decltype(t), false>(q, l, (unsigned)blocks, st); });
}

extern "C" int sempyr_qk_norm_rope_bwd_scratch(const sempyr_rope_desc* d, int64_t* floats)
{
    if (int rc = check_desc(d, "qk_norm_rope_bwd")) return rc;
    if (!floats) SEMPYR_FAIL("qk_norm_rope_bwd: null pointer");
    *floats = (int64_t)MAX_BLOCKS * 2 * d->dim;
    return 0;
}

extern "C" int sempyr_qk_norm_rope_bwd(const sempyr_rope_desc* d, const void* xq, const void* xk, const int32_t* positions,
                                       const uint64_t* freqs, const void* wq, const void* wk, const void* gq, const void* gk,
                                       void* dq, void* dk, void* dwq, void* dwk, float* scratch, void* stream)
{
    if (int rc = check_desc(d, "qk_norm_rope_bwd")) return rc;
    if (!wq != !wk) SEMPYR_FAIL("qk_norm_rope_bwd: norm weights of both or of neither");
    if (wq && (!dwq || !dwk || !scratch)) SEMPYR_FAIL("qk_norm_rope_bwd: null pointer");
    if (d->tokens > 0 && (!xq || !xk || !positions || !freqs || !gq || !gk || !dq || !dk)) SEMPYR_FAIL("qk_norm_rope_bwd: null pointer");
    RopeParams q = {};
    q.x[0] = xq; q.x[1] = xk; q.g[0] = gq; q.g[1] = gk; q.y[0] = dq; q.y[1] = dk; q.w[0] = wq; q.w[1] = wk;
    q.positions = positions; q.freqs = freqs; q.partials = scratch;
    const void* ptrs[] = {xq, xk, gq, gk, dq, dk, wq, wk};
    const Launch l = prepare(d, q, ptrs, 8, BWD_SLICE);
    int64_t blocks = l.blocks;
    if (blocks > MAX_BLOCKS) blocks = MAX_BLOCKS;
    const hipStream_t st = (hipStream_t)stream;
    return with_dtype(d->dtype, [&](auto t) {
        typedef decltype(t) T;
        if (blocks) {
            HbmScope scope("qk_norm_rope_bwd_kernel", 3.0 * d->tokens * (d->heads_q + d->heads_k) * d->dim * dtype_size(d->dtype), st);
            if (int rc = launch<T, true>(q, l, (unsigned)blocks, st)) return rc;
        }
        if (!wq) return 0;
        weight_grad_kernel<T><<<ceil_div(2 * d->dim, 8), 1024, 0, st>>>(scratch, (int)blocks, d->dim, (T*)dwq, (T*)dwk);
        SEMPYR_CHECK_LAUNCH();
        return 0;
    });
}
