// Tiles of the attention kernels (attention_fwd.hip, attention_bwd.hip, attention_split.hip) on gfx950.
//
// Matrix products run on the 32x32 MFMA shapes with the ROWS OF THE RESULT in a lane's registers and one COLUMN per lane pair
// (l, l + 32): register i of lane l holds row 8 (i / 4) + 4 (l / 32) + i % 4 of column l % 32.  Scores are computed transposed
// (keys are rows, a query is a column), so a query's softmax runs over a lane's own registers plus one exchange between the
// lane halves, and the probabilities are, as they lie in the registers, the right operand of the next product: a sum over k
// may run in any order as long as both operands agree, and the order used everywhere is
//     element j of lane half h in the t-th group of 16 = row 16 t + 8 (j / 4) + 4 h + j % 4.
// No probability goes through LDS.
//
// A tile in LDS is [rows][CH chunks of 16 bytes]; chunk c of row r lies at c ^ swz(r).  That spreads both ways of reading over
// the banks: "row fragments" (lane = row, 8 consecutive elements) and "column fragments" (lane = column, 8 rows in the order
// above; 16-bit types by the transposing ds_read_b64_tr_b16, which hands 16 lanes a 4 x 16 block by columns).
// Tiles are filled by LDS DMA (buffer_load_dwordx4 ... lds), which writes a wave's 64 x 16 bytes in lane order: the permutation
// is applied to the addresses that are read.  The buffer descriptor ends with the last valid row, so rows behind a sequence
// and columns behind the head arrive as zeros and nothing outside is ever touched.
#pragma once
#include "tokens.h"

namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
#define LDS_PTR __attribute__((address_space(3)))
// Tells the scheduler how many waves a SIMD will hold, so that it spends the registers on loads ahead of their use.
#define WAVES_PER_SIMD(n) __attribute__((amdgpu_waves_per_eu(n, n)))

struct Params {
    const void *q, *k, *v;                                   // [rows][heads][dim], strides in elements
    int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head;
    void* o;                                                 // contiguous [total_q][heads_q][dim]
    void* o_low;                                             // 16-bit types: what rounding took from o, for delta; or null
    float* stats;                                            // rows' softmax statistics for the backward pass (see Stats), or null
    const void* go;                                          // backward: gradient of o, contiguous
    float* delta;                                            // backward: [heads_q][total_q] rowsum(go * o)
    void *dq, *dk, *dv;                                      // backward: contiguous
    const int32_t *cu_q, *cu_k, *len_k;
    int total_q, total_k, nseq, heads_q, heads_k, group, dim, causal;
    float scale, scale_log2;                                 // scale * log2(e)
};

// ---------------------------------------------------------------------------------------------- element types
template <typename T> struct Elem;
template <> struct Elem<bf16> {
    typedef bf16 Frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <> struct Elem<f16> {
    typedef f16 Frag __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <> struct Elem<float> {
    typedef float Frag __attribute__((ext_vector_type(8)));
    // the group of 16 in eight steps of two (lane half h of step i holds its element i)
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// registers 8 t .. 8 t + 7 of a result as the right operand of the next product.  16-bit types round here: probabilities and
// score gradients enter the matrix pipe in the inputs' type, their sums stay fp32.  A rounding of the results' own size: outputs
// of the packed batch in bf16 are off by 0.0020 (rms, of their norm), 0.0016 of it the one rounding of the result; 0.00027 and
// 0.00020 in fp16.  What it takes can be multiplied, too (rest_of), for half as many products again; that is done where the
// matrix pipe waits for memory anyway.
template <typename T>
__device__ __forceinline__ typename Elem<T>::Frag frag_of(const f32x16& s, int t) {
    typename Elem<T>::Frag f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)s[t * 8 + j];
    return f;
}

// what that rounding took: added as a second product where the matrix pipe has the time, it makes the operand exact to twice
// the type's bits
template <typename T>
__device__ __forceinline__ typename Elem<T>::Frag rest_of(const f32x16& s, const typename Elem<T>::Frag& f, int t) {
    typename Elem<T>::Frag r;
#pragma unroll
    for (int j = 0; j < 8; ++j) r[j] = (T)(s[t * 8 + j] - (float)f[j]);
    return r;
}

// x of the other lane half, combined: gfx950 swaps the halves in the vector unit, no LDS round trip
__device__ __forceinline__ float half_max(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// fp16 backward: P and dS in the type's normal numbers.  P, at most 1, is kept times 2^15 (the statistics carry the shift, see Stats).
// dS has no bound of its own, and the results may fit where it does not or where it falls among the subnormals, so every column
// (lane pair) has a power of two for it, undone in the fp32 sums: whenever a tile's largest |dS| would pass 2^15, the power falls
// to put that at 2^10, and the sums so far follow.  What lies 2^24 below the largest so far is subnormal; its error, 2^-35 of
// the largest, is nothing in the sum.  bf16 has the range of fp32.  (Packed batch of 16 196 tokens, 16/4 heads, causal, fp16: heads of
// 64 dQ 158 -> 168, dK/dV 262 -> 272 us, heads of 128 278 -> 289 and 580 -> 650: a maximum and a product an element.  2^7 takes the same time, 2^12 2 % more.)
template <typename T> constexpr bool NARROW = std::is_same<T, f16>::value;
template <typename T> constexpr int P_BITS = NARROW<T> ? 15 : 0;
struct ColumnScale {
    int bits = 100;                                  // no dS yet
    float f = 0x1p100f;
    template <typename Rescale>
    __device__ __forceinline__ void fit(const f32x16& s, bool counts, Rescale rescale) {
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, fabsf(s[i]));
        mx = counts ? half_max(mx) : 0.f;
        const bool moves = mx * f > 0x1p15f && mx < INFINITY;             // (infinities and NaN go through as they are)
        if (__any(moves)) {
            const int to = moves ? 127 + 10 - (int)(__float_as_uint(mx) >> 23) : bits;
            rescale(ldexpf(1.f, to - bits));
            bits = to;
            f = ldexpf(1.f, to);
        }
    }
};

// ---------------------------------------------------------------------------------------------- tiles
template <typename T, int DPAD, int ROWS>
struct Tile {
    typedef typename Elem<T>::Frag Frag;
    static constexpr int SZ = sizeof(T), ROWB = DPAD * SZ, CH = ROWB / 16, BYTES = ROWS * ROWB;
    static constexpr int LOADS = BYTES / 1024;               // 1 KiB DMA instructions of a tile
    static_assert(CH >= 4 && (CH & (CH - 1)) == 0 && BYTES % 1024 == 0, "tile shape");

    static __device__ __forceinline__ int swz(int r) {
        return CH >= 16 ? (r & 3) << 2 | (r >> 2 & 3) : CH == 8 ? (r >> 1 & 1) << 2 | (r >> 2 & 3) : r >> 2 & 3;
    }
    // byte offset of a lane's row fragment in row block 0, group 0; see row()
    static __device__ __forceinline__ int row_base(int lane) {
        const int r = lane & 31, h = lane >> 5;
        return r * ROWB + (((SZ == 2 ? h : 2 * h) ^ swz(r)) << 4);
    }
    // elements 16 slab + 8 h .. + 8 of row 32 block + lane % 32
    static __device__ __forceinline__ Frag row(const char* tile, int base, int block, int slab) {
        const char* p = tile + block * 32 * ROWB;
        if constexpr (SZ == 2) return *reinterpret_cast<const Frag*>(p + (base ^ slab * 32));
        else {
            typedef float f4 __attribute__((ext_vector_type(4)));
            const f4 a = *reinterpret_cast<const f4*>(p + (base ^ slab * 64)), b = *reinterpret_cast<const f4*>(p + (base ^ slab * 64 ^ 16));
            return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
    static __device__ __forceinline__ int col_base(int lane) {
        const int h = lane >> 5;
        if (SZ == 2) {
            const int r4 = (lane & 15) >> 2, r = h * 4 + r4, c = (lane >> 4 & 1) * 2 + ((lane & 3) >> 1);
            return r * ROWB + ((c ^ swz(r)) << 4) + (lane & 1) * 8;
        }
        return h * 4 * ROWB + (((lane & 31) >> 2 ^ swz(h * 4)) << 4) + (lane & 3) * 4;
    }
    // column 32 block + lane % 32, rows 16 t + 8 (j / 4) + 4 h + j % 4
    static __device__ __forceinline__ Frag col(const char* tile, int base, int block, int t) {
        if constexpr (SZ == 2) {
            typedef T V4 __attribute__((ext_vector_type(4)));
            V4 x[2];                                         // (cast as a whole: __builtin_bit_cast of one element takes element 0)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                x[u] = __builtin_bit_cast(V4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (LDS_PTR s16x4*)(tile + (t * 16 + u * 8) * ROWB + (base ^ block * 64 ^ u * 32))));
            return __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7);
        } else {
            Frag f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int r = (j / 4) * 8 + j % 4;
                f[j] = *reinterpret_cast<const float*>(tile + (t * 16 + r) * ROWB + (base ^ block * 128 ^ swz(r) << 4));
            }
            return f;
        }
    }
};

// LDS DMA of 16 (4) bytes a lane: lane i's bytes from `offset` in the buffer go to lds + 16 i (4 i); behind the buffer's end zeros.
// In assembly, because the compiler, where it knows of a DMA in flight, waits for all of them before a transposing LDS read,
// whatever buffer that reads; the waits are wait_loads() here.  Nothing is returned in registers.
typedef int BufferDesc __attribute__((ext_vector_type(4)));
__device__ __forceinline__ BufferDesc buffer_desc(const void* base, int bytes) {
    const uint64_t at = (uint64_t)base;
    return BufferDesc{__builtin_amdgcn_readfirstlane((int)at), __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xFFFF),
                      __builtin_amdgcn_readfirstlane(bytes), 0x00020000};
}
__device__ __forceinline__ unsigned lds_offset(const void* p) { return (unsigned)(uintptr_t)(LDS_PTR const char*)p; }
// s_nop 4: five wait states, should the compiler have written the descriptor with a vector instruction right before (it does not
// look for that hazard into assembly); m0 needs one.
// (m0, the DMA's LDS address, is a reserved register: the compiler warns that it does not keep a value there across the block,
// which is what the clobber says)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void dma16(BufferDesc rsrc, int offset, const void* lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :: "s"(__builtin_amdgcn_readfirstlane(lds_offset(lds))), "v"(offset), "s"(rsrc) : "memory", "m0");
}
__device__ __forceinline__ void dma4(BufferDesc rsrc, int offset, const void* lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :: "s"(__builtin_amdgcn_readfirstlane(lds_offset(lds))), "v"(offset), "s"(rsrc) : "memory", "m0");
}
#pragma clang diagnostic pop

// Fills tiles from rows of a strided tensor.  `waves` waves share a tile; a lane's source offsets are fixed.
template <typename T, int DPAD, int ROWS, int WAVES>
struct Filler {
    typedef Tile<T, DPAD, ROWS> Tl;
    static constexpr int N = Tl::LOADS / WAVES;              // instructions a wave issues
    static_assert(Tl::LOADS % WAVES == 0, "whole instructions per wave");
    int voff[N];
    int stride_bytes, row_bytes, wave;

    __device__ __forceinline__ void init(int64_t stride_elems, int dim, int wave_, int lane) {
        stride_bytes = (int)stride_elems * Tl::SZ;           // the host has checked that 64 rows stay below 2^31 bytes
        row_bytes = dim * Tl::SZ;
        wave = wave_;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int p = (j * WAVES + wave) * 64 + lane, r = p / Tl::CH, c = (p % Tl::CH) ^ Tl::swz(r);
            voff[j] = c * 16 < row_bytes ? r * stride_bytes + c * 16 : (int)0x80000000;      // behind every buffer's end: zeros
        }
    }
    // rows 0 .. ROWS - 1 from `base` (a wave-uniform address); rows from `valid` on become zeros
    __device__ __forceinline__ void issue(const void* base, int valid, char* tile) const {
        const int rows = valid < ROWS ? valid : ROWS;
        const int bytes = rows > 0 ? (rows - 1) * stride_bytes + row_bytes : 0;
        const BufferDesc rsrc = buffer_desc(base, bytes);
#pragma unroll
        for (int j = 0; j < N; ++j) dma16(rsrc, voff[j], tile + (j * WAVES + wave) * 1024);
    }
};

// waits until at most N of this wave's vector memory accesses are in flight
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }
// waits until this wave's LDS reads have returned: a buffer may be refilled only after that
__device__ __forceinline__ void wait_lds() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// 8 consecutive elements of each group of 16 of a global row, in row-fragment order (zeros for an absent row, behind the head)
template <typename T, int DPAD>
__device__ __forceinline__ void load_row_frags(typename Elem<T>::Frag* f, const T* row, bool present, int dim, int lane) {
    const int h = lane >> 5;
#pragma unroll
    for (int s = 0; s < DPAD / 16; ++s) {
        const int d = s * 16 + h * 8;
        if constexpr (sizeof(T) == 2) {
            typename Elem<T>::Frag z = {};
            f[s] = present && d < dim ? *reinterpret_cast<const typename Elem<T>::Frag*>(row + d) : z;
        } else {
            typedef float f4 __attribute__((ext_vector_type(4)));
            const f4 z = {0.f, 0.f, 0.f, 0.f};
            const f4 a = present && d < dim ? *reinterpret_cast<const f4*>(row + d) : z;
            const f4 b = present && d + 4 < dim ? *reinterpret_cast<const f4*>(row + d + 4) : z;
            f[s] = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
}

// STEPS products from fragments read from LDS, in batches: the next batch is read before this one is used, and the scheduler
// may move neither reads nor products across (left alone, the compiler reads every fragment into the same registers right
// before its product, which then waits for the LDS each time).
template <typename T> constexpr int BATCH = sizeof(T) == 4 ? 2 : 4;
template <typename F, int STEPS, int MOST, typename Load, typename Use>
__device__ __forceinline__ void pipelined(Load load, Use use) {
    constexpr int BATCH = MOST < STEPS ? MOST : STEPS, N = STEPS / BATCH, VALU_SALU_MAY_CROSS = 0x6;
    static_assert(STEPS % BATCH == 0, "whole batches");
    F f[2][BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) f[0][i] = load(i);
#pragma unroll
    for (int s = 0; s < N; ++s) {
        if (s + 1 < N) {
#pragma unroll
            for (int i = 0; i < BATCH; ++i) f[(s + 1) & 1][i] = load((s + 1) * BATCH + i);
        }
        __builtin_amdgcn_sched_barrier(VALU_SALU_MAY_CROSS);
#pragma unroll
        for (int i = 0; i < BATCH; ++i) use(s * BATCH + i, f[s & 1][i]);
        __builtin_amdgcn_sched_barrier(VALU_SALU_MAY_CROSS);
    }
}

// Settles loads into registers before a loop: the compiler would otherwise place their wait inside it, where it would also wait
// for the DMA in flight.
template <typename F, int N>
__device__ __forceinline__ void settle(F (&f)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+v"(f[i]));
}

// 4 consecutive elements
template <typename T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
    typedef T V __attribute__((ext_vector_type(4)));
    *reinterpret_cast<V*>(p) = V{(T)a, (T)b, (T)c, (T)d};
}

// The reference of a row (its maximum at some tile) moves only when a score passes it by REF_SLACK powers of two: until then
// exponentials are at most 2^8, which bf16 and the fp32 sums hold, and the sums need no rescaling.  fp32: always.
// fp16's normal numbers end at 2^-14, and what lies below may be all of the output: a key with nearly all of the weight and no
// value, 20000 others e^-17 below it each -- off by 0.4.  There the slack is 2 and exponentials are taken times 2^13, at most 2^15.
// (Slack 8, 4 or 2: 200.9, 200.5, 202.2 us for the packed batch with heads of 128.)
template <typename T> constexpr float REF_SLACK = sizeof(T) == 4 ? 0.f : NARROW<T> ? 2.f : 8.f;
template <typename T> constexpr int REF_BITS = NARROW<T> ? 13 : 0;
// exponential of a score against a row's reference x (forward: c m for 16-bit types, m for fp32).  fp32 subtracts first: exact
// next to the maximum, so that a row with one key is that key's value to the bit.
template <typename T>
__device__ __forceinline__ float score_exp(float s, float c, float x) {
    return sizeof(T) == 4 ? __builtin_amdgcn_exp2f((s - x) * c) : __builtin_amdgcn_exp2f(fmaf(s, c, -x));
}
// (Not contracted into what it is used in: everywhere the same rounded number.)
template <typename T>
__device__ __forceinline__ float score_ref(float m, float c) {
#pragma clang fp contract(off)
    return m == -INFINITY ? 0.f : sizeof(T) == 4 ? m : m * c - REF_BITS<T>;
}
// what sums taken with the reference m (a row's, a wave's or a workgroup's) are multiplied by to go with another one; 1 where it is
// the same.  (16-bit types: the references as they were used, rounded.)
template <typename T>
__device__ __forceinline__ float score_move(float m, float to, float c) {
#pragma clang fp contract(off)
    if (m == -INFINITY) return 0.f;                  // (no key so far)
    return __builtin_amdgcn_exp2f(sizeof(T) == 4 ? (m - to) * c : score_ref<T>(m, c) - score_ref<T>(to, c));
}

// What the forward leaves of a row's softmax.  16-bit types: lse = c m + log2(sum), from which P = exp2(c s - lse); its rounding
// (2^-24 of about 10; of scores of 10^4, fp16's half step) is far below theirs.  (fp16: lse - 15, see P_BITS.)  fp32: the maximum m and the reciprocal of the sum,
// [2][heads_q][total_q], P = exp2(c (s - m)) / sum: with lse the gradients of 1024 keys were off by 9e-7, twice what the products themselves leave.
template <typename T> struct Stats {
    static constexpr int N = sizeof(T) == 4 ? 2 : 1;
    static __device__ __forceinline__ void store(const Params& p, int64_t at, float m, float sum) {
        if constexpr (N == 1) p.stats[at] = sum == 0.f ? INFINITY : score_ref<T>(m, p.scale_log2) + __log2f(sum) - P_BITS<T>;      // no key: P = exp2(-infinity)
        else {
            p.stats[at] = sum == 0.f ? INFINITY : m;
            p.stats[(int64_t)p.heads_q * p.total_q + at] = sum == 0.f ? 0.f : 1.f / sum;
        }
    }
};

// 4 consecutive elements of the output and, where it is asked for, of what their rounding left
template <typename T>
__device__ __forceinline__ void store_out(const Params& p, int64_t at, float a, float b, float c, float d) {
    store4((T*)p.o + at, a, b, c, d);
    if (sizeof(T) == 2 && p.o_low) store4((T*)p.o_low + at, a - (float)(T)a, b - (float)(T)b, c - (float)(T)c, d - (float)(T)d);
}

// ---------------------------------------------------------------------------------------------- packed sequences
// Sequence s covers rows cu[s] .. cu[s + 1] - 1; the first entry counts as 0, rows behind the last entry form one more,
// key-less sequence (their results are zeros).  Every entry is clamped to the tensor, so a bad table reads nothing outside.
__device__ __forceinline__ int row_bound(const int32_t* cu, int s, int nseq, int total) {
    if (s <= 0) return 0;
    if (s > nseq) return total;
    const int v = cu[s];
    return v < 0 ? 0 : v > total ? total : v;
}

struct Seq { int q0, lq, k0, lk, kcap; };       // first rows, queries, keys that count, rows of the key slot

__device__ __forceinline__ Seq seq_of(const Params& p, int s) {
    Seq q;
    q.q0 = row_bound(p.cu_q, s, p.nseq, p.total_q);
    q.lq = row_bound(p.cu_q, s + 1, p.nseq, p.total_q) - q.q0;
    q.k0 = row_bound(p.cu_k, s, p.nseq, p.total_k);
    q.kcap = row_bound(p.cu_k, s + 1, p.nseq, p.total_k) - q.k0;
    if (q.lq < 0) q.lq = 0;
    if (q.kcap < 0) q.kcap = 0;
    q.lk = q.kcap;
    if (s >= p.nseq) q.lk = 0;
    else if (p.len_k) { const int n = p.len_k[s]; q.lk = n < 0 ? 0 : n < q.kcap ? n : q.kcap; }
    return q;
}

// inclusive prefix sum over the wave (data-parallel primitives: no LDS)
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);      // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);      // last lane of row 0 / 2 into row 1 / 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);      // lane 31 into rows 2 and 3
    return v;
}

// Tile number -> sequence and first row of the tile, for tiles of R rows of the queries (BY_KEYS: of the key slots).
// No table has to be built and lengths may change between replays of a captured graph.
//  * Up to 63 sequences (a lane each, rows behind the last one are one more): tiles are numbered exactly and by falling load
//    -- the keys a query tile sees, the queries that see a key tile -- so that the longest go first.  A tile's load is found by
//    bisection over 32 levels of the loads, each probe counts the tiles of all sequences at or above a level.
//  * More: sequence s owns the numbers cu[s] / R + s .., at least as many as it has tiles (the rest are empty), the numbers
//    run backwards; the search probes 64 entries at a time.  (63 and 64 sequences of 40 to 500 tokens, 16/4 heads of 64, bf16: dK/dV
//    57 and 64 us, the others alike; 63 and 64 tokens against 800 to 10 000 keys, 32/8 heads of 128: 204 and 225 us.)
struct Where { int s, row; bool ok; Seq sq; };

template <bool BY_KEYS>
__device__ __forceinline__ Where locate(const Params& p, int number, int R, int lane) {
    Where w;
    const int total = BY_KEYS ? p.total_k : p.total_q;
    const int32_t* cu = BY_KEYS ? p.cu_k : p.cu_q;
    if (p.nseq > 63) {
        const int slot = total / R + p.nseq - number;
        int lo = 0, hi = p.nseq;
        while (lo < hi) {
            const int step = (hi - lo + 63) / 64, c = lo + (lane + 1) * step;
            const bool ok = c <= hi && row_bound(cu, c, p.nseq, total) / R + c <= slot;
            lo += __popcll(__ballot(ok)) * step;
            hi = lo + step - 1 < hi ? lo + step - 1 : hi;
        }
        w.s = __builtin_amdgcn_readfirstlane(lo);
        w.sq = seq_of(p, w.s);
        w.row = (slot - ((BY_KEYS ? w.sq.k0 : w.sq.q0) / R + w.s)) * R;
        w.ok = slot >= 0 && w.row >= 0 && w.row < (BY_KEYS ? w.sq.kcap : w.sq.lq);
        return w;
    }
    Seq sq = {0, 0, 0, 0, 0};
    if (lane <= p.nseq) sq = seq_of(p, lane);
    const int rows = BY_KEYS ? sq.kcap : sq.lq, n = (rows + R - 1) / R, shift = sq.lk - sq.lq;
    // tiles of this lane's sequence whose load is at least x; the loads fall with the tile's rank
    auto count = [&](int x) {
        if (x <= 0) return n;
        int c;
        if (BY_KEYS) c = x > sq.lq ? 0 : !p.causal ? (sq.lk + R - 1) / R : (min(sq.lk - 1, sq.lq - x + shift) + R) / R;
        else c = !p.causal ? (sq.lk >= x ? n : 0) : n - (max(0, min(x, sq.lk + 1) - shift) + R - 1) / R;      // (the min: 32 bits hold it)
        return max(0, min(n, c));
    };
    const int all = __builtin_amdgcn_readlane(wave_scan(n), 63);
    w.ok = number < all;
    if (!w.ok) return w;
    int top = lane <= p.nseq ? (BY_KEYS ? sq.lq : sq.lk) : 0;            // no load is larger
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = max(top, __shfl_xor(top, o, 64));
    const int level = max(R, top / 32 + 1);
    int lo = 0, hi = 33;                                                 // count(lo level) > number >= count(hi level)
    if (p.nseq == 1 && !BY_KEYS && number < __builtin_amdgcn_readlane(n, 0)) {      // one sequence: late tiles first
        w.s = 0;
        w.row = (__builtin_amdgcn_readlane(n, 0) - 1 - number) * R;
    } else {
        while (hi - lo > 1) {
            const int mid = lo + (hi - lo) / 2;
            if (__builtin_amdgcn_readlane(wave_scan(count(mid * level)), 63) > number) lo = mid; else hi = mid;
        }
        const int above = count((lo + 1) * level), sum_above = __builtin_amdgcn_readlane(wave_scan(above), 63);
        const int mine = count(lo * level) - above, upto = wave_scan(mine), r = number - sum_above;
        const unsigned long long after = __ballot(upto > r);             // first lane that reaches past r
        w.s = __builtin_amdgcn_readfirstlane(__ffsll(after) - 1);
        const int rank = above + r - (upto - mine);                      // in its sequence, by falling load
        w.row = __builtin_amdgcn_readlane(!BY_KEYS && p.causal ? n - 1 - rank : rank, w.s) * R;
    }
    w.ok = w.row >= 0 && w.row < __builtin_amdgcn_readlane(rows, w.s);       // (always, unless the table's entries fall)
    w.sq.q0 = __builtin_amdgcn_readlane(sq.q0, w.s);
    w.sq.lq = __builtin_amdgcn_readlane(sq.lq, w.s);
    w.sq.k0 = __builtin_amdgcn_readlane(sq.k0, w.s);
    w.sq.lk = __builtin_amdgcn_readlane(sq.lk, w.s);
    w.sq.kcap = __builtin_amdgcn_readlane(sq.kcap, w.s);
    return w;
}
// numbers that have to be launched: the exact count is only known on the device
__host__ __device__ inline int num_tiles(int nseq, int total, int R) { return total / R + nseq + 1; }

// Sums p V over keys k0 .. k1 - 1 without the matrix pipe, each query (lane pair) over the keys it sees and no others.  A product
// of a hidden key's probability, 0, with a NaN or an infinity in its V row would be NaN: where a sum is not finite, a causal
// wave redoes it with this.  Slow (a dot product a key), and only ever run on such input.
template <typename T, int DPAD>
__device__ __forceinline__ void sum_seen(f32x16 (&acc)[DPAD / 32], const typename Elem<T>::Frag (&qf)[DPAD / 16], const T* kbase, const T* vbase,
                                         const Params& p, int k0, int k1, int see, float base, int lane) {
    typedef T V4 __attribute__((ext_vector_type(4)));
    const int half = lane >> 5;
    for (int k = k0; k < k1; ++k) {
        typename Elem<T>::Frag kf[DPAD / 16];
        load_row_frags<T, DPAD>(kf, kbase + (int64_t)k * p.k_tok, true, p.dim, lane);
        float s = 0.f;
#pragma unroll
        for (int d = 0; d < DPAD / 16; ++d)
#pragma unroll
            for (int j = 0; j < 8; ++j) s = fmaf((float)qf[d][j], (float)kf[d][j], s);
        const float e = score_exp<T>(half_sum(s), p.scale_log2, base);
#pragma unroll
        for (int b = 0; b < DPAD / 32; ++b)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int d = b * 32 + r * 8 + half * 4;
                if (d >= p.dim) continue;
                const V4 v = *reinterpret_cast<const V4*>(vbase + (int64_t)k * p.v_tok + d);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    acc[b][r * 4 + i] = k < see ? fmaf(e, (float)v[i], acc[b][r * 4 + i]) : acc[b][r * 4 + i];
            }
    }
}
template <int N>
__device__ __forceinline__ bool finite_in_wave(const f32x16 (&acc)[N], bool present) {
    float x = 0.f;
#pragma unroll
    for (int b = 0; b < N; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) x = fmaf(acc[b][i], 0.f, x);
    return !__any(present && x != 0.f);              // (0 times an infinity or a NaN is NaN)
}

// Workgroup -> (tile number, kv head, head in group).  Workgroups go to the 8 XCDs in turn, each with an L2 of its own: an XCD
// gets whole kv heads where there are enough, else every X-th tile of one, so that K and V of a head are read into few L2s;
// within an XCD the heads of a group come next to each other.
struct Work { int number, kvh, g; };
__host__ __device__ inline int xcd_classes(int heads_k) { return heads_k % 8 == 0 ? 8 : heads_k % 4 == 0 ? 4 : heads_k % 2 == 0 ? 2 : 1; }
static inline int64_t work_blocks(int tiles, int heads_k, int inner) {
    const int g = xcd_classes(heads_k), x = 8 / g;
    return 8ll * ((tiles + x - 1) / x) * (heads_k / g) * inner;
}
__device__ __forceinline__ Work work_of(int block, int heads_k, int inner) {
    const int cls = xcd_classes(heads_k), x = 8 / cls, per = heads_k / cls;
    const int xcd = block & 7, j = block >> 3;
    Work w;
    w.g = j % inner;
    w.kvh = xcd % cls + cls * (j / inner % per);
    w.number = j / inner / per * x + xcd / cls;
    return w;
}

}  // namespace attn
