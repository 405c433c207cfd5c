// Launchers of the packed attention (one file each) and what they share with the C entries in attention.hip.
#pragma once
#include "attn_tile.h"

namespace attn {

// Dynamic LDS above 64 KiB has to be asked for, per kernel and device (a host-side attribute, fine under stream capture).
static inline int allow_lds(const void* kernel, int bytes) {
    if (bytes <= 65536) return 0;
    const hipError_t e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != hipSuccess) { sempyr_set_error("attention: %d bytes of LDS: %s", bytes, hipGetErrorString(e)); return (int)e; }
    return 0;
}

// Forward and dQ: queries of a workgroup, keys of a tile, tiles in the LDS ring.  A tile of 64 keys of heads up to 64 takes less
// time than its DMA: two tiles are kept in flight then.
constexpr int BM = 128, BN = 64;
template <typename T, int DPAD> constexpr int stages_of() { return sizeof(T) * DPAD <= 128 ? 3 : 2; }

// Few rows: query heads and queries packed into a tile's 32 columns, keys split (splits 0: the one-pass kernel is taken).
struct SplitPlan { int head_chunks, heads, queries, splits; };
SplitPlan plan_split(const Params& p);
int launch_split(int dtype, const Params& p, const SplitPlan& plan, float* ws, hipStream_t st);

int launch_fwd(int dtype, const Params& p, hipStream_t st);
int launch_bwd(int dtype, const Params& p, hipStream_t st);
}
