// What the cache's page kernels and its attention share.
#pragma once
#include "asrk_common.h"

constexpr int ASRK_KV_EXP_MIN = -64, ASRK_KV_EXP_MAX = 119;

int asrk_kv_check(const asrk_kv_cache* c);

__device__ __forceinline__ int larger(int a, int b) { return a > b ? a : b; }
__device__ __forceinline__ int wave_imax(int v) {  // v >= 0; shifts within rows of 16, then rows broadcast to later ones
    v = larger(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
    v = larger(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
    v = larger(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
    v = larger(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
    v = larger(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
    v = larger(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(v, 63);
}
