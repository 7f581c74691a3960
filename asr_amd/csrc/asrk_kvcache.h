// What the cache's page kernels and its attention share.
#pragma once
#include "asrk_common.h"

constexpr int ASRK_KV_EXP_MIN = -64, ASRK_KV_EXP_MAX = 119;

int asrk_kv_check(const asrk_kv_cache* c);
