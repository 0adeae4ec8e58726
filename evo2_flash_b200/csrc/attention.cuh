// The paged attention cache, shared by kvcache.cu and attention.cu.
#pragma once

#include "common.cuh"

namespace hb {

int check_paged_kv(const hyena_paged_kv& kv);

}  // namespace hb
