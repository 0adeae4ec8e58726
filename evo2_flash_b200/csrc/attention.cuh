// The paged attention cache and the pieces of attention over it, shared by
// kvcache.cu, attention.cu (segments of few rows; joining) and
// attention_shared.cu (shared runs of many rows).
#pragma once

#include "tcgen05.cuh"

namespace hb {

int check_paged_kv(const hyena_paged_kv& kv);

namespace attn {

constexpr int KT = 16;  // a shared run is cut to whole tiles of this many keys

struct Params {
  hyena_paged_attention_args a;
  int groups;      // 0: nothing shared
  int per;         // query heads of one key/value head
  float scale;     // scale * log2(e)
  int slots_s, slots;  // pieces a row may have: of the shared run, of its own keys
  int tc;          // row tiles of the shared kernel, which takes the shared runs (0: none does)
  int planned;     // plan_kernel makes the plan; else each CTA its own
  int warps;       // of the stream kernel
  int ctas;        // of the shared kernel
  // the plan, in the workspace (where not `planned`, what the join kernel reads of it)
  int32_t* head;   // see Head
  int* shared;     // [groups] the shared runs
  int* leader;     // [groups] the requests whose page tables stand for them
  int* tc_first;   // [groups + 1] first items of the shared kernel
  int* first;      // [groups + requests + 1] first items of the stream kernel
  int4* info;      // [groups + requests], see Plan
  float2* ml;      // [T * heads][slots]: (m, l)
  float* o;        // [T * heads][slots][D]
};

enum Head {
  SHARED_TILES,  // KT-key tiles of a piece of a shared run
  CHUNK,         // and of a piece of own keys
  ITEMS,         // of the stream kernel
  NEXT,          // the item that its next free warp takes
  TC_TILES,      // 128-key tiles of an item of the shared kernel
  HEAD_INTS = 8
};

__device__ __forceinline__ int query_begin(const Params& P, int r) {
  return P.a.query_start_loc != nullptr ? __ldg(P.a.query_start_loc + r) : r;
}
// Queries of request r that exist, and their first row; `absent`: further ones that
// it claims beyond the T rows.
__device__ __forceinline__ int queries(const Params& P, int r, int& begin, int& absent) {
  begin = query_begin(P, r);
  const int claimed = query_begin(P, r + 1), end = claimed < P.a.T ? claimed : P.a.T;
  absent = claimed - end;
  return begin >= 0 && end > begin ? end - begin : 0;
}
// Whether query_start_loc gives request r no run of rows inside [0, T].
__device__ __forceinline__ bool bad_queries(const Params& P, int r) {
  if (P.a.query_start_loc == nullptr) return false;
  const int begin = query_begin(P, r), end = query_begin(P, r + 1);
  return begin < 0 || end < begin || end > P.a.T;
}
// Positions that a page table has.
__device__ __forceinline__ int capacity(const Params& P) {
  return P.a.kv.pages_per_request * P.a.kv.page_size;
}
// Keys of request r up to that of its last existing query, which may be more than its
// table has (those are not read): the queries' positions go by this length.
__device__ __forceinline__ int length(const Params& P, int r, int absent) {
  return max(max(__ldg(P.a.seq_lens + r), 0) - absent, 0);
}
// Group of request r, or -1.
__device__ __forceinline__ int group_of(const Params& P, int r) {
  if (P.groups == 0) return -1;
  if (P.a.group_start == nullptr) return 0;
  const int g = find_segment(P.a.group_start, P.groups, r);
  return __ldg(P.a.group_start + g) <= r && r < __ldg(P.a.group_start + g + 1) ? g : -1;
}
__device__ __forceinline__ int group_begin(const Params& P, int g) {
  int r = P.a.group_start != nullptr ? __ldg(P.a.group_start + g) : g == 0 ? 0 : P.a.num_requests;
  r = r < 0 ? 0 : r;
  return r < P.a.num_requests ? r : P.a.num_requests;
}
// Query rows of group g (tokens) and the first of them, inside [0, T).
__device__ __forceinline__ int group_queries(const Params& P, int g, int& begin) {
  begin = min(max(query_begin(P, group_begin(P, g)), 0), P.a.T);
  const int end = min(query_begin(P, group_begin(P, g + 1)), P.a.T);
  return end > begin ? end - begin : 0;
}
__host__ __device__ __forceinline__ int ceil_div(int a, int b) { return a / b + (a % b != 0); }

// The groups' shared runs and the requests whose page tables stand for them
// (leader), in shared memory: shared_lens cut to what every query of the group
// sees, then to whole KT-key tiles.  Padded requests (no keys) do not count.
template <int NTHREADS>
__device__ __forceinline__ void shared_runs(const Params& P, int* shared, int* leader) {
  const int G = P.groups, B = P.a.num_requests, tid = (int)threadIdx.x, cap = capacity(P);
  if (G == 0) return;
  for (int g = tid; g < G; g += NTHREADS) {
    const int n = __ldg(P.a.shared_lens + g);
    shared[g] = n < 0 ? 0 : n < cap ? n : cap;
    leader[g] = 0x7fffffff;
  }
  __syncthreads();
  for (int r = tid; r < B; r += NTHREADS) {
    int begin, absent;
    const int n = queries(P, r, begin, absent), len = length(P, r, absent), g = group_of(P, r);
    if (n > 0 && len > 0 && g >= 0) {
      atomicMin(&shared[g], max(len - n + 1, 0));
      atomicMin(&leader[g], r);
    }
  }
  __syncthreads();
  for (int g = tid; g < G; g += NTHREADS) shared[g] = leader[g] < B ? shared[g] & ~(KT - 1) : 0;
  __syncthreads();
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The kernels scale scores by a positive number after the maximum, where masked
// ones are -inf already: a negative scale's sign, or a zero scale, goes to the
// query (bf16 pairs: xor .x, and .y).
__device__ __forceinline__ uint2 query_sign(float scale) {
  return make_uint2(scale < 0.0f ? 0x80008000u : 0u, scale == 0.0f ? 0u : 0xffffffffu);
}
// ---------------------------------------------------------------- shared kernel
constexpr int TILE_KEYS = 128;
constexpr int ITEM_OVERHEAD = 3;  // tiles that an item's start and end cost

// Its part of the plan: the chunk length (in tiles) that lets its CTAs finish
// soonest, waves x (tiles of an item + its overhead) and the pieces to be joined,
// over the chunk counts of the longest run; then the groups' first items
// (first[groups]: their number).  Every thread of the CTA; thread 0 leaves first
// and the tiles of an item.
template <int NTHREADS>
__device__ __forceinline__ void plan_shared(const Params& P, const int* shared, int* first, int* tiles) {
  __shared__ unsigned long long best_s[NTHREADS / 32];
  const int tid = (int)threadIdx.x, G = P.groups, hkv = P.a.kv.kv_heads, rows_item = P.tc * 128;
  int longest = 0;
  for (int g = 0; g < G; ++g) longest = max(longest, shared[g]);
  const int most = ceil_div(longest, TILE_KEYS);
  // joining: a piece of every query row, there and back, in sixteenths of a tile's
  // time (some 13 MB of memory traffic for two row tiles, 8 MB for one)
  const unsigned long long piece =
      (unsigned long long)((long long)P.a.T * P.a.heads * (P.a.kv.head_dim + 2)) * 8 * 16 /
      (P.tc == 1 ? 8000000u : 13000000u);
  auto units = [&](int g) {
    int begin;
    return ceil_div(group_queries(P, g, begin) * P.per, rows_item) * hkv;
  };
  unsigned long long best = ~0ull;
  for (int c = tid + 1; c <= P.slots_s && c <= max(most, 1); c += NTHREADS) {
    const int n = max(ceil_div(most, c), 1);
    long long items = 0;
    for (int g = 0; g < G; ++g) items += (long long)units(g) * ceil_div(ceil_div(shared[g], TILE_KEYS), n);
    const unsigned long long waves = (unsigned long long)((items + P.ctas - 1) / P.ctas);
    const unsigned long long cost = 16 * waves * (unsigned long long)(n + ITEM_OVERHEAD) + c * piece;
    best = min(best, (cost << 24) | (unsigned long long)min(n, (1 << 24) - 1));
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) best = min(best, __shfl_xor_sync(0xffffffffu, best, d));
  if (tid % 32 == 0) best_s[tid / 32] = best;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < NTHREADS / 32; ++w) best = min(best, best_s[w]);
    const int n = (int)(best & 0xFFFFFFull);
    int at = 0;
    for (int g = 0; g < G; ++g) {
      first[g] = at;
      at += units(g) * ceil_div(ceil_div(shared[g], TILE_KEYS), n);
    }
    first[G] = at;
    *tiles = n;
  }
}

// O is rescaled when weights reach 2^RESCALE_LOG2: below it bf16 and fp32 round
// as well as at 1.
constexpr float RESCALE_LOG2 = 8.0f;
constexpr unsigned long long WAIT_NS = 4000000000ull;  // 4 s

static __device__ int g_wait_timeouts;  // one a source file

// Waits (bounded) for a phase; counts and flags an expired wait.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, int32_t* flags) {
  if (tc::mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = tc::now_ns();
  while (!tc::mbar_try_wait(bar, parity)) {
    if (tc::now_ns() - t0 > WAIT_NS) {
      atomicAdd(&g_wait_timeouts, 1);
      flag_error(flags, HYENA_FLAG_WAIT);
      return false;
    }
  }
  return true;
}

__device__ __forceinline__ void tma_load_4d(const CUtensorMap* map, uint64_t* bar, void* dst, int x,
                                            int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(tc::su32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(tc::su32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

static int read_wait_timeouts(int32_t* count, int reset) {
  int v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_wait_timeouts, sizeof(int));
  if (e == cudaSuccess && reset && v != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(g_wait_timeouts, &zero, sizeof(int));
  }
  if (e != cudaSuccess)
    return fail(HYENA_ERR_CUDA, std::string("attention wait counter: ") + cudaGetErrorString(e));
  *count = v;
  return HYENA_OK;
}

int cache_map(CUtensorMap* m, const hyena_paged_kv& kv, bool keys, int rows);

// Groups the tensor-core kernel of the shared runs takes (its plan's room).
constexpr int MAX_TC_GROUPS = 64;
int shared_launch(const Params& P, const CUtensorMap& k16, const CUtensorMap& v16, cudaStream_t st);
int shared_wait_timeouts(int32_t* count, int reset);

}  // namespace attn
}  // namespace hb
