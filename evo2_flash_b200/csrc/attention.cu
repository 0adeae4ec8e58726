// Attention of a step's queries over the paged key/value cache, the leading keys
// that the requests of a group share read once for the group
// (hyena_paged_attention); the serving form of Evo2Attention's softmax
// attention (model.py:104-152).
//
// For a query at position p of a request, keys j = 0..p of its page table:
//   o = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),   s_j = scale q.k_j,  m = max_j s_j
// The keys are cut into pieces; a piece leaves (m, l = sum exp(s - m),
// O = sum exp(s - m) v), and pieces join exactly:
//   M = max m_i,  o = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i   (m in log2).
//
// Work.  A segment is either the shared keys of a group, seen by every query of
// its requests, or the own keys of one request; a unit is a segment x key/value
// head x 16-row tile (rows = queries x heads of one key/value head), and an item
// is `chunk` 16-key tiles of a unit.  A segment's items are ordered by position,
// then head, and warps take them one after the other: the warps of the GPU sweep
// through the cache together, a page's heads at about the same time.  (Giving each
// warp one long run of tiles instead evens the work out exactly, but spreads the
// warps over the whole cache: 343 us instead of 331 for 32 requests of up to 8000
// keys, items being taken in turn in both.)  A warp's loads run on across its
// items.  Every length is read on the device (one captured graph serves growing
// contexts), and the list of items with it, a prefix sum over segments: by
// plan_kernel, which the warps then ask for their next item (305 us for the 32
// requests: an SM that is further from the memory takes fewer), or, where the items
// are few, by each CTA, its warps taking them in turn.
//
// `shared_lens` says what may be read once, never what is seen: a group's
// shared run is cut to what every query of the group sees and to whole 16-key
// tiles, and the rest of it counts as own keys.  Runs of more than 16 rows a
// key/value head go to attention_shared.cu.
#include <algorithm>
#include <cmath>

#include "attention.cuh"

namespace hb {
namespace attn {

using namespace tc;

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int ROWS = 16;        // rows of a unit
constexpr int STAGES = 3;       // tiles in flight per warp
constexpr int QUEUE = 8;        // items between a warp's loads and its products, at most STAGES
constexpr int MIN_TILES = 2;     // tiles of an item at least
constexpr int ITEMS_PER_WARP = 8;  // that a warp should get
constexpr int MAX_SEGMENTS = 2048;
constexpr int TC_MIN_ROWS = 16;  // mean rows of a group and key/value head
// Without a shared kernel, plan_kernel plans from this many requests and bytes of keys
// and values (as many as their page tables can name) on, else each CTA for itself, its
// warps taking items in turn.  With the plan kernel and without, 32 heads: one request of
// 777 keys 16.7 and 10.5 us; 16 requests of 1024 keys (0.27 GB) 57 and 54 us, 8 of 4096
// (0.54 GB) 94 and 97 us, 8 of 8192 (1.07 GB) 171 and 178, 32 of up to 8000 (2.0 GB of
// keys, 4.2 GB that the tables can name) 305 and 337.  Tables that are half full lose at
// the border: 64 requests of up to 500 keys (0.54 GB) 58 and 53 us.
constexpr int PLANNED_REQUESTS = 5;
constexpr long long PLANNED_BYTES = 512ll << 20;

struct Plan {
  int chunk;   // tiles of an item
  int items;
  int* first;  // [groups + requests + 1] first item of a segment
  int4* info;  // [groups + requests]: first query, queries, keys, {leader | first own key}
  int* shared; // [groups] the shared run
  int* leader; // [groups] the request whose pages stand for it
};

constexpr int PLAN_BYTES = 28;  // of a segment, at most; and 4
// A plan of n segments, G of them groups, at p (16-byte aligned).
__device__ __forceinline__ Plan plan_at(uint8_t* p, int G, int n) {
  Plan L;
  L.chunk = L.items = 0;
  L.info = reinterpret_cast<int4*>(p);
  L.first = reinterpret_cast<int*>(L.info + n);
  L.shared = L.first + n + 1;
  L.leader = L.shared + G;
  return L;
}

__device__ __forceinline__ int row_tiles(const Params& P, int nq) {
  return (int)(((long long)nq * P.per + ROWS - 1) / ROWS);
}
// Tiles of a unit of an own segment.  A request with queries has a tile even
// without keys: its rows are written there.
__device__ __forceinline__ int own_tiles(const Params& P, int len, int k_begin) {
  return max(ceil_div(max(min(len, capacity(P)) - k_begin, 0), KT), 1);
}

// Every thread of the CTA.
template <int NTHREADS>
__device__ void make_plan(const Params& P, Plan& L) {
  constexpr int W = NTHREADS / 32;
  __shared__ long long wsum[W];
  __shared__ int wlong[W], wfirst[W];
  const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = P.groups, n = G + P.a.num_requests;
  shared_runs<NTHREADS>(P, L.shared, L.leader);
  // a thread takes a run of consecutive segments
  const int per = ceil_div(n, NTHREADS);
  const int s0 = min(tid * per, n), s1 = min(s0 + per, n);
  auto tiles_of = [&](int s, const int4& x) { return s < G ? x.z / KT : own_tiles(P, x.z, x.w); };
  long long work = 0;
  int longest = 0;
  for (int s = s0; s < s1; ++s) {
    int4 x;
    if (s < G) {
      x.y = P.tc ? 0 : group_queries(P, s, x.x);
      x.z = L.shared[s];
      x.w = L.leader[s];
    } else {
      const int r = s - G, g = group_of(P, r);
      int absent;
      x.y = queries(P, r, x.x, absent);
      x.z = length(P, r, absent);
      x.w = g >= 0 && x.z > 0 ? L.shared[g] : 0;
    }
    L.info[s] = x;
    const int units = row_tiles(P, x.y) * P.a.kv.kv_heads, tiles = tiles_of(s, x);
    work += (long long)tiles * units;
    if (units > 0) longest = max(longest, tiles);
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) work += __shfl_xor_sync(0xffffffffu, work, d);
  longest = __reduce_max_sync(0xffffffffu, longest);
  if (lane == 0) {
    wsum[warp] = work;
    wlong[warp] = longest;
  }
  __syncthreads();
  work = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    work += wsum[w];
    longest = max(longest, wlong[w]);
  }
  // Some ITEMS_PER_WARP items a warp, for balance; but an item has its start and
  // leaves a piece to be joined (each of its rows 8 D bytes there and back, as much
  // as D / 16 of a tile), so not below 8 tiles and one for each of its rows while
  // every warp still gets one; at most P.slots items a unit.
  const int warps = P.warps;
  const long long even = (work + (long long)warps * ITEMS_PER_WARP - 1) / ((long long)warps * ITEMS_PER_WARP);
  const long long each = (work + warps - 1) / warps;
  const int mean_rows = min(P.a.T / max(P.a.num_requests, 1) * P.per, ROWS);
  const long long few = min(each, (long long)(8 + mean_rows));
  L.chunk = (int)max(max(even, few), (long long)max(ceil_div(longest, P.slots), MIN_TILES));
  int sum = 0;
  for (int s = s0; s < s1; ++s) {
    const int4 x = L.info[s];
    L.first[s] = sum;
    sum += ceil_div(tiles_of(s, x), L.chunk) * row_tiles(P, x.y) * P.a.kv.kv_heads;
  }
  int scan = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += x;
  }
  if (lane == 31) wfirst[warp] = scan;
  __syncthreads();
  int at = scan - sum, total = 0;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    if (w < warp) at += wfirst[w];
    total += wfirst[w];
  }
  for (int s = s0; s < s1; ++s) L.first[s] += at;
  if (tid == 0) L.first[n] = total;
  L.items = total;
  __syncthreads();
}

// The plan in a kernel of its own: one CTA instead of every CTA of the stream
// kernel, and the counter from which that kernel's warps then take their items (an
// SM that is far from its memory, or busy with the shared kernel, takes fewer).
constexpr int PLAN_THREADS = 256;
__global__ void __launch_bounds__(PLAN_THREADS) plan_kernel(const __grid_constant__ Params P) {
  extern __shared__ __align__(16) uint8_t smem_raw[];
  const int tid = (int)threadIdx.x, G = P.groups, n = G + P.a.num_requests;
  pdl_entry();
  Plan L = plan_at(smem_raw, G, n);
  make_plan<PLAN_THREADS>(P, L);
  for (int i = tid; i <= n; i += PLAN_THREADS) {
    P.first[i] = L.first[i];
    if (i < n) P.info[i] = L.info[i];
    if (i < G) P.shared[i] = L.shared[i];
    if (i < G) P.leader[i] = L.leader[i];
  }
  if (tid == 0) {
    P.head[SHARED_TILES] = P.head[CHUNK] = L.chunk;
    P.head[ITEMS] = L.items;
    P.head[NEXT] = 0;
  }
  if (P.tc) {
    plan_shared<PLAN_THREADS>(P, L.shared, P.tc_first, P.head + TC_TILES);
    if (threadIdx.x == 0) P.head[SHARED_TILES] = P.head[TC_TILES] * (TILE_KEYS / KT);
  }
}

// ---------------------------------------------------------------- fragments
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, "
      "{%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int D>
struct Layout {
  static constexpr int HALVES = D / 64;         // 64-column swizzled halves of a row
  static constexpr int HALF = KT * 128;         // bytes of a half's tile
  static constexpr int TILE = HALVES * HALF;    // one operand's tile
  static constexpr int STAGE = 2 * TILE;        // keys, then values
  static constexpr int RING = STAGES * STAGE;   // a warp's ring
  static constexpr int PLAN = WARPS * RING;     // the plan follows
};
// Byte offset of 16-byte chunk c of row `row` in a tile as TMA leaves it
// (SWIZZLE_128B halves): eight rows' same chunk, an ldmatrix phase, lies in
// distinct banks.
__device__ __forceinline__ uint32_t tile_at(int row, int c) {
  return uint32_t((c >> 3) * (KT * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4));
}

__device__ __forceinline__ uint32_t query_word(const bf16* p, uint2 sign) {
  return (*reinterpret_cast<const uint32_t*>(p) ^ sign.x) & sign.y;
}

// An item as a warp meets it (all warp-uniform).
struct Item {
  int seg, index;    // its segment; which chunk of its unit it is
  int n;             // its tiles
  int request, head, begin, rows, row0, nq, len;
  int k0, k1;        // its keys [k0, k1): those some row sees
  int all_see;       // keys below it are seen by every row
  bool only;         // the only piece of its rows
};
__device__ __forceinline__ Item item_at(const Params& P, const Plan& L, int item, int seg) {
  Item I;
  const int G = P.groups;
  if (seg < 0 || item >= L.first[seg + 1]) {
    int lo = seg < 0 ? 0 : seg + 1, hi = G + P.a.num_requests;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (L.first[mid] <= item) lo = mid; else hi = mid;
    }
    seg = lo;
  }
  I.seg = seg;
  const int4 x = L.info[seg];
  const bool own = seg >= G;
  I.begin = x.x;
  I.nq = x.y;
  I.len = x.z;
  I.rows = x.y * P.per;
  I.request = own ? seg - G : x.w;
  const int first_key = own ? x.w : 0, tiles = own ? own_tiles(P, x.z, x.w) : x.z / KT;
  const int tiles_r = ceil_div(I.rows, ROWS), units = tiles_r * P.a.kv.kv_heads;
  const int rem = item - L.first[seg];
  I.index = rem / units;
  const int v = rem - I.index * units;
  I.head = v / tiles_r;
  I.row0 = (v - I.head * tiles_r) * ROWS;
  I.n = min(L.chunk, tiles - I.index * L.chunk);
  I.only = own && x.w == 0 && tiles <= L.chunk;
  I.k0 = first_key + I.index * L.chunk * KT;
  I.k1 = I.all_see = min(min(x.z, capacity(P)), I.k0 + I.n * KT);
  if (own) {
    const int last = min(I.nq - 1, (I.row0 + ROWS - 1) / P.per);
    I.k1 = min(I.k1, I.len - I.nq + last + 1);
    I.all_see = min(I.k1, I.len - I.nq + I.row0 / P.per + 1);
  }
  return I;
}

// A warp walks its tiles with its own ring, maximum, sum and O; no barrier after
// the plan.  The 16 rows of a tensor-core tile are mostly padding for one token
// and ungrouped heads (rows 8-15 are skipped in the softmax where a unit has
// none); the kernel is bound by the keys' bytes as long as the some 130
// instructions of an 8 KB tile stay well under the 2850 cycles that an SM's share
// of HBM gives each of its eight warps for it.  Hence TMA (four instructions a
// tile), masks only in the tiles that need them, and a maximum that is compared
// by one vote: m moves, and O is rescaled, only when a score exceeds it by 2^8
// (the weights stay below 2^8, where bf16 and fp32 round as well as at 1).
template <int D, bool PLANNED>
__global__ void __launch_bounds__(THREADS, 2)
stream_kernel(const __grid_constant__ Params P, const __grid_constant__ CUtensorMap map_k,
              const __grid_constant__ CUtensorMap map_v) {
  using LT = Layout<D>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full_s[WARPS][STAGES];
  __shared__ int queue_s[WARPS][PLANNED ? QUEUE : 1];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~uintptr_t(1023));
  const hyena_paged_attention_args& A = P.a;
  const hyena_paged_kv& kv = A.kv;
  const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = P.groups, B = A.num_requests;
  uint64_t* full = full_s[warp];
  if (lane == 0) {
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (tid == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_k)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_v)) : "memory");
  }
  if (PLANNED && P.tc == 2)
    pdl_trigger();  // the plan is complete: see attention_shared.cu
  else
    pdl_entry();
  Plan L = plan_at(smem + LT::PLAN, G, G + B);
  if (PLANNED) {
    for (int i = tid; i <= G + B; i += THREADS) {
      L.first[i] = __ldcg(P.first + i);
      if (i < G + B) L.info[i] = __ldcg(P.info + i);
    }
    L.chunk = __ldcg(P.head + CHUNK);
    L.items = __ldcg(P.head + ITEMS);
    __syncthreads();
  } else {
    make_plan<THREADS>(P, L);
    if (blockIdx.x == 0) {  // for the join
      if (tid == 0 && !P.tc) P.head[SHARED_TILES] = L.chunk;
      if (tid == 0) P.head[CHUNK] = L.chunk;
      for (int g = tid; g < G; g += THREADS) P.shared[g] = L.shared[g];
    }
  }
  uint8_t* ring = smem + warp * LT::RING;
  const uint32_t ring_u = su32(ring);
  const int g8 = lane >> 2, t4 = lane & 3;
  // Items in turn; or from the counter, the next one asked for when the loads of one
  // begin, and a queue that passes them on from the loads to the products.
  int* queue = queue_s[warp];
  const int first = (int)blockIdx.x * WARPS + warp;
  int asked = 0;
  auto ask = [&]() {
    if (lane == 0) asked = atomicAdd(P.head + NEXT, 1);
  };
  if (PLANNED) ask();
  int next = PLANNED ? __shfl_sync(0xffffffffu, asked, 0) : first;
  if (next >= L.items) {
    if (PLANNED && P.tc == 2) pdl_wait();
    return;
  }
  if (PLANNED) {
    if (lane == 0) queue[0] = next;
    ask();
  }

  // ---- loads, STAGES - 1 tiles ahead; a lane holds the page of one of 32
  // consecutive page-table entries
  Item N = item_at(P, L, next, -1);  // the item being loaded
  int loaded = 0, tile = 0, page_at = 0, page_index = 0, window = -64, window_of = -1, pages = 0;
  uint32_t bad = 0;  // stages whose page is out of range
  int load_stage = 0;
  page_index = N.k0 / kv.page_size;
  page_at = N.k0 - page_index * kv.page_size;
  auto load = [&]() {
    if (next >= L.items) return;
    const int s = load_stage;
    load_stage = s + 1 == STAGES ? 0 : s + 1;
    if (N.k0 + tile * KT < N.k1) {
      if (window_of != N.request || page_index < window || page_index >= window + 32) {
        window = page_index;
        window_of = N.request;
        pages = __ldg(kv.page_table + (long long)N.request * kv.page_table_stride +
                      min(page_index + lane, kv.pages_per_request - 1));
      }
      const int page = __shfl_sync(0xffffffffu, pages, page_index - window);
      const bool ok = page >= 0 && page < kv.num_pages;
      bad = ok ? bad & ~(1u << s) : bad | (1u << s);
      if (lane == 0) {
        if (ok) {
          uint8_t* dst = ring + s * LT::STAGE;
          mbar_expect_tx(&full[s], LT::STAGE);
#pragma unroll
          for (int h = 0; h < LT::HALVES; ++h) {
            tma_load_4d(&map_k, &full[s], dst + h * LT::HALF, h * 64, page_at, N.head, page);
            tma_load_4d(&map_v, &full[s], dst + LT::TILE + h * LT::HALF, h * 64, page_at, N.head, page);
          }
        } else {
          flag_error(A.error_flags, HYENA_FLAG_BLOCK_RANGE);
          mbar_arrive(&full[s]);
        }
      }
      page_at += KT;
      if (page_at == kv.page_size) {
        page_at = 0;
        ++page_index;
      }
    } else if (lane == 0) {
      mbar_arrive(&full[s]);  // nothing to load: the phase completes by itself
    }
    if (++tile == N.n) {
      tile = 0;
      if (PLANNED) {
        next = __shfl_sync(0xffffffffu, asked, 0);
        if (lane == 0) queue[++loaded % QUEUE] = next;
      } else {
        next += P.warps;
      }
      if (next < L.items) {
        if (PLANNED) ask();
        N = item_at(P, L, next, N.seg);
        page_index = N.k0 / kv.page_size;
        page_at = N.k0 - page_index * kv.page_size;
      }
    }
  };
#pragma unroll 1
  for (int i = 0; i < STAGES - 1; ++i) load();

  const float scale = P.scale == 0.0f ? 1.0f : fabsf(P.scale);
  const uint2 sign = query_sign(P.scale);
  uint32_t qf[D / 16][4];
  float o[D / 8][4], m[2], l[2];
  int s = 0, seg = -1;
  uint32_t parity = 0;
#pragma unroll 1
  for (int k = 0;; ++k) {
    if (PLANNED) __syncwarp();
    const int item = PLANNED ? queue[k % QUEUE] : first + k * P.warps;
    if (item >= L.items) break;
    const Item U = item_at(P, L, item, seg);
    seg = U.seg;
    const bool two = U.rows - U.row0 > 8;  // rows 8-15 exist
    // ---- this lane's two rows (g8, g8 + 8) as mma A fragments
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = U.row0 + g8 + 8 * i;
      const bf16* src = nullptr;
      if (row < U.rows) {
        const int qi = row / P.per;
        src = static_cast<const bf16*>(A.q) + (long long)(U.begin + qi) * A.q_token_stride +
              (long long)(U.head * P.per + row - qi * P.per) * A.q_head_stride;
      }
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[ks][i] =
            src != nullptr ? query_word(src + ks * 16 + t4 * 2, sign) : 0u;
        qf[ks][2 + i] =
            src != nullptr ? query_word(src + ks * 16 + 8 + t4 * 2, sign) : 0u;
      }
      m[i] = -INFINITY;
      l[i] = 0.0f;
    }
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;

#pragma unroll 1
    for (int i_tile = 0; i_tile < U.n; ++i_tile) {
      load();
      const int kpos = U.k0 + i_tile * KT;
      if (!__all_sync(0xffffffffu, wait(&full[s], parity, A.error_flags))) {
        // gave up: what else was issued lands (waits bounded too) before the warp leaves
        for (int k = 1; k < STAGES; ++k) {
          if (++s == STAGES) {
            s = 0;
            parity ^= 1u;
          }
          if (s != load_stage) wait(&full[s], parity, A.error_flags);
        }
        if (PLANNED && P.tc == 2) pdl_wait();
        return;
      }
      if (kpos < U.k1 && !((bad >> s) & 1u)) {
        const uint32_t ks_u = ring_u + uint32_t(s * LT::STAGE), vs_u = ks_u + LT::TILE;
        // scores of 16 rows x 16 keys
        float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          uint32_t b[4];  // keys 0-7 (k 0-7, 8-15), keys 8-15 (k 0-7, 8-15)
          ldsm4(ks_u + tile_at((lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)), b);
          mma_bf16(sc[0], qf[ks], b[0], b[1]);
          mma_bf16(sc[1], qf[ks], b[2], b[3]);
        }
        const bool partial = kpos + KT > U.all_see;  // some row does not see some key of the tile
        if (partial) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = U.row0 + g8 + 8 * i;
            int end = U.k1 - kpos;  // keys of the tile this row sees
            if (U.seg >= G && row < U.rows) end = min(end, U.len - U.nq + row / P.per + 1 - kpos);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int key = (e >> 1) * 8 + t4 * 2 + (e & 1);
              if (key >= end) sc[e >> 1][i * 2 + (e & 1)] = -INFINITY;
            }
          }
        }
        float top[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
          top[i] = fmaxf(fmaxf(sc[0][i * 2], sc[0][i * 2 + 1]), fmaxf(sc[1][i * 2], sc[1][i * 2 + 1])) * scale;
        bool grow = top[0] > m[0] + RESCALE_LOG2;
        if (two) grow = grow || top[1] > m[1] + RESCALE_LOG2;
        if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float x = top[i] == top[i] ? top[i] : -INFINITY;
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
            if (x > m[i] + RESCALE_LOG2) {  // by the row alone
              const float keep = exp2_approx(m[i] - x);
              m[i] = x;
              l[i] *= keep;
#pragma unroll
              for (int n = 0; n < D / 8; ++n) {
                o[n][i * 2] *= keep;
                o[n][i * 2 + 1] *= keep;
              }
            }
          }
        }
        // The weights are rounded to bf16 for the product, as the values are; l
        // sums them before that rounding, which is unbiased.
        float p[2][4];
        uint32_t pa[4] = {0u, 0u, 0u, 0u};
        auto weights = [&](int i) {
          const float base = m[i] == -INFINITY ? 0.0f : m[i];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            p[e >> 1][i * 2 + (e & 1)] = exp2_approx(fmaf(sc[e >> 1][i * 2 + (e & 1)], scale, -base));
          l[i] += (p[0][i * 2] + p[0][i * 2 + 1]) + (p[1][i * 2] + p[1][i * 2 + 1]);
          pa[i] = as_u32(pack2_rn(make_float2(p[0][i * 2], p[0][i * 2 + 1])));
          pa[2 + i] = as_u32(pack2_rn(make_float2(p[1][i * 2], p[1][i * 2 + 1])));
        };
        weights(0);
        if (two) weights(1);
        if (partial) {
          // Keys that some row of the tile does not see (a later token of the same
          // step, or beyond the last): those that another row sees are added row by
          // row, so that a masked value, whatever it holds, meets no product; then
          // zeros take their place for the mma.
          const int j0 = max(U.all_see - kpos, 0), j1 = min(U.k1 - kpos, KT);
          uint8_t* vt = ring + s * LT::STAGE + LT::TILE;
          for (int j = j0; j < j1; ++j) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (i == 1 && !two) continue;
              const uint32_t pw0 = __shfl_sync(0xffffffffu, __float_as_uint(j < 8 ? p[0][i * 2] : p[1][i * 2]),
                                               (lane & ~3) | ((j & 7) >> 1));
              const uint32_t pw1 = __shfl_sync(
                  0xffffffffu, __float_as_uint(j < 8 ? p[0][i * 2 + 1] : p[1][i * 2 + 1]),
                  (lane & ~3) | ((j & 7) >> 1));
              const float w = __uint_as_float(j & 1 ? pw1 : pw0);
              const int row = U.row0 + g8 + 8 * i;
              if (row < U.rows && kpos + j < U.len - U.nq + row / P.per + 1) {
#pragma unroll
                for (int n = 0; n < D / 8; ++n) {
                  const float2 v = unpack2(*reinterpret_cast<const bf162*>(vt + tile_at(j, n) + t4 * 4));
                  o[n][i * 2] = fmaf(w, v.x, o[n][i * 2]);
                  o[n][i * 2 + 1] = fmaf(w, v.y, o[n][i * 2 + 1]);
                }
              }
            }
          }
          __syncwarp();
          for (int c = lane; c < (KT - j0) * (D / 8); c += 32)
            *reinterpret_cast<uint4*>(vt + tile_at(j0 + c / (D / 8), c % (D / 8))) = make_uint4(0u, 0u, 0u, 0u);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // before TMA fills the stage again
          __syncwarp();
          const int key = t4 * 2;
          const uint32_t lo0 = key < j0 ? 0xFFFFu : 0u, hi0 = key + 1 < j0 ? 0xFFFF0000u : 0u;
          const uint32_t lo1 = key + 8 < j0 ? 0xFFFFu : 0u, hi1 = key + 9 < j0 ? 0xFFFF0000u : 0u;
          pa[0] &= lo0 | hi0;
          pa[1] &= lo0 | hi0;
          pa[2] &= lo1 | hi1;
          pa[3] &= lo1 | hi1;
        }
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          uint32_t b[4];  // values of keys 0-7 and 8-15, columns 16n + 0-7 then 16n + 8-15
          ldsm4_trans(vs_u + tile_at(lane & 15, n * 2 + (lane >> 4)), b);
          mma_bf16(o[2 * n], pa, b[0], b[1]);
          mma_bf16(o[2 * n + 1], pa, b[2], b[3]);
        }
      }
      __syncwarp();  // the stage is read before it is filled again
      if (++s == STAGES) {
        s = 0;
        parity ^= 1u;
      }

    }
    // ---- the piece is complete
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      const int row = U.row0 + g8 + 8 * i;
      if (row >= U.rows) continue;
      const int qi = row / P.per;
      const long long token = U.begin + qi;
      const int head = U.head * P.per + row - qi * P.per;
      if (U.only) {
        const float inv = l[i] > 0.0f || l[i] != l[i] ? 1.0f / l[i] : 0.0f;
        bf16* dst = static_cast<bf16*>(A.out) + token * A.out_token_stride +
                    (long long)head * A.out_head_stride + t4 * 2;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<uint32_t*>(dst + n * 8) =
              as_u32(pack2_rn(make_float2(o[n][i * 2] * inv, o[n][i * 2 + 1] * inv)));
      } else {
        const long long slot = (token * A.heads + head) * (P.slots_s + P.slots) +
                               (U.seg >= G ? P.slots_s : 0) + U.index;
        if (t4 == 0) P.ml[slot] = make_float2(m[i], l[i]);
        float* dst = P.o + slot * D + t4 * 2;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float2*>(dst + n * 8) = make_float2(o[n][i * 2], o[n][i * 2 + 1]);
      }
    }
  }
  if (PLANNED && P.tc == 2) pdl_wait();  // the shared kernel: the join waits for this one alone
}

// Flags token ranges that are not inside the rows, and lengths beyond the page table.
// (A block of the join's own does it.  In the stream kernel, in every block's plan or
// after one block's, one request of 777 keys takes 10.5 us instead of 9.9.)
__device__ __forceinline__ void flag_ranges(const Params& P) {
  for (int r = (int)threadIdx.x; r < P.a.num_requests; r += THREADS) {
    int begin, absent;
    if (queries(P, r, begin, absent) > 0 && length(P, r, absent) > capacity(P))
      flag_error(P.a.error_flags, HYENA_FLAG_BLOCK_RANGE);
    if (bad_queries(P, r)) flag_error(P.a.error_flags, HYENA_FLAG_SEGMENT);
  }
}
// Out of the way of the code that few rows wait for: one request 9.9 us, inlined 10.1
// (many rows: inlined 90.6 us for 3 prompts being verified, called 91.2).
__device__ __noinline__ void flag_ranges_call(const Params& P) { flag_ranges(P); }

// Joins the pieces of the rows that have more than one: a warp a row, or
// (WPR = 4) the four warps of a block, for few rows of many pieces.
// One block more flags what is wrong with the call's ranges.
template <int D, int WPR>
__global__ void __launch_bounds__(THREADS) join_kernel(const __grid_constant__ Params P) {
  constexpr int E = D / 32;
  __shared__ float red[WPR][D + 2];
  pdl_entry();
  const hyena_paged_attention_args& A = P.a;
  const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
  const long long row = WPR == 1 ? (long long)blockIdx.x * WARPS + warp : (long long)blockIdx.x;
  const int part = WPR == 1 ? 0 : warp;
  if (row >= (long long)A.T * A.heads) {
    if (blockIdx.x + 1 == gridDim.x) {
      if constexpr (WPR == 1) flag_ranges(P);
      else flag_ranges_call(P);
    }
    return;
  }
  const int token = (int)(row / A.heads), head = (int)(row % A.heads);
  int r = token;
  if (A.query_start_loc != nullptr) {
    r = find_segment(A.query_start_loc, A.num_requests, token);
    if (token < __ldg(A.query_start_loc + r) || token >= __ldg(A.query_start_loc + r + 1)) return;
  } else if (r >= A.num_requests) {
    return;
  }
  int begin, absent;
  queries(P, r, begin, absent);
  const int g = group_of(P, r), len = length(P, r, absent);
  // (through L1: read from L2 by every warp, these words cost 4 us of 85)
  const int sh = g >= 0 && len > 0 ? P.shared[g] : 0;
  const int ns = sh > 0 ? ceil_div(sh / KT, P.head[SHARED_TILES]) : 0;
  const int no = ceil_div(own_tiles(P, len, sh), P.head[CHUNK]);
  if (ns == 0 && no == 1) return;  // written already
  // The statistics of 32 pieces at a time, a lane each; then their O, whose weights
  // are known by then, so that UNROLL loads are on their way at once (one request of
  // 777 keys 10.1 us, 11.5 with a piece after the other; a warp that has a row alone
  // usually finds few pieces: 4 at once 91.5 us for 3 prompts being verified, 8 92.3).
  constexpr int UNROLL = WPR == 1 ? 4 : 8;
  const int n = ns + no;
  const long long base = row * (P.slots_s + P.slots);
  auto slot_of = [&](int i) { return base + (i < ns ? i : P.slots_s + i - ns); };
  float m = -INFINITY, l = 0.0f, acc[E];
#pragma unroll
  for (int j = 0; j < E; ++j) acc[j] = 0.0f;
  for (int i0 = part; i0 < n; i0 += 32 * WPR) {
    const int mine = i0 + lane * WPR;
    const float2 x = mine < n ? P.ml[slot_of(mine)] : make_float2(-INFINITY, 0.0f);
    float mx = fmaxf(m, x.x);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
    const float b = mx == -INFINITY ? 0.0f : mx;
    const float keep = exp2_approx(m - b), w = exp2_approx(x.x - b);
    float sum = w * x.y;
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    m = mx;
    l = l * keep + sum;
#pragma unroll
    for (int j = 0; j < E; ++j) acc[j] *= keep;
    for (int k = 0; k < 32 && i0 + k * WPR < n; k += UNROLL) {
      float v[UNROLL][E];
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const int i = i0 + (k + u) * WPR;
        const float* src = P.o + slot_of(i) * D + lane * E;
        if constexpr (E == 4) {
          const float4 y = i < n ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
          v[u][0] = y.x; v[u][1] = y.y; v[u][2] = y.z; v[u][3] = y.w;
        } else {
          const float2 y = i < n ? *reinterpret_cast<const float2*>(src) : make_float2(0.f, 0.f);
          v[u][0] = y.x; v[u][1] = y.y;
        }
      }
#pragma unroll
      for (int u = 0; u < UNROLL; ++u) {
        const float wu = __shfl_sync(0xffffffffu, w, k + u);
#pragma unroll
        for (int j = 0; j < E; ++j) acc[j] = fmaf(wu, v[u][j], acc[j]);
      }
    }
  }
  if constexpr (WPR > 1) {
    if (lane == 0) {
      red[warp][D] = m;
      red[warp][D + 1] = l;
    }
#pragma unroll
    for (int j = 0; j < E; ++j) red[warp][lane * E + j] = acc[j];
    __syncthreads();
    if (warp != 0) return;
    float mx = -INFINITY;
    for (int w = 0; w < WPR; ++w) mx = fmaxf(mx, red[w][D]);
    const float b = mx == -INFINITY ? 0.0f : mx;
    l = 0.0f;
#pragma unroll
    for (int j = 0; j < E; ++j) acc[j] = 0.0f;
    for (int w = 0; w < WPR; ++w) {
      const float k = exp2_approx(red[w][D] - b);
      l += k * red[w][D + 1];
#pragma unroll
      for (int j = 0; j < E; ++j) acc[j] = fmaf(k, red[w][lane * E + j], acc[j]);
    }
  }
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
  bf16* dst = static_cast<bf16*>(A.out) + (long long)token * A.out_token_stride +
              (long long)head * A.out_head_stride + lane * E;
  const uint32_t lo2 = as_u32(pack2_rn(make_float2(acc[0] * inv, acc[1] * inv)));
  if constexpr (E == 4) {
    const uint32_t hi2 = as_u32(pack2_rn(make_float2(acc[2] * inv, acc[3] * inv)));
    *reinterpret_cast<uint2*>(dst) = make_uint2(lo2, hi2);
  } else {
    *reinterpret_cast<uint32_t*>(dst) = lo2;
  }
}

// ---------------------------------------------------------------- host side
int wait_timeouts(int32_t* count, int reset) {
  int n = 0;
  const int rc = read_wait_timeouts(&n, reset);
  return rc ? rc : shared_wait_timeouts(count, reset) ? HYENA_ERR_CUDA : (*count += n, HYENA_OK);
}

// (head_dim, token in page, head, page) over a cache; box: `rows` tokens of one
// page and head, 64 columns.
int cache_map(CUtensorMap* m, const hyena_paged_kv& kv, bool keys, int rows) {
  auto fn = encode_fn();
  if (fn == nullptr) return fail(HYENA_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
  const int64_t page = keys ? kv.k_page_stride : kv.v_page_stride;
  const int64_t token = keys ? kv.k_token_stride : kv.v_token_stride;
  const int64_t head = keys ? kv.k_head_stride : kv.v_head_stride;
  // the stride of a dimension of one is never used; give it a valid one
  cuuint64_t dims[4] = {(cuuint64_t)kv.head_dim, (cuuint64_t)kv.page_size, (cuuint64_t)kv.kv_heads,
                        (cuuint64_t)kv.num_pages};
  cuuint64_t strides[3] = {(cuuint64_t)token * 2, (cuuint64_t)(kv.kv_heads > 1 ? head : 8) * 2,
                           (cuuint64_t)(kv.num_pages > 1 ? page : 8) * 2};
  cuuint32_t boxes[4] = {64, (cuuint32_t)rows, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, keys ? kv.k : kv.v, dims, strides, boxes,
                        estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(HYENA_ERR_CUDA, "cuTensorMapEncodeTiled(cache) failed");
  return HYENA_OK;
}

// Pieces a row may have, from sizes the host knows: enough that one segment
// alone spreads over the GPU (8 pieces an SM over the key/value heads), bounded
// by what its pages can hold and by the workspace.
struct Slots {
  int s, o;
  size_t header, bytes;
};
constexpr size_t WORKSPACE_BYTES = size_t(256) << 20;

static Slots slots_of(const hyena_paged_attention_args& A) {
  const bool shared = A.shared_lens != nullptr;
  const long long rows = (long long)A.T * A.heads;
  const long long row_bytes = (A.kv.head_dim + 2) * 4;
  const long long keys = (long long)A.kv.pages_per_request * A.kv.page_size;
  long long n = (8ll * num_sms() + A.kv.kv_heads - 1) / A.kv.kv_heads;
  n = std::min(n, (keys + MIN_TILES * KT - 1) / (MIN_TILES * KT));
  n = std::min(n, (long long)WORKSPACE_BYTES / (rows * row_bytes * (shared ? 2 : 1)));
  n = std::max(n, 1ll);
  Slots S;
  S.o = (int)n;
  S.s = shared ? (int)n : 0;
  const size_t G = A.num_groups, R = A.num_requests;
  S.header = (4 * (HEAD_INTS + 3 * G + 1 + G + R + 1) + 15) / 16 * 16 + 16 * (G + R);  // the plan
  S.header = (S.header + 255) & ~size_t(255);
  S.bytes = S.header + (size_t)(rows * (S.s + S.o)) * row_bytes;
  return S;
}

static int check(const hyena_paged_attention_args& A) {
  HB_REQUIRE(A.T >= 0 && A.num_requests >= 0, "paged_attention: negative sizes");
  if (A.T == 0 || A.num_requests == 0) return HYENA_OK;
  const int rc = check_paged_kv(A.kv);
  if (rc) return rc;
  HB_REQUIRE(A.q && A.out && A.seq_lens, "paged_attention: null pointer");
  HB_REQUIRE(A.heads > 0 && A.heads % A.kv.kv_heads == 0,
             "paged_attention: heads must be a multiple of kv_heads");
  HB_REQUIRE(aligned16(A.q) && aligned16(A.out), "paged_attention: q and out must be 16-byte aligned");
  HB_REQUIRE(A.q_token_stride % 8 == 0 && A.q_head_stride % 8 == 0 && A.out_token_stride % 8 == 0 &&
                 A.out_head_stride % 8 == 0,
             "paged_attention: strides must be multiples of 8 elements");
  HB_REQUIRE(std::isfinite(A.scale), "paged_attention: scale must be finite");
  HB_REQUIRE((A.shared_lens != nullptr) == (A.num_groups > 0),
             "paged_attention: shared_lens and num_groups go together");
  HB_REQUIRE(A.group_start != nullptr || A.num_groups <= 1,
             "paged_attention: several groups need group_start");
  HB_REQUIRE(A.num_groups >= 0 && (long long)A.num_requests + A.num_groups <= MAX_SEGMENTS,
             "paged_attention: at most 2048 requests and groups");
  HB_REQUIRE((long long)A.T * A.heads < (1ll << 31), "paged_attention: too many query rows");
  return HYENA_OK;
}

template <int D>
static int launch(const hyena_paged_attention_args& A, const Slots& S, void* ws, cudaStream_t st) {
  Params P;
  P.a = A;
  P.groups = A.num_groups;
  P.per = A.heads / A.kv.kv_heads;
  P.scale = A.scale * 1.4426950408889634f;
  P.slots_s = S.s;
  P.slots = S.o;
  // Shared runs of more rows than one 16-row tile go to the tcgen05 kernel, with two
  // row tiles where a group's mean rows need them.
  const long long mean = A.num_groups > 0 ? (long long)A.T * P.per / A.num_groups : 0;
  P.tc = A.num_groups > MAX_TC_GROUPS || mean <= TC_MIN_ROWS ? 0 : mean <= 128 ? 1 : 2;
  const long long most = (long long)A.num_requests * A.kv.pages_per_request * A.kv.page_size;
  P.planned = P.tc == 2 || (P.tc == 0 && A.num_requests >= PLANNED_REQUESTS &&
                            most >= PLANNED_BYTES / (4ll * A.kv.kv_heads * D));
  P.warps = 2 * num_sms() * WARPS;
  P.ctas = (int)std::min<long long>(
      num_sms(), ((long long)A.T * P.per / std::max(P.tc * 128, 1) + A.num_groups) * A.kv.kv_heads *
                     std::max(S.s, 1));
  const long long rows = (long long)A.T * A.heads;
  const int G = A.num_groups, segs = A.num_groups + A.num_requests;
  uint8_t* w = static_cast<uint8_t*>(ws);
  P.head = reinterpret_cast<int32_t*>(w);
  P.shared = P.head + HEAD_INTS;
  P.leader = P.shared + G;
  P.tc_first = P.leader + G;
  P.first = P.tc_first + G + 1;
  P.info = reinterpret_cast<int4*>(w + (4 * (size_t)(HEAD_INTS + 3 * G + 1 + segs + 1) + 15) / 16 * 16);
  P.o = reinterpret_cast<float*>(w + S.header);  // 16-byte pieces first
  P.ml = reinterpret_cast<float2*>(w + S.header + (size_t)(rows * (S.s + S.o)) * D * 4);
  const size_t plan = (size_t)segs * 20 + 4 + (size_t)G * 8, smem = 1024 + Layout<D>::PLAN + plan;
  constexpr int plan_max = MAX_SEGMENTS * PLAN_BYTES + 4, smem_max = 1024 + Layout<D>::PLAN + plan_max;
  if (!smem_attr<stream_kernel<D, false>>(smem_max) || !smem_attr<stream_kernel<D, true>>(smem_max) ||
      !smem_attr<plan_kernel>(plan_max))
    return fail(HYENA_ERR_CUDA, "cudaFuncSetAttribute(paged_attention) failed");
  CUtensorMap map_k, map_v;
  int rc = cache_map(&map_k, A.kv, true, KT);
  if (!rc) rc = cache_map(&map_v, A.kv, false, KT);
  if (rc) return rc;
  // each launch is checked before the next, which reads what it leaves
  if (P.planned) {
    launch_kernel(plan_kernel, dim3(1), dim3(PLAN_THREADS), plan, st, 0u, P);
    if ((rc = check_launch("paged_attention plan"))) return rc;
  }
  if (P.tc == 2 && (rc = shared_launch(P, map_k, map_v, st))) return rc;
  launch_kernel(P.planned ? stream_kernel<D, true> : stream_kernel<D, false>,
                dim3((unsigned)(P.warps / WARPS)), dim3(THREADS), smem, st, 0u, P, map_k, map_v);
  if ((rc = check_launch("paged_attention"))) return rc;
  if (P.tc == 1 && (rc = shared_launch(P, map_k, map_v, st))) return rc;
  // a block a row while there are few (8 an SM), else a warp
  if (rows <= 8ll * num_sms())
    launch_kernel(join_kernel<D, WARPS>, dim3((unsigned)rows + 1), dim3(THREADS), 0, st, 0u, P);
  else
    launch_kernel(join_kernel<D, 1>, dim3((unsigned)((rows + WARPS - 1) / WARPS) + 1), dim3(THREADS), 0, st,
                  0u, P);
  return check_launch("paged_attention");
}

}  // namespace attn

size_t paged_attention_workspace_size(const hyena_paged_attention_args& A) {
  if (attn::check(A) != HYENA_OK || A.T == 0 || A.num_requests == 0) return 0;
  return attn::slots_of(A).bytes;
}

int paged_attention_launch(const hyena_paged_attention_args& A, void* ws, size_t ws_bytes,
                           cudaStream_t st) {
  const int rc = attn::check(A);
  if (rc) return rc;
  if (A.T == 0 || A.num_requests == 0) return HYENA_OK;
  const attn::Slots S = attn::slots_of(A);
  HB_REQUIRE(ws != nullptr && aligned16(ws) && ws_bytes >= S.bytes,
             "paged_attention: workspace missing, misaligned or too small");
  if (A.kv.head_dim == 128) return attn::launch<128>(A, S, ws, st);
  return attn::launch<64>(A, S, ws, st);
}

}  // namespace hb
