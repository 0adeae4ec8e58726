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
// its requests, or the own keys of one request.  Segment x 16-row tile (rows =
// queries x heads of one key/value head) x key/value head x chunk of keys is an
// item; persistent CTAs walk the items.  Every length is read on the device
// (one captured graph serves growing contexts), so each CTA first derives the
// same plan from them: the chunk lengths, a prefix sum of the segments' items.
//
// `shared_lens` says what may be read once, never what is seen: a group's
// shared run is cut to what every query of the group sees and to whole 16-key
// tiles, and the rest of it counts as own keys.
#include <algorithm>

#include "attention.cuh"

namespace hb {
namespace attn {

constexpr int WARPS = 4;
constexpr int THREADS = WARPS * 32;
constexpr int ROWS = 16;        // rows of an item
constexpr int STAGES = 3;       // tiles in flight per warp
constexpr int MIN_CHUNK = 128;  // keys
constexpr int MAX_SEGMENTS = 2048;
constexpr int ITEMS_PER_CTA = 8;
constexpr int TC_MIN_ROWS = 16;  // mean rows of a group and key/value head

struct Plan {
  int chunk_s, chunk_o, items;
  int* first;  // [groups + requests + 1] first item of a segment
  int* shared; // [groups] the shared run
  int* leader; // [groups] the request whose pages stand for it
};

__device__ __forceinline__ int row_tiles(const Params& P, int nq) {
  return (int)(((long long)nq * P.per + ROWS - 1) / ROWS);
}

// Chunk of a kind of segment: the work spread over ITEMS_PER_CTA items a CTA,
// at most `slots` chunks a segment, whole rounds of the four warps.
__device__ __forceinline__ int chunk_keys(long long work, int longest, int slots, int ctas) {
  long long c = (work + (long long)ctas * ITEMS_PER_CTA - 1) / ((long long)ctas * ITEMS_PER_CTA);
  const int floor_slots = ceil_div(longest, slots > 0 ? slots : 1);
  if (c < floor_slots) c = floor_slots;
  if (c < MIN_CHUNK) c = MIN_CHUNK;
  c = (c + WARPS * KT - 1) / (WARPS * KT) * (WARPS * KT);
  return (int)(c < (1ll << 30) ? c : (1ll << 30));
}

// Every thread of the CTA; red: 4 x 4 long longs of scratch.
__device__ void make_plan(const Params& P, Plan& L, long long* red) {
  const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int B = P.a.num_requests, G = P.groups, hkv = P.a.kv.kv_heads;
  shared_runs<THREADS>(P, L.shared, L.leader);
  long long v[4] = {0, 0, 0, 0};  // work and longest, shared and own
  for (int s = tid; s < G + B; s += THREADS) {
    if (s < G) {
      int begin;
      const long long w = (long long)L.shared[s] * row_tiles(P, group_queries(P, s, begin)) * hkv;
      v[0] += w;
      if (w > 0 && L.shared[s] > v[1]) v[1] = L.shared[s];
    } else {
      int begin;
      const int n = queries(P, s - G, begin), g = group_of(P, s - G);
      int own = length(P, s - G) - (g >= 0 ? L.shared[g] : 0);
      own = own > 0 && n > 0 ? own : 0;
      v[2] += (long long)own * row_tiles(P, n) * hkv;
      if (own > v[3]) v[3] = own;
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long long x = __shfl_xor_sync(0xffffffffu, v[k], d);
      v[k] = (k & 1) ? (x > v[k] ? x : v[k]) : v[k] + x;
    }
  }
  if (lane == 0) {
    for (int k = 0; k < 4; ++k) red[warp * 4 + k] = v[k];
  }
  __syncthreads();
  for (int k = 0; k < 4; ++k) {
    v[k] = 0;
    for (int w = 0; w < WARPS; ++w) {
      const long long x = red[w * 4 + k];
      v[k] = (k & 1) ? (x > v[k] ? x : v[k]) : v[k] + x;
    }
  }
  L.chunk_s = chunk_keys(v[0], (int)v[1], P.slots_s, (int)gridDim.x);
  L.chunk_o = chunk_keys(v[2], (int)v[3], P.slots_o, (int)gridDim.x);
  // Items of the segments, then their exclusive prefix sum: a thread sums a run
  // of consecutive segments, the threads' sums are scanned.
  const int per = ceil_div(G + B, THREADS);
  const int s0 = tid * per, s1 = s0 + per < G + B ? s0 + per : G + B;
  int sum = 0;
  for (int s = s0; s < s1; ++s) {
    int items;
    if (s < G) {
      int begin;
      items = P.tc ? 0 : ceil_div(L.shared[s], L.chunk_s) * row_tiles(P, group_queries(P, s, begin)) * hkv;
    } else {
      int begin;
      const int n = queries(P, s - G, begin), g = group_of(P, s - G);
      const int own = length(P, s - G) - (g >= 0 ? L.shared[g] : 0);
      items = (own > 0 ? ceil_div(own, L.chunk_o) : 1) * row_tiles(P, n) * hkv;
    }
    L.first[s] = items;
    sum += items;
  }
  int scan = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, scan, d);
    if (lane >= d) scan += x;
  }
  __syncthreads();
  int* wsum = reinterpret_cast<int*>(red);
  if (lane == 31) wsum[warp] = scan;
  __syncthreads();
  int at = scan - sum, total = 0;
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) at += wsum[w];
    total += wsum[w];
  }
  for (int s = s0; s < s1; ++s) {
    const int items = L.first[s];
    L.first[s] = at;
    at += items;
  }
  if (tid == 0) L.first[G + B] = total;
  L.items = total;
  __syncthreads();
}

// ---------------------------------------------------------------- fragments
__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
// 16 bytes global -> shared, zeros instead where !valid.
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src),
               "r"(valid ? 16 : 0)
               : "memory");
}
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
// Byte offset of 16-byte chunk c of row `row` in a tile of D-element rows, the
// chunks permuted within groups of eight so that eight rows' same chunk (an
// ldmatrix phase) lies in distinct banks.
template <int D>
__device__ __forceinline__ uint32_t tile_at(int row, int c) {
  if constexpr (D == 128) return uint32_t(row * 256 + ((c ^ (row & 7)) << 4));
  return uint32_t(row * 128 + ((c ^ (row & 7)) << 4));
}

template <int D>
struct Layout {
  static constexpr int TILE = KT * D * 2;          // bytes of one operand's tile
  static constexpr int STAGE = 2 * TILE;           // keys, then values
  static constexpr int RING = STAGES * STAGE;      // a warp's ring
  static constexpr int PITCH = D + 4;              // floats of a parked row of O
  static_assert(RING >= ROWS * PITCH * 4, "the ring holds a warp's parked O");
  static constexpr int PLAN = WARPS * RING;        // ints of the plan follow
};

// One CTA walks its items; within an item warp w owns tiles w, w + 4, ... of the
// chunk, with its own ring, maximum, sum and O, and no barrier until the four
// warps' pieces are joined through shared memory.  The 16 rows of a tensor-core
// tile are mostly padding for one token and ungrouped heads; the item is bound
// by its keys' bytes all the same (128 mma for 32 KB of keys and values).
template <int D>
__global__ void __launch_bounds__(THREADS, 2) stream_kernel(const __grid_constant__ Params P) {
  using LT = Layout<D>;
  constexpr int CPR = D / 8;  // 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long red[WARPS * 4];
  __shared__ float2 ml_s[WARPS][ROWS];
  pdl_entry();
  const hyena_paged_attention_args& A = P.a;
  const hyena_paged_kv& kv = A.kv;
  const int tid = (int)threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int G = P.groups, B = A.num_requests, hkv = kv.kv_heads;
  Plan L;
  L.first = reinterpret_cast<int*>(smem + LT::PLAN);
  L.shared = L.first + (G + B + 1);
  L.leader = L.shared + G;
  make_plan(P, L, red);
  if (blockIdx.x == 0 && P.plan != nullptr) {
    if (tid == 0) {
      if (!P.tc) P.plan[0] = L.chunk_s;
      P.plan[1] = L.chunk_o;
    }
    for (int g = tid; g < G; g += THREADS) P.plan[2 + g] = L.shared[g];
  }
  const int slots = P.slots_s + P.slots_o;
  uint8_t* ring = smem + warp * LT::RING;
  const uint32_t ring_u = smem_u32(ring);
  const int g8 = lane >> 2, t4 = lane & 3;

  for (int item = (int)blockIdx.x; item < L.items; item += (int)gridDim.x) {
    // ---- which keys and rows
    int lo = 0, hi = G + B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (L.first[mid] <= item) lo = mid; else hi = mid;
    }
    const int seg = lo;
    const bool own_seg = seg >= G;
    int request, begin, rows, nq = 0, len = 0, k_begin, k_end, chunk, chunks;
    if (own_seg) {
      request = seg - G;
      nq = queries(P, request, begin);
      len = length(P, request);
      rows = nq * P.per;
      const int g = group_of(P, request);
      k_begin = g >= 0 ? L.shared[g] : 0;
      k_end = len > k_begin ? len : k_begin;
      if (len == 0) k_begin = k_end = 0;
      chunk = L.chunk_o;
    } else {
      request = L.leader[seg];
      rows = group_queries(P, seg, begin) * P.per;
      k_begin = 0;
      k_end = L.shared[seg];
      chunk = L.chunk_s;
    }
    chunks = k_end > k_begin ? ceil_div(k_end - k_begin, chunk) : 1;
    const int tiles_r = ceil_div(rows, ROWS);
    int rem = item - L.first[seg];
    const int rt = rem % tiles_r;
    rem /= tiles_r;
    const int h = rem % hkv, c = rem / hkv;
    const int row0 = rt * ROWS;
    int k0 = k_begin + c * chunk;
    int k1 = k_end - k0 > chunk ? k0 + chunk : k_end;
    int all_see = k1;  // keys below it are seen by every row of the tile
    if (own_seg) {
      const int last = min(nq - 1, (row0 + ROWS - 1) / P.per);
      k1 = min(k1, len - nq + last + 1);
      all_see = min(k1, len - nq + row0 / P.per + 1);
    }
    const int tiles = k1 > k0 ? ceil_div(k1 - k0, KT) : 0;

    // ---- this lane's two rows (g8, g8 + 8) as mma A fragments
    uint32_t qf[D / 16][4];
    int limit[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = row0 + g8 + 8 * i;
      limit[i] = 0;
      const bf16* src = nullptr;
      if (row < rows) {
        const int qi = row / P.per;
        limit[i] = own_seg ? len - nq + qi + 1 : 0x7fffffff;
        src = static_cast<const bf16*>(A.q) + (long long)(begin + qi) * A.q_token_stride +
              (long long)(h * P.per + row - qi * P.per) * A.q_head_stride;
      }
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qf[ks][i] = src != nullptr ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + t4 * 2) : 0u;
        qf[ks][2 + i] = src != nullptr ? *reinterpret_cast<const uint32_t*>(src + ks * 16 + 8 + t4 * 2) : 0u;
      }
    }

    // ---- loads
    const int32_t* table = kv.page_table + (long long)request * kv.page_table_stride;
    const int mine = tiles > warp ? (tiles - warp + WARPS - 1) / WARPS : 0;
    auto page_for = [&](int i) {  // page of this warp's tile i
      return i < mine ? __ldg(table + (k0 + (warp + i * WARPS) * KT) / kv.page_size) : 0;
    };
    uint32_t bad = 0;  // stages whose page is out of range
    auto load = [&](int i, int page) {
      if (i < mine) {
        const int kpos = k0 + (warp + i * WARPS) * KT, s = i % STAGES;
        const bool ok = page >= 0 && page < kv.num_pages;
        bad = ok ? bad & ~(1u << s) : bad | (1u << s);
        if (!ok) {
          if (lane == 0) flag_error(A.error_flags, HYENA_FLAG_BLOCK_RANGE);
          page = 0;
        }
        const int at = kpos % kv.page_size;
        const int ch = lane % CPR, r0 = lane / CPR;
        const bf16* ks = static_cast<const bf16*>(kv.k) + page * kv.k_page_stride +
                         (at + r0) * kv.k_token_stride + h * kv.k_head_stride + ch * 8;
        const bf16* vs = static_cast<const bf16*>(kv.v) + page * kv.v_page_stride +
                         (at + r0) * kv.v_token_stride + h * kv.v_head_stride + ch * 8;
        const uint32_t dst = ring_u + uint32_t(s * LT::STAGE);
        const int nvalid = ok ? k1 - kpos : 0;  // rows behind the last key are zeros
#pragma unroll
        for (int r = 0; r < KT; r += 32 / CPR) {
          const uint32_t d = dst + tile_at<D>(r0 + r, ch);
          cp_async16_or_zero(d, ks + r * kv.k_token_stride, r0 + r < nvalid);
          cp_async16_or_zero(d + LT::TILE, vs + r * kv.v_token_stride, r0 + r < nvalid);
        }
      }
      cp_async_commit();
    };
    int page_next = page_for(0);
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
      const int page = page_next;
      page_next = page_for(i + 1);
      load(i, page);
    }

    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    for (int i = 0; i < mine; ++i) {
      {
        const int page = page_next;
        page_next = page_for(i + STAGES);
        load(i + STAGES - 1, page);
      }
      cp_async_wait<STAGES - 1>();
      __syncwarp();
      const int s = i % STAGES;
      const int kpos = k0 + (warp + i * WARPS) * KT;
      const uint32_t ks_u = ring_u + uint32_t(s * LT::STAGE), vs_u = ks_u + LT::TILE;
      const bool is_bad = (bad >> s) & 1u;

      // scores of 16 rows x 16 keys
      float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t b[4];  // keys 0-7 (k 0-7, 8-15), keys 8-15 (k 0-7, 8-15)
        ldsm4(ks_u + tile_at<D>((lane & 7) + ((lane >> 4) << 3), ks * 2 + ((lane >> 3) & 1)), b);
        mma_bf16(sc[0], qf[ks], b[0], b[1]);
        mma_bf16(sc[1], qf[ks], b[2], b[3]);
      }
      float p[2][4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int end = is_bad ? 0 : min(limit[r], k1) - kpos;  // keys of the tile this row sees
        float x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = (e >> 1) * 8 + t4 * 2 + (e & 1);
          x[e] = key < end ? sc[e >> 1][r * 2 + (e & 1)] * P.scale : -INFINITY;
        }
        float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const float mn = fmaxf(m[r], top);
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float keep = exp2_approx(m[r] - base);
        m[r] = mn;
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float w = exp2_approx(x[e] - base);
          sum += w;
          p[e >> 1][r * 2 + (e & 1)] = w;
        }
        l[r] = l[r] * keep + sum;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o[n][r * 2] *= keep;
          o[n][r * 2 + 1] *= keep;
        }
      }
      // Keys that some row of the tile does not see (a later token of the same
      // step): added row by row, so that a masked value, whatever it holds,
      // meets no product; the mma below gets zeros for them.
      if (all_see < kpos + KT && all_see < k1) {
        const int j0 = max(all_see - kpos, 0), j1 = min(k1 - kpos, KT);
        for (int j = j0; j < j1; ++j) {
          const int src = (lane & ~3) | ((j & 7) >> 1);
          const float w00 = __shfl_sync(0xffffffffu, p[0][0], src), w01 = __shfl_sync(0xffffffffu, p[0][1], src);
          const float w02 = __shfl_sync(0xffffffffu, p[0][2], src), w03 = __shfl_sync(0xffffffffu, p[0][3], src);
          const float w10 = __shfl_sync(0xffffffffu, p[1][0], src), w11 = __shfl_sync(0xffffffffu, p[1][1], src);
          const float w12 = __shfl_sync(0xffffffffu, p[1][2], src), w13 = __shfl_sync(0xffffffffu, p[1][3], src);
          const bool upper = j >= 8, odd = j & 1;
          const float wa = upper ? (odd ? w11 : w10) : (odd ? w01 : w00);
          const float wb = upper ? (odd ? w13 : w12) : (odd ? w03 : w02);
          const bool sa = !is_bad && kpos + j < limit[0], sb = !is_bad && kpos + j < limit[1];
#pragma unroll
          for (int n = 0; n < D / 8; ++n) {
            const float2 v = unpack2(*reinterpret_cast<const bf162*>(
                ring + s * LT::STAGE + LT::TILE + tile_at<D>(j, n) + t4 * 4));
            if (sa) {
              o[n][0] = fmaf(wa, v.x, o[n][0]);
              o[n][1] = fmaf(wa, v.y, o[n][1]);
            }
            if (sb) {
              o[n][2] = fmaf(wb, v.x, o[n][2]);
              o[n][3] = fmaf(wb, v.y, o[n][3]);
            }
          }
          __syncwarp();
          if (lane < CPR)
            *reinterpret_cast<uint4*>(ring + s * LT::STAGE + LT::TILE + tile_at<D>(j, lane)) =
                make_uint4(0u, 0u, 0u, 0u);
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = (e >> 1) * 8 + t4 * 2 + (e & 1);
          if (key >= j0) p[e >> 1][e & 1] = p[e >> 1][2 + (e & 1)] = 0.0f;
        }
      }
      // The weights are rounded to bf16 for the product, as the values are; l
      // sums them before that rounding, which is unbiased.
      uint32_t pa[4];
      pa[0] = as_u32(pack2_rn(make_float2(p[0][0], p[0][1])));
      pa[1] = as_u32(pack2_rn(make_float2(p[0][2], p[0][3])));
      pa[2] = as_u32(pack2_rn(make_float2(p[1][0], p[1][1])));
      pa[3] = as_u32(pack2_rn(make_float2(p[1][2], p[1][3])));
#pragma unroll
      for (int n = 0; n < D / 16; ++n) {
        uint32_t b[4];  // values of keys 0-7 and 8-15, columns 16n + 0-7 then 16n + 8-15
        ldsm4_trans(vs_u + tile_at<D>(lane & 15, n * 2 + (lane >> 4)), b);
        mma_bf16(o[2 * n], pa, b[0], b[1]);
        mma_bf16(o[2 * n + 1], pa, b[2], b[3]);
      }
      __syncwarp();  // the stage is read before it is filled again
    }
    cp_async_wait<0>();

    // ---- join the warps' pieces
    float* parked = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
      if (t4 == 0) ml_s[warp][g8 + 8 * r] = make_float2(m[r], l[r]);
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<float2*>(parked + (g8 + 8 * r) * LT::PITCH + n * 8 + t4 * 2) =
            make_float2(o[n][r * 2], o[n][r * 2 + 1]);
    }
    __syncthreads();
    {
      const int row = tid / 8, col = (tid % 8) * (D / 8);
      if (row0 + row < rows) {
        float mx = -INFINITY, lsum = 0.0f, w[WARPS];
#pragma unroll
        for (int k = 0; k < WARPS; ++k) mx = fmaxf(mx, ml_s[k][row].x);
        const float base = mx == -INFINITY ? 0.0f : mx;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) {
          w[k] = exp2_approx(ml_s[k][row].x - base);
          lsum += w[k] * ml_s[k][row].y;
        }
        float acc[D / 8];
#pragma unroll
        for (int j = 0; j < D / 8; ++j) acc[j] = 0.0f;
#pragma unroll
        for (int k = 0; k < WARPS; ++k) {
          const float* src = reinterpret_cast<const float*>(smem + k * LT::RING) + row * LT::PITCH + col;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) acc[j] = fmaf(w[k], src[j], acc[j]);
        }
        const int qi = (row0 + row) / P.per;
        const long long token = begin + qi;
        const int head = h * P.per + row0 + row - qi * P.per;
        if (own_seg && chunks == 1 && k_begin == 0) {  // the row's only piece
          const float inv = lsum > 0.0f || lsum != lsum ? 1.0f / lsum : 0.0f;
          bf16* dst = static_cast<bf16*>(A.out) + token * A.out_token_stride +
                      (long long)head * A.out_head_stride + col;
#pragma unroll
          for (int j = 0; j < D / 8; j += 8) {
            uint4 pk;
            uint32_t* pw = reinterpret_cast<uint32_t*>(&pk);
#pragma unroll
            for (int e = 0; e < 4; ++e)
              pw[e] = as_u32(pack2_rn(make_float2(acc[j + 2 * e] * inv, acc[j + 2 * e + 1] * inv)));
            *reinterpret_cast<uint4*>(dst + j) = pk;
          }
        } else {
          const long long slot = (token * A.heads + head) * slots + (own_seg ? P.slots_s + c : c);
          if (col == 0) P.ml[slot] = make_float2(mx, lsum);
          float* dst = P.o + slot * D + col;
#pragma unroll
          for (int j = 0; j < D / 8; j += 4)
            *reinterpret_cast<float4*>(dst + j) = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
        }
      }
    }
    __syncthreads();  // the rings are free again
  }
}

// Joins the pieces of the rows that have more than one: a warp a row, or
// (WPR = 4) the four warps of a block, for few rows of many pieces.
template <int D, int WPR>
__global__ void __launch_bounds__(THREADS) join_kernel(const __grid_constant__ Params P) {
  constexpr int E = D / 32;
  __shared__ float red[WPR][D + 2];
  pdl_entry();
  const hyena_paged_attention_args& A = P.a;
  const int lane = (int)threadIdx.x & 31, warp = (int)threadIdx.x >> 5;
  const long long row = WPR == 1 ? (long long)blockIdx.x * WARPS + warp : (long long)blockIdx.x;
  const int part = WPR == 1 ? 0 : warp;
  if (row >= (long long)A.T * A.heads) return;
  const int token = (int)(row / A.heads), head = (int)(row % A.heads);
  int r = token;
  if (A.query_start_loc != nullptr) {
    r = find_segment(A.query_start_loc, A.num_requests, token);
    if (token < __ldg(A.query_start_loc + r) || token >= __ldg(A.query_start_loc + r + 1)) return;
  } else if (r >= A.num_requests) {
    return;
  }
  const int chunk_s = P.plan[0], chunk_o = P.plan[1];
  const int g = group_of(P, r), len = length(P, r);
  const int sh = g >= 0 && len > 0 ? P.plan[2 + g] : 0;
  const int ns = ceil_div(sh, chunk_s), no = len > sh ? ceil_div(len - sh, chunk_o) : 1;
  if (ns == 0 && no == 1) return;  // written already
  const long long base = row * (P.slots_s + P.slots_o);
  float m = -INFINITY, l = 0.0f, acc[E];
#pragma unroll
  for (int j = 0; j < E; ++j) acc[j] = 0.0f;
  for (int i = part; i < ns + no; i += WPR) {
    const long long slot = base + (i < ns ? i : P.slots_s + i - ns);
    const float2 x = P.ml[slot];
    const float* src = P.o + slot * D + lane * E;
    float v[E];
    if constexpr (E == 4) {
      const float4 y = *reinterpret_cast<const float4*>(src);
      v[0] = y.x; v[1] = y.y; v[2] = y.z; v[3] = y.w;
    } else {
      const float2 y = *reinterpret_cast<const float2*>(src);
      v[0] = y.x; v[1] = y.y;
    }
    const float mn = fmaxf(m, x.x), b = mn == -INFINITY ? 0.0f : mn;
    const float wa = exp2_approx(m - b), wb = exp2_approx(x.x - b);
    m = mn;
    l = l * wa + x.y * wb;
#pragma unroll
    for (int j = 0; j < E; ++j) acc[j] = acc[j] * wa + v[j] * wb;
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
// Pieces a row may have, from sizes the host knows: enough that one segment
// alone spreads over the GPU, bounded by the chunks its pages can hold and by
// the workspace.
struct Slots {
  int s, o;
  bool join;
  size_t bytes;
};
constexpr size_t WORKSPACE_BYTES = size_t(256) << 20;

static Slots slots_of(const hyena_paged_attention_args& A) {
  const bool shared = A.shared_lens != nullptr;
  const long long rows = (long long)A.T * A.heads;
  const long long row_bytes = (A.kv.head_dim + 2) * 4;
  const long long keys = (long long)A.kv.pages_per_request * A.kv.page_size;
  long long n = (8ll * num_sms() + A.kv.kv_heads - 1) / A.kv.kv_heads;
  n = std::min(n, (keys + MIN_CHUNK - 1) / MIN_CHUNK);
  n = std::min(n, (long long)WORKSPACE_BYTES / (rows * row_bytes * (shared ? 2 : 1)));
  n = std::max(n, 1ll);
  Slots S;
  S.o = (int)n;
  S.s = shared ? (int)n : 0;
  S.join = shared || n > 1;
  const size_t head = 8 + 4 * (size_t)A.num_groups;
  S.bytes = S.join ? ((head + 255) & ~size_t(255)) + (size_t)(rows * (S.s + S.o)) * row_bytes : 0;
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
  P.slots_o = S.o;
  // Shared runs of more rows than one 16-row tile go to the tcgen05 kernel.
  P.tc = S.s > 0 && A.num_groups <= MAX_TC_GROUPS &&
         (long long)A.T * P.per > (long long)TC_MIN_ROWS * A.num_groups;
  P.plan = nullptr;
  P.ml = nullptr;
  P.o = nullptr;
  const long long rows = (long long)A.T * A.heads;
  if (S.join) {
    uint8_t* w = static_cast<uint8_t*>(ws);
    P.plan = reinterpret_cast<int32_t*>(w);
    w += (8 + 4 * (size_t)A.num_groups + 255) & ~size_t(255);
    P.o = reinterpret_cast<float*>(w);  // 16-byte pieces first
    P.ml = reinterpret_cast<float2*>(w + (size_t)(rows * (S.s + S.o)) * D * 4);
  }
  const int segments = A.num_requests + A.num_groups;
  const size_t smem = Layout<D>::PLAN + (size_t)(segments + 1 + 2 * A.num_groups) * 4;
  constexpr int smem_max = Layout<D>::PLAN + (MAX_SEGMENTS + 1 + 2 * MAX_SEGMENTS) * 4;
  if (!smem_attr<stream_kernel<D>>(smem_max))
    return fail(HYENA_ERR_CUDA, "cudaFuncSetAttribute(paged_attention) failed");
  const long long bound = (rows / A.kv.kv_heads / ROWS + segments) * A.kv.kv_heads * (S.s + S.o);
  const long long ctas = std::min<long long>(2ll * num_sms(), bound);
  launch_kernel(stream_kernel<D>, dim3((unsigned)ctas), dim3(THREADS), smem, st, 0u, P);
  if (P.tc) {
    const int rc = shared_launch(P, st);
    if (rc) return rc;
  }
  if (S.join) {
    // a block a row while those fill one wave of 16 blocks an SM
    if (rows <= 16ll * num_sms())
      launch_kernel(join_kernel<D, WARPS>, dim3((unsigned)rows), dim3(THREADS), 0, st, 0u, P);
    else
      launch_kernel(join_kernel<D, 1>, dim3((unsigned)((rows + WARPS - 1) / WARPS)), dim3(THREADS), 0,
                    st, 0u, P);
  }
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
  HB_REQUIRE(S.bytes == 0 || (ws != nullptr && aligned16(ws) && ws_bytes >= S.bytes),
             "paged_attention: workspace missing, misaligned or too small");
  if (A.kv.head_dim == 128) return attn::launch<128>(A, S, ws, st);
  return attn::launch<64>(A, S, ws, st);
}

}  // namespace hb
