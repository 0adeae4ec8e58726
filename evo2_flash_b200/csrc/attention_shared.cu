// Attention over the keys that the requests of a group share: one tcgen05 pass
// for the queries of the whole group (see attention.cu for the decomposition
// into pieces and for the join).
//
// An item is NT x 128 query rows (queries x heads of one key/value head) against
// a chunk of the shared run; one CTA per SM walks its items:
//   warps 0 .. 4 NT - 1  softmax: a thread owns one row; its 128 scores of a key
//                tile come from TMEM, 2^(s - m) goes back as bf16 over the same
//                columns, ready to be the A operand of the value product
//   next warp    tcgen05.mma issue (one thread): S_t = Q_t K^T (K-major operands),
//                O_t += P_t V with P_t in TMEM and V read MN-major as it lies in
//                the cache; O stays in TMEM for the whole item
//   last two     TMA: tiles of 128 keys (256 B rows, SWIZZLE_128B, two 64-column
//                halves) by the largest box that a page holds whole, one warp for
//                the keys and one for the values, which take turns in one ring (a
//                warp needs 50 ns a box, 16 of them a tile in pages of 16: 91 us for
//                verifying 4 tokens of 48 requests on 3 prompts of 2029 keys, 99 us
//                with one warp for both)
// Every row sees every key of the run, so only the run's last tile has a mask.
//
// O is rescaled only when the weights of a row's tile sum to more than 2^8, its
// scores having outgrown the m it is scaled by.  Below that bf16 and fp32 round
// as well as at 1; the pass over O's columns (TMEM -> registers -> TMEM) is rare
// instead of once a tile; m and l leave with the piece, so nothing is lost.
//
// NT = 1 keeps two score buffers (S of the next tile is computed under the
// softmax); NT = 2 (256 rows) reads each key and value once for two row tiles,
// whose softmax and matrix products alternate.  Up to about 128 rows it is bound
// by the keys' bytes.  Beyond, a key tile of 256 rows takes some 3600 cycles, of
// which the tensor pipe works 2300 (2048 at its peak; Q K^T with both operands in
// shared memory reads them at all of its bandwidth): a row tile's chain is 1900
// for the softmax (1024 of them the exponentials alone), 1150 for its two
// products and 500 from one to the other, and TMEM has no room for a second
// score buffer.  Two threads a row, a warp instead of a thread issuing the
// products, 64-key tiles and half tiles of weights all measured the same or worse.
//
// It and the stream kernel share no data, and the second of the two does not wait
// for the first at entry: the first one's CTAs trigger only after their own wait,
// so that all before them is complete when the second starts, whose CTAs take SMs
// as the first one leaves them.  The second waits at its end instead, so that the
// join kernel, which waits for it alone, finds both complete.
//   NT = 2 goes first, after a plan kernel, and the stream kernel's items, which
// are then taken as they come, fill the SMs that its last wave leaves: 353 us for
// 256 samples of one prompt of 32768 keys, 382 us the other way round (332 us now in runs
// of a few ms, 377 in longer ones, for which the power cap lowers the clock).
//   NT = 1 goes second, each CTA of either planning for itself: both are bound by
// the keys' bytes, and this one fills the end of the two better.  85 us for 64
// samples of a prompt of 8192 keys and 99 us for 3 prompts being verified (91 us
// now); with the plan kernel 95 and 112 us, with NT = 2's order 98 and 104 us.
#include <algorithm>
#include <type_traits>

#include "attention.cuh"

namespace hb {
namespace attn {

using namespace tc;

constexpr int BOX_MIN = 16;

template <int D, int NT>
struct Tc {
  static constexpr int HALVES = D / 64;              // 64-column swizzled halves of a row
  static constexpr int HALF_BYTES = TILE_KEYS * 128;
  static constexpr int TILE_BYTES = HALVES * HALF_BYTES;  // 128 rows x D
  static constexpr int FIT = (224 * 1024 - NT * TILE_BYTES) / TILE_BYTES;
  static constexpr int SLOTS = FIT < 8 ? FIT : 8;
  static constexpr int NBUF = NT == 1 ? 2 : 1;       // score buffers of a row tile
  static constexpr int THREADS = NT * 128 + 96;
  static constexpr uint32_t S_COL = 0, O_COL = 256;  // TMEM columns
  static constexpr uint32_t TMEM_COLS = 512;
};

template <int D, int NT>
struct __align__(1024) TcSmem {
  uint8_t q[NT][Tc<D, NT>::TILE_BYTES];
  uint8_t ring[Tc<D, NT>::SLOTS][Tc<D, NT>::TILE_BYTES];
  uint64_t full[Tc<D, NT>::SLOTS], empty[Tc<D, NT>::SLOTS];
  uint64_t q_full;
  uint64_t s_full[NT][2], p_full[NT][2], pv_done[NT], o_done[NT];  // [..][score buffer]
  uint32_t bad[8];  // 16-key blocks of a tile whose page is out of range
  uint32_t tmem;
  int chunk_tiles;
  int first[MAX_TC_GROUPS + 1], shared[MAX_TC_GROUPS], leader[MAX_TC_GROUPS];
};

// D[128 x N] (+)= A[128 x 16] B[N x 16]^T, A in shared memory / in TMEM.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(id), "r"(acc ? 1u : 0u));
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(id), "r"(acc ? 1u : 0u));
}
// SWIZZLE_128B descriptor of an operand whose N (or M) index runs along the
// 128-byte rows: 64-element atoms `lead` bytes apart along N, eight rows (K)
// 1024 bytes.
__device__ __forceinline__ uint64_t sw128_mn_desc(const void* p, uint32_t lead) {
  const uint64_t addr = su32(p);
  return ((addr & 0x3FFFFull) >> 4) | (uint64_t(lead >> 4) << 16) | (uint64_t(1024 >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// bf16 operands, fp32 accumulator, M = 128, N = n; b_mn: B is MN-major.
__host__ __device__ constexpr uint32_t attn_idesc(int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn ? 1u : 0u) << 16) | (uint32_t(n >> 3) << 17) |
         (uint32_t(128 >> 4) << 24);
}

struct Item {
  int group, leader, row0, rows, begin, head, chunk, k0, k1, tiles;
};

template <int D, int NT>
__device__ __forceinline__ Item item_of(const Params& P, const TcSmem<D, NT>& S, int item) {
  Item I;
  int g = 0;
  while (item >= S.first[g + 1]) ++g;
  I.group = g;
  I.leader = S.leader[g];
  I.rows = group_queries(P, g, I.begin) * P.per;
  const int row_tiles = ceil_div(I.rows, NT * 128), hkv = P.a.kv.kv_heads;
  int rem = item - S.first[g];
  I.row0 = rem % row_tiles * (NT * 128);
  rem /= row_tiles;
  I.head = rem % hkv;
  I.chunk = rem / hkv;
  I.k0 = I.chunk * S.chunk_tiles * TILE_KEYS;
  const int end = S.shared[g];
  I.k1 = end - I.k0 > S.chunk_tiles * TILE_KEYS ? I.k0 + S.chunk_tiles * TILE_KEYS : end;
  I.tiles = ceil_div(I.k1 - I.k0, TILE_KEYS);
  return I;
}

template <int D, int NT>
__global__ void __launch_bounds__(Tc<D, NT>::THREADS, 1)
shared_kernel(const __grid_constant__ Params P, const __grid_constant__ CUtensorMap map_k,
              const __grid_constant__ CUtensorMap map_v, const __grid_constant__ CUtensorMap map_k16,
              const __grid_constant__ CUtensorMap map_v16, int box) {
  using T = Tc<D, NT>;
  extern __shared__ uint8_t smem_raw[];
  TcSmem<D, NT>& S = *reinterpret_cast<TcSmem<D, NT>*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const hyena_paged_attention_args& A = P.a;
  const int tid = (int)threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int G = P.groups;

  if (tid == 0) {
    for (int s = 0; s < T::SLOTS; ++s) {
      mbar_init(&S.full[s], 1);
      mbar_init(&S.empty[s], 1);
    }
    mbar_init(&S.q_full, 4 * NT);
    for (int t = 0; t < NT; ++t) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&S.s_full[t][b], 2);
        mbar_init(&S.p_full[t][b], 4);
      }
      mbar_init(&S.pv_done[t], 1);
      mbar_init(&S.o_done[t], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 * NT) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     su32(&S.tmem)),
                 "r"(T::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }

  if (NT == 2) {
    pdl_wait();  // the plan
    pdl_trigger();
    for (int g = tid; g <= G; g += T::THREADS) {
      S.first[g] = __ldcg(P.tc_first + g);
      if (g < G) {
        S.shared[g] = __ldcg(P.shared + g);
        S.leader[g] = __ldcg(P.leader + g);
      }
    }
    if (tid == 0) S.chunk_tiles = __ldcg(P.head + TC_TILES);
  } else {
    shared_runs<T::THREADS>(P, S.shared, S.leader);
    plan_shared<T::THREADS>(P, S.shared, S.first, &S.chunk_tiles);
    if (blockIdx.x == 0 && tid == 0) P.head[SHARED_TILES] = S.chunk_tiles * (TILE_KEYS / KT);
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = S.tmem;
  const int items = S.first[G];

  if (warp > 4 * NT) {
    // ---------------------------------------------------------------- loads
    const int kv = warp - 4 * NT - 1;  // keys, or values
    uint32_t u = (uint32_t)kv, tile_no = 0;
    bool ok = true;
    for (int item = (int)blockIdx.x; item < items && ok; item += (int)gridDim.x) {
      const Item I = item_of<D, NT>(P, S, item);
      const int32_t* table = A.kv.page_table + (long long)I.leader * A.kv.page_table_stride;
      // lane j: page of 16-key block j of a tile, looked up a tile ahead
      auto page_of = [&](int kpos) {
        const int pos = kpos + lane * BOX_MIN;
        return lane < TILE_KEYS / BOX_MIN && pos < I.k1 ? __ldg(table + pos / A.kv.page_size) : 0;
      };
      int next = page_of(I.k0);
      for (int i = 0; i < I.tiles && ok; ++i, ++tile_no, u += 2) {
        const int kpos = I.k0 + i * TILE_KEYS;
        const int keys = min(TILE_KEYS, I.k1 - kpos);
        const int page = next, at = (kpos + lane * BOX_MIN) % A.kv.page_size;
        next = page_of(kpos + TILE_KEYS);
        // whether the block leads a whole box or stands alone in the tail
        const bool mine = lane < TILE_KEYS / BOX_MIN && lane * BOX_MIN < keys;
        const bool good = !mine || (page >= 0 && page < A.kv.num_pages);
        const bool whole = (lane * BOX_MIN / box + 1) * box <= keys;
        if (!good) flag_error(A.error_flags, HYENA_FLAG_BLOCK_RANGE);
        const uint32_t bad = __ballot_sync(0xffffffffu, !good);
        const uint32_t have = __ballot_sync(0xffffffffu, mine && good);
        if (kv == 0 && lane == 0) S.bad[tile_no & 7] = bad;
        const bool leads = mine && good && (whole ? lane * BOX_MIN % box == 0 : true);
        const uint32_t bytes = uint32_t(__popc(have)) * BOX_MIN * D * 2;
        const int s = u % T::SLOTS;
        ok = __all_sync(0xffffffffu, wait(&S.empty[s], ((u / T::SLOTS) & 1) ^ 1, A.error_flags));
        if (!ok) break;
        uint8_t* slot = S.ring[s];
        if (kv == 1 && have != 0xFFu) {
          // weights of absent keys are zero, but so must their values be
          for (int r = lane; r < TILE_KEYS * T::HALVES * 8; r += 32) {
            const int row = r / 8 % TILE_KEYS;
            if (!((have >> (row / BOX_MIN)) & 1u))
              *reinterpret_cast<uint4*>(slot + r * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        if (lane == 0) mbar_expect_tx(&S.full[s], bytes);
        __syncwarp();
        if (leads) {
          const CUtensorMap* map = kv == 0 ? (whole ? &map_k : &map_k16) : (whole ? &map_v : &map_v16);
#pragma unroll
          for (int h = 0; h < T::HALVES; ++h)
            tma_load_4d(map, &S.full[s], slot + h * T::HALF_BYTES + lane * BOX_MIN * 128, h * 64, at,
                        I.head, page);
        }
        __syncwarp();
      }
    }
    // Drain: every issued copy has landed, and every slot's release has arrived,
    // before the CTA can exit.  (u is 2 tile_no + kv: the last SLOTS uses of the ring
    // are those no later use has followed.)
    for (uint32_t i = (uint32_t)kv; i < u; i += 2) {
      if (i + T::SLOTS < 2 * tile_no) continue;
      wait(&S.full[i % T::SLOTS], (i / T::SLOTS) & 1, A.error_flags);
      if (ok) wait(&S.empty[i % T::SLOTS], (i / T::SLOTS) & 1, A.error_flags);
    }
  } else if (warp == 4 * NT) {
    // ---------------------------------------------------------------- products
    if (lane == 0) {
      constexpr uint32_t ID_S = attn_idesc(TILE_KEYS, false), ID_O = attn_idesc(D, true);
      uint32_t u = 0, gi = 0, n_item = 0;
      bool ok = true;
      auto score = [&](int t, uint32_t no, uint32_t slot_u) {  // S_t of tile `no`
        const int b = T::NBUF == 2 ? (no & 1) : 0;
        const uint32_t d = tmem + T::S_COL + uint32_t((T::NBUF == 2 ? b : t) * TILE_KEYS);
        const uint64_t q = sw128_desc(S.q[t]), k = sw128_desc(S.ring[slot_u % T::SLOTS]);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {  // (addresses in descriptors count 16 bytes)
          const uint64_t off = ((ks / 4) * T::HALF_BYTES + (ks % 4) * 32) / 16;
          mma_ss(d, q + off, k + off, ID_S, ks != 0);
        }
        mma_commit(&S.s_full[t][b]);
        mbar_arrive(&S.s_full[t][b]);  // passes on what the loading warp wrote for the tile
      };
      auto values = [&](int t, uint32_t no, uint32_t slot_u, bool acc) {  // O_t += P_t V
        const int b = T::NBUF == 2 ? (no & 1) : 0;
        const uint32_t p = tmem + T::S_COL + uint32_t((T::NBUF == 2 ? b : t) * TILE_KEYS);
        const uint32_t d = tmem + T::O_COL + uint32_t(t * D);
        const uint64_t v = sw128_mn_desc(S.ring[slot_u % T::SLOTS], T::HALF_BYTES);
#pragma unroll
        for (int ks = 0; ks < TILE_KEYS / 16; ++ks)
          mma_ts(d, p + ks * 8, v + ks * (2048 / 16), ID_O, acc || ks != 0);
        // waited for only where O is rescaled, at most one product behind: a parity
        // tells no more than neighbours apart, so the item's end has o_done.  (NT = 2:
        // the tile's next scores come after this product, so s_full tells.)
        if constexpr (NT == 1) mma_commit(&S.pv_done[t]);
      };
      auto slot_full = [&](uint32_t slot_u) {
        ok = ok && wait(&S.full[slot_u % T::SLOTS], (slot_u / T::SLOTS) & 1, A.error_flags);
      };
      for (int item = (int)blockIdx.x; item < items && ok; item += (int)gridDim.x, ++n_item) {
        const Item I = item_of<D, NT>(P, S, item);
        ok = ok && wait(&S.q_full, n_item & 1, A.error_flags);
        slot_full(u);
        if (!ok) break;
        for (int t = 0; t < NT; ++t) score(t, gi, u);
        mma_commit(&S.empty[u % T::SLOTS]);
        for (int i = 0; i < I.tiles && ok; ++i, ++gi, u += 2) {
          const bool more = i + 1 < I.tiles;
          if constexpr (NT == 1) {
            if (more) {
              slot_full(u + 2);
              if (!ok) break;
              score(0, gi + 1, u + 2);
              mma_commit(&S.empty[(u + 2) % T::SLOTS]);
            }
          }
          // (before the weights are awaited, while products are under way)
          slot_full(u + 1);
          if (NT > 1 && more) slot_full(u + 2);
          for (int t = 0; t < NT && ok; ++t) {
            // (a barrier a buffer: a warp without rows is done with the next tile's
            // scores before the others are with this one's)
            ok = ok && wait(&S.p_full[t][T::NBUF == 2 ? (gi & 1) : 0],
                            T::NBUF == 2 ? (gi >> 1) & 1 : gi & 1, A.error_flags);
            if (!ok) break;
            fence_after();
            values(t, gi, u + 1, i != 0);
            if (!more) mma_commit(&S.o_done[t]);
            if (t == NT - 1) mma_commit(&S.empty[(u + 1) % T::SLOTS]);
            if constexpr (NT > 1) {
              if (more) {
                score(t, gi + 1, u + 2);
                if (t == NT - 1) mma_commit(&S.empty[(u + 2) % T::SLOTS]);
              }
            }
          }
        }
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax
    const int t = warp / 4, row_in = tid % 128;
    const uint32_t lanes = uint32_t(32 * (warp % 4)) << 16;
    const float scale = P.scale == 0.0f ? 1.0f : fabsf(P.scale);
    const uint2 sign = query_sign(P.scale);
    const int slots = P.slots_s + P.slots;
    uint32_t gi = 0, n_item = 0;
    bool ok = true;
    auto warp_arrive = [&](uint64_t* bar) {
      __syncwarp();
      if (lane == 0) mbar_arrive(bar);
    };
    for (int item = (int)blockIdx.x; item < items && ok; item += (int)gridDim.x) {
      const Item I = item_of<D, NT>(P, S, item);
      const int row = I.row0 + t * 128 + row_in;
      const int qi = row / P.per;
      const long long token = I.begin + qi;
      const int head = I.head * P.per + row - qi * P.per;
      {
        const uint4* src = reinterpret_cast<const uint4*>(
            static_cast<const bf16*>(A.q) + token * A.q_token_stride + (long long)head * A.q_head_stride);
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (row < I.rows) x = src[c];
          x.x = (x.x ^ sign.x) & sign.y;
          x.y = (x.y ^ sign.x) & sign.y;
          x.z = (x.z ^ sign.x) & sign.y;
          x.w = (x.w ^ sign.x) & sign.y;
          *reinterpret_cast<uint4*>(S.q[t] + (c / 8) * T::HALF_BYTES + row_in * 128 +
                                    (((c & 7) ^ (row_in & 7)) << 4)) = x;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        warp_arrive(&S.q_full);
      }
      const bool active = I.row0 + t * 128 + 32 * (warp % 4) < I.rows;  // some row of the warp exists
      float m = -INFINITY, l = 0.0f;  // m: what O and l are scaled by (log2)
      for (int i = 0; i < I.tiles && ok; ++i, ++gi) {
        const int b = T::NBUF == 2 ? (gi & 1) : 0;
        const uint32_t parity = T::NBUF == 2 ? (gi >> 1) & 1 : gi & 1;
        ok = __all_sync(0xffffffffu, wait(&S.s_full[t][b], parity, A.error_flags));
        if (!ok) break;
        fence_after();
        if (active) {
          const uint32_t scol = tmem + lanes + T::S_COL + uint32_t((T::NBUF == 2 ? b : t) * TILE_KEYS);
          const int keys = I.k1 - (I.k0 + i * TILE_KEYS);
          const uint32_t bad = S.bad[gi & 7];
          const bool partial = keys < TILE_KEYS || bad != 0;
          uint32_t x[2][32], p[TILE_KEYS / 2];
          // The next 32 scores are on their way from TMEM while these are used.
          // (Tiles with a mask have code of their own: a branch a chunk keeps the
          // compiler from overlapping the chunks.)
          auto scores = [&](auto masked, auto&& use) {
            tmem_ld32_async(scol, x[0]);
#pragma unroll
            for (int c = 0; c < TILE_KEYS / 32; ++c) {
              tmem_wait_ld(x[c & 1]);
              if (c + 1 < TILE_KEYS / 32) tmem_ld32_async(scol + (c + 1) * 32, x[(c + 1) & 1]);
              if constexpr (decltype(masked)::value) {
#pragma unroll
                for (int j = 0; j < 32; ++j)
                  if (c * 32 + j >= keys || ((bad >> ((c * 32 + j) / BOX_MIN)) & 1u))
                    x[c & 1][j] = 0xff800000u;  // -inf
              }
              use(c, x[c & 1]);
            }
          };
          auto set_m = [&]() {  // m: the row's largest score of this tile
            float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            scores(std::true_type{}, [&](int, const uint32_t (&v)[32]) {
#pragma unroll
              for (int j = 0; j < 32; ++j) top[j & 3] = fmaxf(top[j & 3], __uint_as_float(v[j]));
            });
            return fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
          };
          float part;      // sum of the weights
          auto weights = [&](auto masked) {
            const float base = m == -INFINITY ? 0.0f : m;
            const f2 sc2 = f2_make(scale, scale), nb2 = f2_make(-base, -base);
            f2 sum[2] = {f2_make(0.0f, 0.0f), f2_make(0.0f, 0.0f)};
            scores(masked, [&](int c, const uint32_t (&v)[32]) {
#pragma unroll
              for (int j = 0; j < 32; j += 2) {
                const float2 y =
                    f2_split(f2_fma(f2_make(__uint_as_float(v[j]), __uint_as_float(v[j + 1])), sc2, nb2));
                const float2 w = make_float2(exp2_approx(y.x), exp2_approx(y.y));
                sum[(j >> 1) & 1] = f2_add(sum[(j >> 1) & 1], f2_make(w.x, w.y));
                p[c * 16 + j / 2] = as_u32(pack2_rn(w));
              }
            });
            const float2 a = f2_split(f2_add(sum[0], sum[1]));
            part = a.x + a.y;
          };
          if (i == 0) m = set_m();
          if (partial) weights(std::true_type{});
          else weights(std::false_type{});
          if (i > 0) {
            // A sum above 2^RESCALE_LOG2 (the row's m is that far behind): the rare
            // tile where m moves, O and l follow, and the weights are made again.  So
            // too where no tile had a score yet: weights against 0 may all vanish.
            const bool grow = part > exp2_approx(RESCALE_LOG2) || m == -INFINITY;
            if (__any_sync(0xffffffffu, grow)) {
              float keep = 1.0f;
              const float mx = set_m();
              if (grow && mx > m) {
                keep = exp2_approx(m - mx);
                m = mx;
              }
              l *= keep;
              weights(std::true_type{});
              if constexpr (NT == 1) {
                ok = __all_sync(0xffffffffu, wait(&S.pv_done[t], (gi - 1) & 1, A.error_flags));
                if (!ok) break;
              }
              fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                const uint32_t col = tmem + lanes + T::O_COL + uint32_t(t * D + c * 32);
                tmem_ld32(col, o);
#pragma unroll
                for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * keep);
                tmem_st32(col, o);
              }
            }
          }
          l += part;
          tmem_st32(scol, p);
          tmem_st32(scol + 32, p + 32);
          tmem_wait_st();
        }
        fence_before();
        warp_arrive(&S.p_full[t][b]);
      }
      if (!ok) break;
      ok = __all_sync(0xffffffffu, wait(&S.o_done[t], n_item & 1, A.error_flags));
      ++n_item;
      if (!ok) break;
      fence_after();
      if (active) {
        const long long slot = (token * A.heads + head) * slots + I.chunk;
        if (row < I.rows) P.ml[slot] = make_float2(m, l);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(tmem + lanes + T::O_COL + uint32_t(t * D + c * 32), o);
          if (row < I.rows) {
            float4* dst = reinterpret_cast<float4*>(P.o + slot * D + c * 32);
#pragma unroll
            for (int j = 0; j < 8; ++j)
              dst[j] = make_float4(__uint_as_float(o[4 * j]), __uint_as_float(o[4 * j + 1]),
                                   __uint_as_float(o[4 * j + 2]), __uint_as_float(o[4 * j + 3]));
          }
        }
      }
      fence_before();
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 4 * NT) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                 "r"(T::TMEM_COLS)
                 : "memory");
  }
  if (NT == 1) {
    pdl_trigger();
    pdl_wait();  // the stream kernel: the join waits for this one alone
  }
}

// ---------------------------------------------------------------- host side
template <int D, int NT>
static int launch_tc(const Params& P, const CUtensorMap& k16, const CUtensorMap& v16, cudaStream_t st) {
  const hyena_paged_kv& kv = P.a.kv;
  int box = BOX_MIN;
  while (box < TILE_KEYS && kv.page_size % (2 * box) == 0) box *= 2;
  CUtensorMap k, v;
  int rc = cache_map(&k, kv, true, box);
  if (!rc) rc = cache_map(&v, kv, false, box);
  if (rc) return rc;
  const size_t smem = sizeof(TcSmem<D, NT>) + 1024;
  static_assert(sizeof(TcSmem<D, NT>) + 1024 <= 232448, "shared memory of a CTA");
  if (!smem_attr<shared_kernel<D, NT>>((int)smem))
    return fail(HYENA_ERR_CUDA, "cudaFuncSetAttribute(paged_attention shared) failed");
  launch_kernel(shared_kernel<D, NT>, dim3((unsigned)P.ctas), dim3(Tc<D, NT>::THREADS), smem, st, 0u, P,
                k, v, k16, v16, box);
  return check_launch("paged_attention shared");
}

int shared_launch(const Params& P, const CUtensorMap& k16, const CUtensorMap& v16, cudaStream_t st) {
  if (P.a.kv.head_dim == 128)
    return P.tc == 2 ? launch_tc<128, 2>(P, k16, v16, st) : launch_tc<128, 1>(P, k16, v16, st);
  return P.tc == 2 ? launch_tc<64, 2>(P, k16, v16, st) : launch_tc<64, 1>(P, k16, v16, st);
}

int shared_wait_timeouts(int32_t* count, int reset) { return read_wait_timeouts(count, reset); }

}  // namespace attn
}  // namespace hb
