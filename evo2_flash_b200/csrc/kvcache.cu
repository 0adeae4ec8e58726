// Appending a step's keys and values to the paged attention cache, with the
// rotary embedding of queries and keys on the way (hyena_kv_append): the
// rotation of Evo2Attention (model.py:104-152, neox halves) and the cache write
// that follows it, one pass over q, k and v.
//
//   a = x[i], b = x[i + D/2], i < D/2, at position p:
//   x'[i] = a cos(p f_i) - b sin(p f_i),  x'[i + D/2] = b cos(p f_i) + a sin(p f_i),
//   f_i = theta^(-2i/D)
//
// in fp32, rounded once to bf16 (the caches hold bf16, as every activation of
// the model).  The angle is formed in turns in fp64, t = p f_i / 2 pi, and
// reduced to t - rint(t) before it is narrowed: an fp32 p f_i is off by up to
// 2^-24 p radians, 0.06 at a position of one million.
//
// HBM-bound: 12 bytes an element pair of heads read and written once.  A block
// owns TB tokens, KV_THREADS / TB threads each; their cos / sin are formed once
// for all heads, in shared memory, and a thread, which stays with eight pairs of its
// token, keeps theirs in registers (16-byte accesses; the first head's loads under
// way before the cos / sin are formed).  TB is 1 up to 8 tokens an SM, so that short
// steps spread over the GPU, else 4.  65536 tokens of 32 heads take 495 us (499 at the
// measured copy rate), 4099 tokens of 32 query and 8 key/value heads 19-21 us (15.6),
// one token 3.3 us (a launch).  With cos / sin read from shared memory for every head:
// 509, 20 and 3.8 us; TB of 2 494, of 8 501 us; blocks of 128 threads 500, of 512 554.
#include <cmath>

#include "attention.cuh"

namespace hb {

constexpr int KV_THREADS = 256;
constexpr int KV_MAX_HALF = 64;  // head_dim / 2

struct KvAppendParams {
  hyena_kv_append_args a;
  double turns[KV_MAX_HALF];  // f_i / (2 pi)
};

// Page of `pos` of request r, or -1 (flagged) where the table does not have it.
__device__ __forceinline__ int page_of(const hyena_paged_kv& kv, int r, int page_index,
                                       int32_t* flags) {
  int page = -1;
  if (page_index < kv.pages_per_request)
    page = __ldg(kv.page_table + (long long)r * kv.page_table_stride + page_index);
  if (page < 0 || page >= kv.num_pages) {
    flag_error(flags, HYENA_FLAG_BLOCK_RANGE);
    return -1;
  }
  return page;
}

template <int TB>
__global__ void __launch_bounds__(KV_THREADS) kv_append_kernel(const __grid_constant__ KvAppendParams P) {
  __shared__ __align__(16) float2 cs[TB][KV_MAX_HALF];
  __shared__ long long koff[TB], voff[TB];  // element offset of the token's row; -1: not written
  __shared__ int live[TB];
  pdl_entry();
  const hyena_kv_append_args& A = P.a;
  const int tid = (int)threadIdx.x;
  const int half = A.kv.head_dim / 2;
  const long long t0 = (long long)blockIdx.x * TB;
  // A thread's items: 8 + 8 elements (piece `oct` of both halves) of every step-th
  // head of one token.
  constexpr int TPT = KV_THREADS / TB;
  const int oct_bits = half == 64 ? 3 : 2;  // 8-element pieces of a half
  const int tok = tid / TPT, oct = tid & ((1 << oct_bits) - 1), step = TPT >> oct_bits;
  const int hq = A.q != nullptr ? A.heads : 0, hkv = A.kv.kv_heads, all = hq + 2 * hkv;
  const int h0 = (tid % TPT) >> oct_bits;
  const long long t = t0 + tok;
  uint4 a, b;
  auto load = [&](int h) {
    if (h >= all || t >= A.T) return;
    const bf16* src;
    if (h < hq)
      src = static_cast<const bf16*>(A.q) + t * A.q_token_stride + h * A.q_head_stride;
    else if (h < hq + hkv)
      src = static_cast<const bf16*>(A.k) + t * A.k_token_stride + (h - hq) * A.k_head_stride;
    else
      src = static_cast<const bf16*>(A.v) + t * A.v_token_stride + (h - hq - hkv) * A.v_head_stride;
    a = *reinterpret_cast<const uint4*>(src + oct * 8);
    b = *reinterpret_cast<const uint4*>(src + half + oct * 8);
  };
  load(h0);  // before anything else: it waits for nothing but the previous kernel

  if (tid < TB) {
    const long long t = t0 + tid;
    int ok = 0;
    long long ko = -1, vo = -1;
    if (t < A.T) {
      int r = (int)t;
      bool owned = r < A.num_requests;
      if (A.query_start_loc != nullptr) {
        r = find_segment(A.query_start_loc, A.num_requests, (int)t);
        owned = __ldg(A.query_start_loc + r) <= t && t < __ldg(A.query_start_loc + r + 1);
      }
      const int pos = owned ? __ldg(A.positions + t) : -1;
      if (pos >= 0) {
        ok = 1;
        const int pi = pos / A.kv.page_size, at = pos - pi * A.kv.page_size;
        const int page = page_of(A.kv, r, pi, A.error_flags);
        if (page >= 0) {
          ko = page * A.kv.k_page_stride + at * A.kv.k_token_stride;
          vo = page * A.kv.v_page_stride + at * A.kv.v_token_stride;
        }
      }
    }
    live[tid] = ok;
    koff[tid] = ko;
    voff[tid] = vo;
  }
  for (int i = tid; i < TB * half; i += KV_THREADS) {
    const int k = i / half, p = i - k * half;
    if (t0 + k < A.T) {
      const double turn = (double)__ldg(A.positions + t0 + k) * P.turns[p];
      float s, c;
      sincospif(2.0f * (float)(turn - rint(turn)), &s, &c);
      cs[k][p] = make_float2(c, s);
    }
  }
  __syncthreads();

  if (!live[tok]) return;
  float4 rot[4];  // cos, sin of this thread's pairs
#pragma unroll
  for (int w = 0; w < 4; ++w) rot[w] = reinterpret_cast<const float4*>(&cs[tok][oct * 8])[w];
  for (int h = h0; h < all; h += step) {
    if (h != h0) load(h);
    bf16* dst;
    if (h < hq) {
      dst = static_cast<bf16*>(A.q_out) + t * A.q_out_token_stride + h * A.q_out_head_stride;
    } else if (h < hq + hkv) {
      if (koff[tok] < 0) continue;
      dst = static_cast<bf16*>(A.kv.k) + koff[tok] + (h - hq) * A.kv.k_head_stride;
    } else {
      if (voff[tok] < 0) continue;
      dst = static_cast<bf16*>(A.kv.v) + voff[tok] + (h - hq - hkv) * A.kv.v_head_stride;
    }
    if (h < hq + hkv) {
      uint32_t* aw = reinterpret_cast<uint32_t*>(&a);
      uint32_t* bw = reinterpret_cast<uint32_t*>(&b);
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float4 r = rot[w];
        const float2 x = unpack2(as_bf162(aw[w])), y = unpack2(as_bf162(bw[w]));
        aw[w] = as_u32(pack2_rn(make_float2(x.x * r.x - y.x * r.y, x.y * r.z - y.y * r.w)));
        bw[w] = as_u32(pack2_rn(make_float2(y.x * r.x + x.x * r.y, y.y * r.z + x.y * r.w)));
      }
    }
    *reinterpret_cast<uint4*>(dst + oct * 8) = a;
    *reinterpret_cast<uint4*>(dst + half + oct * 8) = b;
  }
}

int check_paged_kv(const hyena_paged_kv& kv) {
  HB_REQUIRE(kv.k != nullptr && kv.v != nullptr && kv.page_table != nullptr, "paged cache: null pointer");
  HB_REQUIRE(aligned16(kv.k) && aligned16(kv.v), "paged cache: k / v must be 16-byte aligned");
  HB_REQUIRE(kv.k_page_stride % 8 == 0 && kv.k_token_stride % 8 == 0 && kv.k_head_stride % 8 == 0 &&
                 kv.v_page_stride % 8 == 0 && kv.v_token_stride % 8 == 0 && kv.v_head_stride % 8 == 0,
             "paged cache: strides must be multiples of 8 elements");
  HB_REQUIRE(kv.page_size > 0 && kv.page_size % 16 == 0, "paged cache: page_size must be a positive multiple of 16");
  HB_REQUIRE(kv.num_pages > 0 && kv.pages_per_request > 0 && kv.page_table_stride >= 0,
             "paged cache: no pages");
  HB_REQUIRE((long long)kv.pages_per_request * kv.page_size < (1ll << 31) - 65536,
             "paged cache: a request's pages must hold fewer than 2^31 - 65536 positions");
  HB_REQUIRE(kv.kv_heads > 0, "paged cache: kv_heads must be positive");
  HB_REQUIRE(kv.head_dim == 64 || kv.head_dim == 128, "paged cache: head_dim must be 64 or 128");
  return HYENA_OK;
}

int kv_append_launch(const hyena_kv_append_args& A, cudaStream_t st) {
  HB_REQUIRE(A.T >= 0 && A.num_requests >= 0, "kv_append: negative sizes");
  if (A.T == 0 || A.num_requests == 0) return HYENA_OK;
  const int rc = check_paged_kv(A.kv);
  if (rc) return rc;
  HB_REQUIRE(A.k && A.v && A.positions, "kv_append: null pointer");
  HB_REQUIRE((A.q == nullptr) == (A.q_out == nullptr), "kv_append: q and q_out go together");
  HB_REQUIRE(A.q == nullptr || A.heads > 0, "kv_append: heads must be positive");
  HB_REQUIRE(aligned16(A.q) && aligned16(A.q_out) && aligned16(A.k) && aligned16(A.v),
             "kv_append: q, k, v must be 16-byte aligned");
  HB_REQUIRE(A.q_token_stride % 8 == 0 && A.q_head_stride % 8 == 0 && A.q_out_token_stride % 8 == 0 &&
                 A.q_out_head_stride % 8 == 0 && A.k_token_stride % 8 == 0 && A.k_head_stride % 8 == 0 &&
                 A.v_token_stride % 8 == 0 && A.v_head_stride % 8 == 0,
             "kv_append: strides must be multiples of 8 elements");
  HB_REQUIRE(A.rope_theta > 0.0 && std::isfinite(A.rope_theta), "kv_append: rope_theta must be positive");
  KvAppendParams P;
  P.a = A;
  const int half = A.kv.head_dim / 2;
  const double step = std::pow(A.rope_theta, -1.0 / half);
  double f = 1.0 / (2.0 * 3.14159265358979323846);
  for (int i = 0; i < half; ++i, f *= step) P.turns[i] = f;
  // One token a block until the GPU has a few blocks an SM, then four.
  if (A.T <= 8 * num_sms()) {
    launch_kernel(kv_append_kernel<1>, dim3((unsigned)A.T), dim3(KV_THREADS), 0, st, 0u, P);
  } else {
    launch_kernel(kv_append_kernel<4>, dim3((unsigned)((A.T + 3) / 4)), dim3(KV_THREADS), 0, st, 0u, P);
  }
  return check_launch("kv_append_kernel");
}

}  // namespace hb
