// Rotary positions: q rotated, k rotated and stored with v in the pages of a
// paged cache that the tokens' slots name.
//
// Pair i of a head, (x0, x1), at position n becomes (x0 cos a - x1 sin a,
// x1 cos a + x0 sin a) times a factor, a = 2 pi turns_i n. The angle is formed
// in turns in 64 bits, where its whole part can be dropped exactly, and only
// the remaining part of a turn is taken to 32 bits: half an ulp of it is
// 2^-26 turns however far the position. Everything after that is 32-bit, rounded once to the 16-bit
// result.
//
// Bound by memory: q is read and written, k and v read and written, once. 8
// threads take a (token, head) row of 128 dims, 16 dims each, in two 16-byte
// pieces: the dims of thread j's 8 pairs are dims 8j .. and rotary/2 + 8j ..
// (halves) or 16j .. 16j + 15 (interleaved). The 8 angles of a thread depend on
// the token alone, so with many tokens a thread keeps them for several heads.
// 40007 tokens of 32 + 2 x 8 heads (984 MB) take 214 us, 4.6 TB/s, a large copy's
// rate; 48 tokens 3.4 us, the launch.

#include "serve_common.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int ROTARY_THREADS = 256;
constexpr int ROW_THREADS = 8;              // threads of a (token, head) row

struct RotaryArgs {
  const uint16_t *q, *k, *v;
  uint16_t *q_out, *k_cache, *v_cache;
  const int *positions, *slots;
  const double* turns;
  int64_t qs[2], os[2], ks[2], vs[2];       // strides of tokens and heads
  int64_t kc[3], vc[3];                     // of pages, tokens and heads
  int64_t slots_all;                        // slots of the cache
  int tokens, heads_q, heads_kv, half, shift, heads_each;
  float factor, sign;
};

template <bool BF>
__device__ __forceinline__ float widen(uint16_t x) {
  if constexpr (BF)
    return __uint_as_float((uint32_t)x << 16);
  else
    return (float)__builtin_bit_cast(_Float16, x);
}
template <bool BF>
__device__ __forceinline__ uint16_t narrow(float x) {
  if constexpr (BF)
    return __builtin_bit_cast(uint16_t, (__bf16)x);
  else
    return __builtin_bit_cast(uint16_t, (_Float16)x);
}

union Piece {
  u32x4 words;
  uint16_t x[8];
};

template <bool BF, bool HALF>
__global__ void __launch_bounds__(ROTARY_THREADS) fa_serve_rotary_kernel(RotaryArgs a) {
  const int64_t unit = ((int64_t)blockIdx.x * ROTARY_THREADS + threadIdx.x) / ROW_THREADS;
  const int j = threadIdx.x % ROW_THREADS;
  if (unit >= a.tokens) return;
  const int64_t t = unit;
  const int heads = a.heads_q + 2 * a.heads_kv;
  const int h0 = blockIdx.y * a.heads_each, h1 = min(heads, h0 + a.heads_each);
  // This thread's pairs 8j .. 8j + 7, and the dims of its two pieces. Threads
  // past the rotated pairs copy 16 of the dims that stay.
  const bool turned = 8 * j < a.half;
  const int lo = HALF && turned ? 8 * j : 16 * j;
  const int hi = HALF && turned ? a.half + 8 * j : 16 * j + 8;
  float c[8], s[8];
  if (turned && h0 < a.heads_q + a.heads_kv) {
    const double n = a.positions[t];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      double turn = n * a.turns[8 * j + i];
      turn -= rint(turn);
      float sn, cs;
      sincospif(2.f * (float)turn, &sn, &cs);
      c[i] = cs * a.factor;
      s[i] = sn * (a.factor * a.sign);
    }
  }
  const int64_t slot = a.heads_kv ? a.slots[t] : -1;
  const bool stored = slot >= 0 && slot < a.slots_all;
  const int64_t page = slot >> a.shift, in_page = slot & (((int64_t)1 << a.shift) - 1);
  for (int h = h0; h < h1; ++h) {
    const uint16_t* src;
    uint16_t* dst;
    bool rotate = turned;
    if (h < a.heads_q) {
      src = a.q + t * a.qs[0] + h * a.qs[1];
      dst = a.q_out + t * a.os[0] + h * a.os[1];
    } else if (!stored) {
      break;
    } else if (h < a.heads_q + a.heads_kv) {
      const int hk = h - a.heads_q;
      src = a.k + t * a.ks[0] + hk * a.ks[1];
      dst = a.k_cache + page * a.kc[0] + in_page * a.kc[1] + hk * a.kc[2];
    } else {
      const int hk = h - a.heads_q - a.heads_kv;
      src = a.v + t * a.vs[0] + hk * a.vs[1];
      dst = a.v_cache + page * a.vc[0] + in_page * a.vc[1] + hk * a.vc[2];
      rotate = false;
    }
    Piece x0, x1;
    x0.words = *reinterpret_cast<const u32x4*>(src + lo);
    x1.words = *reinterpret_cast<const u32x4*>(src + hi);
    if (rotate) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        // Pair i: one element of each piece, or two neighbours of one.
        uint16_t* const e0 = HALF ? &x0.x[i] : i < 4 ? &x0.x[2 * i] : &x1.x[2 * i - 8];
        uint16_t* const e1 = HALF ? &x1.x[i] : e0 + 1;
        const float u = widen<BF>(*e0), w = widen<BF>(*e1);
        *e0 = narrow<BF>(__builtin_fmaf(u, c[i], -(w * s[i])));
        *e1 = narrow<BF>(__builtin_fmaf(w, c[i], u * s[i]));
      }
    }
    *reinterpret_cast<u32x4*>(dst + lo) = x0.words;
    *reinterpret_cast<u32x4*>(dst + hi) = x1.words;
  }
}

// Threads a launch should have before a thread takes more than one head. With one, 16 and
// this number of heads a thread (12 + 2 heads or 32 + 16): 300 tokens 4.0, 8.4 and 4.1 us;
// 8000 tokens 14.6, 14.0 and 12.2; 40007 tokens of 48 heads 227, 216 and 215.
constexpr int64_t ROTARY_WIDE = 256 * 1024;

}  // namespace

extern "C" {

int fa_rotary_append(const fa_rotary* p, const void* q, void* q_out, const void* k, const void* v,
                     const int32_t* positions, const int32_t* slots, const double* turns,
                     void* k_cache, void* v_cache, void* stream) {
  if (!p) return FA_SERVE_ERR_NULL;
  const int64_t limit = (int64_t)1 << 30;
  // 8 threads a token, and fewer than 2^32 threads in a dimension of a launch.
  if (p->tokens < 0 || p->tokens > limit / 4 || p->heads_q < 0 || p->heads_kv < 0 || p->heads_q > 4096 ||
      p->heads_kv > 4096 || p->heads_q + p->heads_kv < 1)
    return FA_SERVE_ERR_GEOMETRY;
  if (p->type != FA_SERVE_FP16 && p->type != FA_SERVE_BF16) return FA_SERVE_ERR_TYPE;
  if (p->rotary_dim < 16 || p->rotary_dim > 128 || p->rotary_dim % 16 ||
      (p->layout != FA_ROTARY_HALF && p->layout != FA_ROTARY_INTERLEAVED))
    return FA_SERVE_ERR_ROTARY;
  int shift = 0;
  int rc = check_strides(p->q, 2);
  if (!rc) rc = check_strides(p->q_out, 2);
  if (p->heads_kv) {
    shift = page_shift(p->page_size);
    if (shift < 0) return FA_SERVE_ERR_PAGE;
    if (p->pages < 0 || p->pages > limit) return FA_SERVE_ERR_GEOMETRY;
    for (const int64_t* s : {p->k, p->v})
      if (!rc) rc = check_strides(s, 2);
    for (const int64_t* s : {p->k_cache, p->v_cache})
      if (!rc) rc = check_strides(s, 3);
  }
  if (rc) return rc;
  if (p->tokens == 0) return FA_SERVE_OK;
  if (!positions || !turns || (p->heads_q && (!q || !q_out)) ||
      (p->heads_kv && (!k || !v || !slots || !k_cache || !v_cache)))
    return FA_SERVE_ERR_NULL;
  for (const void* ptr : {q, (const void*)q_out, k, v, (const void*)k_cache, (const void*)v_cache})
    if (!aligned(ptr, 16)) return FA_SERVE_ERR_ALIGN;
  if (!aligned(positions, 4) || !aligned(slots, 4) || !aligned(turns, 8)) return FA_SERVE_ERR_ALIGN;
  rc = check_stream_device(stream);
  if (rc) return rc;
  RotaryArgs a{};
  a.q = static_cast<const uint16_t*>(q);
  a.k = static_cast<const uint16_t*>(k);
  a.v = static_cast<const uint16_t*>(v);
  a.q_out = static_cast<uint16_t*>(q_out);
  a.k_cache = static_cast<uint16_t*>(k_cache);
  a.v_cache = static_cast<uint16_t*>(v_cache);
  a.positions = positions;
  a.slots = slots;
  a.turns = turns;
  memcpy(a.qs, p->q, sizeof(a.qs));
  memcpy(a.os, p->q_out, sizeof(a.os));
  memcpy(a.ks, p->k, sizeof(a.ks));
  memcpy(a.vs, p->v, sizeof(a.vs));
  memcpy(a.kc, p->k_cache, sizeof(a.kc));
  memcpy(a.vc, p->v_cache, sizeof(a.vc));
  a.slots_all = p->heads_kv ? p->pages << shift : 0;
  a.tokens = (int)p->tokens;
  a.heads_q = (int)p->heads_q;
  a.heads_kv = (int)p->heads_kv;
  a.half = (int)p->rotary_dim / 2;
  a.shift = shift;
  a.factor = p->factor;
  a.sign = p->backward ? -1.f : 1.f;
  const int64_t heads = p->heads_q + 2 * p->heads_kv;
  int64_t each = p->tokens * ROW_THREADS * heads / ROTARY_WIDE;
  each = each < 1 ? 1 : each > 16 ? 16 : each;
  a.heads_each = (int)each;
  void* args[] = {&a};
  const dim3 grid((unsigned)((p->tokens * ROW_THREADS + ROTARY_THREADS - 1) / ROTARY_THREADS),
                  (unsigned)((heads + each - 1) / each));
  const bool bf = p->type == FA_SERVE_BF16, half = p->layout == FA_ROTARY_HALF;
  const void* fn = bf ? half ? reinterpret_cast<const void*>(&fa_serve_rotary_kernel<true, true>)
                             : reinterpret_cast<const void*>(&fa_serve_rotary_kernel<true, false>)
                   : half ? reinterpret_cast<const void*>(&fa_serve_rotary_kernel<false, true>)
                          : reinterpret_cast<const void*>(&fa_serve_rotary_kernel<false, false>);
  return enqueue(fn, grid, dim3(ROTARY_THREADS), args, 0, stream);
}

}  // extern "C"
