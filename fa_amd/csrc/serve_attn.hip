// Attention of new tokens over a paged cache, and with a causal sliding window
// and sinks, paged or contiguous: GQA, 128 dims, FP16 or BF16, FP32 softmax
// statistics and O.
//
// A request has n new rows per head behind its earlier keys; row i stands at
// position p and sees key j iff j <= p and (j > p - W or j < S). One pass over
// the keys per row, with the running maximum m and sum l of the softmax (base
// 2, scale folded in, c = scale log2 e):
//   m' = max(m, max_j s_j), a = 2^((m - m') c), P_j = 2^(s_j c - m' c),
//   l' = a l + sum_j P_j, O' = a O + sum_j P_j v_j,
// at the end o = O / l, lse = ln l + scale m.
//
// Rows are packed: the n * group rows of the query heads that share a KV head
// form one sequence, position by position, of which a tile is a run of
// consecutive rows. A tile needs keys [0, min(S, hi)) and [lo, hi), lo the first key
// its first row's window holds and hi one past its last row's position: a list
// of 128-key blocks, the blocks that all its rows see whole and those that take
// the mask. A block's keys may lie in any pages: the loads from a 16-key
// group, which no page end cuts, go through a buffer descriptor of its own,
// with the page's address as a 64-bit base and its range ending behind the
// request's last key. So caches may be of any size, and what lies behind the
// last key is never read: it arrives in LDS as zeros.
//
// Matrix products run transposed, S^T = K Q^T and O^T += V^T P^T, so that a lane
// holds one row's scores and sums; the P^T operand is the S^T registers,
// converted, and V^T comes from V in its natural layout through transposing LDS
// reads (v_mfma 32x32x16, ds_read_b64_tr_b16; operand layouts at `Fragments`).
//
// A key that the mask hides has its score replaced by -inf, so NaN in its K has
// no effect; NaN or an infinity in its V would get into O through the product
// 0 * NaN in the blocks that take the mask. That is found at the end (l is a
// number and O is not) and the row computed again key by key, if no visible key
// accounts for the NaN (spoiled_row, repair_row).

#include <math.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>

#include "fa_device.h"
#include "serve_common.h"

namespace {

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

constexpr int HD = 128;
constexpr int ROW_BYTES = HD * 2;
constexpr int BLOCK = 128;                  // keys of a block of the lists below
constexpr double LOG2E = 1.4426950408889634;
constexpr float LN2 = 0.6931471805599453f;
constexpr int NO_WINDOW = 1 << 30;
constexpr int kUncut = 1 << 30;
// The maximum is raised when a score exceeds it by more than this (in powers of
// two), so P <= 2^8 and O is rescaled rarely.
constexpr float TAU = 8.f;

struct AttnArgs {
  const char *q, *k, *v;
  char* o;
  float* lse;
  const int *table, *starts, *lengths;      // paged; null: contiguous
  int64_t table_stride;
  int64_t qs_b, qs_n, qs_h, os_b, os_n, os_h;             // byte strides of q and o
  int64_t ks_b, vs_b, ks_h, vs_h;                         // of a page (or batch entry), a head
  int ks_n, vs_n;                                         // of a key
  int64_t ls_b, ls_n, ls_h;                               // strides of lse
  int batch, heads_kv, group, tokens, pages, shift, max_pages;
  int seq_q, seq_k, off;                    // contiguous: lengths, position of row 0
  int window, sinks;
  float c;
  int rows_max;                             // packed rows of a request that the row kernel takes
  int split;                                // tile kernel: there is room for parts
  int length;                               // contiguous: blocks of a part (uncut: kUncut)
  int tile_groups;                          // workgroups of the tile kernel that take tiles
  float *opart, *lpart;                     // row kernel's parts
  int* desc;
  float *topart, *tlpart;                   // tile kernel's parts
  int* tdesc;
  int groups;                               // workgroups of the row kernel
};

// The kernel's arguments through an address that the compiler cannot follow: read
// again where they are needed instead of staying in scalar registers (or spilling)
// across a key loop.
typedef const AttnArgs __attribute__((address_space(4))) ConstArgs;
__device__ __forceinline__ ConstArgs& fresh_args() {
  uint64_t addr = reinterpret_cast<uint64_t>(__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(addr));
  return *reinterpret_cast<ConstArgs*>(addr);
}

// A value every lane of the wave has, in a scalar register (integer divisions, for
// one, are made in vector registers).
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ uint32_t uniform(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

// Sum over this lane and the lanes before it.
__device__ __forceinline__ uint32_t lanes_sum(uint32_t x) {
#define ADD_DPP(ctrl, rows) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rows, 0xf, false)
  ADD_DPP(0x111, 0xf);                      // row_shr 1, 2, 4, 8: within 16 lanes
  ADD_DPP(0x112, 0xf);
  ADD_DPP(0x114, 0xf);
  ADD_DPP(0x118, 0xf);
  ADD_DPP(0x142, 0xa);                      // the last of a row to the next one
  ADD_DPP(0x143, 0xc);                      // and of the lower to the upper half
#undef ADD_DPP
  return x;
}

// A batch entry: the first of its rows in q, their number, the position of
// row 0, its keys, and whether its table row is too short for them.
struct Request {
  int row0, n, pos, keys, bad;
};
template <bool PAGED>
__host__ __device__ __forceinline__ Request request(const AttnArgs& a, int b) {
  Request r;
  if constexpr (PAGED) {
    const int s0 = min(max(a.starts[b], 0), a.tokens), s1 = min(max(a.starts[b + 1], s0), a.tokens);
    const int len = max(a.lengths[b], 0);
    const int64_t cap = (int64_t)a.max_pages << a.shift;
    r.row0 = s0;
    r.n = s1 - s0;
    r.pos = len - r.n;
    r.bad = len > cap;
    r.keys = r.bad ? (int)cap : len;
  } else {
    r.row0 = 0;
    r.n = a.seq_q;
    r.pos = a.off;
    r.keys = a.seq_k;
    r.bad = 0;
  }
  return r;
}

// The request of a whole workgroup, in scalar registers: descriptors and loop
// bounds are made from it.
__device__ __forceinline__ Request uniform(const Request& r) {
  return Request{uniform(r.row0), uniform(r.n), uniform(r.pos), uniform(r.keys), uniform(r.bad)};
}

// The key blocks that rows at positions first .. last see: blocks [0, ns) and
// [w0, w1), of which [f0, f1) (within [w0, w1)) are seen whole by every row.
struct Blocks {
  int ns, w0, w1, f0, f1;
  __host__ __device__ __forceinline__ int total() const { return ns + w1 - w0; }
};
__host__ __device__ __forceinline__ Blocks blocks(const AttnArgs& a, const Request& r, int first, int last) {
  Blocks k;
  const int hi = min(last + 1, r.keys);
  if (hi <= 0) return Blocks{0, 0, 0, 0, 0};
  const int lo = min(max(first - a.window + 1, 0), hi);
  k.w0 = lo / BLOCK;
  k.w1 = (hi + BLOCK - 1) / BLOCK;
  if (lo == hi) k.w0 = k.w1;
  k.ns = min((min(a.sinks, hi) + BLOCK - 1) / BLOCK, k.w0);
  // Whole for all: from the last row's window start to the first row's position.
  const int full_hi = min(first + 1, r.keys), full_lo = max(last - a.window + 1, 0);
  k.f0 = min(max((full_lo + BLOCK - 1) / BLOCK, k.w0), k.w1);
  k.f1 = max(min(full_hi > 0 ? full_hi / BLOCK : 0, k.w1), k.f0);
  return k;
}

// ---------------------------------------------------------------------------
// Fragments. The 32x32 output layout gives lane l column l % 32 and rows
// 8g + 4(l / 32) + e (register 4g + e): of S^T, query row l % 32 and those keys.
// The PV step over keys 16s .. 16s + 15 takes P^T from registers 8s .. 8s + 7
// converted, so its k slots 8h .. 8h + 7 (h = l / 32) hold keys 16s + 4h + {0..3}
// and 16s + 8 + 4h + {0..3}; the V^T operand follows that order with two
// transposing reads of 4 keys each.
template <bool BF>
__device__ __forceinline__ f32x16 mma(h8 x, h8 y, f32x16 acc) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b8, x), __builtin_bit_cast(b8, y), acc,
                                                   0, 0, 0);
  else
    return mfma32(x, y, acc);
}
// Two probabilities rounded to the element type (the matrix operand), as one word.
// l sums them unrounded: it becomes the FP32 log-sum-exp, and rounding P to 8 or
// 11 bits leaves O = sum P16 v / l off by at most half a step of the type times
// sum P |v| / l, the size of its own rounding at the end.
template <bool BF>
__device__ __forceinline__ uint32_t pack_p(float p0, float p1) {
  if constexpr (BF)
    return __builtin_bit_cast(uint32_t, b2{(__bf16)p0, (__bf16)p1});
  else
    return __builtin_bit_cast(uint32_t, h2{(_Float16)p0, (_Float16)p1});
}
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

// Ones in the low n bits, n from anything below 0 to anything above 32.
__device__ __forceinline__ uint32_t low_bits(int n) {
  return (uint32_t)(((uint64_t)1 << min(max(n, 0), 32)) - 1);
}
// Replaces the scores of the keys a row does not see by -inf: those past hi, and those
// that are neither from lo on nor before sink, all relative to the lane's first key
// (register r of 32-key tile t holds key 32t + 8 (r / 4) + r % 4 from there). The
// keys of a tile become a word with a bit for each key seen, of which a score takes its own:
// two instructions a score. Compares and selects would keep a scalar register
// pair a score alive; sign arithmetic with its three differences a score made a
// block with the mask take 2.3 us longer than one without.
template <int T>
__device__ __forceinline__ void hide(f32x16 (&s)[T], int hi, int lo, int sink) {
#pragma unroll
  for (int t = 0; t < T; ++t) {
    const uint32_t seen = low_bits(hi + 1 - 32 * t) & (~low_bits(lo - 32 * t) | low_bits(sink - 32 * t));
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const uint32_t keep = (uint32_t)__builtin_amdgcn_sbfe((int)seen, 8 * (r >> 2) + (r & 3), 1);
      s[t][r] = __uint_as_float((__float_as_uint(s[t][r]) & keep) | (0xff800000u & ~keep));
    }
  }
}

// One step of the online softmax over 16 T scores of the lane's row (the other
// half of the keys is with lane + 32): raises m, rescales l and O if some row of
// the wave needs it, and turns the scores into P fragments. at(i) runs before
// the exponentials of pair i.
template <bool BF, int T, typename At>
__device__ __forceinline__ void softmax_step(f32x16 (&s)[T], h8 (&p)[2 * T], float& m, float& l,
                                             f32x16 (&acc)[4], float c, At&& at) {
  float mv[16 * T];
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int r = 0; r < 16; ++r) mv[16 * t + r] = s[t][r];
#pragma unroll
  for (int n = 16 * T; n > 1; n = (n + 2) / 3) {
#pragma unroll
    for (int i = 0; 3 * i < n; ++i) {
      float x = mv[3 * i];
      if (3 * i + 1 < n) x = smax(x, mv[3 * i + 1]);
      if (3 * i + 2 < n) x = smax(x, mv[3 * i + 2]);
      mv[i] = x;
    }
  }
  const float mx = half_max(mv[0]);
  // False where both are -inf (no key seen yet) and for NaN, which then shows in P.
  const bool need = (mx - m) * c > TAU;
  if (__builtin_amdgcn_ballot_w64(need)) {
    const float alpha = need ? __builtin_amdgcn_exp2f((m - mx) * c) : 1.f;
    m = need ? mx : m;
    l *= alpha;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) acc[dt] *= alpha;
  }
  const float mc = m == -INFINITY ? 0.f : m * c;
  float ls[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      u32x4 frag;
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        at((2 * t + g) * 4 + e / 2);
        const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][8 * g + e], c, -mc));
        const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][8 * g + e + 1], c, -mc));
        frag[e / 2] = pack_p<BF>(p0, p1);
        ls[e & 2] += p0;
        ls[(e & 2) + 1] += p1;
      }
      p[2 * t + g] = __builtin_bit_cast(h8, frag);
    }
  l += (ls[0] + ls[1]) + (ls[2] + ls[3]);
}

// Keys of one KV head of a request: descriptors for the loads of a 16-key group.
template <bool PAGED>
struct Stream {
  const char *k, *v;                        // of the head
  const int __attribute__((address_space(4)))* table;     // the request's row
  uint32_t ks_b, vs_b;
  int ks_n, vs_n, keys, pages, shift;
  __device__ __forceinline__ Stream(const AttnArgs& a, const Request& r, int b, int hk) {
    k = a.k + hk * a.ks_h;
    v = a.v + hk * a.vs_h;
    if constexpr (PAGED) {
      table = (const int __attribute__((address_space(4)))*)(uintptr_t)(a.table + b * a.table_stride);
      ks_b = (uint32_t)a.ks_b;
      vs_b = (uint32_t)a.vs_b;
    } else {
      k += b * a.ks_b;
      v += b * a.vs_b;
    }
    ks_n = a.ks_n;
    vs_n = a.vs_n;
    keys = r.keys;
    pages = a.pages;
    shift = a.shift;
  }
  // The page of the group at `key` (for a group past the last key, of that key).
  __device__ __forceinline__ int page(int key) const {
    if constexpr (PAGED)
      return table[max(min(key, keys - 1), 0) >> shift];
    else
      return 0;
  }
  // Keys of the group at `key` that may be read: none if the page does not exist.
  __device__ __forceinline__ int valid(int key, int id) const {
    int n = min(max(keys - key, 0), 16);
    if constexpr (PAGED) n = (uint32_t)id < (uint32_t)pages ? n : 0;
    return n;
  }
  __device__ __forceinline__ bool missing(int key, int id) const {
    return PAGED && key < keys && (uint32_t)id >= (uint32_t)pages;
  }
  // Without a branch: a range of 0 fetches nothing, whatever the base.
  __device__ __forceinline__ i32x4 rsrc(const char* base, uint32_t page_bytes, int pitch, int key, int id) const {
    const int n = valid(key, id);
    if constexpr (PAGED)
      base += (uint64_t)(uint32_t)id * page_bytes + (uint64_t)(uint32_t)(key & ((1 << shift) - 1)) * (uint32_t)pitch;
    else
      base += (int64_t)key * pitch;
    const int range = (n - 1) * pitch + ROW_BYTES;
    const i32x4 rs = buffer_rsrc(base, n > 0 ? range : 0);
    return i32x4{uniform(rs[0]), uniform(rs[1]), uniform(rs[2]), rs[3]};
  }
  __device__ __forceinline__ i32x4 k_rsrc(int key, int id) const { return rsrc(k, ks_b, ks_n, key, id); }
  __device__ __forceinline__ i32x4 v_rsrc(int key, int id) const { return rsrc(v, vs_b, vs_n, key, id); }
  // A key's row (a key the request has, in a page that exists).
  __device__ __forceinline__ int64_t at(int key, int64_t page_bytes, int pitch) const {
    if constexpr (PAGED)
      return table[key >> shift] * page_bytes + (int64_t)(key & ((1 << shift) - 1)) * pitch;
    else
      return (int64_t)key * pitch;
  }
};

// Exponent all ones: infinity or NaN, in the lower (1) and the upper (2) element of a word.
template <bool BF>
__device__ __forceinline__ int not_finite(uint32_t w) {
  constexpr uint32_t E = BF ? 0x7f80u : 0x7c00u;
  return ((w & E) == E ? 1 : 0) | ((w >> 16 & E) == E ? 2 : 0);
}

// Whether a row whose O has NaN in it must be computed again: some dim has infinity or
// NaN in the V of a key that the row does not see (in the blocks [s0, s1) of a list, which
// it was computed from), and the keys that it sees hold neither NaN nor infinities of both
// signs there, which would be the row's own NaN. The whole wave works on one row, 2 dims
// a lane. Both passes end early: a V that is NaN all over costs a row a few keys.
template <bool BF, bool PAGED, typename Args, typename BlockAt>
__device__ __forceinline__ bool spoiled_row(const Args& a, const Stream<PAGED>& st, int pos, int s0, int s1,
                                            BlockAt&& block_at) {
  constexpr int STEP = 4;                   // keys whose loads are in flight together
  const int lane = threadIdx.x & 63;
  const int hi = min(pos, st.keys - 1);
  int hidden = 0;                           // dims (a bit each) not finite at a hidden key
  float seen[2] = {0.f, 0.f};               // the sum of what is not finite at visible ones
  for (int pass = 0; pass < 2; ++pass) {
    for (int s = s0; s < s1; ++s) {
      const int key0 = block_at(s) * BLOCK;
      if (pass == 0 && key0 + BLOCK - 1 <= hi && (key0 > pos - a.window || key0 + BLOCK <= a.sinks)) continue;
      for (int key = key0; key < key0 + BLOCK && key < st.keys; key += STEP) {
        uint32_t w[STEP];
#pragma unroll
        for (int e = 0; e < STEP; ++e)
          w[e] = *reinterpret_cast<const uint32_t*>(st.v + st.at(min(key + e, st.keys - 1), a.vs_b, a.vs_n) + 4 * lane);
#pragma unroll
        for (int e = 0; e < STEP; ++e) {
          if (key + e >= st.keys) continue;
          const bool visible = key + e <= hi && (key + e > pos - a.window || key + e < a.sinks);
          const int odd = not_finite<BF>(w[e]);
          if (!visible) {
            hidden |= odd;
          } else if (pass) {
            seen[0] += odd & 1 ? widen<BF>((uint16_t)w[e]) : 0.f;
            seen[1] += odd & 2 ? widen<BF>((uint16_t)(w[e] >> 16)) : 0.f;
          }
        }
        const int left = hidden & ((seen[0] == seen[0] ? 1 : 0) | (seen[1] == seen[1] ? 2 : 0));
        if (pass && !__builtin_amdgcn_ballot_w64(left != 0)) return false;
      }
    }
    if (!pass && !__builtin_amdgcn_ballot_w64(hidden != 0)) return false;
  }
  return true;
}

// A row again, one key at a time, over the blocks [s0, s1) of a list: o (dims
// 2 lane, 2 lane + 1) and lse of the keys it sees, which alone are read; for the rare
// rows that spoiled_row finds.
template <bool BF, bool PAGED, typename Args, typename BlockAt>
__device__ __forceinline__ void repair_row(const Args& a, const Stream<PAGED>& st, const char* qrow, int pos,
                                           int s0, int s1, BlockAt&& block_at, float (&o)[2], float& lse) {
  const int lane = threadIdx.x & 63;
  const uint32_t qw = *reinterpret_cast<const uint32_t*>(qrow + 4 * lane);
  const float q0 = widen<BF>((uint16_t)qw), q1 = widen<BF>((uint16_t)(qw >> 16));
  float m = -INFINITY, l = 0.f;
  o[0] = o[1] = 0.f;
  const int hi = min(pos, st.keys - 1);
  for (int s = s0; s < s1; ++s) {
    const int key0 = block_at(s) * BLOCK;
    for (int key = key0; key < key0 + BLOCK && key <= hi; ++key) {
      if (key <= pos - a.window && key >= a.sinks) continue;
      const uint32_t kw = *reinterpret_cast<const uint32_t*>(st.k + st.at(key, a.ks_b, a.ks_n) + 4 * lane);
      const uint32_t vw = *reinterpret_cast<const uint32_t*>(st.v + st.at(key, a.vs_b, a.vs_n) + 4 * lane);
      float x = __builtin_fmaf(q0, widen<BF>((uint16_t)kw), q1 * widen<BF>((uint16_t)(kw >> 16)));
#pragma unroll
      for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d);
      if ((x - m) * a.c > TAU) {
        const float alpha = __builtin_amdgcn_exp2f((m - x) * a.c);
        m = x;
        l *= alpha;
        o[0] *= alpha;
        o[1] *= alpha;
      }
      const float p = __builtin_amdgcn_exp2f(m == -INFINITY ? x * a.c : (x - m) * a.c);
      l += p;
      o[0] = __builtin_fmaf(p, widen<BF>((uint16_t)vw), o[0]);
      o[1] = __builtin_fmaf(p, widen<BF>((uint16_t)(vw >> 16)), o[1]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : l;  // NaN stays
  o[0] *= inv;
  o[1] *= inv;
  lse = (__builtin_amdgcn_logf(l) + m * a.c) * LN2;
}

__device__ __forceinline__ bool is_nan(float x) { return !(x == x); }

// ---------------------------------------------------------------------------
// The row kernel: requests of few rows (decode, a few tokens behind a cache).
// Every key is read once and that read is the bound, so the kernel is laid out
// for bytes in flight and even shares. A workgroup is 4 waves, two of them to a CU
// (64 KiB of LDS each), or beside the tile kernel's 8 waves, every other block
// for each half; a wave takes 32 of a block's 128 keys for itself, its own
// LDS slots (8 KiB of K, 8 KiB of V), statistics and O, so the key loop has no
// barrier: K(j + 1) is loaded once K(j) is in registers, V(j + 1) after the
// products of block j. The four results are joined in LDS at an item's end.
//
// An item is a 32-row tile of one KV head of a request. The blocks of all items,
// in order, are one long axis of which each workgroup takes an equal share,
// whatever the requests' lengths; a share starts and ends anywhere in an item. A
// piece of an item leaves its normalised O and lse in the workspace (a
// workgroup has at most two, its first and its last), and the merge kernel joins
// an item's pieces. Measured, with the joins: 64 requests of 100-8005 keys, 64 heads on 8
// (470 MB of K and V), 112 us, 4.2 TB/s; 131072 keys of one KV head (67 MB) 22 us, of
// which the start takes 4 and the join 5; one request of 4099 keys 13 us, all latency.
constexpr int RT = 32;
constexpr int RSLOT = 32 * ROW_BYTES;       // 32 keys of K or V
constexpr int rows_lds(int waves) { return waves * 2 * RSLOT; }
constexpr int kRowsGroups = 512;            // of 4 waves, two a CU; half as many of 8 waves
// Blocks a share holds at least. 1, 2, 3: 19.1, 13.1, 13.5 us for 4099 keys of one KV head
// (one: 33 pieces), 17.8, 16.8, 17.6 for 8 requests of a window of 1024 keys and 8 heads.
constexpr int kMinShare = 2;
constexpr int DESC_INTS = 8;                // ints of a descriptor

template <bool PAGED>
__device__ __forceinline__ int row_tiles(const AttnArgs& a, const Request& r) {
  const int64_t rows = (int64_t)r.n * a.group;
  return rows <= a.rows_max ? (int)((rows + RT - 1) / RT) : 0;
}
// Blocks of every item of a request: those any of its rows sees, at least one (an
// item whose rows see nothing still writes zeros).
__device__ __forceinline__ int row_blocks(const AttnArgs& a, const Request& r) {
  return max(blocks(a, r, r.pos, r.pos + r.n - 1).total(), 1);
}

__device__ __forceinline__ Blocks uniform(const Blocks& k) {
  return Blocks{uniform(k.ns), uniform(k.w0), uniform(k.w1), uniform(k.f0), uniform(k.f1)};
}

template <bool BF, bool PAGED, int RW>
__device__ __forceinline__ void row_item(const AttnArgs& a, const Request& r, int b, int hk, int tile, int s0, int s1,
                                         int nblk, int slot, char* lds, float* st_m, float* st_l) {
  // Opaque, so that nothing derived from it is kept across the items.
  int tid;
  asm volatile("v_mov_b32 %0, %1" : "=v"(tid) : "v"((int)threadIdx.x));
  const int lane = tid & 63, l32 = lane & 31, hf = lane >> 5, lr = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int rows = r.n * a.group;
  const int row = min(tile * RT + l32, rows - 1);
  const int i = row / a.group, head = hk * a.group + row % a.group;
  const int pos = r.pos + i;
  const Blocks bl = uniform(blocks(a, r, r.pos, r.pos + r.n - 1));
  auto block_at = [&](int s) { return s < bl.ns ? s : bl.w0 + s - bl.ns; };
  // Whether the keys [key, key + 32) are seen whole by every row of the tile.
  const int first = uniform(r.pos + tile * RT / a.group);
  const int last = uniform(r.pos + min(tile * RT + RT - 1, rows - 1) / a.group);
  auto whole = [&](int key) {
    return key + 31 <= min(first, r.keys - 1) && (key > last - a.window || key + 32 <= a.sinks);
  };
  const Stream<PAGED> st(a, r, b, hk);

  // A load instruction fills 4 rows of 256 bytes: lane l brings row l / 16, the
  // chunk its place holds. K keeps chunk c of row n at c ^ n % 16 (the 32 rows
  // an operand read takes one chunk column from then lie in different banks), V
  // at c ^ 4 (n % 4) (a transposing read's 4 rows in the 4 quarters of the banks).
  int koff[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) koff[x] = lr * st.ks_n + ((lane & 15) ^ (4 * x + lr)) * 16;
  const int voff = lr * st.vs_n + ((lane & 15) ^ (4 * lr)) * 16;
  char* kslot = lds + wave * 2 * RSLOT;
  char* vslot = kslot + RSLOT;
  const uint32_t kdst = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)kslot;
  const uint32_t vdst = kdst + RSLOT;
  bool bad = r.bad;
  // Keys of this wave in block s of the list (past the piece: no keys).
  auto key_of = [&](int s) { return s < s1 ? block_at(s) * BLOCK + (wave & 3) * 32 : 1 << 30; };
  auto load_k = [&](int key, const int (&id)[2]) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      bad |= st.missing(key + 16 * g, id[g]);
      const i32x4 rs = st.k_rsrc(key + 16 * g, id[g]);
#pragma unroll
      for (int x = 0; x < 4; ++x) dma_to_lds_late(rs, kdst + (4 * g + x) * 1024, koff[x], 4 * x * st.ks_n);
    }
  };
  auto load_v = [&](int key, const int (&id)[2]) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const i32x4 rs = st.v_rsrc(key + 16 * g, id[g]);
#pragma unroll
      for (int x = 0; x < 4; ++x) dma_to_lds_late(rs, vdst + (4 * g + x) * 1024, voff, 4 * x * st.vs_n);
    }
  };
  auto pages_of = [&](int key, int (&id)[2]) {
    id[0] = uniform(st.page(key));
    id[1] = uniform(st.page(key + 16));
  };

  const char* qrow = a.q + b * a.qs_b + (int64_t)(r.row0 + i) * a.qs_n + head * a.qs_h;
  int id[2], next[2];
  int key = key_of(s0 + (wave >> 2));
  pages_of(key, id);
  h8 qf[8];
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) qf[kk] = *reinterpret_cast<const h8*>(qrow + (kk * 2 + hf) * 16);
  load_k(key, id);
  load_v(key, id);
  constexpr int STEP = RW / 4;              // blocks a round of the waves covers
  int key_next = key_of(s0 + (wave >> 2) + STEP);
  pages_of(key_next, next);
  // The compiler waits for its own loads here, before the key loop.
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) asm volatile("" ::"v"(qf[kk]));

  const int k_lane = l32 * ROW_BYTES + ((hf ^ (l32 & 15)) << 4);
  int v_lane[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) {
    const int e = (lane & 15) >> 2;
    v_lane[dt] = (4 * hf + e) * ROW_BYTES + (4 * (dt ^ e) + 2 * (lr & 1) + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;
  }
  f32x16 acc[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) acc[dt] = f32x16{};
  float m = -INFINITY, l = 0.f;
  for (int s = s0 + (wave >> 2); s < s1; s += STEP) {
    wait_loads<8>();                        // K has landed; V may be in flight
    f32x16 sc[1];
    sc[0] = f32x16{};
#pragma unroll
    for (int kk = 0; kk < 8; ++kk)
      sc[0] = mma<BF>(*reinterpret_cast<const h8*>(kslot + (k_lane ^ (kk << 5))), qf[kk], sc[0]);
    wait_lds();
    load_k(key_next, next);
    if (!whole(key)) {
      const int base = key + 4 * hf;
      const int hi = min(pos, r.keys - 1) - base, lo = pos - a.window + 1 - base, sink = a.sinks - base;
      hide(sc, hi, lo, sink);
    }
    h8 p[2];
    softmax_step<BF, 1>(sc, p, m, l, acc, a.c, [](int) {});
    wait_loads<8>();                        // V has landed; the next K may be in flight
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) {
        const char* at = vslot + v_lane[dt] + ks * 16 * ROW_BYTES;
        const h8 x = __builtin_shufflevector(lds_read_tr(at), lds_read_tr(at + 8 * ROW_BYTES), 0, 1, 2, 3, 4, 5, 6, 7);
        acc[dt] = mma<BF>(x, p[ks], acc[dt]);
      }
    wait_lds();
    load_v(key_next, next);
    key = key_next;
    key_next = key_of(s + 2 * STEP);
    pages_of(key_next, next);
  }

  // Join the waves: O goes to the wave's own 16 KiB of slots once its loads have
  // landed, 512-byte rows with chunk c of row n at c ^ n, m and l beside them.
  wait_loads<0>();
  const float lw = bad ? NAN : half_sum(l);
  if (hf == 0) {
    st_m[wave * RT + l32] = m;
    st_l[wave * RT + l32] = lw;
  }
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const float4 val = {acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]};
      *reinterpret_cast<float4*>(kslot + l32 * 512 + (((dt * 8 + 2 * g + hf) ^ l32) << 4)) = val;
    }
  __syncthreads();
  // The first 4 waves: 8 threads a row, 16 dims each, 8 at 8t and 8 at 64 + 8t.
  if (RW > 4 && wave >= 4) {
    __syncthreads();
    return;
  }
  const int n = tid >> 3, t = tid & 7;
  const int orow = tile * RT + n;
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < RW; ++w) M = smax(M, st_m[w * RT + n]);
  float L = 0.f, o[16];
#pragma unroll
  for (int x = 0; x < 16; ++x) o[x] = 0.f;
#pragma unroll
  for (int w = 0; w < RW; ++w) {
    const float mw = st_m[w * RT + n];
    const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((mw - M) * a.c);
    L = __builtin_fmaf(f, st_l[w * RT + n], L);
    const char* base = lds + w * 2 * RSLOT + n * 512;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int chunk = (x >> 1) * 16 + 2 * t + (x & 1);
      const float4 val = *reinterpret_cast<const float4*>(base + ((chunk ^ n) << 4));
      o[4 * x] = __builtin_fmaf(f, val.x, o[4 * x]);
      o[4 * x + 1] = __builtin_fmaf(f, val.y, o[4 * x + 1]);
      o[4 * x + 2] = __builtin_fmaf(f, val.z, o[4 * x + 2]);
      o[4 * x + 3] = __builtin_fmaf(f, val.w, o[4 * x + 3]);
    }
  }
  __syncthreads();                          // the slots may be filled again
  const bool inside = orow < rows;
  const int orc = inside ? orow : rows - 1;
  const int oi = orc / a.group, ohead = hk * a.group + orc % a.group;
  const bool part = s0 > 0 || s1 < nblk;
  float* prow = a.opart + ((int64_t)slot * RT + n) * HD;
  char* out = a.o + b * a.os_b + (int64_t)(r.row0 + oi) * a.os_n + ohead * a.os_h;
  float* out_lse = a.lse + b * a.ls_b + (int64_t)(r.row0 + oi) * a.ls_n + ohead * a.ls_h;
  // O is not a number though every weight is: a hidden key's V (see above).
  float sum = 0.f;
#pragma unroll
  for (int x = 0; x < 16; ++x) sum += o[x] * 0.f;
  uint64_t sick = __builtin_amdgcn_ballot_w64(inside && is_nan(sum) && !is_nan(L));
  bool again = false;
  while (sick) {
    const int at = __ffsll((unsigned long long)sick) - 1;
    sick &= ~(0xffull << (at & ~7));
    const int row = tile * RT + __builtin_amdgcn_readfirstlane(__shfl(n, at));
    const int ri = row / a.group, rh = hk * a.group + row % a.group;
    if (!spoiled_row<BF, PAGED>(a, st, r.pos + ri, s0, s1, block_at)) continue;
    again |= (lane >> 3) == (at >> 3);
    float x[2], rl;
    repair_row<BF, PAGED>(a, st, a.q + b * a.qs_b + (int64_t)(r.row0 + ri) * a.qs_n + rh * a.qs_h, r.pos + ri, s0, s1,
                          block_at, x, rl);
    if (part) {
      float* dst = a.opart + ((int64_t)slot * RT + row - tile * RT) * HD;
      dst[2 * lane] = x[0];
      dst[2 * lane + 1] = x[1];
      if (lane == 0) a.lpart[(int64_t)slot * RT + row - tile * RT] = rl;
    } else {
      char* dst = a.o + b * a.os_b + (int64_t)(r.row0 + ri) * a.os_n + rh * a.os_h;
      *reinterpret_cast<uint32_t*>(dst + 4 * lane) = narrow<BF>(x[0]) | (uint32_t)narrow<BF>(x[1]) << 16;
      if (a.lse && lane == 0) a.lse[b * a.ls_b + (int64_t)(r.row0 + ri) * a.ls_n + rh * a.ls_h] = rl;
    }
  }
  if (!inside || again) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const float lse = (__builtin_amdgcn_logf(L) + M * a.c) * LN2;
  if (part) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int chunk = (x >> 1) * 16 + 2 * t + (x & 1);
      *reinterpret_cast<float4*>(prow + 4 * chunk) =
          float4{o[4 * x] * inv, o[4 * x + 1] * inv, o[4 * x + 2] * inv, o[4 * x + 3] * inv};
    }
    if (t == 0) a.lpart[(int64_t)slot * RT + n] = lse;
  } else {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      u16x8 val;
#pragma unroll
      for (int e = 0; e < 8; ++e) val[e] = narrow<BF>(o[8 * x + e] * inv);
      *reinterpret_cast<u16x8*>(out + (64 * x + 8 * t) * 2) = val;
    }
    if (a.lse && t == 0) *out_lse = lse;
  }
}

// The share of workgroup g, of RW waves.
template <bool BF, bool PAGED, int RW>
__device__ __forceinline__ void rows_share(const AttnArgs& a, int g, char* lds) {
  constexpr int RTHREADS = RW * 64;
  __shared__ float st_m[RW * RT], st_l[RW * RT];
  __shared__ uint32_t wave_sum[RW][2];
  __shared__ int found[2];
  __shared__ Request found_r;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // Blocks of all items before this thread's run of requests, and of all.
  const int per = (a.batch + RTHREADS - 1) / RTHREADS;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  auto cost = [&](const Request& r) {
    const int tiles = row_tiles<PAGED>(a, r);
    return tiles ? (uint32_t)(a.heads_kv * tiles * row_blocks(a, r)) : 0u;
  };
  Request own{};                            // of request b0
  uint64_t all = 0;
  for (int b = b0; b < b1; ++b) {
    const Request r = request<PAGED>(a, b);
    if (b == b0) own = r;
    all += cost(r);
  }
  const uint32_t mine = (uint32_t)all, sum = lanes_sum(mine), upper = lanes_sum((uint32_t)(all >> 16));
  if (lane == 63) {
    wave_sum[wave][0] = sum;
    wave_sum[wave][1] = upper;
  }
  __syncthreads();
  uint32_t before = sum - mine, total = 0, large = 0;
#pragma unroll
  for (int w = 0; w < RW; ++w) {
    if (w < wave) before += wave_sum[w][0];
    total += wave_sum[w][0];
    large += wave_sum[w][1];
  }
  total = uniform(total);
  // Workgroup g takes blocks [g total / groups, (g + 1) total / groups): shares that
  // differ by one block at most, so that every CU's two workgroups have as much.
  const uint32_t groups = max(min((uint32_t)a.groups, (total + kMinShare - 1) / kMinShare), 1u);
  const bool narrow = total < 1u << 22;     // products with `groups` fit 32 bits
  auto start_of = [&](uint32_t n) {
    return uniform(narrow ? n * total / groups : (uint32_t)((uint64_t)n * total / groups));
  };
  auto taker_of = [&](uint32_t block) {
    return (int)(narrow ? ((block + 1) * groups - 1) / total : (((uint64_t)block + 1) * groups - 1) / total);
  };
  uint32_t x = (uint32_t)g < groups ? start_of(g) : total;
  const uint32_t end = (uint32_t)g < groups ? start_of(g + 1) : total;
  int* desc = a.desc + g * DESC_INTS;
  if (tid == 0) desc[3] = -1;               // no item that began earlier, so far
  // Uniform. (`large`: requests that overlap, beyond what 32 bits count.)
  if (x >= total || large >= 1 << 15) return;
  if (before <= x && x < before + mine) {
    int b = b0;
    uint32_t at = before;
    Request r = own;
    while (true) {
      const uint32_t n = cost(r);
      if (x < at + n || b + 1 >= b1) break;
      at += n;
      r = request<PAGED>(a, ++b);
    }
    found[0] = b;
    found[1] = (int)at;
    found_r = r;
  }
  __syncthreads();
  int b = uniform(found[0]);
  uint32_t at = uniform((uint32_t)found[1]);          // where request b's blocks start
  Request r = uniform(found_r);
  bool head = true;
  while (true) {
    const int tiles = row_tiles<PAGED>(a, r);
    if (tiles) {
      const int nblk = uniform(row_blocks(a, r));
      const uint32_t stop = at + (uint32_t)a.heads_kv * tiles * nblk;
      while (x < end && x < stop) {
        const uint32_t rel = x - at, item = uniform(rel / (uint32_t)nblk);
        const int s0 = uniform((int)(rel - item * (uint32_t)nblk));
        const int s1 = uniform((int)min((uint32_t)nblk, s0 + (end - x)));
        const int hk = uniform((int)(item / (uint32_t)tiles)), tile = uniform((int)(item - (uint32_t)hk * tiles));
        if (head && s0 > 0 && tid == 0) {
          // An item that began before this one's share: what the merge kernel needs.
          const uint32_t start = x - s0;
          desc[0] = b;
          desc[1] = hk;
          desc[2] = tile;
          desc[3] = taker_of(start);        // the workgroups that share it
          desc[4] = taker_of(start + nblk - 1);
          desc[5] = r.row0;
          desc[6] = r.n * a.group;
        }
        head = false;
        row_item<BF, PAGED, RW>(a, r, b, hk, tile, s0, s1, nblk, 2 * g + (s0 == 0), lds, st_m, st_l);
        x += s1 - s0;
      }
      at = stop;
    }
    if (x >= end) break;
    if (++b >= a.batch) break;
    r = uniform(request<PAGED>(a, b));
  }
}

template <bool BF, bool PAGED>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2)))
fa_serve_rows_kernel(AttnArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  rows_share<BF, PAGED, 4>(a, blockIdx.x, lds);
}

// Joins the pieces of the items that several workgroups share:
//   O = sum w_s O_s / sum w_s, w_s = exp(lse_s - M), M = max lse_s, lse = M + ln sum w_s.
// Workgroup g > 0 whose share starts inside an item is one of the K = pieces - 1 that
// do, and they share its join, so that a launch's joins are spread evenly however
// many pieces an item has. Up to kFewPieces pieces, 32 lanes take a row (4 dims each),
// 8 rows at once; up to kSomePieces the workgroup takes a row, 8 groups of 32 lanes
// reading an 8th of the pieces each; beyond, a quarter of a row, 32 groups of 8 lanes.
// So every workgroup has one row or quarter to join at most, and all its loads are in
// flight at once. Both launches for 8400 keys of 12 rows (33 pieces) take 12.1 us, with
// quarters (of which there are 48) 20.0; for 4000 keys (16 pieces) 12.6, a row a workgroup
// 13.4; for 131072 keys (512 pieces) 22.0, of which the join in quarters has 5, where
// the first form alone took 23.6. The launch is short, so the length of its code counts:
// expf instead of exp2, unrolled, cost 4 us at 64000 keys (18.5, not 14.7).
constexpr int kFewPieces = 32, MERGE_EACH = 16, kSomePieces = 8 * MERGE_EACH;
static_assert(32 * MERGE_EACH >= kRowsGroups, "every piece has a load");
// e^(x - M), 0 for a part that saw no key (also where M is -inf). The product with log2 e
// is off by half a step of |x - M| log2 e, which the weight it goes with makes
// smaller than 2^-24.
__device__ __forceinline__ float weight(float x, float M) {
  return x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((x - M) * (float)LOG2E);
}
template <bool BF, bool PAGED>
__device__ __forceinline__ void merge_rows(const AttnArgs& a, int block) {
  __shared__ __attribute__((aligned(16))) float red[32 * 36];   // results of 32 (or 8) groups
  const int* desc = a.desc + (block + 1) * DESC_INTS;
  const int first = desc[3];
  if (first < 0) return;
  const int b = desc[0], hk = desc[1], tile = desc[2], last = desc[4], row0 = desc[5];
  const int tid = threadIdx.x;
  const int boundaries = last - first, pieces = boundaries + 1, mine = block - first;
  const int rows = min(desc[6] - tile * RT, RT);
  auto piece = [&](int s) { return 2 * (first + s) + (s == 0); };
  auto out_row = [&](int n) {
    const int row = tile * RT + n, i = row / a.group, head = hk * a.group + row % a.group;
    return a.o + b * a.os_b + (int64_t)(row0 + i) * a.os_n + head * a.os_h;
  };
  auto out_lse = [&](int n, float M, float total) {
    if (!a.lse) return;
    const int row = tile * RT + n, i = row / a.group, head = hk * a.group + row % a.group;
    a.lse[b * a.ls_b + (int64_t)(row0 + i) * a.ls_n + head * a.ls_h] = M == -INFINITY ? M : M + logf(total);
  };
  if (pieces <= kFewPieces) {
    const int l32 = tid & 31;
    for (int n = mine + (tid >> 5) * boundaries; n < rows; n += 8 * boundaries) {
      // The first pieces' rows beside their lse (past the last piece, that one again).
      float4 v[8];
      auto read = [&](int s0) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          v[e] = *reinterpret_cast<const float4*>(a.opart + (piece(min(s0 + e, boundaries)) * RT + n) * HD + 4 * l32);
      };
      const float x = l32 < pieces ? a.lpart[piece(l32) * RT + n] : -INFINITY;
      read(0);
      float M = x;
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) M = smax(M, __shfl_xor(M, d, 32));
      const float w = weight(x, M);
      float total = w;
#pragma unroll
      for (int d = 16; d >= 1; d >>= 1) total += __shfl_xor(total, d, 32);
      float4 o = {0.f, 0.f, 0.f, 0.f};
      for (int s0 = 0; s0 < pieces; s0 += 8) {
        if (s0) read(s0);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          // Past the last piece both factors are 0: that piece, read again, may hold an
          // infinity. (Leaving the loop there makes the loads wait for each other:
          // 7.2 us instead of 4.0 for 17 pieces.)
          const bool on = s0 + e < pieces;
          const float ws = on ? __shfl(w, min(s0 + e, 31), 32) : 0.f;
          o.x = __builtin_fmaf(ws, on ? v[e].x : 0.f, o.x);
          o.y = __builtin_fmaf(ws, on ? v[e].y : 0.f, o.y);
          o.z = __builtin_fmaf(ws, on ? v[e].z : 0.f, o.z);
          o.w = __builtin_fmaf(ws, on ? v[e].w : 0.f, o.w);
        }
      }
      const float inv = total == 0.f ? 0.f : 1.f / total;
      *reinterpret_cast<u16x4*>(out_row(n) + 8 * l32) =
          u16x4{narrow<BF>(o.x * inv), narrow<BF>(o.y * inv), narrow<BF>(o.z * inv), narrow<BF>(o.w * inv)};
      if (l32 == 0) out_lse(n, M, total);
    }
    return;
  }
  auto many = [&](auto lanes) {
    constexpr int LANES = decltype(lanes)::value, GROUPS = 256 / LANES, SLICES = 32 / LANES;
    constexpr int PITCH = 4 * LANES + 4;    // the dims, the maximum and the sum of a group
    for (int u = mine; u < SLICES * rows; u += boundaries) {
      const int n = u / SLICES, dim0 = u % SLICES * 4 * LANES, grp = tid / LANES, l = tid % LANES;
      // The group's pieces, s = grp, grp + GROUPS, .., joined on their own; all loads at once.
      float4 v[MERGE_EACH];
      float x[MERGE_EACH], M = -INFINITY, total = 0.f;
#pragma unroll
      for (int k = 0; k < MERGE_EACH; ++k) {
        const int at = piece(min(grp + GROUPS * k, boundaries)) * RT + n;
        x[k] = a.lpart[at];
        v[k] = *reinterpret_cast<const float4*>(a.opart + (int64_t)at * HD + dim0 + 4 * l);
      }
#pragma unroll
      for (int k = 0; k < MERGE_EACH; ++k) {
        x[k] = grp + GROUPS * k < pieces ? x[k] : -INFINITY;
        M = smax(M, x[k]);
      }
      float4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < MERGE_EACH; ++k) {
        const bool on = x[k] != -INFINITY;  // such a piece, and with a visible key
        const float w = weight(x[k], M);
        total += w;
        o.x = __builtin_fmaf(w, on ? v[k].x : 0.f, o.x);
        o.y = __builtin_fmaf(w, on ? v[k].y : 0.f, o.y);
        o.z = __builtin_fmaf(w, on ? v[k].z : 0.f, o.z);
        o.w = __builtin_fmaf(w, on ? v[k].w : 0.f, o.w);
      }
      __syncthreads();                      // the last unit's LDS has been read
      float* const own = red + grp * PITCH;
      *reinterpret_cast<float4*>(own + 4 * l) = o;
      if (l == 0) {
        own[4 * LANES] = M;
        own[4 * LANES + 1] = total;
      }
      __syncthreads();
      if (tid < 4 * LANES) {
        M = -INFINITY;
#pragma unroll
        for (int s = 0; s < GROUPS; ++s) M = smax(M, red[s * PITCH + 4 * LANES]);
        float sum = 0.f;
        total = 0.f;
#pragma unroll
        for (int s = 0; s < GROUPS; ++s) {
          const float* const other = red + s * PITCH;
          const float m = other[4 * LANES];
          const float w = weight(m, M);
          total = __builtin_fmaf(w, other[4 * LANES + 1], total);
          sum = __builtin_fmaf(w, other[tid], sum);
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        reinterpret_cast<uint16_t*>(out_row(n))[dim0 + tid] = narrow<BF>(sum * inv);
        if (dim0 == 0 && tid == 0) out_lse(n, M, total);
      }
    }
  };
  if (pieces <= kSomePieces)
    many(std::integral_constant<int, 32>());
  else
    many(std::integral_constant<int, 8>());
}

// ---------------------------------------------------------------------------
// The tile kernel: requests of many rows (prompts, chunks of them), bound by the
// matrix cores. A tile is 256 packed rows, 8 waves x 32. Two groups of four
// waves, one wave of each on a SIMD, run a phase apart: a wave alternates an
// MFMA step (S^T(j) = K(j) Q^T interleaved with O^T += V^T(j-1) P^T(j-1)) with a
// softmax step (S(j) into P(j)), so that on every SIMD one wave feeds the matrix
// pipe while the other does its softmax; the phases are separated by barriers. LDS
// holds two K and two V blocks of 128 keys, 256-byte rows placed as in the row
// kernel. Group 1 loads the K blocks, group 0 the V blocks; their page numbers are
// fetched (scalar loads) a step earlier.
//
// The blocks that every row of the tile sees whole come first, in a loop without
// mask code, then the others: the order of keys is free in the online softmax.
//
// With fewer tiles than CUs (a chunk behind a long cache) the lists of blocks are
// cut into parts, a workgroup each, joined by a merge kernel. The lengths are
// known on the GPU alone, so it decides there.
//
// Measured: a block of 128 keys takes a CU 3.6 us with all of them busy (16.8 MFLOP each,
// 1190 TFLOP/s: the board's power limit; 3.1 in short launches), a tile 8 us besides: 2.5 until
// it starts after the one before, 4.5 for its first loads, 1 for its stores. 32768 tokens of 12 heads, a window of 4096: 745 us, 1040
// TFLOP/s of visible scores; 2048 tokens behind 30001, 12 heads: 391 us, 1000 TFLOP/s.
constexpr int TT = 256;                     // rows of a tile
constexpr int TTHREADS = 512;
constexpr int TBLOCK = BLOCK * ROW_BYTES;   // bytes of a K or V block
constexpr int kTileLds = 4 * TBLOCK;
constexpr int kTileItems = 512;             // parts of a launch that cuts tiles, at most
constexpr int kTileGroups = 256;            // CUs: launches of fewer tiles may cut them
constexpr int kCuts = 24;                   // parts of the longest tile, at most
// Costs in units of a key block (3.6 us on a CU): what an item takes besides its
// blocks if it is a whole tile, or a part (256 rows of FP32 O to write), a merge
// kernel, and every part's share of it (128 KiB to read).
constexpr float kWholeCost = 2.f, kPartCost = 5.f, kMergeCost = 2.f, kMergeShare = 0.014f;

template <bool PAGED>
__device__ __forceinline__ int tile_count(const AttnArgs& a, const Request& r) {
  const int64_t rows = (int64_t)r.n * a.group;
  return rows > a.rows_max ? (int)((rows + TT - 1) / TT) : 0;
}
// At least the blocks of any tile of the request.
__host__ __device__ __forceinline__ int tile_blocks(const AttnArgs& a, const Request& r) {
  const Blocks all = blocks(a, r, r.pos, r.pos + r.n - 1);
  const int span = min(TT / a.group + 2, r.n);
  const int64_t near = ((int64_t)a.window + span + BLOCK - 1) / BLOCK + 1 + (a.sinks + BLOCK - 1) / BLOCK;
  return max((int)min((int64_t)all.total(), near), 1);
}

// What a workgroup of the tile kernel does: a part of a tile's blocks.
struct Item {
  int b, hk, tile, part, parts, length;     // length: blocks of a part
  int index, tile_index;                    // place among all parts, all tiles
  Request r;
};

template <bool BF, bool PAGED>
__device__ __forceinline__ void tile_item(const AttnArgs& a, const Item& it, char* lds, int* flag) {
  int tid;
  asm volatile("v_mov_b32 %0, %1" : "=v"(tid) : "v"((int)threadIdx.x));
  const int lane = tid & 63, l32 = lane & 31, hf = lane >> 5, lr = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int grp = wave >> 2, dw = wave & 3;
  const Request& r = it.r;
  const int b = it.b, hk = it.hk;
  const int rows = r.n * a.group;
  const int row0 = it.tile * TT + wave * 32;
  const int row = min(row0 + l32, rows - 1);
  const bool row_ok = row0 + l32 < rows;
  const int group = a.group, window = a.window, sinks = a.sinks;
  const float c = a.c;
  const int i = row / group, head = hk * group + row % group;
  const int pos = r.pos + i;
  const int tile_last = min(it.tile * TT + TT, rows) - 1;
  const Blocks bl = uniform(blocks(a, r, uniform(r.pos + it.tile * TT / a.group), uniform(r.pos + tile_last / a.group)));
  // The list: whole blocks, then those with the mask in order.
  const int nfull_all = bl.f1 - bl.f0;
  auto list = [&](int s) {
    int x = s - nfull_all;
    if (x < 0) return bl.f0 + s;
    if (x < bl.ns) return x;
    x += bl.w0 - bl.ns;
    return x < bl.f0 ? x : x + nfull_all;
  };
  const int total = bl.total();
  const int s0 = min(it.part * it.length, total);
  const int nblk = min(it.length, total - s0);        // of this part
  const int nfull = min(max(nfull_all - s0, 0), nblk);
  const bool part = it.parts > 1;
  auto block_at = [&](int s) { return list(s0 + s); };

  if (nblk <= 0) {                          // uniform: no row sees a key of this part
    const float bad = r.bad ? NAN : 0.f;
    if (!row_ok) return;
    if (part) {                             // the merge reads no O of weight 0
      if (hf == 0) a.tlpart[(int64_t)it.index * TT + wave * 32 + l32] = r.bad ? NAN : -INFINITY;
      return;
    }
    u16x8 z;
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = narrow<BF>(bad);
    char* out = a.o + b * a.os_b + (int64_t)(r.row0 + i) * a.os_n + head * a.os_h;
#pragma unroll
    for (int x = 0; x < 8; ++x) *reinterpret_cast<u16x8*>(out + (2 * x + hf) * 16) = z;
    if (a.lse && hf == 0) a.lse[b * a.ls_b + (int64_t)(r.row0 + i) * a.ls_n + head * a.ls_h] = r.bad ? NAN : -INFINITY;
    return;
  }

  const Stream<PAGED> st(a, r, b, hk);
  // Loads: wave dw of group 1 fills rows 32 dw .. + 31 of the K blocks, that of group 0
  // those of the V blocks: two 16-key groups, and so two descriptors for the 8
  // instructions of 4 rows each. The descriptor of the next load is made after a load.
  const char* const lbase = grp ? st.k : st.v;
  const uint32_t lpage = grp ? st.ks_b : st.vs_b;
  const int lpitch = grp ? st.ks_n : st.vs_n;
  int loff[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) loff[x] = lr * lpitch + ((lane & 15) ^ (grp ? 4 * x + lr : 4 * lr)) * 16;
  const uint32_t ldst = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds + dw * (32 * ROW_BYTES) +
                        (grp ? 0 : 2 * TBLOCK);
  bool bad = r.bad;
  int id[2], key = 0, nid[2], nkey = 0;     // pages and first key (this wave's) of the next block to load, and the one after
  i32x4 rs;
  auto fetch = [&](int s) {
    nkey = s < nblk ? block_at(s) * BLOCK + 32 * dw : 1 << 30;
#pragma unroll
    for (int g = 0; g < 2; ++g) nid[g] = uniform(st.page(nkey + 16 * g));
  };
  auto describe = [&](int g) {
    bad |= st.missing(key + 16 * g, id[g]);
    rs = st.rsrc(lbase, lpage, lpitch, key + 16 * g, id[g]);
  };
  auto advance = [&]() {                    // what was fetched is next
    key = nkey;
    id[0] = nid[0];
    id[1] = nid[1];
    describe(0);
  };
  auto load = [&](int x, int slot) {
    dma_to_lds_late(rs, ldst + slot * TBLOCK + x * 1024, loff[x & 3], 4 * (x & 3) * lpitch);
    if (x == 3) describe(1);
  };
  auto load_all = [&](int slot) {
#pragma unroll
    for (int x = 0; x < 8; ++x) load(x, slot);
  };

  h8 qf[8];
  f32x16 acc[4], s[4];
  h8 p[8];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) acc[dt] = f32x16{};
  float m = -INFINITY, l = 0.f;

  // Operands: K row 32t + l32, chunk 2kk + hf; V as described at Fragments.
  const int k_lane = l32 * ROW_BYTES + ((hf ^ (l32 & 15)) << 4);
  int v_lane[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) {
    const int e = (lane & 15) >> 2;
    v_lane[dt] = (4 * hf + e) * ROW_BYTES + (4 * (dt ^ e) + 2 * (lr & 1) + ((lane & 3) >> 1)) * 16 + (lane & 1) * 8;
  }
  // Operand x of a step: even x QK product n = x / 2 (score tile n % 4, k-step n / 4),
  // odd x PV product n (O tile n % 4, 16-key step n / 4), so consecutive
  // products of a kind go to different accumulators.
  constexpr int BOTH = 0, QK = 1, PV = 2, PF = 4;
  auto ld = [&](const char* kb, const char* vb, int x) -> h8 {
    const int n = x >> 1;
    if ((x & 1) == 0)
      return *reinterpret_cast<const h8*>(kb + (k_lane ^ ((n / 4) << 5)) + (n % 4) * 32 * ROW_BYTES);
    const char* at = vb + v_lane[n % 4] + (n / 4) * 16 * ROW_BYTES;
    return __builtin_shufflevector(lds_read_tr(at), lds_read_tr(at + 8 * ROW_BYTES), 0, 1, 2, 3, 4, 5, 6, 7);
  };
  h8 fr[PF];
  auto operand = [](int kind, int x) constexpr { return kind == BOTH ? x : 2 * x + (kind == PV); };
  auto preload = [&](const char* kb, const char* vb, auto kind) {
#pragma unroll
    for (int x = 0; x < PF; ++x) fr[x] = ld(kb, vb, operand(decltype(kind)::value, x));
  };
  // load_at(x) runs after product N / 8 * x + 1 of the step, 0 <= x < 8.
  auto mfma_step = [&](const char* kb, const char* vb, auto preloaded, auto kind, auto&& load_at) {
    constexpr int KIND = decltype(kind)::value;
    constexpr int N = KIND == BOTH ? 64 : 32;
    if constexpr (!decltype(preloaded)::value) preload(kb, vb, kind);
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const h8 f = fr[x % PF];
      const int op = operand(KIND, x), n = op >> 1;
      if ((op & 1) == 0)
        s[n % 4] = mma<BF>(f, qf[n / 4], n < 4 ? f32x16{} : s[n % 4]);
      else
        acc[n % 4] = mma<BF>(f, p[n / 4], acc[n % 4]);
      if (x + PF < N) fr[x % PF] = ld(kb, vb, operand(KIND, x + PF));
      if (x % (N / 8) == 1) load_at(x / (N / 8));
      __builtin_amdgcn_sched_barrier(0);    // operand reads stay PF products ahead
    }
  };
  auto softmax = [&](int j, auto with_mask, auto&& at) {
    if constexpr (decltype(with_mask)::value) {
      const int base = block_at(j) * BLOCK + 4 * hf;
      const int hi = min(pos, r.keys - 1) - base, lo = pos - window + 1 - base, sink = sinks - base;
      hide(s, hi, lo, sink);
    }
    softmax_step<BF, 4>(s, p, m, l, acc, c, at);
  };
  const std::integral_constant<bool, false> loads, whole;
  const std::integral_constant<bool, true> preloaded, with_mask;
  const std::integral_constant<int, BOTH> both;
  const std::integral_constant<int, QK> qk;
  const std::integral_constant<int, PV> pv;
  auto kslot = [&](int j) { return lds + (j & 1) * TBLOCK; };
  auto vslot = [&](int j) { return lds + (2 + (j & 1)) * TBLOCK; };

  // Phase 2j + grp is a wave's MFMA step for block j, phase 2j + grp + 1 its
  // softmax; all waves pass the same 2 nblk + 3 barriers. K(j) and V(j) are in
  // slots j % 2. Group 1 loads K(0) before the first barrier, K(1) in phase 0 and
  // K(j + 2) in phase 2j + 2, its softmax, into the slot of K(j), which both groups'
  // MFMA steps j have read. Group 0 loads V(j) in phase 2j, its MFMA step, into the
  // slot of V(j - 2), which was last read in phase 2j - 1. A group waits for its loads
  // at the end of the next phase, before the barrier that publishes them.
  // (All loads in group 1's softmax made that step the longest of a phase.)
  if (tid == 0) *flag = 0;
  const bool idle = row0 >= rows;           // this wave has no row: it loads and waits only
  auto nothing = [](int) {};
  fetch(0);
  advance();
  if (grp == 1) load_all(0);
  const char* qrow = a.q + b * a.qs_b + (int64_t)(r.row0 + i) * a.qs_n + head * a.qs_h;
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) qf[kk] = *reinterpret_cast<const h8*>(qrow + (kk * 2 + hf) * 16);
  if (grp == 1) {
    fetch(1);
    advance();
    wait_loads<0>();
  }
  // The compiler waits for its own loads here, before the key loop.
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) asm volatile("" ::"v"(qf[kk]));
  lds_barrier();
  if (grp == 0) {
    if (idle) {
      for (int j = 0; j < nblk; ++j) {
        load_all(j & 1);
        fetch(j + 1);
        lds_barrier();
        wait_loads<0>();
        advance();
        lds_barrier();
      }
      lds_barrier();
      lds_barrier();
    } else {
      auto step = [&](int j, auto kind, auto mask) {
        mfma_step(kslot(j), vslot(j + 1), loads, kind, [&](int x) { load(x, j & 1); });
        lds_barrier();
        fetch(j + 1);
        softmax(j, mask, nothing);
        wait_loads<0>();
        advance();
        lds_barrier();
      };
      if (nfull > 0)
        step(0, qk, whole);
      else
        step(0, qk, with_mask);
      int j = 1;
      for (; j < nfull; ++j) step(j, both, whole);
      for (; j < nblk; ++j) step(j, both, with_mask);
      mfma_step(kslot(nblk), vslot(nblk + 1), loads, pv, nothing);
      lds_barrier();
      lds_barrier();
    }
  } else {
    load_all(1);                            // phase 0
    fetch(2);
    advance();
    if (idle) {
      lds_barrier();
      for (int j = 0; j < nblk; ++j) {
        wait_loads<0>();
        lds_barrier();
        load_all(j & 1);
        fetch(j + 3);
        advance();
        lds_barrier();
      }
      wait_loads<0>();
      lds_barrier();
    } else {
      preload(kslot(0), vslot(0), qk);
      lds_barrier();
      auto step = [&](int j, auto kind, auto mask) {
        mfma_step(kslot(j), vslot(j + 1), preloaded, kind, nothing);
        wait_loads<0>();
        lds_barrier();
        fetch(j + 3);
        softmax(j, mask, [&](int x) {       // 8 loads over the 32 pairs of exponentials
          if (x % 4) return;
          __builtin_amdgcn_sched_barrier(0);
          load(x / 4, j & 1);
          __builtin_amdgcn_sched_barrier(0);
        });
        advance();
        preload(kslot(j + 1), vslot(j), both);
        lds_barrier();
      };
      if (nfull > 0)
        step(0, qk, whole);
      else
        step(0, qk, with_mask);
      int j = 1;
      for (; j < nfull; ++j) step(j, both, whole);
      for (; j < nblk; ++j) step(j, both, with_mask);
      mfma_step(kslot(nblk), vslot(nblk + 1), loads, pv, nothing);
      wait_loads<0>();
      lds_barrier();
    }
  }
  if (bad && lane == 0) *flag = 1;
  lds_barrier();                            // nobody reads the ring any more; flag is set
  const bool poisoned = *flag != 0 || r.bad;

  // Results. l is 0 for a row that saw no key.
  ConstArgs& f = fresh_args();
  float lsum = half_sum(l);
  if (poisoned) lsum = NAN;
  const float inv = lsum == 0.f ? 0.f : 1.f / lsum;
  const float lse = (__builtin_amdgcn_logf(lsum) + m * f.c) * LN2;
  float check = 0.f;
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int x = 0; x < 16; ++x) check += acc[dt][x] * 0.f;
  const bool sick = row_ok && is_nan(check) && !is_nan(lsum);
  uint64_t again = __builtin_amdgcn_ballot_w64(sick);
  again |= again >> 32;
  again &= 0xffffffffull;                   // a bit a row
  uint32_t repaired = 0;
  while (again) {
    const int n = __ffsll((unsigned long long)again) - 1;
    again &= again - 1;
    const int rr = row0 + n, ri = rr / f.group, rh = hk * f.group + rr % f.group;
    if (!spoiled_row<BF, PAGED>(f, st, r.pos + ri, 0, nblk, block_at)) continue;
    repaired |= 1u << n;
    float x[2], rl;
    repair_row<BF, PAGED>(f, st, f.q + b * f.qs_b + (int64_t)(r.row0 + ri) * f.qs_n + rh * f.qs_h, r.pos + ri, 0, nblk,
                          block_at, x, rl);
    if (part) {
      float* dst = f.topart + ((int64_t)it.index * TT + wave * 32 + n) * HD;
      dst[2 * lane] = x[0];
      dst[2 * lane + 1] = x[1];
      if (lane == 0) f.tlpart[(int64_t)it.index * TT + wave * 32 + n] = rl;
    } else {
      char* dst = f.o + b * f.os_b + (int64_t)(r.row0 + ri) * f.os_n + rh * f.os_h;
      *reinterpret_cast<uint32_t*>(dst + 4 * lane) = narrow<BF>(x[0]) | (uint32_t)narrow<BF>(x[1]) << 16;
      if (f.lse && lane == 0) f.lse[b * f.ls_b + (int64_t)(r.row0 + ri) * f.ls_n + rh * f.ls_h] = rl;
    }
  }
  const bool done = repaired >> l32 & 1;
  const int orow = min(row0 + l32, rows - 1), oi = orow / f.group, ohead = hk * f.group + orow % f.group;
  if (part) {
    if (!row_ok || done) return;
    if (hf == 0) f.tlpart[(int64_t)it.index * TT + wave * 32 + l32] = lse;
    float* const prow = f.topart + ((int64_t)it.index * TT + wave * 32 + l32) * HD;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<float4*>(prow + dt * 32 + 8 * g + 4 * hf) =
            float4{acc[dt][4 * g] * inv, acc[dt][4 * g + 1] * inv, acc[dt][4 * g + 2] * inv, acc[dt][4 * g + 3] * inv};
    return;
  }
  if (f.lse && hf == 0 && row_ok && !done) f.lse[b * f.ls_b + (int64_t)(r.row0 + oi) * f.ls_n + ohead * f.ls_h] = lse;
  // A lane holds 4 dims here and there of one row; the wave turns its rows around
  // in 8 KiB of the ring, chunk c of row n at c ^ n % 16, and stores whole rows.
  const int64_t obase = b * f.os_b + (int64_t)(r.row0 + oi) * f.os_n + ohead * f.os_h;
  char* turn = lds + wave * (32 * ROW_BYTES);
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      u16x4 out;
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = narrow<BF>(acc[dt][4 * g + e] * inv);
      *reinterpret_cast<u16x4*>(turn + l32 * ROW_BYTES + (((4 * dt + g) ^ (l32 & 15)) << 4) + hf * 8) = out;
    }
  // All reads before the stores, which a branch each would keep apart (0.85 us a tile, not 1.5).
  u32x4 val[8];
  uint32_t lo[8], hi[8];
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const int n = 4 * x + lr;
    val[x] = *reinterpret_cast<const u32x4*>(turn + n * ROW_BYTES + (((lane & 15) ^ (n & 15)) << 4));
    lo[x] = (uint32_t)__shfl((int)obase, n);
    hi[x] = (uint32_t)__shfl((int)(obase >> 32), n);
  }
#pragma unroll
  for (int x = 0; x < 8; ++x) asm volatile("" : "+v"(val[x]), "+v"(lo[x]), "+v"(hi[x]));
  char* const out = f.o + (lane & 15) * 16;
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const int n = 4 * x + lr;
    const int64_t dst = (int64_t)(lo[x] | (uint64_t)hi[x] << 32);
    if (row0 + n < rows && !(repaired >> n & 1)) *reinterpret_cast<u32x4*>(out + dst) = val[x];
  }
}

// Cost of a launch whose tiles, the longest of `longest` blocks, are cut into
// parts of `length` blocks, `items` of them (p = 1: uncut, all of them in the one round
// that fewer tiles than CUs take).
__host__ __device__ inline float cut_cost(int p, int longest, int length, int64_t items) {
  if (p == 1) return longest + kWholeCost;
  if (items > kTileItems) return 1e30f;
  const float rounds = (float)((items + kTileGroups - 1) / kTileGroups);
  return rounds * (length + kPartCost) + kMergeCost + kMergeShare * items;
}
__host__ __device__ inline int cut_length(int p, int longest) {
  const int n = (longest + p - 1) / p;
  return n > 1 ? n : 1;
}

// Which item a workgroup has. The 8 dies take workgroups in turn (die = workgroup
// % 8), and the tiles that read the same keys should be on one die at a time, so
// that its L2 fetches them once, while every die gets its share of long and short
// tiles. Whole tiles: with h = gcd(8, KV heads), die x takes the KV heads hk = x mod h
// and, of request b's tiles counted from the last (the longest come first), those
// with number (x / h + b) mod (8 / h). Parts: the tiles of a part are consecutive,
// and each die has an eighth of all parts, consecutive ones.
struct Dies {
  int die, h, step, heads_kv;
  __device__ __forceinline__ Dies(int die, int heads_kv)
      : die(die), h(min(heads_kv & -heads_kv, 8)), step(8 / h), heads_kv(heads_kv) {}
  __device__ __forceinline__ int first(int b) const { return (die / h + b) & (step - 1); }
  // Whole tiles of request b that the die takes of one head, and of all its heads.
  __device__ __forceinline__ int tiles_of(int b, int tiles) const {
    return max(0, (tiles - first(b) + step - 1) / step);
  }
  __device__ __forceinline__ int items_of(int b, int tiles) const { return heads_kv / h * tiles_of(b, tiles); }
  // The rel-th of these.
  __device__ __forceinline__ Item whole(const Request& r, int b, int tiles, int rel) const {
    const int here = tiles_of(b, tiles), unit = rel / here;
    return Item{b, unit * h + die % h, tiles - 1 - (first(b) + (rel - unit * here) * step), 0, 1, kUncut, 0, 0, r};
  }
  // The rel-th part of request b, whose parts and tiles others precede.
  __device__ __forceinline__ Item part(const Request& r, int b, int tiles, int parts, int length, int rel, int before,
                                       int tiles_before) const {
    const int unit = rel / tiles, hk = unit / parts, at = unit - hk * parts;
    const int tile = tiles - 1 - (rel - unit * tiles), place = hk * tiles + tile;
    return Item{b, hk, tile, at, parts, length, before + place * parts + at, tiles_before + place, r};
  }
  // This die's part number `slot` of `total`; total if it has no such part.
  __device__ __forceinline__ uint32_t eighth(uint32_t slot, uint32_t total) const {
    const uint32_t n = (total + 7) / 8;
    return slot < n ? die * n + slot : total;
  }
};

// The item of workgroup `slot` of its die; b < 0 if it has none. Contiguous: every
// request is alike, and the host has chosen the cut.
template <bool BF, bool PAGED>
__device__ __forceinline__ Item find_item(const AttnArgs& a, const Dies& d, uint32_t slot, char* lds) {
  const int tid = threadIdx.x;
  const Item none{-1, 0, 0, 0, 0, 0, 0, 0, Request{}};
  if constexpr (!PAGED) {
    const Request r = request<PAGED>(a, 0);
    const int tiles = tile_count<PAGED>(a, r);
    if (a.length < kUncut) {
      const int parts = (tile_blocks(a, r) + a.length - 1) / a.length, each = a.heads_kv * tiles * parts;
      const uint32_t total = (uint32_t)a.batch * each, x = d.eighth(slot, total);
      if (x >= total) return none;
      const int b = x / each;
      return d.part(r, b, tiles, parts, a.length, (int)(x - b * each), b * each, b * a.heads_kv * tiles);
    } else {
      // `step` consecutive requests' tiles of a head are dealt to the dies evenly.
      const uint32_t each = (uint32_t)(a.heads_kv / d.h * tiles);
      int b = (int)(slot / each) * d.step, rel = (int)(slot % each);
      while (b < a.batch && rel >= d.items_of(b, tiles)) rel -= d.items_of(b++, tiles);
      return b < a.batch ? d.whole(r, b, tiles, rel) : none;
    }
  } else {
    __shared__ uint32_t wave_sum[TTHREADS / 64][3];
    __shared__ float costs[kCuts];
    __shared__ int longest;
    __shared__ Item found;
    const int lane = tid & 63, wave = tid >> 6;
    const int per = (a.batch + TTHREADS - 1) / TTHREADS;
    const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
    if (tid == 0) {
      longest = 0;
      found.b = -1;
    }
    __syncthreads();
    // All tiles (at most 256 a request: only fewer in all matter) and this die's
    // whole ones before this thread's run of requests.
    uint32_t tiles_mine = 0, whole_mine = 0;
    int2* const loads = reinterpret_cast<int2*>(lds);   // of every request: tiles, blocks
    Request own{};                          // of request b0
    for (int b = b0; b < b1; ++b) {
      const Request r = request<PAGED>(a, b);
      if (b == b0) own = r;
      const int tiles = tile_count<PAGED>(a, r), n = tiles ? tile_blocks(a, r) : 0;
      tiles_mine += min((int64_t)a.heads_kv * tiles, (int64_t)kTileGroups);
      whole_mine += tiles ? d.items_of(b, tiles) : 0;
      if (a.split) {
        loads[b] = int2{(int)min((int64_t)a.heads_kv * tiles, (int64_t)kTileGroups), n};
        if (n) atomicMax(&longest, n);
      }
    }
    const uint32_t scan_t = lanes_sum(tiles_mine), scan_w = lanes_sum(whole_mine);
    if (lane == 63) {
      wave_sum[wave][0] = scan_t;
      wave_sum[wave][1] = scan_w;
    }
    __syncthreads();
    uint32_t all_tiles = 0, tiles_before = scan_t - tiles_mine, before = scan_w - whole_mine, total = 0;
#pragma unroll
    for (int w = 0; w < TTHREADS / 64; ++w) {
      if (w < wave) {
        tiles_before += wave_sum[w][0];
        before += wave_sum[w][1];
      }
      all_tiles += wave_sum[w][0];
      total += wave_sum[w][1];
    }
    // Fewer tiles than CUs: cut them if that is modelled to be faster. Wave w looks
    // at cuts of the longest tile into w + 1, w + 9, .. parts.
    int length = kUncut;
    const bool few = a.split && all_tiles < kTileGroups;     // uniform
    if (few) {
      for (int p = wave + 1; p <= kCuts; p += TTHREADS / 64) {
        const int n = cut_length(p, longest);
        int items = 0;
        for (int b = lane; b < a.batch; b += 64) items += loads[b].x * ((loads[b].y + n - 1) / n);
        items = (int)lanes_sum((uint32_t)items);
        if (lane == 63) costs[p - 1] = cut_cost(p, longest, n, items);
      }
      __syncthreads();
      int best = 1;
      float least = costs[0];
#pragma unroll
      for (int p = 2; p <= kCuts; ++p) {    // unrolled: its reads do not wait for each other
        const float x = costs[p - 1];
        best = x < least ? p : best;
        least = x < least ? x : least;
      }
      if (best > 1) length = cut_length(best, longest);
    }
    const bool cut = length < kUncut;
    if (a.split && blockIdx.x == 0 && tid == 0) a.tdesc[0] = cut ? (int)all_tiles : 0;
    uint32_t mine = whole_mine, x = slot;
    if (cut) {
      mine = 0;
      for (int b = b0; b < b1; ++b) mine += loads[b].x * ((loads[b].y + length - 1) / length);
      const uint32_t scan = lanes_sum(mine);
      if (lane == 63) wave_sum[wave][2] = scan;
      __syncthreads();
      before = scan - mine;
      total = 0;
#pragma unroll
      for (int w = 0; w < TTHREADS / 64; ++w) {
        if (w < wave) before += wave_sum[w][2];
        total += wave_sum[w][2];
      }
      x = d.eighth(slot, total);
    }
    if (x >= total) return none;            // uniform
    if (before <= x && x - before < mine) {
      uint32_t rel = x - before;
      Request r = own;
      for (int b = b0; b < b1; ++b) {
        if (b > b0) r = request<PAGED>(a, b);
        const int tiles = tile_count<PAGED>(a, r);
        if (!tiles) continue;
        const int parts = cut ? (loads[b].y + length - 1) / length : 1;
        const uint32_t n = cut ? (uint32_t)(a.heads_kv * tiles * parts) : (uint32_t)d.items_of(b, tiles);
        if (rel >= n) {
          rel -= n;
          before += n;
          tiles_before += a.heads_kv * tiles;
          continue;
        }
        found = cut ? d.part(r, b, tiles, parts, length, (int)rel, (int)before, (int)tiles_before)
                    : d.whole(r, b, tiles, (int)rel);
        break;
      }
    }
    __syncthreads();
    // None: requests that overlap, counted past 32 bits.
    return found.b < 0 ? none : found;
  }
}

// In a mixed launch the workgroups from a.tile_groups on do the row kernel's work, in
// 8 waves: they fill the CUs that have no long tile (22 decoding requests beside two
// chunks of 1000 tokens: 136 us, one kernel after the other 166).
template <bool BF, bool PAGED, bool MIXED>
__global__ void __launch_bounds__(TTHREADS) __attribute__((amdgpu_waves_per_eu(2, 2)))
fa_serve_tiles_kernel(AttnArgs a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ int flag;
  if constexpr (MIXED)
    if ((int)blockIdx.x >= a.tile_groups) {
      rows_share<BF, PAGED, 8>(a, blockIdx.x - a.tile_groups, lds);
      return;
    }
  const Dies d(blockIdx.x & 7, a.heads_kv);
  const Item found = find_item<BF, PAGED>(a, d, blockIdx.x >> 3, lds);
  const Item it{uniform(found.b),      uniform(found.hk),    uniform(found.tile),       uniform(found.part), uniform(found.parts),
                uniform(found.length), uniform(found.index), uniform(found.tile_index), uniform(found.r)};
  if (!PAGED && blockIdx.x == 0 && threadIdx.x == 0 && a.split)
    a.tdesc[0] = a.length < kUncut ? a.batch * a.heads_kv * tile_count<PAGED>(a, request<PAGED>(a, 0)) : 0;
  if (it.b < 0) return;                     // no item
  if (it.length < kUncut && it.part == 0 && threadIdx.x == 0) {
    int* desc = a.tdesc + (it.tile_index + 1) * DESC_INTS;
    desc[0] = it.b;
    desc[1] = it.hk;
    desc[2] = it.tile;
    desc[3] = it.index;
    desc[4] = it.parts;
  }
  __syncthreads();                          // the LDS that find_item used is free
  tile_item<BF, PAGED>(a, it, lds, &flag);
}

// Joins the parts of the tiles, 8 rows a workgroup, 32 lanes a row (4 dims each). Bound by
// memory: 480 parts of 96 tiles (63 MB) 17 us, 3.7 TB/s.
template <bool BF, bool PAGED>
__device__ __forceinline__ void merge_tiles(const AttnArgs& a, int block) {
  const int t = block >> 5;
  if (t >= a.tdesc[0]) return;
  const int* d = a.tdesc + (t + 1) * DESC_INTS;
  const int parts = d[4];
  if (parts < 2) return;
  const int b = d[0], hk = d[1], n = (block & 31) * 8 + (threadIdx.x >> 5), dim = (threadIdx.x & 31) * 4;
  const Request r = request<PAGED>(a, b);
  const int row = d[2] * TT + n;
  if (row >= r.n * a.group) return;
  const int64_t at = (int64_t)d[3] * TT + n;
  float M = -INFINITY;
  for (int s = 0; s < parts; ++s) M = smax(M, a.tlpart[at + (int64_t)s * TT]);
  float total = 0.f;
  float4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < parts; ++s) {
    const float x = a.tlpart[at + (int64_t)s * TT];
    const float4 v = *reinterpret_cast<const float4*>(a.topart + (at + (int64_t)s * TT) * HD + dim);
    if (x == -INFINITY) continue;           // such a part has written no O
    const float w = weight(x, M);
    total += w;
    o.x = __builtin_fmaf(w, v.x, o.x);
    o.y = __builtin_fmaf(w, v.y, o.y);
    o.z = __builtin_fmaf(w, v.z, o.z);
    o.w = __builtin_fmaf(w, v.w, o.w);
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  const int i = row / a.group, head = hk * a.group + row % a.group;
  const u16x4 val = {narrow<BF>(o.x * inv), narrow<BF>(o.y * inv), narrow<BF>(o.z * inv), narrow<BF>(o.w * inv)};
  *reinterpret_cast<u16x4*>(a.o + b * a.os_b + (int64_t)(r.row0 + i) * a.os_n + head * a.os_h + dim * 2) = val;
  if (a.lse && dim == 0)
    a.lse[b * a.ls_b + (int64_t)(r.row0 + i) * a.ls_n + head * a.ls_h] = M == -INFINITY ? M : M + logf(total);
}

// The joins of a launch: of the row kernel's pieces (a.groups - 1 workgroups), of the
// tiles' parts, or both.
template <bool BF, bool PAGED>
__global__ void __launch_bounds__(256) fa_serve_rows_merge_kernel(AttnArgs a) {
  merge_rows<BF, PAGED>(a, blockIdx.x);
}
template <bool BF, bool PAGED>
__global__ void __launch_bounds__(256) fa_serve_tiles_merge_kernel(AttnArgs a) {
  merge_tiles<BF, PAGED>(a, blockIdx.x);
}
template <bool BF>
__global__ void __launch_bounds__(256) fa_serve_mixed_merge_kernel(AttnArgs a) {
  const int rows = a.groups - 1;
  if ((int)blockIdx.x < rows)
    merge_rows<BF, true>(a, blockIdx.x);
  else
    merge_tiles<BF, true>(a, blockIdx.x - rows);
}

// ---------------------------------------------------------------------------
// Host side.

// Which kernel takes a request (row kernel against tile kernel, FP16, 8 query heads a
// KV head, 64 heads where not said):
//   - One row tile: the row kernel. 32 rows of 32 requests of 1000-8000 keys 135 us
//     against 163, of one request of 8000 keys 21 against 37, of 64 requests of
//     4000 keys with one KV head 32 against 53.
//   - More than kRowsMax rows: the tile kernel, as the row kernel reads the keys once a
//     row tile. 96 rows of 32 requests 288 against 172, of one request 28 against 40, but
//     of 4 requests of 60000 keys with one KV head 84 against 69.
//   - In between: the row kernel if the launch has few row tiles. 64 rows of
//     one request (16 tiles) 26 against 38, of 8 requests of 4000 keys (128) 52 against 47,
//     of 64 with one KV head (128) 52 against 55, of the 32 (512) 226 against 171; also
//     beside longer requests, where it fills CUs that have no tile: 20 requests of 48
//     rows (12 heads, one KV head) and two chunks of 1000 tokens 129 against 149, 10 of
//     64 rows and two of 2000 tokens 387 against 490; but 58 of 40 rows (8 KV heads)
//     and two of 300 tokens 261 against 196.
constexpr int64_t kRowsMax = 64, kRowsItems = 128;

struct Kernels {
  const void *rows, *tiles, *mixed, *rows_merge, *tiles_merge, *mixed_merge;
};
template <bool BF, bool PAGED>
constexpr Kernels kernels_of() {
  return {reinterpret_cast<const void*>(&fa_serve_rows_kernel<BF, PAGED>),
          reinterpret_cast<const void*>(&fa_serve_tiles_kernel<BF, PAGED, false>),
          reinterpret_cast<const void*>(&fa_serve_tiles_kernel<BF, true, true>),
          reinterpret_cast<const void*>(&fa_serve_rows_merge_kernel<BF, PAGED>),
          reinterpret_cast<const void*>(&fa_serve_tiles_merge_kernel<BF, PAGED>),
          reinterpret_cast<const void*>(&fa_serve_mixed_merge_kernel<BF>)};
}
const Kernels kKernels[2][2] = {{kernels_of<false, false>(), kernels_of<false, true>()},
                                {kernels_of<true, false>(), kernels_of<true, true>()}};

// Raises the LDS limit of every attention kernel on the current device, once.
constexpr int kMaxDevices = 64;
int ensure_lds_limits() {
  static std::atomic<bool> done[kMaxDevices];
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return FA_SERVE_ERR_LAUNCH;
  const bool known = dev >= 0 && dev < kMaxDevices;
  if (known && done[dev].load(std::memory_order_acquire)) return FA_SERVE_OK;
  for (const auto& type : kKernels)
    for (const Kernels& k : type) {
      if (hipFuncSetAttribute(k.rows, hipFuncAttributeMaxDynamicSharedMemorySize, rows_lds(4)) != hipSuccess ||
          hipFuncSetAttribute(k.tiles, hipFuncAttributeMaxDynamicSharedMemorySize, kTileLds) != hipSuccess ||
          hipFuncSetAttribute(k.mixed, hipFuncAttributeMaxDynamicSharedMemorySize, kTileLds) != hipSuccess)
        return FA_SERVE_ERR_LAUNCH;
    }
  if (known) done[dev].store(true, std::memory_order_release);
  return FA_SERVE_OK;
}

// What a call launches, from what the host knows: bounds on the rows.
struct LaunchPlan {
  bool rows = false, tiles = false, split = false;
  int rows_max = 0;                         // for the kernels: see AttnArgs
  int64_t tiles_max = 0;                    // tiles, if the requests are all consistent
  int length = kUncut;
  uint64_t opart = 0, lpart = 0, desc = 0, topart = 0, tlpart = 0, tdesc = 0, end = 0;   // offsets
};
LaunchPlan launch_plan(int64_t batch, int64_t heads_kv, int64_t group, int64_t tokens, int64_t max_new, bool even) {
  LaunchPlan p;
  const int64_t most = max_new * group;     // rows of a request
  const int64_t items = heads_kv * std::min(batch * (kRowsMax / RT), tokens * group / RT + batch);
  p.tiles = most > (items > kRowsItems ? RT : kRowsMax);
  p.rows_max = (int)(most > kRowsMax ? kRowsMax : RT);
  // One kernel takes every request if all have few rows, or all as many, or
  // there is one request.
  p.rows = !p.tiles || (batch > 1 && !even);
  if (!p.rows) p.rows_max = 0;
  if (!p.tiles) p.rows_max = INT32_MAX;
  p.tiles_max = heads_kv * (even ? batch * ((max_new * group + TT - 1) / TT) : tokens * group / TT + batch);
  p.split = p.tiles && (!even || p.tiles_max < kTileGroups);
  auto take = [&](uint64_t bytes) {
    const uint64_t at = p.end;
    p.end += (bytes + 255) / 256 * 256;
    return at;
  };
  if (p.rows) {
    p.opart = take((uint64_t)2 * kRowsGroups * RT * HD * 4);
    p.lpart = take((uint64_t)2 * kRowsGroups * RT * 4);
    p.desc = take((uint64_t)kRowsGroups * DESC_INTS * 4);
  }
  if (p.split) {
    p.topart = take((uint64_t)kTileItems * TT * HD * 4);
    p.tlpart = take((uint64_t)kTileItems * TT * 4);
    p.tdesc = take((uint64_t)(kTileGroups + 1) * DESC_INTS * 4);
  }
  return p;
}

int check_heads(int64_t heads_q, int64_t heads_kv) {
  return heads_q < 1 || heads_kv < 1 || heads_q > 4096 || heads_q % heads_kv ? FA_SERVE_ERR_GEOMETRY : FA_SERVE_OK;
}
int check_mask(int64_t window, int64_t sinks) {
  return window < 0 || sinks < 0 || (sinks && !window) ? FA_SERVE_ERR_WINDOW : FA_SERVE_OK;
}
// c = scale log2 e: scores times c must neither vanish nor overflow for ordinary scores.
int check_scale(float scale) { return scale > 0.f && isfinite(scale) ? FA_SERVE_OK : FA_SERVE_ERR_SCALE; }
int check_type(int32_t type) {
  return type == FA_SERVE_FP16 || type == FA_SERVE_BF16 ? FA_SERVE_OK : FA_SERVE_ERR_TYPE;
}
// Rows of K and V within a page (or of a contiguous tensor) are 32-bit apart.
int check_rows(int64_t stride) { return stride < HD || stride >= 1 << 25 ? FA_SERVE_ERR_STRIDE : FA_SERVE_OK; }

// A workgroup for every item there can be: each die's share of whole tiles rounds
// up once a request and head.
int64_t tile_groups(const LaunchPlan& lp, int64_t batch, int64_t heads_kv) {
  const int64_t h = std::min<int64_t>(heads_kv & -heads_kv, 8);
  const int64_t grid = 8 * (lp.tiles_max / 8 + heads_kv / h * batch + 1);
  return std::max<int64_t>(grid, lp.split ? kTileItems : 8);
}

int run(const AttnArgs& filled, const LaunchPlan& lp, int32_t type, bool paged, void* workspace, void* stream) {
  AttnArgs a = filled;
  int rc = check_stream_device(stream);
  if (!rc) rc = ensure_lds_limits();
  if (rc) return rc;
  char* ws = static_cast<char*>(workspace);
  a.opart = reinterpret_cast<float*>(ws + lp.opart);
  a.lpart = reinterpret_cast<float*>(ws + lp.lpart);
  a.desc = reinterpret_cast<int*>(ws + lp.desc);
  a.topart = reinterpret_cast<float*>(ws + lp.topart);
  a.tlpart = reinterpret_cast<float*>(ws + lp.tlpart);
  a.tdesc = reinterpret_cast<int*>(ws + lp.tdesc);
  a.rows_max = lp.rows_max;
  a.split = lp.split;
  a.length = lp.length;
  a.groups = !lp.rows ? 0 : lp.tiles ? kRowsGroups / 2 : kRowsGroups;
  const Kernels& k = kKernels[type == FA_SERVE_BF16][paged];
  void* args[] = {&a};
  if (lp.tiles) {
    a.tile_groups = (int)tile_groups(lp, a.batch, a.heads_kv);
    rc = enqueue(lp.rows ? k.mixed : k.tiles, dim3((unsigned)(a.tile_groups + a.groups)), dim3(TTHREADS), args,
                 kTileLds, stream);
  } else {
    rc = enqueue(k.rows, dim3(a.groups), dim3(256), args, rows_lds(4), stream);
  }
  const unsigned joins = (a.groups ? a.groups - 1 : 0) + (lp.split ? kTileGroups * 32 : 0);
  if (!rc && joins)
    rc = enqueue(!lp.tiles ? k.rows_merge : lp.rows ? k.mixed_merge : k.tiles_merge, dim3(joins), dim3(256), args, 0, stream);
  return rc;
}

// The row kernel counts the key blocks of all its items in 32 bits; the tile
// kernel's launch has fewer than 2^32 threads.
int check_work(const LaunchPlan& lp, int64_t batch, int64_t heads_kv, int64_t group, int64_t rows, int64_t keys) {
  if (lp.tiles && tile_groups(lp, batch, heads_kv) + kRowsGroups >= ((int64_t)1 << 32) / TTHREADS)
    return FA_SERVE_ERR_GEOMETRY;
  if (!lp.rows) return FA_SERVE_OK;
  const int64_t tiles = lp.tiles ? batch * (kRowsMax / RT) : rows * group / RT + batch;
  return tiles <= ((int64_t)1 << 31) / heads_kv / (keys / BLOCK + 2) ? FA_SERVE_OK : FA_SERVE_ERR_GEOMETRY;
}

int check_paged(const fa_paged* p, LaunchPlan* lp) {
  if (!p) return FA_SERVE_ERR_NULL;
  const int64_t limit = (int64_t)1 << 30;
  int rc = check_heads(p->heads_q, p->heads_kv);
  if (rc) return rc;
  if (p->batch < 1 || p->batch > 4096 || p->tokens < 0 || p->max_new < 1 || p->pages < 0 || p->pages > limit ||
      p->max_pages < 1 || p->max_pages > limit)
    return FA_SERVE_ERR_GEOMETRY;
  if (page_shift(p->page_size) < 0) return FA_SERVE_ERR_PAGE;
  // Rows and keys are counted in 32 bits, packed rows too.
  if (p->tokens >= limit / (p->heads_q / p->heads_kv) || p->max_pages > limit / p->page_size)
    return FA_SERVE_ERR_GEOMETRY;
  rc = check_type(p->type);
  if (!rc) rc = check_mask(p->window, p->sinks);
  if (!rc) rc = check_scale(p->scale);
  if (rc) return rc;
  *lp = launch_plan(p->batch, p->heads_kv, p->heads_q / p->heads_kv, p->tokens,
                    std::min(p->max_new, std::max<int64_t>(p->tokens, 1)), false);
  return check_work(*lp, p->batch, p->heads_kv, p->heads_q / p->heads_kv, p->tokens, p->max_pages * p->page_size);
}

AttnArgs mask_args(int64_t window, int64_t sinks, float scale) {
  AttnArgs a{};
  a.window = window ? (int)std::min<int64_t>(window, NO_WINDOW) : NO_WINDOW;
  a.sinks = (int)std::min<int64_t>(sinks, NO_WINDOW);
  a.c = (float)((double)scale * LOG2E);
  return a;
}

AttnArgs window_args(const fa_window* p) {
  AttnArgs a = mask_args(p->window, p->sinks, p->scale);
  a.batch = (int)p->batch;
  a.heads_kv = (int)p->heads_kv;
  a.group = (int)(p->heads_q / p->heads_kv);
  a.seq_q = (int)p->seq_q;
  a.seq_k = (int)p->seq_k;
  a.off = p->causal == FA_WINDOW_BOTTOM_RIGHT ? (int)(p->seq_k - p->seq_q) : 0;
  return a;
}

int check_window(const fa_window* p, LaunchPlan* lp) {
  if (!p) return FA_SERVE_ERR_NULL;
  const int64_t limit = (int64_t)1 << 30;
  int rc = check_heads(p->heads_q, p->heads_kv);
  if (rc) return rc;
  if (p->batch < 1 || p->batch > 65536 || p->seq_q < 1 || p->seq_k < 1 || p->seq_k >= limit ||
      p->seq_q >= limit / (p->heads_q / p->heads_kv))
    return FA_SERVE_ERR_GEOMETRY;
  rc = check_type(p->type);
  if (!rc && (p->window < 1 || p->sinks < 0)) rc = FA_SERVE_ERR_WINDOW;
  if (!rc) rc = check_scale(p->scale);
  if (!rc && p->causal != FA_WINDOW_TOP_LEFT && p->causal != FA_WINDOW_BOTTOM_RIGHT) rc = FA_SERVE_ERR_CAUSAL;
  if (rc) return rc;
  *lp = launch_plan(p->batch, p->heads_kv, p->heads_q / p->heads_kv, p->batch * p->seq_q, p->seq_q, true);
  if (lp->split) {
    const AttnArgs a = window_args(p);
    const int longest = tile_blocks(a, request<false>(a, 0));
    float least = 0.f;
    for (int cut = 1; cut <= kCuts; ++cut) {
      const int n = cut_length(cut, longest);
      const float cost = cut_cost(cut, longest, n, lp->tiles_max * ((longest + n - 1) / n));
      if (cut == 1 || cost < least) {
        least = cost;
        lp->length = cut == 1 ? kUncut : n;
      }
    }
    lp->split = lp->length < kUncut;
    if (!lp->split) lp->end = lp->topart;   // nothing but the parts is behind them
  }
  return check_work(*lp, p->batch, p->heads_kv, p->heads_q / p->heads_kv, p->batch * p->seq_q, p->seq_k);
}

}  // namespace

extern "C" {

int fa_paged_workspace_bytes(const fa_paged* p, uint64_t* bytes) {
  LaunchPlan lp;
  const int rc = check_paged(p, &lp);
  if (rc) return rc;
  if (!bytes) return FA_SERVE_ERR_NULL;
  *bytes = lp.end;
  return FA_SERVE_OK;
}

int fa_paged_fwd(const fa_paged* p, const void* q, const void* k_cache, const void* v_cache, const int32_t* table,
                 const int32_t* starts, const int32_t* lengths, void* o, float* lse, void* workspace,
                 uint64_t workspace_bytes, void* stream) {
  LaunchPlan lp;
  int rc = check_paged(p, &lp);
  if (rc) return rc;
  if (p->table_stride < p->max_pages || p->table_stride > (int64_t)1 << 30) return FA_SERVE_ERR_STRIDE;
  for (const int64_t* s : {p->q, p->o})
    if (!rc) rc = check_strides(s, 2);
  for (const int64_t* s : {p->k_cache, p->v_cache}) {
    if (!rc) rc = check_strides(s, 3);
    if (!rc) rc = check_rows(s[1]);
    // The page's byte stride is a 32-bit factor of a 64-bit product.
    if (!rc && s[0] >= (int64_t)1 << 31) rc = FA_SERVE_ERR_STRIDE;
  }
  if (rc) return rc;
  if (!k_cache || !v_cache || !table || !starts || !lengths || (p->tokens && (!q || !o))) return FA_SERVE_ERR_NULL;
  for (const void* ptr : {q, k_cache, v_cache, (const void*)o, (const void*)workspace})
    if (!aligned(ptr, 16)) return FA_SERVE_ERR_ALIGN;
  for (const void* ptr : {(const void*)table, (const void*)starts, (const void*)lengths, (const void*)lse})
    if (!aligned(ptr, 4)) return FA_SERVE_ERR_ALIGN;
  if ((lp.end && !workspace) || workspace_bytes < lp.end) return FA_SERVE_ERR_WORKSPACE;
  if (p->tokens == 0) return FA_SERVE_OK;
  AttnArgs a = mask_args(p->window, p->sinks, p->scale);
  a.q = static_cast<const char*>(q);
  a.k = static_cast<const char*>(k_cache);
  a.v = static_cast<const char*>(v_cache);
  a.o = static_cast<char*>(o);
  a.lse = lse;
  a.table = table;
  a.starts = starts;
  a.lengths = lengths;
  a.table_stride = p->table_stride;
  a.qs_n = 2 * p->q[0];
  a.qs_h = 2 * p->q[1];
  a.os_n = 2 * p->o[0];
  a.os_h = 2 * p->o[1];
  a.ks_b = 2 * p->k_cache[0];
  a.ks_n = (int)(2 * p->k_cache[1]);
  a.ks_h = 2 * p->k_cache[2];
  a.vs_b = 2 * p->v_cache[0];
  a.vs_n = (int)(2 * p->v_cache[1]);
  a.vs_h = 2 * p->v_cache[2];
  a.ls_n = p->heads_q;
  a.ls_h = 1;
  a.batch = (int)p->batch;
  a.heads_kv = (int)p->heads_kv;
  a.group = (int)(p->heads_q / p->heads_kv);
  a.tokens = (int)p->tokens;
  a.pages = (int)p->pages;
  a.shift = page_shift(p->page_size);
  a.max_pages = (int)p->max_pages;
  return run(a, lp, p->type, true, workspace, stream);
}

int fa_window_workspace_bytes(const fa_window* p, uint64_t* bytes) {
  LaunchPlan lp;
  const int rc = check_window(p, &lp);
  if (rc) return rc;
  if (!bytes) return FA_SERVE_ERR_NULL;
  *bytes = lp.end;
  return FA_SERVE_OK;
}

int fa_window_fwd(const fa_window* p, const void* q, const void* k, const void* v, void* o, float* lse,
                  void* workspace, uint64_t workspace_bytes, void* stream) {
  LaunchPlan lp;
  int rc = check_window(p, &lp);
  if (rc) return rc;
  for (const int64_t* s : {p->q, p->k, p->v, p->o})
    if (!rc) rc = check_strides(s, 3);
  if (!rc) rc = check_rows(p->k[2]);
  if (!rc) rc = check_rows(p->v[2]);
  if (rc) return rc;
  if (!q || !k || !v || !o) return FA_SERVE_ERR_NULL;
  for (const void* ptr : {q, k, v, (const void*)o, (const void*)workspace})
    if (!aligned(ptr, 16)) return FA_SERVE_ERR_ALIGN;
  if (!aligned(lse, 4)) return FA_SERVE_ERR_ALIGN;
  if ((lp.end && !workspace) || workspace_bytes < lp.end) return FA_SERVE_ERR_WORKSPACE;
  AttnArgs a = window_args(p);
  a.q = static_cast<const char*>(q);
  a.k = static_cast<const char*>(k);
  a.v = static_cast<const char*>(v);
  a.o = static_cast<char*>(o);
  a.lse = lse;
  a.qs_b = 2 * p->q[0];
  a.qs_h = 2 * p->q[1];
  a.qs_n = 2 * p->q[2];
  a.os_b = 2 * p->o[0];
  a.os_h = 2 * p->o[1];
  a.os_n = 2 * p->o[2];
  a.ks_b = 2 * p->k[0];
  a.ks_h = 2 * p->k[1];
  a.ks_n = (int)(2 * p->k[2]);
  a.vs_b = 2 * p->v[0];
  a.vs_h = 2 * p->v[1];
  a.vs_n = (int)(2 * p->v[2]);
  a.ls_b = p->heads_q * p->seq_q;
  a.ls_h = p->seq_q;
  a.ls_n = 1;
  return run(a, lp, p->type, false, workspace, stream);
}

const char* fa_serve_strerror(int status) {
  switch (status) {
    case FA_SERVE_OK: return "ok";
    case FA_SERVE_ERR_NULL: return "a required pointer is NULL";
    case FA_SERVE_ERR_GEOMETRY: return "a size is out of range, or heads_q is no multiple of heads_kv";
    case FA_SERVE_ERR_TYPE: return "unknown element type";
    case FA_SERVE_ERR_PAGE: return "page size must be a power of two from 16 to 65536";
    case FA_SERVE_ERR_ALIGN: return "a pointer or stride is not aligned";
    case FA_SERVE_ERR_WORKSPACE: return "workspace missing or too small";
    case FA_SERVE_ERR_WINDOW: return "invalid window or sinks";
    case FA_SERVE_ERR_SCALE: return "scale must be finite and positive";
    case FA_SERVE_ERR_ROTARY: return "rotary dims must be a multiple of 16 from 16 to 128, in a known layout";
    case FA_SERVE_ERR_LAUNCH: return "the HIP runtime rejected a launch";
    case FA_SERVE_ERR_STRIDE: return "a stride is out of range";
    case FA_SERVE_ERR_CAUSAL: return "unknown causal alignment";
    case FA_SERVE_ERR_DEVICE: return "the stream belongs to another device than the current one";
    default: return "unknown status";
  }
}

}  // extern "C"
