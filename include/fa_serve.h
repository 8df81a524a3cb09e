/*
 * fa_serve.h -- C ABI of libfa_serve.so, the operators a serving program needs
 * next to the attention forward of fa_hip.h on MI355X (gfx950): block tables
 * and slot maps built on the GPU from request lengths, rotary positions
 * written straight into a paged cache, attention of every request's new tokens
 * over that cache, and attention with a sliding window and sinks on contiguous
 * tensors. The reference has none of them.
 *
 * The conventions are fa_hip.h's: every entry point returns 0 on success and a
 * nonzero code otherwise (fa_serve_strerror() names it); everything that can
 * be refused on the host is refused before anything is enqueued; nothing
 * allocates device memory, aborts or synchronises; a call is asynchronous on
 * its stream (a hipStream_t passed as void*, NULL for the default stream),
 * which belongs to the current device, and only launches kernels, so it can be
 * captured in a HIP graph once each attention entry point has been called
 * outside a capture on that device (the first call raises the kernels' LDS
 * limit). Calls on different streams with different workspaces and outputs are
 * independent.
 *
 * Strides are in elements, sizes of 128 dims per head; q, k, v, o and the
 * caches are FP16 or BF16 (enum fa_serve_type) with contiguous dims, 16-byte
 * aligned pointers and non-negative strides that are multiples of 8. Integers
 * in device memory are int32.
 *
 * A paged cache is a pair of buffers (k and v) of `pages` pages of `page_size`
 * tokens of `heads_kv` heads. Slot s of it is token s % page_size of page
 * s / page_size. Request b's tokens 0, 1, ... lie in the pages its row of the
 * block table lists, in order.
 */
#ifndef FA_SERVE_H
#define FA_SERVE_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum fa_serve_status {
  FA_SERVE_OK = 0,
  FA_SERVE_ERR_NULL = 1,       /* a required pointer is NULL */
  FA_SERVE_ERR_GEOMETRY = 2,   /* a size out of range, or heads_q % heads_kv != 0 */
  FA_SERVE_ERR_TYPE = 3,       /* unknown element type */
  FA_SERVE_ERR_PAGE = 4,       /* page size not a power of two in 16 .. 65536 */
  FA_SERVE_ERR_ALIGN = 5,      /* a pointer or stride that is not aligned */
  FA_SERVE_ERR_WORKSPACE = 6,  /* workspace missing or too small */
  FA_SERVE_ERR_WINDOW = 7,     /* negative window or sinks, or sinks without a window */
  FA_SERVE_ERR_SCALE = 8,      /* scale not finite and positive */
  FA_SERVE_ERR_ROTARY = 9,     /* rotary dims not a multiple of 16 in 16 .. 128, or unknown layout */
  FA_SERVE_ERR_LAUNCH = 10,    /* the HIP runtime rejected a launch */
  FA_SERVE_ERR_STRIDE = 11,    /* a stride out of range */
  FA_SERVE_ERR_CAUSAL = 12,    /* unknown alignment of the window's diagonal */
  FA_SERVE_ERR_DEVICE = 16     /* the stream belongs to another device than the current one */
};

enum fa_serve_type { FA_SERVE_FP16 = 0, FA_SERVE_BF16 = 1 };

/*
 * Block tables and slot maps from request lengths: request b holds past[b]
 * tokens and gets fresh[b] more. Its first ceil(past / page_size) table entries
 * are there already; the new tokens' further pages are taken from pages[],
 * from index *taken on, request by request in order, and entered in the
 * table. Writes
 *   table[b][j]   the new entries (others are left alone)
 *   starts[b]     sum of fresh[0 .. b-1]; starts[batch] is the sum of all
 *   lengths[b]    past[b] + fresh[b]
 *   positions[t]  past[b] + i for token i of request b, t = starts[b] + i
 *   slots[t]      where that token is stored
 *   *taken_out    *taken plus the pages needed
 * Tokens t >= starts[batch] get position 0 and slot -1. With too few pages
 * left (*taken_out > pages_count) the entries and slots past the last page are
 * -1; so are the slots of tokens that do not fit a table row (max_pages).
 * Negative lengths count as 0. The call may be repeated: nothing it reads is
 * overwritten but with the same values (taken_out is not taken).
 */
typedef struct fa_page_plan {
  int64_t batch;          /* requests, 1 .. 4096 */
  int64_t tokens;         /* entries of positions and slots */
  int64_t page_size;
  int64_t max_pages;      /* entries of a table row */
  int64_t table_stride;   /* elements from one table row to the next, >= max_pages */
  int64_t pages_count;    /* entries of pages[] */
} fa_page_plan;
int fa_plan_pages(const fa_page_plan* p, const int32_t* past, const int32_t* fresh, int32_t* table,
                  const int32_t* pages, const int32_t* taken, int32_t* starts, int32_t* lengths,
                  int32_t* positions, int32_t* slots, int32_t* taken_out, void* stream);

/*
 * Rotary positions. Token t's pair i of a head, (x0, x1), becomes
 *   ((x0 cos a - x1 sin a) factor, (x1 cos a + x0 sin a) factor),
 *   a = 2 pi turns[i] positions[t], i < rotary_dim / 2,
 * where the pair is dims (i, i + rotary_dim / 2) (FA_ROTARY_HALF) or
 * (2i, 2i + 1) (FA_ROTARY_INTERLEAVED); dims from rotary_dim on stay. With
 * `backward` the sign of a is turned, which makes the map its own transpose:
 * the gradient of the rotation. turns[] (FP64, device) is the rotation per
 * position in turns, so the angle of a far position loses nothing.
 *
 * q [tokens, heads_q, 128] goes to q_out. k [tokens, heads_kv, 128] goes
 * rotated to k_cache, v unrotated to v_cache, at slots[t]; a token whose slot
 * is negative or past the cache is not stored. Slots of one call that are
 * stored are distinct. heads_kv = 0 leaves out k, v, the caches and slots.
 * q_out may be q, with q's strides; no other two tensors overlap.
 */
enum fa_rotary_layout { FA_ROTARY_HALF = 0, FA_ROTARY_INTERLEAVED = 1 };
typedef struct fa_rotary {
  int64_t tokens, heads_q, heads_kv, rotary_dim;
  int64_t pages, page_size;
  float factor;
  int32_t type;                      /* enum fa_serve_type */
  int32_t layout;                    /* enum fa_rotary_layout */
  int32_t backward;
  int64_t q[2], q_out[2], k[2], v[2];      /* strides of tokens and heads */
  int64_t k_cache[3], v_cache[3];          /* strides of pages, tokens and heads */
} fa_rotary;
int fa_rotary_append(const fa_rotary* p, const void* q, void* q_out, const void* k, const void* v,
                     const int32_t* positions, const int32_t* slots, const double* turns,
                     void* k_cache, void* v_cache, void* stream);

/*
 * Attention of new tokens over a paged cache that holds them already. Request
 * b's new tokens are rows starts[b] .. starts[b+1]-1 of q and o [tokens,
 * heads_q, 128], the last of its lengths[b] tokens: row i stands at position
 * p = lengths[b] - (starts[b+1] - starts[b]) + i and sees key j iff j <= p and,
 * with a window, j > p - window or j < sinks. o = softmax(q k^T scale) v over
 * the visible keys, query head h with KV head h / (heads_q / heads_kv); a row
 * that sees no key gets o = 0 and lse = -inf. lse [tokens, heads_q] (FP32) may
 * be NULL. What the cache holds at keys a row does not see has no influence on
 * it, NaN and infinities included. Scores are FP32 and may reach 1e7 in magnitude
 * (scale q.k); a row that sees an infinite or NaN score gets NaN.
 *
 * max_new is a bound on the new tokens of a request, known to the caller; it
 * chooses kernels only, a larger request is still computed. Rows outside
 * every request (t >= starts[batch]) are left as they were. starts[] values
 * outside 0 .. tokens are clamped. A row gets NaN if its request is longer than
 * its table row (max_pages * page_size) or a page its tile reads is outside
 * 0 .. pages-1.
 *
 * o overlaps nothing that the call reads: rows are written while others are read.
 *
 * Workspace: fa_paged_workspace_bytes(); its contents on entry do not matter.
 * Calls that may overlap need a workspace each.
 */
typedef struct fa_paged {
  int64_t batch, tokens, heads_q, heads_kv;
  int64_t max_new;
  int64_t pages, page_size, max_pages, table_stride;
  int64_t window;                    /* 0: none */
  int64_t sinks;
  float scale;
  int32_t type;                      /* enum fa_serve_type */
  int64_t q[2], o[2];                /* strides of tokens and heads */
  int64_t k_cache[3], v_cache[3];    /* strides of pages, tokens and heads */
} fa_paged;
int fa_paged_workspace_bytes(const fa_paged* p, uint64_t* bytes);
int fa_paged_fwd(const fa_paged* p, const void* q, const void* k_cache, const void* v_cache,
                 const int32_t* table, const int32_t* starts, const int32_t* lengths, void* o,
                 float* lse, void* workspace, uint64_t workspace_bytes, void* stream);

/*
 * Attention with a causal sliding window and sinks on q [B, Hq, Nq, 128] and
 * k, v [B, Hkv, Nk, 128]: row i at position p = i (FA_WINDOW_TOP_LEFT) or
 * i + Nk - Nq (FA_WINDOW_BOTTOM_RIGHT) sees key j iff j <= p and (j > p -
 * window or j < sinks). Everything else as in fa_paged_fwd(); lse [B, Hq, Nq]
 * contiguous, or NULL.
 */
enum fa_window_causal { FA_WINDOW_TOP_LEFT = 1, FA_WINDOW_BOTTOM_RIGHT = 2 };
typedef struct fa_window {
  int64_t batch, heads_q, heads_kv, seq_q, seq_k;
  int64_t window, sinks;
  float scale;
  int32_t type;                      /* enum fa_serve_type */
  int32_t causal;                    /* enum fa_window_causal */
  int64_t q[3], k[3], v[3], o[3];    /* strides of dims B, H and N */
} fa_window;
int fa_window_workspace_bytes(const fa_window* p, uint64_t* bytes);
int fa_window_fwd(const fa_window* p, const void* q, const void* k, const void* v, void* o,
                  float* lse, void* workspace, uint64_t workspace_bytes, void* stream);

/* Static message for a status code. */
const char* fa_serve_strerror(int status);

#ifdef __cplusplus
}
#endif

#endif /* FA_SERVE_H */
