// Argument blocks of the rotary and paged-cache entries of the library, filled in by ops/rotary.py and ops/paged.py and by the
// native host part (host_ext.cpp). All fields are 64 bits wide; strides are in elements.
#pragma once

// One tensor of a rotary launch: [batch, tokens, heads, dim], or rows of a paged cache as destination
// (dst_batch, dst_token: of a page, and of a token in it).
struct UaRotPart {
  const void* src;
  void* dst;
  long heads;
  long rotate;               // 0: copied
  long paged;                // 1: dst is a cache, rows by slot
  long src_batch, src_token, src_head;
  long dst_batch, dst_token, dst_head;
};

struct UaRotary {
  UaRotPart part[3];
  long n_parts;
  long batch, per_batch;     // sequences and tokens of one
  const void* pos;           // position of every token
  long pos64;                // 1: 64-bit positions, 0: 32-bit
  long pos_batch, pos_token;
  const int* slots;          // paged parts: page * page size + offset in it; negative: the token is not written
  long page_shift, n_slots;
  const double* inv_freq;    // angle per position of every pair
  long pairs, dim;
  long interleaved, inverse;
  long dtype;                // 0 bf16, 1 fp16, 2 fp32
};
// Attention of new tokens over a paged cache.
struct UaPagedAttn {
  const void* q;             // [tokens, heads, 128] bf16
  long tokens, heads;
  long q_token, q_head;
  const void *k, *v;         // [pages, page size, kv heads, 128] bf16
  long pages, kv_heads;
  long k_page, k_token, k_head;
  long v_page, v_token, v_head;
  long page_shift;
  const int* table;          // [requests, columns] pages of a request, in order
  long table_stride, columns;
  const int* context;        // [requests] keys of a request, the new tokens among them
  const int* cu_new;         // [requests + 1] first new token of a request
  long requests;
  long most_new;             // no request has more new tokens
  long left, sink;           // window: keys from position p - left on (negative: all), and the first `sink`
  void* o;                   // [tokens, heads, 128] bf16
  long o_token, o_head;
  float* lse;                // [heads, tokens]
  long lse_head;
};
static_assert(sizeof(UaPagedAttn) == 30 * 8, "ops/paged.py packs 30 words");
static_assert(sizeof(UaRotary) == (33 + 16) * 8, "ops/rotary.py packs 49 words");
