// Arguments of the paged key/value cache kernels (kvcache.hip), filled by the bindings.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace zoo {

constexpr int kKvMaxGroup = 256;        // query heads that may share one kv head
constexpr int kKvMaxSlots = 1 << 30;    // slots one sequence may name
constexpr int kEvictHeld = 16384;       // slots of a row that one workgroup selects from, its keys in LDS
constexpr int kEvictSeg = 1024;         // slots of a workgroup where a row is shared out
constexpr int kEvictRow = 16 + 3 * 2048;  // ints of a row's selection state where it is shared out

// unsigned n / d for n < 2^31 as (mulhi(n, m) + n) >> s (Granlund and Montgomery's round-up method)
struct FastDiv {
  uint32_t d, m, s;
};

// element strides of a pool [pages, kv_heads, page, ...]
struct PoolStride {
  long page, head, row;
};

struct PagedAttnArgs {
  const void* q;             // [B, H * G, D], strides q_b / q_h
  const void* k;
  const void* v;
  const int* table;          // [B, width], row stride table_b
  const int* len;            // [B]
  const float* scores;       // pools [pages, H, page], or null: no weights wanted
  float* scores_out;
  void* o;                   // [B, H * G, D]
  float* logits;             // [B, H * G, pitch] raw products q.k (weights only)
  float* part_o;             // [items, gs, D] partial sums of a split sequence
  float* part_ml;            // [items, wide, 2] their running maximum (log2 units) and sum
  int4* plan;                // [items, 2] who does what, for the join; null where there is none
  long q_b, q_h, table_b;
  PoolStride ks, vs, ss, sos;
  FastDiv page;
  int B, H, G, D, pages, cap;
  int pitch;                 // cap rounded up to 16
  int dtype;                 // 0 bf16, 1 fp16, 2 fp32
  int wide;                  // query heads of a workgroup: 16 or 32
  int gs;                    // min(G, wide)
  int single;                // 1: every sequence is one work item
  int held;                  // 1: no `logits`, an unsplit sequence's products stay in LDS
  int hbs;                   // workgroups to the query heads of a kv head
  FastDiv step;              // H * hbs: items from one chunk to the next
  float per_target;          // 0.999 / target: the chunks to aim at over the batch, per head block
  float cached;              // slots of the batch up to which keys and values are left in the caches
  int big;                   // whether there can be more, for sequences of one work item each
  int at_once;               // chunks per head block that the chip can run at once, 0: fewer than B
  float c;                   // scale * log2(e)
};

struct PagedAppendArgs {
  const void* k;             // [B, T, H, D]
  const void* v;
  void* kp;
  void* vp;
  const int* table;
  const int* len;
  const int* counts;         // [B] or null: T tokens each
  const int* seen;           // [B] or null: the position of a token is its slot
  float* scores;             // pools or null
  int* positions;
  int* len_out;
  long k_b, k_t, k_h, v_b, v_t, v_h, table_b;
  PoolStride ks, vs, ss, ps;
  FastDiv page, vec, heads;  // vec: 16-byte pieces of a row
  int B, T, H, pages, cap, es;
};

struct PagedEvictArgs {
  void* kp;
  void* vp;
  const float* scores;
  const int* positions;
  float* scores_out;
  int* positions_out;
  const int* table;
  const int* len;
  const int* seen;
  int* len_out;
  int* moves;                // [B, H, 2, most]: slots given up below the budget, and the kept ones that take them
  int* count;                // [B, H] how many of each
  int* hist;                 // rows shared out: [B * H, kEvictRow] zeroed, then [B * H, segs * 4] Counts
  int* keys;                 // rows shared out: [B * H, cap]
  long table_b;
  PoolStride ks, vs, ss, ps, sos, pos;
  FastDiv page, vec;
  int B, H, pages, cap, es, budget, recent, most;
  int over;                  // budget + slack (at most cap): rows of more slots are cut down
  int fused;                 // 1: so little moves that the selecting workgroup does it
  int segs;                  // workgroups to a row, 0: one, its keys in LDS
};

}  // namespace zoo
