// The key/value cache of generation: attention of one new token over a paged cache, appending
// tokens to it, evicting from it by gathered attention weight.
//
// Cache. Keys and values lie in pools [pages, H, page, D]; slot s of sequence b is row s % page of
// page table[b, s / page]. A page id that names no page, or a length outside the table, is never
// followed: that sequence's attention comes out NaN, its tokens are not written and it is not
// evicted from. Nothing here waits for another workgroup and no order of atomics matters, so results
// repeat bit for bit.
//
// Attention. For one kv head and the G query heads that share it
//   s_gj = scale q_g.k_j,   w_gj = exp(s_gj - lse_g),   o_g = sum_j w_gj v_j,   lse_g = log sum_j exp s_gj
// in one pass over the slots with a running maximum and sum. Every byte of K and V is used for G
// products, so the pass is bound by HBM. The work goes to the matrix cores (heads padded to 16
// columns) because a VALU form would need 2G fma per element and reductions across lanes.
//
// One wave streams tiles of slots straight from memory into MFMA operands, without LDS:
//   S = K Q^T   A = 16 slots x 32 dims of K: lane l holds slot l % 16, dims 8 (l / 16) .. + 8, which is a
//               16-byte load. The C layout leaves head l % 16 and slots 4 (l / 16) + r in the lane.
//   O = V^T P   B = P in the order in which S left it: the k index of an MFMA may name the slots in any
//               order as long as A uses the same one. So the lane needs slots 4 (l / 16) + r of two
//               16-slot halves for one dim; it loads 8 dims of each of these 8 slots (16 bytes a row, 16
//               lanes to a row, 256 bytes contiguous) and transposes the 8 x 8 block in its registers
//               with v_perm: MFMA e takes dim 8 (l % 16) + e.
// P is fed as the sum of three bfloat16 numbers, which hold all 24 bits of it, or of two float16 numbers (22 bits):
// rounding it to one would cost an error as large as the output's own rounding, and two bfloat16 numbers (16 bits) still
// turn one in 200 of the outputs' roundings. The third costs nothing where HBM is the bound (64 sequences of 16k slots 633 us
// with two and three), and some where latency is (32 of up to 512 with weights 12.6 us and 13.1, 200 of 500 with pages of 7
// 50 and 55).
//
// The slots of all sequences are cut into equal chunks, one per workgroup, whose number aims at
// filling the chip whatever the batch and the lengths (find_work): lengths are only known on the
// device, so every workgroup derives the cut from them itself. A join kernel merges a sequence's
// chunks and, where weights are wanted, turns the stored products into sum_g w_gj.
//
// Measured on one MI355X (a large copy: 4.8 TB/s): 64 sequences of 16k slots, 8 kv heads of 128, 64 query heads, bf16:
// 633 us, 6.8 TB/s; 24 of up to 8k, fp16: 78 us, 5.4 TB/s; one of 131k with weights: 111 us with the join, 4.9 TB/s;
// 32 of up to 512, 12 heads of 64, with weights: 13 us, of which 5 are the chain of look-ups, loads and the epilogue that
// a call over 77 slots takes alone.
#include <math.h>

#include <type_traits>

#include "common.h"
#include "kvcache.h"

namespace zoo {
namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// NT: past the caches, for what will not be read again before it would have left them anyway
template <bool NT>
ZOO_DEV uint4 load16(const void* p) {
  if constexpr (NT) return __builtin_bit_cast(uint4, __builtin_nontemporal_load((const u32x4*)p));
  return *(const uint4*)p;
}
template <bool NT>
ZOO_DEV uint2 load8(const void* p) {
  if constexpr (NT) return __builtin_bit_cast(uint2, __builtin_nontemporal_load((const u32x2*)p));
  return *(const uint2*)p;
}

enum { kBf16 = 0, kF16 = 1, kF32 = 2 };

// v_exp_f32: one instruction, within an ulp; results under 2^-126 are 0
ZOO_DEV float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

ZOO_DEV uint32_t fdiv(uint32_t n, const FastDiv& f) { return (__umulhi(n, f.m) + n) >> f.s; }

// Lengths and tables, which nothing writes while a kernel here runs, are read through the constant address
// space: wave-uniform look-ups become scalar loads, which answer sooner and do not queue behind the vector loads
// in flight.
typedef const __attribute__((address_space(4))) int* cint;
ZOO_DEV cint fixed(const int* p) { return (cint)p; }

// slots of sequence b, or -1 where its length does not fit its table
ZOO_DEV int seq_len(const int* len, int b, int cap) {
  const int n = fixed(len)[b];
  return n < 0 || n > cap ? -1 : n;
}

ZOO_DEV int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// inclusive prefix sum over the wave: shifts within rows of 16 lanes, then each row's total to the ones behind it
#define ZOO_DPP(x, ctrl, rows) __builtin_amdgcn_update_dpp(0, (x), ctrl, rows, 0xf, false)
ZOO_DEV int wave_prefix(int x) {
  x += ZOO_DPP(x, 0x111, 0xf);
  x += ZOO_DPP(x, 0x112, 0xf);
  x += ZOO_DPP(x, 0x114, 0xf);
  x += ZOO_DPP(x, 0x118, 0xf);
  x += ZOO_DPP(x, 0x142, 0xa);
  x += ZOO_DPP(x, 0x143, 0xc);
  return x;
}
ZOO_DEV float wave_total(float x) {
  x += __int_as_float(ZOO_DPP(__float_as_int(x), 0x111, 0xf));
  x += __int_as_float(ZOO_DPP(__float_as_int(x), 0x112, 0xf));
  x += __int_as_float(ZOO_DPP(__float_as_int(x), 0x114, 0xf));
  x += __int_as_float(ZOO_DPP(__float_as_int(x), 0x118, 0xf));
  x += __int_as_float(ZOO_DPP(__float_as_int(x), 0x142, 0xa));
  x += __int_as_float(ZOO_DPP(__float_as_int(x), 0x143, 0xc));
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), 63));
}
#undef ZOO_DPP

struct Work {
  int b, hk, hb;    // sequence, kv head, block of query heads
  int chunk, n;     // which of the sequence's n chunks
  int s0, s1;       // its slots
  int len;          // the sequence's slots, -1: bad
  int first;        // item of the sequence's chunk 0, same head block
  bool big;         // the batch's keys and values do not fit the last-level cache
};

ZOO_DEV int chunks_of(int len, int size) { return len <= size ? 1 : (int)(((unsigned)len + size - 1) / (unsigned)size); }

// `want` slots rounded up to grains (a power of two), at least one; a sequence has 2^30 slots at most
ZOO_DEV int chunk_size(float want, int grain) {
  return max((int)ceilf(fminf(want, 0x1p30f) / grain), 1) * grain;
}

// The logical item of this workgroup. Blocks of query heads of one kv head read the same keys and values: they are
// put 8 workgroups apart, on one XCD, so that its L2 serves all but the first (there are 8 XCDs, and
// workgroups go to them in turn).
ZOO_DEV int item_of(const PagedAttnArgs& a) {
  const int x = blockIdx.x;
  if (a.hbs == 1) return x;
  const int group = 8 * a.hbs, g = x / group, in = x - g * group;
  return (g + 1) * group <= (int)gridDim.x ? g * group + (in & 7) * a.hbs + (in >> 3) : x;
}

// Cuts the batch into chunks of `size` slots, a multiple of `grain`, such that there are at most
// target (1 + 1 / 512) + B of them per head block, and finds the chunk of this workgroup; every wave does so alone.
// Every sequence has a chunk, if an empty one. False for the items that are not needed.
ZOO_DEV bool find_work(const PagedAttnArgs& a, int grain, Work& w) {
  const int lane = threadIdx.x & 63;
  const int item = item_of(a);
  const int t = fdiv(item, a.step), hh = item - t * a.step.d;
  w.hb = 0, w.hk = hh;
  if (a.hbs > 1) w.hk = hh / a.hbs, w.hb = hh - w.hk * a.hbs;
  if (a.single) {
    w.b = uni(t), w.chunk = 0, w.n = 1, w.first = item, w.big = a.big;
    w.len = seq_len(a.len, w.b, a.cap);
    w.s0 = 0, w.s1 = w.len;
    return true;
  }
  const int mine0 = lane < a.B ? seq_len(a.len, lane, a.cap) : 0;
  float total = (float)max(mine0, 0);
  for (int b = lane + 64; b < a.B; b += 64) total += (float)max(seq_len(a.len, b, a.cap), 0);
  total = wave_total(total);
  w.big = total > a.cached;
  // per_target is 0.999 / target, so that a total that divides evenly is not rounded up to another grain
  int size = chunk_size(total * a.per_target, grain);
  // Sequences end inside chunks, so there are more chunks than the total asks for: if they would
  // not all run at once, longer ones (twice, as this is a fixed point's iteration).
  for (int i = 0; i < 2 && a.at_once > 0; ++i) {
    int n = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
      const int mine = b0 == 0 ? mine0 : b0 + lane < a.B ? seq_len(a.len, b0 + lane, a.cap) : 0;
      n += __builtin_amdgcn_readlane(wave_prefix(b0 + lane < a.B ? chunks_of(mine, size) : 0), 63);
    }
    if (n <= a.at_once) break;
    size = chunk_size((float)size * n / a.at_once, grain);
  }
  int at = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int mine = b0 == 0 ? mine0 : b0 + lane < a.B ? seq_len(a.len, b0 + lane, a.cap) : 0;
    const int chunks = b0 + lane < a.B ? chunks_of(mine, size) : 0;
    const int upto = wave_prefix(chunks);
    const unsigned long long hit = __ballot(at + upto > t);
    if (hit) {
      const int who = __ffsll(hit) - 1;
      w.b = b0 + who;
      w.n = __builtin_amdgcn_readlane(chunks, who);
      w.len = __builtin_amdgcn_readlane(mine, who);
      at += __builtin_amdgcn_readlane(upto, who) - w.n;
      w.chunk = t - at;
      w.first = at * (int)a.step.d + hh;
      w.s0 = w.chunk * size;
      w.s1 = min(w.len, w.s0 + size);
      return true;
    }
    at += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// what find_work found, for the join kernel: n = 0 where there is nothing
ZOO_DEV void put_work(const PagedAttnArgs& a, const Work& w, bool found) {
  if (a.plan != nullptr && threadIdx.x == 0) {
    a.plan[2 * item_of(a)] = make_int4(w.b, w.chunk, found ? w.n : 0, w.len);
    a.plan[2 * item_of(a) + 1] = make_int4(w.s0, w.s1, w.first, 0);
  }
}
ZOO_DEV bool get_work(const PagedAttnArgs& a, Work& w) {
  const int4 x = a.plan[2 * blockIdx.x], y = a.plan[2 * blockIdx.x + 1];
  w.b = uni(x.x), w.chunk = uni(x.y), w.n = uni(x.z), w.len = uni(x.w);
  w.s0 = uni(y.x), w.s1 = uni(y.y), w.first = uni(y.z);
  const int hh = blockIdx.x - fdiv(blockIdx.x, a.step) * a.step.d;
  w.hk = hh / a.hbs, w.hb = hh - w.hk * a.hbs;
  return w.n > 0;
}

template <int DT, int DP>
struct Tile {
  static constexpr int ES = DT == kF32 ? 4 : 2;
  static constexpr int NS = DT == kF32 ? (DP == 64 ? 2 : 1) : (DP == 64 ? 4 : 2);  // 16-slot subtiles
  static constexpr int TS = 16 * NS;
  static constexpr int KL = DP * ES / 64;                  // 16-byte loads of a lane per K subtile
  static constexpr int VB = DP * ES / 16 < 16 ? DP * ES / 16 : 16;  // bytes of one V load
  static constexpr int VC = DP * ES / 16 / VB;             // V loads of a lane per row
  static constexpr int VW = VB / 4;
  static constexpr int VE = VB / ES;                       // dims of one V load
  static constexpr int NA = DP / 16;                       // 16-dim tiles of O
  static constexpr int GRAIN = 4 * TS;
};

template <int DT>
ZOO_DEV f32x4 mma16(const uint4& x, const uint4& y, const f32x4& c) {
  if constexpr (DT == kBf16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0,
                                                  0);
}

// Weights of a sequence of len slots are held times 2 to the power of this. In bfloat16 and float32 it is the first power
// below 1 / len, so that sums of the type's largest values stay finite and those of small ones keep their bits; in
// float16, whose values are far from the ends of float32's range, 2^15 (below its 65504): its parts then hold weights down
// to 2^-38 of the wave's largest.
ZOO_DEV int weight_log(int dt, int len) { return dt == kF16 ? 15 : __clz(len) - 32; }

ZOO_DEV uint32_t high16(float x, float y) { return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u); }
// the upper 16 bits of the float next to x on the side of zero; of 0 for 0
ZOO_DEV float below16(float x) { return __uint_as_float(__builtin_elementwise_sub_sat(__float_as_uint(x), 1u) & 0xffff0000u); }

// Two weights as packed 16-bit numbers whose sum they are. Each part is cut off so that something is left for the
// next one: an infinite value times a weight is then infinite in every part, where a part of 0 would make it NaN.
// Only a weight of 0 has parts of 0, or one so small that its parts leave the type's range (held in float16 below 2^-23, in
// bfloat16 below 2^-102).
// bfloat16: 8 bits in each of three parts, nothing is lost. float16: 11 bits in each of two, an error of 2^-22 of the weight
// and 2^-25 (2^-40 of the wave's largest weight, in either direction, with no sign to add up in); what is below 2^-23
// goes into the second part alone.
template <int DT>
constexpr int kParts = DT == kBf16 ? 3 : 2;

template <int DT>
ZOO_DEV void split(float x, float y, uint32_t (&part)[kParts<DT>]) {
  if constexpr (DT == kBf16) {
    const float x0 = below16(x), y0 = below16(y), xr = x - x0, yr = y - y0;
    const float x1 = below16(xr), y1 = below16(yr);
    part[0] = high16(x0, y0);
    part[1] = high16(x1, y1);
    part[2] = high16(xr - x1, yr - y1);
  } else {
    constexpr float kLess = 1.f - 0x1p-22f;
    const auto h = __builtin_amdgcn_cvt_pkrtz(fmaxf(fmaf(x, kLess, -0x1p-24f), 0.f), fmaxf(fmaf(y, kLess, -0x1p-24f), 0.f));
    part[0] = __builtin_bit_cast(uint32_t, h);
    part[1] = __builtin_bit_cast(uint32_t, f16x2{(_Float16)(x - (float)h[0]), (_Float16)(y - (float)h[1])});
  }
}

template <int DT>
ZOO_DEV void store_out(void* o, long at, float x) {
  if constexpr (DT == kBf16)
    ((uint16_t*)o)[at] = f2bf(x);
  else if constexpr (DT == kF16)
    ((_Float16*)o)[at] = (_Float16)x;
  else
    ((float*)o)[at] = x;
}

ZOO_DEV void store_any(int dt, void* o, long at, float x) {
  if (dt == kBf16)
    store_out<kBf16>(o, at, x);
  else if (dt == kF16)
    store_out<kF16>(o, at, x);
  else
    store_out<kF32>(o, at, x);
}

// scores_out = scores + sum_g 2^(c x_g - lse_g) for the slots s0 .. s1 of one kv head, x the stored products
// of its heads with the slot. A thread has kWays slots under way at a time, and the first of them can
// be asked for (ahead) long before the lse are known: a chain of two loads that would otherwise end the kernel.
constexpr int kWays = 4;
struct Ahead {
  int page[kWays];     // -1: nothing to do
  float was[kWays];
};

ZOO_DEV const float* logits_of(const PagedAttnArgs& a, int b, int hk) {
  return a.logits + ((long)b * a.H + hk) * a.G * a.pitch;
}

ZOO_DEV Ahead weights_ahead(const PagedAttnArgs& a, int b, int hk, int s, int s1) {
  const int* table = a.table + (long)b * a.table_b;
  const float* in = a.scores + (long)hk * a.ss.head;
  Ahead x;
#pragma unroll
  for (int u = 0; u < kWays; ++u) x.page[u] = table[fdiv(min(s + u * (int)blockDim.x, s1 - 1), a.page)];
#pragma unroll
  for (int u = 0; u < kWays; ++u) {
    const int at = s + u * blockDim.x;
    if ((unsigned)x.page[u] >= (unsigned)a.pages || at >= s1) x.page[u] = -1;
    x.was[u] = x.page[u] < 0 ? 0.f : in[x.page[u] * a.ss.page + (long)(at - fdiv(at, a.page) * a.page.d) * a.ss.row];
  }
  return x;
}

// The log of the sums that stands for a sequence with a bad page: its slots gather nothing, on good pages either. What
// data can give is finite, -inf or NaN. (Where it is summed from, a maximum of NaN stands for one: a maximum that fmaxf
// found is never NaN.)
constexpr float kBadLse = INFINITY;

// `logit`: of the kv head's first query head, in memory or in LDS
ZOO_DEV void gather_weights(const PagedAttnArgs& a, int b, int hk, int s0, int s1, Ahead x, const float* lse,
                            const float* logit) {
  if (lse[0] == kBadLse) return;    // pages are a sequence's: all its heads say so
  const int G = a.G, step = blockDim.x;
  float* out = a.scores_out + (long)hk * a.sos.head;
  for (int s = s0 + threadIdx.x; s < s1; s += kWays * step) {
    float sum[kWays];
#pragma unroll
    for (int u = 0; u < kWays; ++u) sum[u] = 0.f;
#pragma unroll 4
    for (int g = 0; g < G; ++g) {
#pragma unroll
      for (int u = 0; u < kWays; ++u)
        sum[u] += pow2(fmaf(logit[(long)g * a.pitch + min(s + u * step, s1 - 1)], a.c, -lse[g]));
    }
    Ahead y = x;
    if (s + kWays * step < s1) x = weights_ahead(a, b, hk, s + kWays * step, s1);
#pragma unroll
    for (int u = 0; u < kWays; ++u)
      if (y.page[u] >= 0) {
        const int at = s + u * step;
        out[y.page[u] * a.sos.page + (long)(at - fdiv(at, a.page) * a.page.d) * a.sos.row] = y.was[u] + sum[u];
      }
  }
}

// DP: the head width rounded up; PAD: it was rounded; P16: pages of a multiple of 16 rows, so that a
// 16-slot subtile lies in one page and its address is wave-uniform. Other page sizes look up a page per
// slot. NB: blocks of 16 query heads that share what was loaded. Three workgroups to a CU where the registers allow it; in 16
// bits with pages of any size they do not without spilling (200 sequences of 500 slots, pages of 7: two 55 us, three 60).
template <int DT, int DP, bool PAD, bool P16, int NB>
__global__ __launch_bounds__(256, DP == 256 ? 1 : NB == 2 || (DT != kF32 && !P16) || (DT == kF32 && DP == 128 && PAD) ? 2 : 3) void paged_attn_kernel(
    const PagedAttnArgs a) {
  using T = Tile<DT, DP>;
  constexpr int NS = T::NS, KL = T::KL, VC = T::VC, VW = T::VW, VE = T::VE, NA = T::NA, ES = T::ES;
  constexpr int W = 16 * NB;
  // Dims that only the padding has: left out in 32 bits, where their products take time (16 of 64 dims 194 us and 216 with
  // them, 136 of 256 136 and 156); in 16 bits the branches cost more (16 of 64 139 and 111).
  constexpr bool SKIP = PAD && DT == kF32;
  extern __shared__ float lds[];  // [4][gb][DP + 4] sums, then [4][W][2] maximum and sum
  __shared__ float lse[W];
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  // An unsplit sequence's first page can be looked up before its length is known: the look-up that counts then
  // finds it in the scalar cache.
  int early = 0;
  if (P16 && a.single && a.cap > 0)
    early = fixed(a.table + (long)fdiv(item_of(a), a.step) * a.table_b)[fdiv(min(wave * T::TS, a.cap - 1), a.page)];
  Work w{};
  const bool found = find_work(a, T::GRAIN, w);
  asm volatile("" ::"s"(early));   // keeps the look-up
  put_work(a, w, found);
  if (!found) return;
  const int row = lane & 15, quad = lane >> 4;
  const int gb = min(W, a.G - W * w.hb), D = a.D;
  const int head0 = w.hk * a.G + W * w.hb;
  const long out0 = ((long)w.b * a.H * a.G + head0) * D;
  const int up = weight_log(DT, w.len);
  const float up2 = __uint_as_float((uint32_t)(127 + up) << 23);
  if (w.len <= 0) {
    const float x = w.len < 0 ? __builtin_nanf("") : 0.f;
    for (int i = threadIdx.x; i < gb * D; i += 256) store_out<DT>(a.o, out0 + i, x);
    return;
  }

  // Q^T: heads row, 16 + row, the dims that K's loads bring. Heads and dims that are not there are zero.
  uint4 q[NB][KL];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const int h = 16 * n + row;
    const char* qp = (const char*)a.q + ((long)w.b * a.q_b + (long)(head0 + min(h, gb - 1)) * a.q_h) * ES;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int at = i * 64 + quad * 16;
      const bool in = h < gb && (!PAD || at < D * ES);
      q[n][i] = mask4(*(const uint4*)(qp + (!PAD || at < D * ES ? at : 0)), in);
    }
  }
  const int* table = a.table + (long)w.b * a.table_b;
  const char* kb = (const char*)a.k + (long)w.hk * a.ks.head * ES;
  const char* vb = (const char*)a.v + (long)w.hk * a.vs.head * ES;
  const long klane = (long)row * a.ks.row * ES + quad * 16;
  const long vlane = (long)(quad * 4) * a.vs.row * ES;
  const int vdim = row * T::VB;  // PAD: dims past D load the row's first ones, and no result of theirs is stored
  bool bad = false;

  uint4 kr[NS][KL];
  uint32_t vr[NS][4][VC][VW];

  [[maybe_unused]] auto page_of = [&](int slot) {
    const int p = fixed(table)[fdiv(slot, a.page)];
    const bool ok = (unsigned)p < (unsigned)a.pages;
    bad |= !ok;
    return ok ? p : 0;
  };
  // Pages of any size: lane l looks up slot l of the tile, the page number one tile ahead, and the rows' offsets go from
  // lane to lane (54 rows of up to 29k slots, 24 heads of 64, pages of 100: 55 us; with look-ups by every lane for itself,
  // five a subtile, 100; pages of 64 53).
  int ahead_id = 0;
  long k_at = 0, v_at = 0;
  auto slot_of = [&](int base) { return min(base + (lane & (T::TS - 1)), w.s1 - 1); };
  auto load_k = [&](int base, auto nt) {
    constexpr bool NT = decltype(nt)::value;
    if constexpr (!P16) {
      const int s = slot_of(base);
      const bool ok = (unsigned)ahead_id < (unsigned)a.pages;
      bad |= !ok;
      const long id = ok ? ahead_id : 0, off = s - fdiv(s, a.page) * a.page.d;
      k_at = (id * a.ks.page + off * a.ks.row) * ES;
      v_at = (id * a.vs.page + off * a.vs.row) * ES;
      ahead_id = table[fdiv(slot_of(base + T::GRAIN), a.page)];
    }
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      const char* p;
      if constexpr (P16) {
        const int s = min(base + 16 * u, (w.s1 - 1) & ~15);
        p = kb + ((long)uni(page_of(s)) * a.ks.page + (long)(s - fdiv(s, a.page) * a.page.d) * a.ks.row) * ES + klane;
      } else {
        p = kb + __shfl(k_at, 16 * u + row, 64) + quad * 16;
      }
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        if constexpr (PAD) {
          if (SKIP && i * 64 >= D * ES) break;
          const bool in = i * 64 + quad * 16 < D * ES;
          kr[u][i] = mask4(load16<NT>(p + (in ? i * 64 : -quad * 16)), in);
        } else {
          kr[u][i] = load16<NT>(p + i * 64);
        }
      }
    }
  };
  auto load_v = [&](int base, auto nt) {
    constexpr bool NT = decltype(nt)::value;
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      const char* p0 = vb;
      if constexpr (P16) {
        const int s = min(base + 16 * u, (w.s1 - 1) & ~15);
        p0 += ((long)uni(page_of(s)) * a.vs.page + (long)(s - fdiv(s, a.page) * a.page.d) * a.vs.row) * ES + vlane;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const char* p = p0;
        if constexpr (P16) {
          p += (long)r * a.vs.row * ES;
        } else {
          p += __shfl(v_at, 16 * u + 4 * quad + r, 64);
        }
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          const int at = c * 256 + vdim;
          const char* pc = p + (!PAD || at < D * ES ? at : 0);
          if constexpr (VW == 4) {
            const uint4 x = load16<NT>(pc);
            vr[u][r][c][0] = x.x, vr[u][r][c][1] = x.y, vr[u][r][c][2] = x.z, vr[u][r][c][3] = x.w;
          } else {
            const uint2 x = load8<NT>(pc);
            vr[u][r][c][0] = x.x, vr[u][r][c][1] = x.y;
          }
        }
      }
    }
  };

  f32x4 acc[NB][NA];
  float m[NB], l[NB];  // of heads 16 n + row; l of this lane's slots only
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    m[n] = -INFINITY, l[n] = 0.f;
#pragma unroll
    for (int i = 0; i < NA; ++i) acc[n][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  float* logit = a.logits ? a.logits + ((long)w.b * a.H * a.G + head0 + row) * a.pitch + 4 * quad : nullptr;
  float* held = lds + 4 * gb * (DP + 4) + 8 * W;   // [gb][pitch] where the products fit

  auto stream = [&](auto nt) {
    int base = w.s0 + wave * T::TS;
    if (base < w.s1) {
      if constexpr (!P16) ahead_id = table[fdiv(slot_of(base), a.page)];
      load_k(base, nt);
      load_v(base, nt);
    }
    for (; base < w.s1; base += T::GRAIN) {
      const bool more = base + T::GRAIN < w.s1, tail = base + T::TS > w.s1;
      f32x4 s[NB][NS];
#pragma unroll
      for (int n = 0; n < NB; ++n)
#pragma unroll
        for (int u = 0; u < NS; ++u) {
          f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 0; i < KL; ++i) {
            if (SKIP && i * 64 >= D * ES) break;
            if constexpr (DT == kF32) {
              const uint4 &k = kr[u][i], &y = q[n][i];
              x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.x), __uint_as_float(y.x), x, 0, 0, 0);
              x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.y), __uint_as_float(y.y), x, 0, 0, 0);
              x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.z), __uint_as_float(y.z), x, 0, 0, 0);
              x = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k.w), __uint_as_float(y.w), x, 0, 0, 0);
            } else {
              x = mma16<DT>(kr[u][i], q[n][i], x);
            }
          }
          s[n][u] = x;
        }
      if (more) load_k(base + T::GRAIN, nt);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        if (a.held && 16 * n + row < gb) {
#pragma unroll
          for (int u = 0; u < NS; ++u)
            if (base + 16 * u < w.s1) *(f32x4*)(held + (16 * n + row) * a.pitch + base + 16 * u + 4 * quad) = s[n][u];
        }
        if (logit != nullptr && 16 * n + row < gb) {
          // rows are padded to whole subtiles, so 4 slots go at once
#pragma unroll
          for (int u = 0; u < NS; ++u)
            if (base + 16 * u < w.s1) *(f32x4*)(logit + (long)(16 * n) * a.pitch + base + 16 * u) = s[n][u];
        }
        float top = m[n];
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[n][u][r] *= a.c;
            if (tail && base + 16 * u + 4 * quad + r >= w.s1) s[n][u][r] = -INFINITY;
            top = fmaxf(top, s[n][u][r]);
          }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float mu = top == -INFINITY ? 0.f : top;  // nothing but -inf so far: every weight is 0, not NaN
        const float old = pow2(m[n] - mu);
        m[n] = top;
        l[n] *= old;
        if (__any(old != 1.f)) {
#pragma unroll
          for (int i = 0; i < NA; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[n][i][r] *= old;
        }
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            s[n][u][r] = pow2(s[n][u][r] - mu) * up2;
            l[n] += s[n][u][r];
          }
      }
      // a slot behind the last has weight 0, but 0 times what its row happens to hold may be NaN
      if (tail) {
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t keep = base + 16 * u + 4 * quad + r < w.s1 ? 0xffffffffu : 0u;
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
              for (int i = 0; i < VW; ++i) vr[u][r][c][i] &= keep;
          }
      }
      if constexpr (DT == kF32) {
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int c = 0; c < VC; ++c)
#pragma unroll
              for (int e = 0; e < VE; ++e)
#pragma unroll
                for (int n = 0; n < NB; ++n)
                  acc[n][c * VE + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                      __uint_as_float(vr[u][r][c][e]), s[n][u][r], acc[n][c * VE + e], 0, 0, 0);
      } else {
#pragma unroll
        for (int u = 0; u < NS; u += 2) {
          uint32_t w2[NB][4][kParts<DT>];
#pragma unroll
          for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int i = 0; i < 4; ++i) split<DT>(s[n][u + i / 2][2 * (i & 1)], s[n][u + i / 2][2 * (i & 1) + 1], w2[n][i]);
#pragma unroll
          for (int c = 0; c < VC; ++c)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
              const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
              uint4 x;
              x.x = __builtin_amdgcn_perm(vr[u][1][c][e / 2], vr[u][0][c][e / 2], sel);
              x.y = __builtin_amdgcn_perm(vr[u][3][c][e / 2], vr[u][2][c][e / 2], sel);
              x.z = __builtin_amdgcn_perm(vr[u + 1][1][c][e / 2], vr[u + 1][0][c][e / 2], sel);
              x.w = __builtin_amdgcn_perm(vr[u + 1][3][c][e / 2], vr[u + 1][2][c][e / 2], sel);
#pragma unroll
              for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int p = 0; p < kParts<DT>; ++p)
                  acc[n][c * VE + e] =
                      mma16<DT>(x, make_uint4(w2[n][0][p], w2[n][1][p], w2[n][2][p], w2[n][3][p]), acc[n][c * VE + e]);
            }
        }
      }
      if (more) load_v(base + T::GRAIN, nt);
    }
  };
  // Rows that were padded share cache lines with their neighbours, which a load past the caches reads again (16 heads, 64
  // sequences, bf16: 80 dims, 4096 slots 240 us through the caches and 301 past them, 200 dims 578 and 718, 96 277 and 304;
  // 16 dims, 16384 slots 355 and 351).
  if (!PAD && w.big)
    stream(std::bool_constant<!PAD>{});
  else
    stream(std::false_type{});
  const bool weights = a.held || (w.n == 1 && a.logits != nullptr && a.G <= W);
  Ahead ahead;
  if (weights && threadIdx.x < w.s1) ahead = weights_ahead(a, w.b, w.hk, threadIdx.x, w.s1);
  // the four waves' sums meet in LDS
  constexpr int LD = DP + 4;
  float* ml = lds + 4 * gb * LD;
  const bool wrong = __any(bad);
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    l[n] += __shfl_xor(l[n], 16, 64);
    l[n] += __shfl_xor(l[n], 32, 64);
    const int h = 16 * n + row;
    if (h < gb) {
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          lds[(wave * gb + h) * LD + (i / VE) * (16 * VE) + (quad * 4 + r) * VE + i % VE] = acc[n][i][r];
      if (quad == 0) {
        ml[(wave * W + h) * 2] = wrong ? __builtin_nanf("") : m[n];   // and so everything that is summed with it
        ml[(wave * W + h) * 2 + 1] = l[n];
      }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < gb * DP; i += 256) {
    const int g = i / DP, d = i & (DP - 1);
    float top = -INFINITY;
    bool bad_page = false;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      top = fmaxf(top, ml[(x * W + g) * 2]);
      bad_page |= isnan(ml[(x * W + g) * 2]);
    }
    const float mu = top == -INFINITY ? 0.f : top;
    float sum = 0.f, o = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float f = pow2(ml[(x * W + g) * 2] - mu);
      sum += f * ml[(x * W + g) * 2 + 1];
      o += f * lds[(x * gb + g) * LD + d];
    }
    if (!PAD || d < D) {
      if (w.n == 1)
        store_out<DT>(a.o, out0 + (long)g * D + d, o / sum);
      else
        a.part_o[((long)item_of(a) * a.gs + g) * D + d] = o;
    }
    if (d == 0) {
      if (a.part_ml != nullptr) {
        a.part_ml[((long)item_of(a) * W + g) * 2] = bad_page ? __builtin_nanf("") : top;
        a.part_ml[((long)item_of(a) * W + g) * 2 + 1] = sum;
      }
      lse[g] = bad_page ? kBadLse : top + log2f(sum) - up;
    }
  }
  if (weights) {
    __syncthreads();    // orders the waves' products, which this workgroup reads back, as well
    if (a.held)
      gather_weights(a, w.b, w.hk, 0, w.s1, ahead, lse, held);
    else
      gather_weights(a, w.b, w.hk, 0, w.s1, ahead, lse, logits_of(a, w.b, w.hk));
  }
}

// folds the running maximum and sum (m2, l2), and what is weighted with them, into (m, l)
ZOO_DEV void merge(float& m, float& l, float& x, float m2, float l2, float x2) {
  const float top = fmaxf(m, m2), mu = top == -INFINITY ? 0.f : top;
  const float f = pow2(m - mu), f2 = pow2(m2 - mu);
  l = l * f + l2 * f2;
  x = x * f + x2 * f2;
  m = top;
}

// Joins the chunks of a sequence: chunk c of n writes the c-th part of the outputs, and the gathered
// weights of its own slots. Bound by the latency of its chain of loads, not by bytes: so every thread
// takes the maxima and sums along with the partial outputs instead of waiting for their total first.
constexpr int kJoinThreads = 512;

__global__ __launch_bounds__(kJoinThreads) void paged_attn_join_kernel(const PagedAttnArgs a) {
  __shared__ float lse[kKvMaxGroup], sm[kJoinThreads], sl[kJoinThreads], sx[kJoinThreads];
  Work w;
  if (!get_work(a, w)) return;
  // an unsplit sequence is ready but for the weights of kv heads with more than one block of query heads
  const bool weights = a.logits != nullptr && w.hb == 0 && (w.n > 1 || a.hbs > 1);
  if (w.len <= 0 || (w.n == 1 && !weights)) return;
  const int tid = threadIdx.x;
  const long next = (long)a.step.d * a.wide * 2;   // from one chunk's maxima and sums to the next one's
  Ahead ahead;
  if (weights) {
    if (w.s0 + tid < w.s1) ahead = weights_ahead(a, w.b, w.hk, w.s0 + tid, w.s1);
    // log2 of the sum of exponentials of all heads, 16 threads to a head
    for (int g0 = 0; g0 < a.G; g0 += kJoinThreads / 16) {
      const int g = g0 + (tid >> 4);
      const float* ml = a.part_ml + ((long)(w.first + g / a.wide) * a.wide + g % a.wide) * 2;
      float m = -INFINITY, l = 0.f, x = 0.f;
      bool bad_page = false;
      if (g < a.G) {
#pragma unroll 4
        for (int i = tid & 15; i < w.n; i += 16) {
          const float top = ml[i * next];
          bad_page |= isnan(top);
          merge(m, l, x, top, ml[i * next + 1], 0.f);
        }
      }
      bad_page = __ballot(bad_page) >> (tid & 48) & 0xffff;   // of the 16 threads of this head
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) merge(m, l, x, __shfl_xor(m, o, 64), __shfl_xor(l, o, 64), 0.f);
      if (g < a.G && (tid & 15) == 0) lse[g] = bad_page ? kBadLse : m + log2f(l) - weight_log(a.dtype, w.len);
    }
    if (w.n == 1) __syncthreads();
  }
  if (w.n > 1) {
    const int E = min(a.wide, a.G - a.wide * w.hb) * a.D;
    const int per = ((E + w.n - 1) / w.n + 15) & ~15;
    const int e0 = w.chunk * per, e1 = min(E, e0 + per);
    int wide = 16;
    while (wide < per && wide < kJoinThreads) wide *= 2;
    const int ways = kJoinThreads / wide, who = tid / wide;
    const float* po = a.part_o + (long)w.first * a.gs * a.D;
    const float* ml = a.part_ml + (long)w.first * a.wide * 2;
    const long step_o = (long)a.step.d * a.gs * a.D;
    const long out0 = ((long)w.b * a.H * a.G + w.hk * a.G + a.wide * w.hb) * a.D;
    if (e0 >= e1) __syncthreads();
    for (int e = e0; e < e1; e += wide) {
      const int at = e + (tid & (wide - 1));
      float m = -INFINITY, l = 0.f, x = 0.f;
      if (at < e1) {
        const int g = at / a.D;
#pragma unroll 4
        for (int i = who; i < w.n; i += ways)
          merge(m, l, x, ml[i * next + g * 2], ml[i * next + g * 2 + 1], po[i * step_o + at]);
      }
      // threads of a wave with the same element first: lanes that are `wide` apart
      for (int o = wide; o < 64; o *= 2) merge(m, l, x, __shfl_xor(m, o, 64), __shfl_xor(l, o, 64), __shfl_xor(x, o, 64));
      sm[tid] = m, sl[tid] = l, sx[tid] = x;
      __syncthreads();
      if (who == 0 && at < e1) {
        const int apart = max(wide, 64);
        for (int i = apart + tid; i < kJoinThreads; i += apart) merge(m, l, x, sm[i], sl[i], sx[i]);
        store_any(a.dtype, a.o, out0 + at, x / l);
      }
      __syncthreads();
    }
  }
  if (weights) gather_weights(a, w.b, w.hk, w.s0, w.s1, ahead, lse, logits_of(a, w.b, w.hk));
}

// ---- append: one thread moves 16 bytes of a token's key row and of its value row ----
// Bound by HBM: 16 prompts of up to 2048 tokens, 8 heads of 128, bf16: 144 MB in 28 us, 5.1 TB/s. Neighbouring threads take
// the pieces, then the heads of a token, as a packed projection has them side by side; 32 single tokens: 3.2 us.
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendArgs a, int blocks_per_seq) {
  const int b = blockIdx.x / blocks_per_seq;
  const uint32_t i = (uint32_t)(blockIdx.x - b * blocks_per_seq) * 256 + threadIdx.x;
  const int len = seq_len(a.len, b, a.cap);
  const int count = a.counts ? max(0, min(a.T, a.counts[b])) : a.T;
  if (i == 0) a.len_out[b] = len < 0 ? a.len[b] : len + count;
  const uint32_t hv = fdiv(i, a.vec), piece = i - hv * a.vec.d;
  const int t = fdiv(hv, a.heads), h = hv - t * a.heads.d;
  if (len < 0 || t >= count || t >= a.cap - len) return;
  const int slot = len + t;
  const int pi = fdiv(slot, a.page), p = a.table[b * a.table_b + pi];
  if ((unsigned)p >= (unsigned)a.pages) return;
  const long off = slot - pi * a.page.d;
  const uint4 x = load16<true>((const char*)a.k + (b * a.k_b + t * a.k_t + h * a.k_h) * a.es + piece * 16);
  const uint4 y = load16<true>((const char*)a.v + (b * a.v_b + t * a.v_t + h * a.v_h) * a.es + piece * 16);
  *(uint4*)((char*)a.kp + (p * a.ks.page + h * a.ks.head + off * a.ks.row) * a.es + piece * 16) = x;
  *(uint4*)((char*)a.vp + (p * a.vs.page + h * a.vs.head + off * a.vs.row) * a.es + piece * 16) = y;
  if (piece == 0) {
    if (a.scores) a.scores[p * a.ss.page + h * a.ss.head + off * a.ss.row] = 0.f;
    if (a.positions)
      a.positions[p * a.ps.page + h * a.ps.head + off * a.ps.row] = (a.seen ? a.seen[b] : len) + t;
  }
}

// ---- evict ----
// Order of a slot among those of its head: recent ones first, then by weight; NaN last. As an
// unsigned number that grows with the rank: -0 counts as 0.
ZOO_DEV uint32_t rank_key(float score, bool late) {
  if (late) return 0xffffffffu;
  if (score != score) return 0u;
  const uint32_t u = __float_as_uint(score + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kEvictBins = 2048;
constexpr int kEvictFew = 4;        // so many are found one after the other

// exclusive prefix sum over the workgroup in thread order. Two barriers.
template <int NT>
ZOO_DEV int block_prefix(int x, int* tmp) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int upto = wave_prefix(x);
  if (lane == 63) tmp[wave] = upto;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int i = 0; i < NT / 64; ++i) before += i < wave ? tmp[i] : 0;
  __syncthreads();
  return before + upto - x;
}

// The cut between kept and evicted: a slot is kept if its key is above `key`, or if it equals it and it is among
// the first `ties` of those.
struct Cut {
  uint32_t key;
  int ties;
};

// One digit of a radix selection: finds the bin, from the top, that holds the `left`-th largest of the keys counted
// in `hist`, puts it into the key at `shift` and takes those above it off `left`. True if the bin is kept whole, and
// the selection is finished: then everything from the bin's lowest key on is kept.
template <int NT>
ZOO_DEV bool pick_bin(const int* hist, int shift, uint32_t& key, int& left, int* tmp, int* res) {
  constexpr int PER = kEvictBins / NT;
  int n[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) sum += n[i] = hist[kEvictBins - 1 - (int)threadIdx.x * PER - i];
  int before = block_prefix<NT>(sum, tmp);
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (before < left && before + n[i] >= left) {
      res[0] = kEvictBins - 1 - (int)threadIdx.x * PER - i;
      res[1] = left - before;
      res[2] = n[i];
    }
    before += n[i];
  }
  __syncthreads();
  key |= (uint32_t)res[0] << shift;
  left = res[1];
  const bool whole = res[1] == res[2];
  __syncthreads();
  return whole;
}
// with every slot of the bin kept, the cut lies below its lowest key (which is not 0: then all would be kept)
ZOO_DEV Cut cut_of(uint32_t key, int left, bool whole) { return whole ? Cut{key - 1u, 0} : Cut{key, left}; }

constexpr int kShift[3] = {21, 10, 0};
constexpr uint32_t kAbove[3] = {0u, 0xffe00000u, 0xfffffc00u};   // the digits already known
constexpr uint32_t kDigit[3] = {2047u, 2047u, 1023u};

// where slot s of a row lies
struct Row {
  const int* table;
  FastDiv page;
  int h;
  ZOO_DEV long at(int s, int p, const PoolStride& st) const {
    return p * st.page + h * st.head + (long)(s - (int)(fdiv(s, page) * page.d)) * st.row;
  }
  ZOO_DEV int id(int s) const { return table[fdiv(s, page)]; }
};

// counts of a stretch of slots: key above the cut or equal to it, below the budget or behind it
struct Counts {
  int gt_lo, eq_lo, gt_hi, eq_hi;
};

template <class Key>
ZOO_DEV Counts count_range(int s0, int s1, int K, const Cut& cut, Key key) {
  Counts c{0, 0, 0, 0};
#pragma unroll 4
  for (int s = s0; s < s1; s += 64) {
    const int at = s + (threadIdx.x & 63);
    const bool in = at < s1;
    const uint32_t k = in ? key(at) : 0u;
    const unsigned long long gt = __ballot(in && k > cut.key), eq = __ballot(in && k == cut.key);
    const unsigned long long lo = __ballot(at < K);
    c.gt_lo += __popcll(gt & lo), c.gt_hi += __popcll(gt & ~lo);
    c.eq_lo += __popcll(eq & lo), c.eq_hi += __popcll(eq & ~lo);
  }
  return c;
}

// Lists, for the slots s0 .. s1 of one wave, those given up below the budget K and those kept behind it, in
// order. `b`: the counts of all slots before s0; `eq_lo`: of the whole row; `masks`: this wave's room in LDS for a bit
// to each of its slots.
template <class Key>
ZOO_DEV void list_range(const PagedEvictArgs& a, const Row& row, int s0, int s1, int K, const Counts& b, int eq_lo,
                        const Cut& cut, int* give, int* take, unsigned long long* masks, Key key) {
  const int lane = threadIdx.x & 63;
  const unsigned long long below = (1ull << lane) - 1;
  int equal = b.eq_lo + b.eq_hi;
  int gave = min(s0, K) - b.gt_lo - min(cut.ties, b.eq_lo);
  int took = b.gt_hi + min(max(cut.ties - eq_lo, 0), b.eq_hi);
  for (int t = s0; t < s1; t += 256) {
    uint32_t keys[4];   // four at a time: the compiler cannot know that the lists are no keys
#pragma unroll
    for (int u = 0; u < 4; ++u) keys[u] = t + 64 * u + lane < s1 ? key(t + 64 * u + lane) : 0u;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = t + 64 * u + lane;
      const bool in = at < s1;
      const unsigned long long eq = __ballot(in && keys[u] == cut.key);
      const bool kept =
          in && (keys[u] > cut.key || (keys[u] == cut.key && equal + __popcll(eq & below) < cut.ties));
      equal += __popcll(eq);
      const bool hole = in && !kept && at < K, tail = kept && at >= K;
      const unsigned long long holes = __ballot(hole), tails = __ballot(tail), stay = __ballot(kept && at < K);
      if (hole) give[gave + __popcll(holes & below)] = at;
      if (tail) take[took + __popcll(tails & below)] = at;
      gave += __popcll(holes);
      took += __popcll(tails);
      if (lane == 0 && t + 64 * u < s1) masks[(t - s0 + 64 * u) >> 6] = stay;
    }
  }
  if (a.scores_out == a.scores && a.positions_out == a.positions) return;
  // scores and positions that stay where they are, in other pools: four slots of a lane under way at a time
  for (int s = s0; s < min(s1, K); s += 256) {
    int p[4], pos[4];
    float score[4];
    bool on[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int at = s + 64 * u + lane;
      on[u] = s + 64 * u < s1 && (masks[(s - s0 + 64 * u) >> 6] >> lane & 1);
      p[u] = on[u] ? row.id(at) : 0;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (on[u]) {
        const int at = s + 64 * u + lane;
        score[u] = a.scores[row.at(at, p[u], a.ss)];
        pos[u] = a.positions[row.at(at, p[u], a.ps)];
      }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (on[u]) {
        const int at = s + 64 * u + lane;
        a.scores_out[row.at(at, p[u], a.sos)] = score[u];
        a.positions_out[row.at(at, p[u], a.pos)] = pos[u];
      }
  }
}

// calls take(slot, key) for the slots s0 + tid, s0 + tid + threads, .. below s1, and returns whether one of their
// pages is bad. Four slots of a thread are under way at a time, without a branch in between: each is a chain of
// two loads (32 x 8 rows of up to 8192 slots 20.6 us, one by one 26).
template <class Take>
ZOO_DEV bool each_key(const PagedEvictArgs& a, const Row& row, int s0, int s1, long oldest, Take take) {
  bool bad = false;
  const int step = blockDim.x;
  for (int s = s0 + threadIdx.x; s < s1; s += 4 * step) {
    int p[4], pos[4];
    float score[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) p[u] = row.id(min(s + u * step, s1 - 1));
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const bool ok = (unsigned)p[u] < (unsigned)a.pages;
      bad |= !ok;
      p[u] = ok ? p[u] : 0;
      const int at = min(s + u * step, s1 - 1);
      score[u] = a.scores[row.at(at, p[u], a.ss)];
      pos[u] = a.positions[row.at(at, p[u], a.ps)];
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (s + u * step < s1) take(s + u * step, rank_key(score[u], pos[u] >= oldest));
  }
  return bad;
}

// Moves the n slots that the lists of row r say, 16 bytes of a key row and of a value row at a time: the pieces first,
// first + step, ..
ZOO_DEV void move_rows(const PagedEvictArgs& a, const Row& row, int r, int n, uint32_t first, uint32_t step) {
  const int* give = a.moves + (long)r * 2 * a.most;
  const uint32_t total = (uint32_t)n * a.vec.d;
  char *kp = (char*)a.kp, *vp = (char*)a.vp;
  for (uint32_t i = first; i < total; i += step) {
    const int m = fdiv(i, a.vec);
    const long piece = (i - m * a.vec.d) * 16;
    const int to = give[m], from = give[a.most + m];
    const int tp = row.id(to), fp = row.id(from);
    const uint4 x = load16<true>(kp + row.at(from, fp, a.ks) * a.es + piece);
    const uint4 y = load16<true>(vp + row.at(from, fp, a.vs) * a.es + piece);
    *(uint4*)(kp + row.at(to, tp, a.ks) * a.es + piece) = x;
    *(uint4*)(vp + row.at(to, tp, a.vs) * a.es + piece) = y;
    if (piece == 0) {
      a.scores_out[row.at(to, tp, a.sos)] = a.scores[row.at(from, fp, a.ss)];
      a.positions_out[row.at(to, tp, a.pos)] = a.positions[row.at(from, fp, a.ps)];
    }
  }
}

// slots that a row of len may keep: one that is within the slack keeps all of them
ZOO_DEV int row_budget(const PagedEvictArgs& a, int len) { return len > a.over ? a.budget : max(len, a.budget); }

// One workgroup per row (sequence and kv head), its keys in LDS: a radix selection of the budget-th largest by
// digits of 11, 11 and 10 bits, then the lists, each wave a stretch of the slots. Bound by its barriers and the latency
// of its loads: 256 rows of up to 8192 slots 21 us, where reading them takes 2. Rows of up to 2048 slots go to 256
// threads, whose barriers are cheaper, longer ones to 1024 (the whole eviction, 384 rows of 513 slots: 8.8 us and with
// 1024 threads 16.4; of 2048: 36.0 and 40.7; of 4096: 60.3 and 58.0; 256 rows of 8192: 87.9 and 65.0).
template <int NT>
__global__ __launch_bounds__(NT) void paged_evict_select_kernel(const PagedEvictArgs a) {
  extern __shared__ uint32_t keys[];
  __shared__ int hist[kEvictBins];
  __shared__ int tmp[NT / 64], res[3], s_bad;
  __shared__ unsigned long long low[2][NT / 64], masks[kEvictHeld / 64 + NT / 64];
  __shared__ Counts counts[NT / 64];
  const int b = blockIdx.x / a.H, tid = threadIdx.x, wave = uni(tid >> 6);
  const Row row{a.table + (long)b * a.table_b, a.page, (int)blockIdx.x - b * a.H};
  const int len = seq_len(a.len, b, a.cap), K = row_budget(a, len);
  const long oldest = (long)a.seen[b] - a.recent;
  const bool digits = len - K > kEvictFew;
  if (tid == 0) s_bad = len < 0;
  if (digits)
    for (int i = tid; i < kEvictBins; i += NT) hist[i] = 0;
  __syncthreads();
  const bool bad = each_key(a, row, 0, len, oldest, [&](int s, uint32_t k) {
    keys[s] = k;
    if (digits) atomicAdd(&hist[k >> kShift[0]], 1);
  });
  if (bad) s_bad = 1;
  __syncthreads();
  const bool leave = s_bad;
  if (tid == 0) {
    a.count[blockIdx.x] = 0;
    if (row.h == 0) a.len_out[b] = leave ? a.len[b] : min(len, K);
  }
  if (leave || len == 0) return;
  auto key = [&](int s) { return keys[s]; };
  Cut cut{0u, len};   // no longer than the budget: all are kept
  int gone = 0;       // slots equal to the cut that go, where that is known rather than how many stay
  if (len > K && !digits) {
    // One slot over the budget at a time is what a decoding step brings. The lowest key, the last of its slots, as
    // many times as slots have to go: each round is one pass and one barrier. 1 of 513: 8.0 us, by digits 11.2.
    unsigned long long last = 0;
    for (int i = 0; i < len - K; ++i) {
      unsigned long long mine = ~0ull;
      for (int s = tid; s < len; s += NT) {
        const unsigned long long x = ((unsigned long long)keys[s] << 32) | (0xffffffffu - (uint32_t)s);
        if ((i == 0 || x > last) && x < mine) mine = x;
      }
#pragma unroll
      for (int o = 32; o > 0; o >>= 1) {
        const unsigned long long x = __shfl_xor(mine, o, 64);
        mine = x < mine ? x : mine;
      }
      if ((tid & 63) == 0) low[i & 1][wave] = mine;
      __syncthreads();
      unsigned long long best = low[i & 1][0];
#pragma unroll
      for (int x = 1; x < NT / 64; ++x) best = low[i & 1][x] < best ? low[i & 1][x] : best;
      const uint32_t k = (uint32_t)(best >> 32);
      gone = k == cut.key && i > 0 ? gone + 1 : 1;
      cut.key = k;
      last = best;
    }
  } else if (len > K) {
    uint32_t known = 0;
    int left = K;
    bool whole = pick_bin<NT>(hist, kShift[0], known, left, tmp, res);
    for (int pass = 1; pass < 3 && !whole; ++pass) {
      for (int i = tid; i < kEvictBins; i += NT) hist[i] = 0;
      __syncthreads();
      for (int s = tid; s < len; s += NT)
        if ((keys[s] & kAbove[pass]) == known) atomicAdd(&hist[(keys[s] >> kShift[pass]) & kDigit[pass]], 1);
      __syncthreads();
      whole = pick_bin<NT>(hist, kShift[pass], known, left, tmp, res);
    }
    cut = cut_of(known, left, whole);
  }
  const int per = ((len + NT - 1) / NT) * 64, s0 = min(len, wave * per), s1 = min(len, s0 + per);
  const Counts mine = count_range(s0, s1, K, cut, key);
  if ((tid & 63) == 0) counts[wave] = mine;
  __syncthreads();
  Counts before{0, 0, 0, 0};
  int eq_lo = 0, eq_all = 0;
  for (int i = 0; i < NT / 64; ++i) {
    const Counts c = counts[i];
    eq_lo += c.eq_lo;
    eq_all += c.eq_lo + c.eq_hi;
    if (i < wave) before.gt_lo += c.gt_lo, before.eq_lo += c.eq_lo, before.gt_hi += c.gt_hi, before.eq_hi += c.eq_hi;
  }
  if (gone > 0) cut.ties = eq_all - gone;
  int* give = a.moves + (long)blockIdx.x * 2 * a.most;
  list_range(a, row, s0, s1, K, before, eq_lo, cut, give, give + a.most, masks + wave * ((len + NT - 1) / NT), key);
  int gt = 0, eq = 0;   // as many are kept behind the budget as are given up below it
  for (int i = 0; i < NT / 64; ++i) gt += counts[i].gt_hi, eq += counts[i].eq_hi;
  const int n = gt + min(max(cut.ties - eq_lo, 0), eq);
  if (a.fused) {
    __syncthreads();
    move_rows(a, row, blockIdx.x, n, tid, NT);
  } else if (tid == 0) {
    a.count[blockIdx.x] = n;
  }
}

// Rows of more slots than one workgroup should take: the same selection with a row shared out in segments of
// kEvictSeg, a launch for each step that needs all of the row before it. Histograms of a row add
// up in memory (whole numbers, so in any order). 8 rows of 131k slots: 35 us in five launches, one workgroup each 590. The
// whole eviction from 8 rows of 16384 slots takes 31 us so and 33 with a workgroup each, from 256 rows 127 and 85: the
// border, kEvictHeld, is where a row's keys stop fitting LDS beside a second workgroup, and suits few long rows, not many.
// STEP 0 .. 2: the digits, 3: counts of each wave's stretch, 4: the lists.
template <int STEP>
__global__ __launch_bounds__(256) void paged_evict_long_kernel(const PagedEvictArgs a) {
  __shared__ int hist[kEvictBins];
  __shared__ int tmp[4], res[3];
  __shared__ unsigned long long masks[kEvictSeg / 64];
  const int r = blockIdx.x / a.segs, seg = blockIdx.x - r * a.segs, b = r / a.H, tid = threadIdx.x;
  const Row row{a.table + (long)b * a.table_b, a.page, r - b * a.H};
  const int len = seq_len(a.len, b, a.cap), K = row_budget(a, len);
  int* flag = a.hist + (long)r * kEvictRow;     // a page of the row is bad
  int* state = flag + 1;                        // [3][3] known bits, left, whole, after each digit
  int* sums = flag + 16;                        // [3][kEvictBins]
  if (STEP == 0 && seg == 0 && tid == 0) a.count[r] = 0;
  if (STEP > 0 && seg == 0 && tid == 0 && STEP == 4 && row.h == 0) a.len_out[b] = len < 0 || *flag ? a.len[b] : min(len, K);
  const int s0 = seg * kEvictSeg, s1 = min(len, s0 + kEvictSeg);
  if (s0 >= s1) return;
  uint32_t* keys = (uint32_t*)a.keys + (long)r * a.cap;
  if constexpr (STEP == 0) {
    const long oldest = (long)a.seen[b] - a.recent;
    for (int i = tid; i < kEvictBins; i += 256) hist[i] = 0;
    __syncthreads();
    const bool bad = each_key(a, row, s0, s1, oldest, [&](int s, uint32_t k) {
      keys[s] = k;
      atomicAdd(&hist[k >> kShift[0]], 1);
    });
    if (bad) atomicOr(flag, 1);
  } else {
    if (*flag) return;
    uint32_t known = 0;
    int left = K;
    bool whole = false;
    if (len > K) {
      if (STEP > 1) {
        const int* st = state + 3 * (min(STEP, 4) - 2);
        known = st[0], left = st[1], whole = st[2];
      }
      if (STEP <= 3 && !whole) {
        // the histogram that the step before filled
        constexpr int d = STEP <= 3 ? STEP - 1 : 0;
        for (int i = tid; i < kEvictBins; i += 256) hist[i] = sums[d * kEvictBins + i];
        __syncthreads();
        whole = pick_bin<256>(hist, kShift[d], known, left, tmp, res);
      }
      if (STEP <= 3 && seg == 0 && tid == 0) {
        int* st = state + 3 * (STEP - 1);
        st[0] = known, st[1] = left, st[2] = whole;
      }
    }
    if constexpr (STEP <= 2) {
      if (len <= K || whole) return;
      for (int i = tid; i < kEvictBins; i += 256) hist[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (int s = s0 + tid; s < s1; s += 256) {
        const uint32_t k = keys[s];
        if ((k & kAbove[STEP]) == known) atomicAdd(&hist[(k >> kShift[STEP]) & kDigit[STEP]], 1);
      }
    } else {
      const Cut cut = len > K ? cut_of(known, left, whole) : Cut{0u, len};
      const int wave = uni(tid >> 6), w0 = min(s1, s0 + wave * (kEvictSeg / 4)), w1 = min(s1, w0 + kEvictSeg / 4);
      auto key = [&](int s) { return keys[s]; };
      Counts* counts = (Counts*)(a.hist + (long)a.B * a.H * kEvictRow) + (long)r * a.segs * 4;
      if constexpr (STEP == 3) {
        const Counts c = count_range(w0, w1, K, cut, key);
        if ((tid & 63) == 0) counts[seg * 4 + wave] = c;
      } else {
        // the stretches before this wave's, and those of the whole row, a few to each lane
        const int used = ((len - 1) / kEvictSeg + 1) * 4, here = seg * 4 + wave;
        Counts before{0, 0, 0, 0}, all{0, 0, 0, 0};
#pragma unroll 4
        for (int i = tid & 63; i < used; i += 64) {
          const Counts c = counts[i];
          all.eq_lo += c.eq_lo, all.gt_hi += c.gt_hi, all.eq_hi += c.eq_hi;
          if (i < here) before.gt_lo += c.gt_lo, before.eq_lo += c.eq_lo, before.gt_hi += c.gt_hi, before.eq_hi += c.eq_hi;
        }
        auto sum = [](int x) { return __builtin_amdgcn_readlane(wave_prefix(x), 63); };
        before = {sum(before.gt_lo), sum(before.eq_lo), sum(before.gt_hi), sum(before.eq_hi)};
        const int eq_lo = sum(all.eq_lo), gt_hi = sum(all.gt_hi), eq_hi = sum(all.eq_hi);
        int* give = a.moves + (long)r * 2 * a.most;
        list_range(a, row, w0, w1, K, before, eq_lo, cut, give, give + a.most, masks + wave * (kEvictSeg / 256), key);
        if (seg == 0 && tid == 0) a.count[r] = gt_hi + min(max(cut.ties - eq_lo, 0), eq_hi);
      }
    }
  }
  if constexpr (STEP <= 2) {
    __syncthreads();
    for (int i = tid; i < kEvictBins; i += 256)
      if (hist[i] != 0) atomicAdd(&sums[STEP * kEvictBins + i], hist[i]);
  }
}

// The moves of a row by many workgroups. Bound by HBM: 131k -> 16k slots of 8 heads of 128 move 117 MB in 26 us, 4.5
// TB/s (a large copy: 4.8).
__global__ __launch_bounds__(256) void paged_evict_move_kernel(const PagedEvictArgs a, int blocks_per_row) {
  const int r = blockIdx.x / blocks_per_row, b = r / a.H;
  const Row row{a.table + (long)b * a.table_b, a.page, r - b * a.H};
  move_rows(a, row, r, a.count[r], (blockIdx.x - r * blocks_per_row) * 256 + threadIdx.x, blocks_per_row * 256);
}

template <int DT, int DP, bool PAD, bool P16, int NB>
hipError_t attn_launch(const PagedAttnArgs& a, int items, hipStream_t st) {
  const size_t lds = (size_t)(4 * a.gs * (DP + 4) + 4 * 16 * NB * 2 + (a.held ? a.gs * a.pitch : 0)) * sizeof(float);
  if (lds > 49152) {
    const hipError_t e = hipFuncSetAttribute((const void*)paged_attn_kernel<DT, DP, PAD, P16, NB>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  paged_attn_kernel<DT, DP, PAD, P16, NB><<<items, 256, lds, st>>>(a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && (!a.single || (a.logits != nullptr && a.hbs > 1))) {
    paged_attn_join_kernel<<<items, kJoinThreads, 0, st>>>(a);
    e = hipGetLastError();
  }
  return e;
}

template <int DT, int DP, int NB>
hipError_t attn_pick(const PagedAttnArgs& a, int items, hipStream_t st) {
  const bool p16 = a.page.d % 16 == 0;
  if (a.D == DP)
    return p16 ? attn_launch<DT, DP, false, true, NB>(a, items, st) : attn_launch<DT, DP, false, false, NB>(a, items, st);
  return p16 ? attn_launch<DT, DP, true, true, NB>(a, items, st) : attn_launch<DT, DP, true, false, NB>(a, items, st);
}

template <int DT, int NB>
hipError_t attn_width(const PagedAttnArgs& a, int items, hipStream_t st) {
  if (a.D <= 64) return attn_pick<DT, 64, NB>(a, items, st);
  if (a.D <= 128) return attn_pick<DT, 128, NB>(a, items, st);
  // 32 heads of 256 dims in 32 bits do not fit the registers: the bindings never ask for them
  return attn_pick<DT, 256, DT == kF32 ? 1 : NB>(a, items, st);
}

template <int DT>
hipError_t attn_dims(const PagedAttnArgs& a, int items, hipStream_t st) {
  return a.wide == 16 ? attn_width<DT, 1>(a, items, st) : attn_width<DT, 2>(a, items, st);
}

}  // namespace
}  // namespace zoo

extern "C" hipError_t zoo_paged_attn(const zoo::PagedAttnArgs* a, int items, hipStream_t st) {
  if (a->dtype == zoo::kBf16) return zoo::attn_dims<zoo::kBf16>(*a, items, st);
  if (a->dtype == zoo::kF16) return zoo::attn_dims<zoo::kF16>(*a, items, st);
  return zoo::attn_dims<zoo::kF32>(*a, items, st);
}

extern "C" hipError_t zoo_paged_append(const zoo::PagedAppendArgs* a, hipStream_t st) {
  const long rows = ((long)a->T * a->H * a->vec.d + 255) / 256, per = rows > 0 ? rows : 1;
  zoo::paged_append_kernel<<<(unsigned)(per * a->B), 256, 0, st>>>(*a, (int)per);
  return hipGetLastError();
}

extern "C" long zoo_paged_evict_scratch(const zoo::PagedEvictArgs* a) {
  return a->segs > 0 ? (long)a->B * a->H * (zoo::kEvictRow + a->segs * 16) : 0;
}

extern "C" hipError_t zoo_paged_evict(const zoo::PagedEvictArgs* a, hipStream_t st) {
  const int rows = a->B * a->H;
  hipError_t e;
  if (a->segs > 0) {
    const unsigned grid = (unsigned)rows * a->segs;
    zoo::paged_evict_long_kernel<0><<<grid, 256, 0, st>>>(*a);
    zoo::paged_evict_long_kernel<1><<<grid, 256, 0, st>>>(*a);
    zoo::paged_evict_long_kernel<2><<<grid, 256, 0, st>>>(*a);
    zoo::paged_evict_long_kernel<3><<<grid, 256, 0, st>>>(*a);
    zoo::paged_evict_long_kernel<4><<<grid, 256, 0, st>>>(*a);
  } else {
    const size_t lds = (size_t)(a->cap > 0 ? a->cap : 1) * 4;
    if (a->cap <= 2048) {
      zoo::paged_evict_select_kernel<256><<<rows, 256, lds, st>>>(*a);
    } else {
      if (lds > 32768) {
        e = hipFuncSetAttribute((const void*)zoo::paged_evict_select_kernel<1024>,
                                hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
      }
      zoo::paged_evict_select_kernel<1024><<<rows, 1024, lds, st>>>(*a);
    }
  }
  e = hipGetLastError();
  if (e != hipSuccess || a->most <= 0 || a->fused) return e;
  // a workgroup for 256 pieces, up to 2^22 of them; more pieces are taken in turn
  const long want = ((long)a->most * a->vec.d + 255) / 256, room = (1 << 22) / rows;
  const int per = (int)(want < room ? want : room > 0 ? room : 1);
  zoo::paged_evict_move_kernel<<<(unsigned)per * rows, 256, 0, st>>>(*a, per);
  return hipGetLastError();
}
