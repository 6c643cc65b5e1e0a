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
// P is fed as the sum of two 16-bit numbers: rounding it to one would cost an error as large as the
// output's own rounding.
//
// The slots of all sequences are cut into equal chunks, one per workgroup, whose number aims at
// filling the chip whatever the batch and the lengths (find_work): lengths are only known on the
// device, so every workgroup derives the cut from them itself. A join kernel merges a sequence's
// chunks and, where weights are wanted, turns the stored products into sum_g w_gj.
#include <math.h>

#include "common.h"
#include "kvcache.h"

namespace zoo {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

enum { kBf16 = 0, kF16 = 1, kF32 = 2 };

// v_exp_f32: one instruction, within an ulp; results under 2^-126 are 0
ZOO_DEV float pow2(float x) { return __builtin_amdgcn_exp2f(x); }

ZOO_DEV uint32_t fdiv(uint32_t n, const FastDiv& f) { return (__umulhi(n, f.m) + n) >> f.s; }

// slots of sequence b, or -1 where its length does not fit its table
ZOO_DEV int seq_len(const int* len, int b, int cap) {
  const int n = len[b];
  return n < 0 || n > cap ? -1 : n;
}

ZOO_DEV int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

struct Work {
  int b, hk, hb;    // sequence, kv head, block of 16 query heads
  int chunk, n;     // which of the sequence's n chunks
  int s0, s1;       // its slots
  int len;          // the sequence's slots, -1: bad
  int first;        // item of the sequence's chunk 0, same head block
  int step;         // items from one chunk to the next
};

// Cuts the batch into chunks of `size` slots, a multiple of `grain`, such that there are at most
// target + B of them per head block, and finds the chunk of this workgroup; every wave does so alone.
// Every sequence has a chunk, if an empty one. Returns false for the items that are not needed.
ZOO_DEV bool find_work(const PagedAttnArgs& a, int grain, Work& w) {
  const int lane = threadIdx.x & 63;
  const int hbs = (a.G + 15) >> 4, step = a.H * hbs;
  const int t = blockIdx.x / step, hh = blockIdx.x - t * step;
  w.hk = hh / hbs;
  w.hb = hh - w.hk * hbs;
  w.step = step;
  int at = 0, size = kKvMaxSlots;
  if (!a.single) {
    long total = 0;
    for (int b = lane; b < a.B; b += 64) total += max(seq_len(a.len, b, a.cap), 0);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) total += __shfl_xor(total, o, 64);
    // a chunk is at least one grain and at most a whole sequence, so this fits an int
    const long want = (total + a.target - 1) / a.target;
    size = (int)min((long)kKvMaxSlots, max((want + grain - 1) / grain, 1L) * grain);
  }
  int b = 0, chunk = 0, n = 0, len = 0;
  bool found = false;
  for (int b0 = 0; b0 < a.B && !found; b0 += 64) {
    const int mine = b0 + lane < a.B ? seq_len(a.len, b0 + lane, a.cap) : 0;
    const int chunks = b0 + lane < a.B ? max((max(mine, 0) + size - 1) / size, 1) : 0;
    int upto = chunks;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_up(upto, o, 64);
      if (lane >= o) upto += x;
    }
    const unsigned long long hit = __ballot(at + upto > t);
    if (hit) {
      const int who = __ffsll(hit) - 1;
      b = b0 + who;
      n = __shfl(chunks, who, 64);
      len = __shfl(mine, who, 64);
      at += __shfl(upto, who, 64) - n;
      chunk = t - at;
      found = true;
    } else {
      at += __shfl(upto, 63, 64);
    }
  }
  if (!found) return false;
  w.b = uni(b);
  w.chunk = uni(chunk);
  w.n = uni(n);
  w.len = uni(len);
  w.first = uni(at) * step + hh;
  w.s0 = w.chunk * size;
  w.s1 = min(w.len, w.s0 + size);
  return true;
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

// Two weights as packed 16-bit numbers, rounded towards zero, and what that left over, packed too. The rest is
// kept above zero (by less than 2^-35 of the largest weight), so that an infinite value times a weight stays
// infinite: a rest of 0, or a negative one, would make it NaN.
template <int DT>
ZOO_DEV void split2(float x, float y, uint32_t& hi, uint32_t& lo) {
  if constexpr (DT == kBf16) {
    const uint32_t xi = __float_as_uint(x), yi = __float_as_uint(y);
    hi = __builtin_amdgcn_perm(yi, xi, 0x07060302u);
    lo = pack2bf(fmaxf(x - __uint_as_float(xi & 0xffff0000u), 0x1p-126f),
                 fmaxf(y - __uint_as_float(yi & 0xffff0000u), 0x1p-126f));
  } else {
    const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
    const auto r = __builtin_amdgcn_cvt_pkrtz(fmaxf(x - (float)h[0], 0x1p-24f), fmaxf(y - (float)h[1], 0x1p-24f));
    hi = __builtin_bit_cast(uint32_t, h);
    lo = __builtin_bit_cast(uint32_t, r);
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

// DP: the head width rounded up; PAD: it was rounded; P16: pages of a multiple of 16 rows, so that a
// 16-slot subtile lies in one page and its address is wave-uniform. Other page sizes look up a page per
// slot.
template <int DT, int DP, bool PAD, bool P16>
__global__ __launch_bounds__(256) void paged_attn_kernel(const PagedAttnArgs a) {
  using T = Tile<DT, DP>;
  constexpr int NS = T::NS, KL = T::KL, VC = T::VC, VW = T::VW, VE = T::VE, NA = T::NA, ES = T::ES;
  extern __shared__ float lds[];  // [4][gb][DP + 4] sums, then [4][16][2] maximum and sum
  Work w;
  if (!find_work(a, T::GRAIN, w)) return;
  const int lane = threadIdx.x & 63, wave = uni(threadIdx.x >> 6);
  const int row = lane & 15, quad = lane >> 4;
  const int gb = min(16, a.G - 16 * w.hb), D = a.D;
  const int head0 = w.hk * a.G + 16 * w.hb;
  const long out0 = ((long)w.b * a.H * a.G + head0) * D;
  if (w.len <= 0) {
    const float x = w.len < 0 ? __builtin_nanf("") : 0.f;
    for (int i = threadIdx.x; i < gb * D; i += 256) store_out<DT>(a.o, out0 + i, x);
    return;
  }
  // fp16 cannot hold small weights: they are kept times 2^12 (their maximum is 1, and 16 * 2^12 < 2^16)
  constexpr float kUp = DT == kF16 ? 12.f : 0.f;

  // Q^T: head `row`, the dims that K's loads bring. Heads and dims that are not there are zero.
  uint4 q[KL];
  {
    const char* qp = (const char*)a.q + ((long)w.b * a.q_b + (long)(head0 + min(row, gb - 1)) * a.q_h) * ES;
#pragma unroll
    for (int i = 0; i < KL; ++i) {
      const int at = i * 64 + quad * 16;
      const bool in = row < gb && (!PAD || at < D * ES);
      q[i] = mask4(*(const uint4*)(qp + (!PAD || at < D * ES ? at : 0)), in);
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

  // nothing writes the table while the kernel runs: the constant address space lets a wave-uniform look-up
  // be a scalar load, which does not queue behind the vector loads in flight
  const auto* page_ids = (const __attribute__((address_space(4))) int*)table;
  auto page_of = [&](int slot) {
    const int p = page_ids[fdiv(slot, a.page)];
    const bool ok = (unsigned)p < (unsigned)a.pages;
    bad |= !ok;
    return ok ? p : 0;
  };
  auto load_k = [&](int base) {
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      const char* p;
      if constexpr (P16) {
        const int s = min(base + 16 * u, (w.s1 - 1) & ~15);
        p = kb + ((long)uni(page_of(s)) * a.ks.page + (long)(s - fdiv(s, a.page) * a.page.d) * a.ks.row) * ES + klane;
      } else {
        const int s = min(base + 16 * u + row, w.s1 - 1);
        p = kb + ((long)page_of(s) * a.ks.page + (long)(s - fdiv(s, a.page) * a.page.d) * a.ks.row) * ES + quad * 16;
      }
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        if constexpr (PAD) {
          const bool in = i * 64 + quad * 16 < D * ES;
          kr[u][i] = mask4(*(const uint4*)(p + (in ? i * 64 : -quad * 16)), in);
        } else {
          kr[u][i] = *(const uint4*)(p + i * 64);
        }
      }
    }
  };
  auto load_v = [&](int base) {
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
          const int s = min(base + 16 * u + 4 * quad + r, w.s1 - 1);
          p += ((long)page_of(s) * a.vs.page + (long)(s - fdiv(s, a.page) * a.page.d) * a.vs.row) * ES;
        }
#pragma unroll
        for (int c = 0; c < VC; ++c) {
          const int at = c * 256 + vdim;
          const char* pc = p + (!PAD || at < D * ES ? at : 0);
          if constexpr (VW == 4) {
            const uint4 x = *(const uint4*)pc;
            vr[u][r][c][0] = x.x, vr[u][r][c][1] = x.y, vr[u][r][c][2] = x.z, vr[u][r][c][3] = x.w;
          } else {
            const uint2 x = *(const uint2*)pc;
            vr[u][r][c][0] = x.x, vr[u][r][c][1] = x.y;
          }
        }
      }
    }
  };

  f32x4 acc[NA];
#pragma unroll
  for (int i = 0; i < NA; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;  // of head `row`; l of this lane's slots only
  float* logit =
      a.logits ? a.logits + (((long)w.b * a.H + w.hk) * a.cap) * a.G + 16 * w.hb + row : nullptr;

  int base = w.s0 + wave * T::TS;
  if (base < w.s1) {
    load_k(base);
    load_v(base);
  }
  for (; base < w.s1; base += T::GRAIN) {
    const bool more = base + T::GRAIN < w.s1, tail = base + T::TS > w.s1;
    f32x4 s[NS];
#pragma unroll
    for (int u = 0; u < NS; ++u) {
      s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KL; ++i) {
        if constexpr (DT == kF32) {
          s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[u][i].x), __uint_as_float(q[i].x), s[u], 0, 0, 0);
          s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[u][i].y), __uint_as_float(q[i].y), s[u], 0, 0, 0);
          s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[u][i].z), __uint_as_float(q[i].z), s[u], 0, 0, 0);
          s[u] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kr[u][i].w), __uint_as_float(q[i].w), s[u], 0, 0, 0);
        } else {
          s[u] = mma16<DT>(kr[u][i], q[i], s[u]);
        }
      }
    }
    if (more) load_k(base + T::GRAIN);
    if (logit != nullptr && row < gb) {
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = base + 16 * u + 4 * quad + r;
          if (at < w.s1) logit[(long)at * a.G] = s[u][r];
        }
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[u][r] *= a.c;
        if (tail && base + 16 * u + 4 * quad + r >= w.s1) s[u][r] = -INFINITY;
        top = fmaxf(top, s[u][r]);
      }
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    const float mu = top == -INFINITY ? 0.f : top;  // nothing but -inf so far: every weight is 0, not NaN
    const float old = pow2(m - mu);
    m = top;
    l *= old;
    if (__any(old != 1.f)) {
#pragma unroll
      for (int i = 0; i < NA; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] *= old;
    }
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[u][r] = pow2(s[u][r] - mu + kUp);
        l += s[u][r];
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
              acc[c * VE + e] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vr[u][r][c][e]), s[u][r],
                                                                     acc[c * VE + e], 0, 0, 0);
    } else {
#pragma unroll
      for (int u = 0; u < NS; u += 2) {
        uint4 hi, lo;
        split2<DT>(s[u][0], s[u][1], hi.x, lo.x);
        split2<DT>(s[u][2], s[u][3], hi.y, lo.y);
        split2<DT>(s[u + 1][0], s[u + 1][1], hi.z, lo.z);
        split2<DT>(s[u + 1][2], s[u + 1][3], hi.w, lo.w);
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
            acc[c * VE + e] = mma16<DT>(x, hi, acc[c * VE + e]);
            acc[c * VE + e] = mma16<DT>(x, lo, acc[c * VE + e]);
          }
      }
    }
    if (more) load_v(base + T::GRAIN);
  }
  // the four waves' sums meet in LDS
  l += __shfl_xor(l, 16, 64);
  l += __shfl_xor(l, 32, 64);
  if (__any(bad)) l = __builtin_nanf("");
  constexpr int LD = DP + 4;
  float* ml = lds + 4 * gb * LD;
  if (row < gb) {
#pragma unroll
    for (int i = 0; i < NA; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        lds[(wave * gb + row) * LD + (i / VE) * (16 * VE) + (quad * 4 + r) * VE + i % VE] = acc[i][r];
    if (quad == 0) {
      ml[(wave * 16 + row) * 2] = m;
      ml[(wave * 16 + row) * 2 + 1] = l;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < gb * DP; i += 256) {
    const int g = i / DP, d = i & (DP - 1);
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < 4; ++x) top = fmaxf(top, ml[(x * 16 + g) * 2]);
    const float mu = top == -INFINITY ? 0.f : top;
    float sum = 0.f, o = 0.f;
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float f = pow2(ml[(x * 16 + g) * 2] - mu);
      sum += f * ml[(x * 16 + g) * 2 + 1];
      o += f * lds[(x * gb + g) * LD + d];
    }
    if (!PAD || d < D) {
      if (w.n == 1)
        store_out<DT>(a.o, out0 + (long)g * D + d, o / sum);
      else
        a.part_o[((long)blockIdx.x * a.gs + g) * D + d] = o;
    }
    if (d == 0 && a.part_ml != nullptr) {
      a.part_ml[((long)blockIdx.x * 16 + g) * 2] = top;
      a.part_ml[((long)blockIdx.x * 16 + g) * 2 + 1] = sum;
    }
  }
}

// Joins the chunks of a sequence: chunk c of n writes the c-th part of the outputs, and the gathered
// weights of its own slots.
__global__ __launch_bounds__(256) void paged_attn_join_kernel(const PagedAttnArgs a, int grain) {
  __shared__ float lse[kKvMaxGroup], part[256];
  Work w;
  if (!find_work(a, grain, w)) return;
  const bool weights = a.logits != nullptr && w.hb == 0;
  if (w.len <= 0 || (w.n == 1 && !weights)) return;
  const int tid = threadIdx.x;
  const int hbs = (a.G + 15) >> 4;
  const float up = a.dtype == kF16 ? 12.f : 0.f;
  // log2 of the sum of exponentials of the heads that this workgroup needs, 16 threads to a head
  const int heads = weights ? a.G : min(16, a.G - 16 * w.hb);
  for (int g0 = 0; g0 < heads; g0 += 16) {
    const int g = g0 + (tid >> 4);
    const float* ml = a.part_ml + ((long)(w.first + (weights ? g >> 4 : 0)) * 16 + (g & 15)) * 2;
    const long next = (long)w.step * 32;
    float m = -INFINITY, l = 0.f;
    if (g < heads)
      for (int i = tid & 15; i < w.n; i += 16) {
        const float mi = ml[i * next], li = ml[i * next + 1];
        const float top = fmaxf(m, mi), mu = top == -INFINITY ? 0.f : top;
        l = l * pow2(m - mu) + li * pow2(mi - mu);
        m = top;
      }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      const float mi = __shfl_xor(m, o, 64), li = __shfl_xor(l, o, 64);
      const float top = fmaxf(m, mi), mu = top == -INFINITY ? 0.f : top;
      l = l * pow2(m - mu) + li * pow2(mi - mu);
      m = top;
    }
    if (g < heads && (tid & 15) == 0) lse[g] = m + log2f(l);
  }
  __syncthreads();
  if (w.n > 1) {
    const int gb = min(16, a.G - 16 * w.hb), E = gb * a.D;
    int per = ((E + w.n - 1) / w.n + 15) & ~15;
    const int e0 = w.chunk * per, e1 = min(E, e0 + per);
    int wide = 16;
    while (wide < per && wide < 256) wide *= 2;
    const int ways = 256 / wide, who = tid / wide;
    const float* po = a.part_o + (long)w.first * a.gs * a.D;
    const float* ml = a.part_ml + (long)w.first * 32;
    const long step_o = (long)w.step * a.gs * a.D, step_m = (long)w.step * 32;
    const long out0 = ((long)w.b * a.H * a.G + w.hk * a.G + 16 * w.hb) * a.D;
    for (int e = e0; e < e1; e += wide) {
      const int at = e + (tid & (wide - 1));
      float sum = 0.f;
      if (at < e1) {
        const int g = at / a.D;
        const float ref = lse[g];
        for (int i = who; i < w.n; i += ways) sum += po[i * step_o + at] * pow2(ml[i * step_m + g * 2] - ref);
      }
      part[tid] = sum;
      __syncthreads();
      if (who == 0 && at < e1) {
        for (int i = 1; i < ways; ++i) sum += part[i * wide + tid];
        store_any(a.dtype, a.o, out0 + at, sum);
      }
      __syncthreads();
    }
  }
  if (weights) {
    const int* table = a.table + (long)w.b * a.table_b;
    const float* logit = a.logits + ((long)w.b * a.H + w.hk) * a.cap * a.G;
    for (int s = w.s0 + tid; s < w.s1; s += 256) {
      const int p = table[fdiv(s, a.page)];
      if ((unsigned)p >= (unsigned)a.pages) continue;
      const long off = s - fdiv(s, a.page) * a.page.d;
      float sum = 0.f;
      for (int g = 0; g < a.G; ++g) sum += pow2(logit[(long)s * a.G + g] * a.c - lse[g] + up);
      a.scores_out[p * a.sos.page + w.hk * a.sos.head + off * a.sos.row] =
          a.scores[p * a.ss.page + w.hk * a.ss.head + off * a.ss.row] + sum;
    }
  }
}

// ---- append: one thread moves 16 bytes of a token's key row and of its value row ----
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
  const uint4 x = *(const uint4*)((const char*)a.k + (b * a.k_b + t * a.k_t + h * a.k_h) * a.es + piece * 16);
  const uint4 y = *(const uint4*)((const char*)a.v + (b * a.v_b + t * a.v_t + h * a.v_h) * a.es + piece * 16);
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

constexpr int kEvictThreads = 1024;
constexpr int kEvictBins = 2048;

// exclusive prefix sum over the workgroup in thread order; total for everybody. Two barriers.
ZOO_DEV int block_prefix(int x, int* tmp, int& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  int upto = x;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(upto, o, 64);
    if (lane >= o) upto += y;
  }
  if (lane == 63) tmp[wave] = upto;
  __syncthreads();
  int before = 0;
  total = 0;
  for (int i = 0; i < waves; ++i) {
    const int t = tmp[i];
    before += i < wave ? t : 0;
    total += t;
  }
  __syncthreads();
  return before + upto - x;
}

// One workgroup per (sequence, kv head): a radix selection of the budget-th largest key (11 + 11 + 10
// bits, histograms in LDS, the keys too as far as they fit), then one ordered pass that lists the slots
// given up below the budget and the kept ones behind it, which will take their places.
__global__ __launch_bounds__(kEvictThreads) void paged_evict_select_kernel(const PagedEvictArgs a, int held) {
  extern __shared__ uint32_t sh[];  // [held] keys
  __shared__ int hist[kEvictBins];
  __shared__ int tmp[kEvictThreads / 64];
  __shared__ int s_bin, s_left, s_bad;
  const int b = blockIdx.x / a.H, h = blockIdx.x - b * a.H, tid = threadIdx.x;
  const int len = seq_len(a.len, b, a.cap);
  const int* table = a.table + (long)b * a.table_b;
  if (tid == 0) s_bad = len < 0;
  __syncthreads();
  if (len > 0) {
    bool bad = false;
    for (int i = tid; i <= (int)fdiv(len - 1, a.page); i += kEvictThreads) bad |= (unsigned)table[i] >= (unsigned)a.pages;
    if (bad) s_bad = 1;
  }
  __syncthreads();
  const bool bad = s_bad;
  if (tid == 0) {
    a.count[blockIdx.x] = 0;
    // every kv head writes the same number only if no page is bad, and that is the sequence's matter
    if (h == 0) a.len_out[b] = bad ? a.len[b] : min(len, a.budget);
  }
  if (bad || len == 0) return;
  auto at = [&](int s, const PoolStride& st) {
    const int pi = fdiv(s, a.page);
    return table[pi] * st.page + h * st.head + (long)(s - pi * (int)a.page.d) * st.row;
  };
  const long oldest = (long)a.seen[b] - a.recent;
  auto key_of = [&](int s) { return rank_key(a.scores[at(s, a.ss)], a.positions[at(s, a.ps)] >= oldest); };
  const int K = a.budget;
  uint32_t cut = 0;
  int ties = len;  // keys equal to `cut` that are kept, lowest slots first
  if (len > K) {
    uint32_t prefix = 0;
    int left = K;
    for (int pass = 0; pass < 3; ++pass) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t mask = pass == 2 ? 1023u : 2047u;
      const uint32_t above = pass == 0 ? 0u : pass == 1 ? 0xffe00000u : 0xfffffc00u;
      for (int i = tid; i < kEvictBins; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      for (int s = tid; s < len; s += kEvictThreads) {
        uint32_t k;
        if (pass == 0 || s >= held) {
          k = key_of(s);
          if (s < held) sh[s] = k;
        } else {
          k = sh[s];
        }
        if ((k & above) == prefix) atomicAdd(&hist[(k >> shift) & mask], 1);
      }
      __syncthreads();
      // bins from the top: thread t owns bins 2047 - 2t and 2046 - 2t
      const int b0 = hist[kEvictBins - 1 - 2 * tid], b1 = hist[kEvictBins - 2 - 2 * tid];
      int total;
      const int before = block_prefix(b0 + b1, tmp, total);
      if (before < left && before + b0 >= left) s_bin = kEvictBins - 1 - 2 * tid, s_left = left - before;
      if (before + b0 < left && before + b0 + b1 >= left) s_bin = kEvictBins - 2 - 2 * tid, s_left = left - before - b0;
      __syncthreads();
      prefix |= (uint32_t)s_bin << shift;
      left = s_left;
      __syncthreads();
    }
    cut = prefix;
    ties = left;
  }
  int* give = a.moves + (long)blockIdx.x * 2 * a.most;
  int* take = give + a.most;
  const bool copy = a.scores_out != a.scores || a.positions_out != a.positions;
  int equal = 0, gave = 0, took = 0;
  for (int s0 = 0; s0 < len; s0 += kEvictThreads) {
    const int s = s0 + tid;
    const bool in = s < len;
    const uint32_t k = len <= K ? 0xffffffffu : !in ? 0u : s < held ? sh[s] : key_of(s);
    int n;
    const bool eq = in && k == cut;
    const int nth = equal + block_prefix(eq, tmp, n);
    equal += n;
    const bool kept = in && (k > cut || (eq && nth < ties));
    // gives in the low half, takes in the high half of one sum
    const bool hole = in && s < K && !kept, tail = kept && s >= K;
    const int rank = block_prefix((int)hole | ((int)tail << 16), tmp, n);
    if (hole) give[gave + (rank & 0xffff)] = s;
    if (tail) take[took + (rank >> 16)] = s;
    gave += n & 0xffff;
    took += n >> 16;
    if (copy && kept && s < K) {
      a.scores_out[at(s, a.sos)] = a.scores[at(s, a.ss)];
      a.positions_out[at(s, a.pos)] = a.positions[at(s, a.ps)];
    }
  }
  if (tid == 0) a.count[blockIdx.x] = gave;
}

// moves what the lists say: 256 / vec rows at a time
__global__ __launch_bounds__(256) void paged_evict_move_kernel(const PagedEvictArgs a, int blocks_per_row) {
  const int r = blockIdx.x / blocks_per_row, b = r / a.H, h = r - b * a.H;
  const uint32_t i = (uint32_t)(blockIdx.x - r * blocks_per_row) * 256 + threadIdx.x;
  const int n = fdiv(i, a.vec), piece = i - n * a.vec.d;
  if (n >= a.count[r]) return;
  const int* give = a.moves + (long)r * 2 * a.most;
  const int to = give[n], from = give[a.most + n];
  const int* table = a.table + (long)b * a.table_b;
  const int ti = fdiv(to, a.page), fi = fdiv(from, a.page);
  const long tp = table[ti], fp = table[fi];
  const long to_off = to - ti * (int)a.page.d, from_off = from - fi * (int)a.page.d;
  const uint4 x = *(const uint4*)((char*)a.kp + (fp * a.ks.page + h * a.ks.head + from_off * a.ks.row) * a.es + piece * 16);
  const uint4 y = *(const uint4*)((char*)a.vp + (fp * a.vs.page + h * a.vs.head + from_off * a.vs.row) * a.es + piece * 16);
  *(uint4*)((char*)a.kp + (tp * a.ks.page + h * a.ks.head + to_off * a.ks.row) * a.es + piece * 16) = x;
  *(uint4*)((char*)a.vp + (tp * a.vs.page + h * a.vs.head + to_off * a.vs.row) * a.es + piece * 16) = y;
  if (piece == 0) {
    a.scores_out[tp * a.sos.page + h * a.sos.head + to_off * a.sos.row] =
        a.scores[fp * a.ss.page + h * a.ss.head + from_off * a.ss.row];
    a.positions_out[tp * a.pos.page + h * a.pos.head + to_off * a.pos.row] =
        a.positions[fp * a.ps.page + h * a.ps.head + from_off * a.ps.row];
  }
}

template <int DT, int DP, bool PAD, bool P16>
hipError_t attn_launch(const PagedAttnArgs& a, int items, hipStream_t st) {
  const int gb = a.G < 16 ? a.G : 16;
  const size_t lds = (size_t)(4 * gb * (DP + 4) + 128) * sizeof(float);
  if (lds > 65536) {
    const hipError_t e = hipFuncSetAttribute((const void*)paged_attn_kernel<DT, DP, PAD, P16>,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  paged_attn_kernel<DT, DP, PAD, P16><<<items, 256, lds, st>>>(a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && (!a.single || a.logits != nullptr)) {
    paged_attn_join_kernel<<<items, 256, 0, st>>>(a, Tile<DT, DP>::GRAIN);
    e = hipGetLastError();
  }
  return e;
}

template <int DT, int DP>
hipError_t attn_pick(const PagedAttnArgs& a, int items, hipStream_t st) {
  const bool p16 = a.page.d % 16 == 0;
  if (a.D == DP) return p16 ? attn_launch<DT, DP, false, true>(a, items, st) : attn_launch<DT, DP, false, false>(a, items, st);
  return p16 ? attn_launch<DT, DP, true, true>(a, items, st) : attn_launch<DT, DP, true, false>(a, items, st);
}

template <int DT>
hipError_t attn_dims(const PagedAttnArgs& a, int items, hipStream_t st) {
  if (a.D <= 64) return attn_pick<DT, 64>(a, items, st);
  if (a.D <= 128) return attn_pick<DT, 128>(a, items, st);
  return attn_pick<DT, 256>(a, items, st);
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

extern "C" hipError_t zoo_paged_evict(const zoo::PagedEvictArgs* a, hipStream_t st) {
  const int held = a->cap < 32768 ? a->cap : 32768;
  const size_t lds = (size_t)held * 4;
  if (lds > 32768) {
    const hipError_t e = hipFuncSetAttribute((const void*)zoo::paged_evict_select_kernel,
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  zoo::paged_evict_select_kernel<<<a->B * a->H, zoo::kEvictThreads, lds, st>>>(*a, held);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a->most <= 0) return e;
  const long per = ((long)a->most * a->vec.d + 255) / 256;
  zoo::paged_evict_move_kernel<<<(unsigned)(per * a->B * a->H), 256, 0, st>>>(*a, (int)per);
  return hipGetLastError();
}
