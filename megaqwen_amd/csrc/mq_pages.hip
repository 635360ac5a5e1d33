// A paged K/V cache on MI355X (gfx950): moving pages, appending rows, and the attentions that
// read it. The reference keeps one contiguous cache (csrc/megakernel/megakernel_decode.py:140-146)
// and has no counterpart of these.
//
// A pool holds [layers, pages, kv heads, page size, head dim] of 16-bit values for K and as many for
// V, so that one page of one layer is one contiguous run and one page's rows of one head are one
// inside it: an attention workgroup reads whole runs of page size * head dim, and a fork or a
// compaction moves a layer's page as a single run. Page ids hold for every layer. `bounds`
// [layers, pages, kv heads, 2, head dim] are a page's least and greatest key entries.

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "megaqwen_amd.h"
#include "mq_common.h"
#include "mq_pages.h"

namespace mq {
namespace pg {

// ------------------------------------------------------------------ moving pages
// Page ids travel in the argument block, so that no copy from host memory waits for the device and a
// captured launch keeps them: a block of 4 KB holds 448 pairs and the rest of the arguments; a small
// one holds 32, which costs the host less to fill and send.
constexpr int LIST_LONG = 448, LIST_SHORT = 32;

template <int N>
struct CopyArgs {
  void* base[3];         // K, V, bounds (or null)
  uint32_t page_bytes;   // one page of one layer of K or V
  uint32_t bounds_bytes; // one page of one layer of the bounds
  uint32_t per_page;     // workgroups a page of K or V
  int num_pages;
  int2 ids[N];           // (from, to)
};

constexpr int CT = 256;              // threads
constexpr int CU = 4;                // 16-byte units a thread
constexpr uint32_t CB = CT * CU * 16;  // bytes a workgroup

// Workgroup (part of a page, pair, layer): a run of at most 16 KB of K or V, or the page's bounds. Bound by memory:
// 120 pages of 7.3 MB read and written at 5.3 TB/s, past the caches.
template <int N>
__global__ void __launch_bounds__(CT) copy_kernel(CopyArgs<N> A) {
  const uint32_t part = blockIdx.x, which = part < A.per_page ? 0 : part < 2 * A.per_page ? 1 : 2;
  const uint32_t bytes = which == 2 ? A.bounds_bytes : A.page_bytes;
  const uint32_t off = (which == 2 ? part - 2 * A.per_page : which ? part - A.per_page : part) * CB;
  const int2 id = A.ids[blockIdx.y];
  const size_t layer = (size_t)blockIdx.z * A.num_pages;
  const char* src = static_cast<const char*>(A.base[which]) + (layer + id.x) * bytes;
  char* dst = static_cast<char*>(A.base[which]) + (layer + id.y) * bytes;
  u32x4 w[CU];
#pragma unroll
  for (int u = 0; u < CU; u++) {
    const uint32_t o = off + 16 * (threadIdx.x + CT * u);
    if (o < bytes) w[u] = __builtin_nontemporal_load((gu32x4*)(src + o));
  }
#pragma unroll
  for (int u = 0; u < CU; u++) {
    const uint32_t o = off + 16 * (threadIdx.x + CT * u);
    if (o < bytes) __builtin_nontemporal_store(w[u], reinterpret_cast<u32x4*>(dst + o));
  }
}

template <int N>
struct MoveArgs {
  uint16_t *k, *v, *bounds;  // the pool
  uint16_t *kc, *vc;         // the contiguous cache [layers, kv heads, max_seq, head dim]
  int num_pages, hkv, page, d, max_seq, first, length;  // first: position of the list's first page
  int ids[N];
};

// the least (greatest) of two values; a value that is not a number wins, as in torch.amin
__device__ __forceinline__ float least(float a, float x) { return x < a || x != x ? x : a; }
__device__ __forceinline__ float greatest(float a, float x) { return x > a || x != x ? x : a; }

template <bool F16>
__device__ __forceinline__ float to_f32(uint32_t b) {
  return F16 ? (float)__builtin_bit_cast(_Float16, (unsigned short)b) : bf2f(b & 0xffffu);
}
template <bool F16>
__device__ __forceinline__ void to_f32x8(const u32x4 w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; i++) {
    f[2 * i] = to_f32<F16>(w[i] & 0xffffu);
    f[2 * i + 1] = to_f32<F16>(w[i] >> 16);
  }
}
// values that came from 16 bits go back without rounding
template <bool F16>
__device__ __forceinline__ u32x4 from_f32x8(const float (&f)[8]) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; i++)
    w[i] = F16 ? (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)f[2 * i]) |
                     (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)f[2 * i + 1]) << 16
               : pack_bf2(f[2 * i], f[2 * i + 1]);
  return w;
}

// Workgroup (kv head, page, layer): the page's filled rows between the contiguous cache and the
// pool, K and V, and on the way in the bounds of its keys. Thread t takes 8 dims of rows t / (d / 8),
// ... in steps of CT / (d / 8) rows. Bound by memory (3000 positions of 28 layers at 5.5 TB/s).
template <int N, bool IN, bool F16>
__global__ void __launch_bounds__(CT) move_kernel(MoveArgs<N> A) {
  __shared__ float s_lo[CT][9], s_hi[CT][9];  // (9: a column of eight lanes' rows lies in distinct banks)
  const int h = blockIdx.x, j = blockIdx.y, l = blockIdx.z, cpr = A.d / 8, c = threadIdx.x % cpr, step = CT / cpr;
  const int first = A.first + j * A.page, rows = min(A.page, A.length - first);
  const size_t in_pool = (((size_t)l * A.num_pages + A.ids[j]) * A.hkv + h) * A.page * A.d + 8 * c;
  const size_t flat = (((size_t)l * A.hkv + h) * A.max_seq + first) * A.d + 8 * c;
  float lo[8], hi[8];
#pragma unroll
  for (int i = 0; i < 8; i++) lo[i] = INFINITY, hi[i] = -INFINITY;
  for (int r = threadIdx.x / cpr; r < rows; r += step) {
    const size_t p = in_pool + (size_t)r * A.d, q = flat + (size_t)r * A.d;
    const u32x4 kw = ldw(IN ? A.kc + q : A.k + p), vw = ldw(IN ? A.vc + q : A.v + p);
    __builtin_nontemporal_store(kw, reinterpret_cast<u32x4*>(IN ? A.k + p : A.kc + q));
    __builtin_nontemporal_store(vw, reinterpret_cast<u32x4*>(IN ? A.v + p : A.vc + q));
    if (IN && A.bounds) {
      float f[8];
      to_f32x8<F16>(kw, f);
#pragma unroll
      for (int i = 0; i < 8; i++) lo[i] = least(lo[i], f[i]), hi[i] = greatest(hi[i], f[i]);
    }
  }
  if (!IN || !A.bounds) return;
#pragma unroll
  for (int i = 0; i < 8; i++) s_lo[threadIdx.x][i] = lo[i], s_hi[threadIdx.x][i] = hi[i];
  __syncthreads();
  if ((int)threadIdx.x >= cpr) return;
  for (int t = threadIdx.x + cpr; t < CT; t += cpr)
#pragma unroll
    for (int i = 0; i < 8; i++) lo[i] = least(lo[i], s_lo[t][i]), hi[i] = greatest(hi[i], s_hi[t][i]);
  uint16_t* b = A.bounds + (((size_t)l * A.num_pages + A.ids[j]) * A.hkv + h) * 2 * A.d + 8 * c;
  *reinterpret_cast<u32x4*>(b) = from_f32x8<F16>(lo);
  *reinterpret_cast<u32x4*>(b + A.d) = from_f32x8<F16>(hi);
}

// Workgroup b: sequence b's new K and V row to its position lens[b], and the page's bounds: the row
// itself where it is the page's first, the least and greatest with it otherwise. A position behind
// the table or a page outside the pool: nothing is written. 2 us for one sequence, 3.1 for 200: length, page id and
// bounds are read one behind the other.
template <bool F16>
__global__ void __launch_bounds__(CT) append_kernel(AppendArgs A) {
  const int b = blockIdx.x, len = A.lens[b], at = len >> A.lp;
  if (len < 0 || at >= A.width) return;
  const int id = A.tables[(size_t)b * A.t_sb + at], slot = len & ((1 << A.lp) - 1);
  if (id < 0 || id >= A.num_pages) return;
  const int cpr = A.d / 8;
  for (int t = threadIdx.x; t < A.hkv * cpr; t += CT) {
    const int h = t / cpr, c = t % cpr;
    const u32x4 kw = *(gu32x4*)(A.kr + (size_t)b * A.k_sb + (size_t)h * A.k_sh + 8 * c);
    const u32x4 vw = *(gu32x4*)(A.vr + (size_t)b * A.v_sb + (size_t)h * A.v_sh + 8 * c);
    const size_t head = (size_t)id * A.hkv + h, p = ((head << A.lp) + slot) * A.d + 8 * c;
    if (A.bounds) {
      uint16_t* bd = A.bounds + head * 2 * A.d + 8 * c;
      u32x4 lo = kw, hi = kw;
      if (slot > 0) {
        float f[8], lf[8], hf[8];
        to_f32x8<F16>(kw, f);
        to_f32x8<F16>(*(gu32x4*)bd, lf);
        to_f32x8<F16>(*(gu32x4*)(bd + A.d), hf);
#pragma unroll
        for (int i = 0; i < 8; i++) lf[i] = least(lf[i], f[i]), hf[i] = greatest(hf[i], f[i]);
        lo = from_f32x8<F16>(lf);
        hi = from_f32x8<F16>(hf);
      }
      *reinterpret_cast<u32x4*>(bd) = lo;
      *reinterpret_cast<u32x4*>(bd + A.d) = hi;
    }
    *reinterpret_cast<u32x4*>(A.k + p) = kw;
    *reinterpret_cast<u32x4*>(A.v + p) = vw;
  }
}

// ------------------------------------------------------------------ attention over pages
// One query token a sequence: o = softmax(scale q K^T) V over keys in pages, one pass with a running
// maximum m, sum l and unnormalised output, in base 2 (scores times scale * log2 e). A workgroup takes
// a part of the keys for a tile of query rows of one kv head and leaves (m, l, o) of it; combine_kernel
// joins the parts. Rows that read the same keys share a tile: the queries of all sequences for the
// shared prefix, so its K and V are read once for 128 rows, the query heads of one kv head for a
// sequence's own rows.
//
// K and V rows go to LDS by 1 KB DMA instructions; a row's 16-byte pieces are XOR-swizzled with the row
// (applied where the DMA reads), so that the 16 rows of a fragment read fall in distinct banks. Every
// form takes 64 KB of LDS and at most 256 registers (D = 128), so that two workgroups are resident on a
// CU: while one starts, waits or joins its waves, the other streams, and parts of the prefix, which
// are bound by the matrix units, run beside own rows, which are bound by memory.
//
// Scores come transposed, S^T = K Q^T: a lane holds 4 keys of each 16-key tile for one query row, so
// the softmax needs one reduction over the four lane groups, and its probabilities are already the
// operand of O^T = V^T P^T, whose V^T comes from LDS by transpose reads in the same key order. The
// probabilities are rounded to the type for that product (at most a relative 2^-8 of a term in bf16, 2^-11
// in fp16, as much as the output's own rounding; the sum they are divided by is that of the rounded
// ones); maxima, sums and outputs stay in 32 bits.
constexpr int NUM_CUS = 256;
constexpr int AW = 4;   // waves
constexpr int KS = 32;  // keys a wave takes at a time, of own rows
constexpr int TS = 64;  // keys a workgroup takes at a time, of a prefix whose rows its waves share out

#define PG_AWAIT(n) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(n) : "memory")
// this wave's LDS reads are done
#define PG_READ() asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory")
// this wave's DMAs have landed and its LDS reads are done, for every wave of the workgroup
#define PG_BARRIER() asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory")

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
template <bool F16>
__device__ __forceinline__ f32x4 mma(const u32x4& a, const u32x4& b, f32x4 c) {
  if constexpr (F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return mfma_16x16x32(a, b, c);
}
template <bool F16>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (F16)
    return (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)lo) |
           (uint32_t)__builtin_bit_cast(unsigned short, (_Float16)hi) << 16;
  else
    return pack_bf2(lo, hi);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
// maximum over the four 16-lane groups (lanes l, l + 16, l + 32, l + 48), in every group
__device__ __forceinline__ float groups_max(float v) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s lds_v4s;
typedef const __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) f32x4 lds_f32x4;
typedef __attribute__((address_space(3))) uint8_t lds_byte;
typedef const __attribute__((address_space(1))) int gint;

// The swizzle of a row's 16-byte pieces (D / 8 of them), by XOR with the piece's number: the rows that one read
// takes together fall in distinct banks. 256-byte rows all start at the same bank, 128-byte ones in pairs. K is
// read 16 rows of a piece at a time, V by transpose reads, 8 rows of two neighbouring pieces at a time. No read
// of either meets another one's bank (counted: SQ_LDS_BANK_CONFLICT 0).
template <int D>
__device__ __forceinline__ int swz_k(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D>
__device__ __forceinline__ int swz_v(int row) { return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 3); }

// A value that a plain load brought, used here: the compiler, which does not count the DMA instructions, waits
// for it at this place, and not (for every load and DMA under way) at its next use inside a loop
template <class T>
__device__ __forceinline__ void settled(T& x) { asm volatile("" : "+v"(x)); }

// The page ids of a run of keys, 64 at a time, one a lane; asked for in ascending order.
struct Pages {
  const int* table;
  int first, last, ids, num_pages;
  bool bad;  // an id was outside the pool (page 0 is read in its place)
  __device__ __forceinline__ Pages(const int* t, int n, int page_lo, int page_last, int lane, bool any)
      : table(t), first(page_lo), last(page_last), ids(0), num_pages(n), bad(false) {
    if (!any) return;  // (a run without keys may have no table)
    ids = *(gint*)(table + min(first + lane, last));
    settled(ids);
  }
  __device__ __forceinline__ int operator()(int page, int lane) {
    if (page - first >= 64) {
      first = page;
      ids = *(gint*)(table + min(first + lane, last));
      settled(ids);
    }
    const int id = __builtin_amdgcn_readlane(ids, page - first);
    if (id >= 0 && id < num_pages) return id;
    bad = true;
    return 0;
  }
};

// One DMA instruction: lane l's 16 bytes at base + off to LDS byte lds + 16 l (dma16 with a uniform base, so that a
// step's addresses cost no vector instruction; ONCE: past the caches)
template <bool ONCE>
__device__ __forceinline__ void dma16_at(const uint16_t* base, uint32_t off, uint32_t lds) {
  uint32_t saved;
  if constexpr (ONCE)
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\tglobal_load_lds_dwordx4 %1, %2 nt\n\ts_mov_b32 m0, %0"
                 : "=&s"(saved)
                 : "v"(off), "s"(base), "s"(lds)
                 : "memory");
  else
    asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %3\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b32 m0, %0"
                 : "=&s"(saved)
                 : "v"(off), "s"(base), "s"(lds)
                 : "memory");
}

// Byte offsets, from a 16-key tile's first row, of the pieces that a lane brings: instruction i moves rows RPI i ..,
// lane l -> row RPI i + l / CPR, slot l % CPR, which takes the piece that the swizzle puts there
template <int D, bool V>
struct Lanes {
  static constexpr int CPR = D / 8, RPI = 64 / CPR, NI = 16 / RPI;  // pieces a row, rows an instruction, instructions
  uint32_t off[NI];
  __device__ __forceinline__ explicit Lanes(int lane) {
#pragma unroll
    for (int i = 0; i < NI; i++) {
      const int row = RPI * i + lane / CPR;
      off[i] = row * (2 * D) + 16 * ((lane % CPR) ^ (V ? swz_v<D>(row) : swz_k<D>(row)));
    }
  }
  // the tile at `base` to LDS; rows past `last` repeat it (their scores are masked; a row that is not there is never read)
  template <bool ONCE>
  __device__ __forceinline__ void fetch(const uint16_t* base, int last, uint32_t dst, int lane) const {
#pragma unroll
    for (int i = 0; i < NI; i++) {
      uint32_t o = off[i];
      if (last < 15) o -= max(0, RPI * i + lane / CPR - last) * (2 * D);
      dma16_at<ONCE>(base, o, __builtin_amdgcn_readfirstlane(dst + 1024u * i));
    }
  }
};

// Where the 16-key tile at key k0 (or, past the last key, that key's tile) lies in a layer's K (and V), and the last
// row of it that is there
struct Tile {
  size_t at;
  int last;
  __device__ __forceinline__ Tile(Pages& pages, const AttnArgs& A, int h, int d, int k0, int k_last, int lane) {
    const int k = min(k0, k_last & ~15);
    at = (((((size_t)pages(k >> A.lp, lane) * A.hkv + h) << A.lp) + (k & ((1 << A.lp) - 1))) * d);
    last = k_last - k;
  }
};

// Fragment addresses in 16-key tiles of LDS rows: K row r16, pieces 4 ks + kg; V keys 4 kg + r16 / 4, dims
// 16 dt + 4 (r16 % 4) .. + 3 (a tile t adds 32 t D bytes; ks and dt come in by XOR)
template <int D>
__device__ __forceinline__ uint32_t k_frag(int r16, int kg) { return r16 * (2 * D) + 16 * (kg ^ swz_k<D>(r16)); }
template <int D>
__device__ __forceinline__ uint32_t v_frag(int r16, int kg) {
  const int row = 4 * kg + (r16 >> 2);
  return row * (2 * D) + 16 * (((r16 & 3) >> 1) ^ swz_v<D>(row)) + 8 * (r16 & 1);
}

// m is the maximum that a row's probabilities are taken relative to. Where the matrix units are the bound
// (prefix_part) it follows the true one only once that is 2^SLACK times as large, so that few steps have to rescale l
// and o (64 products a 64-key step, 40% of all vector instructions there; the prefix of 16384 rows for 512 query rows
// 61.0 us at 0, 58.8 at 1, 57.8 at 8). Where memory is (own_part) it is the maximum. The nearer it is, the less
// the heaviest terms, just below 1 then, round: bf16 outputs are a relative 2.3e-3 from the 64-bit ones at 8, 2.1e-3 at 0
// (the output's own rounding alone: 1.7e-3).
constexpr float SLACK = 1.f;

// One step of NT key tiles (K and V rows in LDS at kb and vb) for RB * 16 query rows: running maximum m of
// query row r16 of each block, sum l (four equal values) and output o (lane: dims 16 dt + 4 kg + e of row r16).
// `left`: keys of the step that are there. before_v() runs between the scores and the product with V.
// The vector units are the tighter bound here (the products of a 64-key step of 32 rows cost the matrix units 1024
// cycles), so the sum of the probabilities is another row of the product, with ones
// for V, and the maximum takes three operands (v_maximum3_f32; a score that is not a number
// makes its row's output not a number either way).
template <bool F16, int D, int RB, int NT, class BeforeV>
__device__ __forceinline__ void attend_step(uint32_t kb, uint32_t vb, int left, float scale, float slack, int kg, uint32_t ka,
                                            uint32_t va, const u32x4 (&qf)[RB][D / 32], float (&m)[RB], f32x4 (&l)[RB],
                                            f32x4 (&o)[RB][D / 16], BeforeV before_v) {
  f32x4 sc[RB][NT];
  // two key tiles at a time (2 RB chains of products that do not wait for each other); a pair's K fragments are
  // read each as soon as its registers are free, beside the products of the pair before
  u32x4 kf[2][D / 32];
  auto load_k = [&](int t, int ks) {
    kf[t & 1][ks] = *(lds_u32x4*)((const lds_byte*)(uintptr_t)(kb + (ka ^ (64u * ks))) + 32 * D * t);
  };
#pragma unroll
  for (int ks = 0; ks < D / 32; ks++) load_k(0, ks), load_k(1, ks);
#pragma unroll
  for (int t = 0; t < NT; t += 2) {
#pragma unroll
    for (int rb = 0; rb < RB; rb++) sc[rb][t] = sc[rb][t + 1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < D / 32; ks++) {
#pragma unroll
      for (int rb = 0; rb < RB; rb++) {
        sc[rb][t] = mma<F16>(kf[0][ks], qf[rb][ks], sc[rb][t]);
        sc[rb][t + 1] = mma<F16>(kf[1][ks], qf[rb][ks], sc[rb][t + 1]);
      }
      if (t + 2 < NT) load_k(t + 2, ks), load_k(t + 3, ks);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  if (left < 16 * NT) {
    asm volatile("");  // (a branch: as selects it would cost every step)
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (16 * t + 4 * kg + e >= left)
#pragma unroll
          for (int rb = 0; rb < RB; rb++) sc[rb][t][e] = -INFINITY;
  }
  float mx[RB];
  bool raise = false;
#pragma unroll
  for (int rb = 0; rb < RB; rb++) {
    mx[rb] = -INFINITY;
#pragma unroll
    for (int t = 0; t < NT; t++)
      mx[rb] = max3(max3(mx[rb], sc[rb][t][0], sc[rb][t][1]), sc[rb][t][2], sc[rb][t][3]);
    mx[rb] = fmaxf(m[rb], groups_max(mx[rb]) * scale);
    raise |= mx[rb] > m[rb] + slack;
  }
  if (__any(raise)) {
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
      const float al = mx[rb] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[rb] - mx[rb]);
#pragma unroll
      for (int e = 0; e < 4; e++) l[rb][e] *= al;
#pragma unroll
      for (int dt = 0; dt < D / 16; dt++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[rb][dt][e] *= al;
      m[rb] = mx[rb];
    }
  }
  before_v();
  constexpr uint32_t ONE = F16 ? 0x3c003c00u : 0x3f803f80u;
  const u32x4 ones = u32x4{ONE, ONE, ONE, ONE};
  // straight-line from here: the V fragments of a 32-key half are read before its exponentials, those of the
  // next one each as soon as its registers are free, beside the products of this one
  u32x4 vf[D / 16];
  auto load_v = [&](int j, int dt) {
    lds_byte* at = (lds_byte*)(uintptr_t)(vb + (va ^ (32u * dt))) + 64 * D * j;
    const u32x2 lo = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)at));
    const u32x2 hi = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(at + 32 * D)));
    vf[dt] = u32x4{lo.x, lo.y, hi.x, hi.y};
  };
#pragma unroll
  for (int dt = 0; dt < D / 16; dt++) load_v(0, dt);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int j = 0; j < NT / 2; j++) {
    u32x4 pf[RB];
#pragma unroll
    for (int rb = 0; rb < RB; rb++) {
      const float base = m[rb] == -INFINITY ? 0.f : m[rb];
#pragma unroll
      for (int t = 0; t < 2; t++) {
        float p[4];
#pragma unroll
        for (int e = 0; e < 4; e++) p[e] = __builtin_amdgcn_exp2f(fmaf(sc[rb][2 * j + t][e], scale, -base));
        pf[rb][2 * t] = pack2<F16>(p[0], p[1]);
        pf[rb][2 * t + 1] = pack2<F16>(p[2], p[3]);
      }
    }
#pragma unroll
    for (int rb = 0; rb < RB; rb++) l[rb] = mma<F16>(ones, pf[rb], l[rb]);
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++) {
#pragma unroll
      for (int rb = 0; rb < RB; rb++) o[rb][dt] = mma<F16>(vf[dt], pf[rb], o[rb][dt]);
      if (j + 1 < NT / 2) {
        load_v(j + 1, dt);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
}

// Query fragments of rows row0 + 16 rb + r16 (row r of a kv head: its query r % G of sequence b0 + r / G)
template <int D, int RB>
__device__ __forceinline__ void load_q(const AttnArgs& A, int h, int b0, int row0, int rows, int r16, int kg,
                                       u32x4 (&qf)[RB][D / 32]) {
#pragma unroll
  for (int rb = 0; rb < RB; rb++) {
    const int r = min(row0 + 16 * rb + r16, rows - 1);  // (rows past the end repeat the last one and are not stored)
    const uint16_t* q = A.q + (size_t)(b0 + r / A.g) * A.q_sb + (size_t)(h * A.g + r % A.g) * A.q_sh;
#pragma unroll
    for (int ks = 0; ks < D / 32; ks++) qf[rb][ks] = *(gu32x4*)(q + 32 * ks + 8 * kg);
  }
#pragma unroll
  for (int rb = 0; rb < RB; rb++)
#pragma unroll
    for (int ks = 0; ks < D / 32; ks++) settled(qf[rb][ks]);
}

// Device-scope accesses, for what one workgroup leaves to another of the same launch, maybe on another XCD: they pass
// the L2, which holds no other XCD's stores.
__device__ __forceinline__ void put_dev(void* p, u32x2 x) {
  __hip_atomic_store(static_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ u32x2 get_dev(const void* p) {
  return __builtin_bit_cast(u32x2, __hip_atomic_load(static_cast<const uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Where row r's result goes: part `slot` of the partial results, or, as the only part, the output. DEV: the parts are
// joined in the same launch.
template <bool F16, int D, bool DEV>
__device__ __forceinline__ void store_o(const AttnArgs& A, int slot, bool only, int h, int b0, int r, int d0, f32x4 x, float m,
                                        float l) {
  const int b = b0 + r / A.g, hq = h * A.g + r % A.g;
  if (only) {
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    *reinterpret_cast<u32x2*>(A.out + (size_t)b * A.o_sb + (size_t)hq * A.o_sh + d0) =
        u32x2{pack2<F16>(x[0] * inv, x[1] * inv), pack2<F16>(x[2] * inv, x[3] * inv)};
    return;
  }
  const size_t at = ((size_t)slot * A.batch + b) * A.hq + hq;
  if constexpr (DEV) {
    put_dev(A.part_o + at * D + d0, u32x2{__float_as_uint(x[0]), __float_as_uint(x[1])});
    put_dev(A.part_o + at * D + d0 + 2, u32x2{__float_as_uint(x[2]), __float_as_uint(x[3])});
    if (d0 == 0) put_dev(A.part_ml + at, u32x2{__float_as_uint(m), __float_as_uint(l)});
  } else {
    *reinterpret_cast<f32x4*>(A.part_o + at * D + d0) = x;
    if (d0 == 0) A.part_ml[at] = make_float2(m, l);
  }
}

// A run of keys: positions [lo, hi) of the sequence (or prefix) with page table `table`
struct Run {
  const int* table;
  int lo, hi;
};

// The 32-key steps of a run from key k0 on, every `stride` keys, for 16 query rows, by one wave with 16 KB of LDS, half
// for K and half for V: it asks for the next step's K as soon as it has the scores of this one, for its V once this one's is multiplied.
// load() brings the query fragments. The rows are read once (or, of several runs, by few workgroups), past the caches:
// non-temporal, 6.1 against 5.4 TB/s. True if a page was outside the pool.
template <bool F16, int D, class Load>
__device__ __forceinline__ bool walk(const AttnArgs& A, const Run& run, int h, int k0, int stride, uint32_t mine, int lane,
                                     const Lanes<D, false>& lk, const Lanes<D, true>& lv, u32x4 (&qf)[1][D / 32],
                                     float (&m)[1], f32x4 (&l)[1], f32x4 (&o)[1][D / 16], Load load) {
  constexpr uint32_t HALF = KS * D * 2;  // bytes of a step's K (or V)
  constexpr int NI = KS * D * 2 / 1024;  // DMA instructions of it
  const uint32_t ka = k_frag<D>(lane & 15, lane >> 4), va = v_frag<D>(lane & 15, lane >> 4);
  const int k_hi = run.hi;
  const bool any = k0 < k_hi;  // (the wave's)
  Pages pages(run.table, A.num_pages, run.lo >> A.lp, max(run.lo, k_hi - 1) >> A.lp, lane, any);
  size_t at[2];  // a step's two tiles
  int last[2];
  auto find = [&](int k0) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const Tile t(pages, A, h, D, k0 + 16 * i, k_hi - 1, lane);
      at[i] = t.at;
      last[i] = t.last;
    }
  };
  auto fetch_k = [&] {
#pragma unroll
    for (int i = 0; i < 2; i++) lk.template fetch<true>(A.k + at[i], last[i], mine + HALF / 2 * i, lane);
  };
  auto fetch_v = [&] {
#pragma unroll
    for (int i = 0; i < 2; i++) lv.template fetch<true>(A.v + at[i], last[i], mine + HALF + HALF / 2 * i, lane);
  };
  if (any) {
    find(k0);
    fetch_k();
    fetch_v();
  }
  load();
  for (; k0 < k_hi; k0 += stride) {
    const int next = k0 + stride;
    PG_AWAIT(NI);  // K is there (V may be in flight)
    attend_step<F16, D, 1, KS / 16>(mine, mine + HALF, k_hi - k0, A.scale_log2, 0.f, lane >> 4, ka, va, qf, m, l, o, [&] {
      PG_READ();  // (K is in registers)
      if (next < k_hi) {
        find(next);
        fetch_k();
        PG_AWAIT(NI);  // V is there (the next K may be in flight)
      } else {
        PG_AWAIT(0);
      }
    });
    PG_READ();
    if (next < k_hi) fetch_v();
  }
  return pages.bad;
}

template <int RB, int N>
__device__ __forceinline__ void clear(float (&m)[RB], f32x4 (&l)[RB], f32x4 (&o)[RB][N]) {
#pragma unroll
  for (int rb = 0; rb < RB; rb++) {
    m[rb] = -INFINITY;
    l[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < N; dt++) o[rb][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
}

// The keys of one run for up to 16 query rows, by one wave.
template <bool F16, int D>
__device__ __forceinline__ void wave_part(const AttnArgs& A, const Run& run, int h, int b, int row0, int rows, int slot, bool only,
                                          uint32_t mine, int lane) {
  const Lanes<D, false> lk(lane);
  const Lanes<D, true> lv(lane);
  u32x4 qf[1][D / 32];
  float m[1];
  f32x4 l[1], o[1][D / 16];
  clear(m, l, o);
  const bool bad = walk<F16, D>(A, run, h, run.lo, KS, mine, lane, lk, lv, qf, m, l, o,
                                   [&] { load_q<D, 1>(A, h, b, row0, rows, lane & 15, lane >> 4, qf); });
  const int r = row0 + (lane & 15);
  if (r < rows)
#pragma unroll
    for (int dt = 0; dt < D / 16; dt++)
      store_o<F16, D, false>(A, slot, only, h, b, r, 16 * dt + 4 * (lane >> 4), o[0][dt], m[0], bad ? NAN : l[0][0]);
}

// The keys of N runs for up to 16 query rows, by a workgroup: its waves take steps in turn and do not wait for each
// other until the end.
template <bool F16, int D, int N, bool DEV>
__device__ __forceinline__ void own_part(const AttnArgs& A, const Run (&runs)[N], int h, int b0, int row0, int rows, int slot,
                                         bool only, uint32_t lds, float (*s_m)[16], float (*s_l)[16]) {
  constexpr uint32_t WAVE = 2 * KS * D * 2;  // bytes of a wave
  static_assert(16 * D * 4 <= (int)WAVE, "a wave's output fits its LDS");
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, kg = lane >> 4;
  const uint32_t mine = lds + WAVE * wv;
  const Lanes<D, false> lk(lane);
  const Lanes<D, true> lv(lane);
  u32x4 qf[1][D / 32];
  float m[1];
  f32x4 l[1], o[1][D / 16];
  clear(m, l, o);
  bool bad = false;
#pragma unroll
  for (int n = 0; n < N; n++)
    bad |= walk<F16, D>(A, runs[n], h, runs[n].lo + KS * wv, KS * AW, mine, lane, lk, lv, qf, m, l, o, [&] {
      if (n == 0) load_q<D, 1>(A, h, b0, row0, rows, r16, kg, qf);
    });
  // ---- join the waves: each scales its output to the rows' common maximum and leaves it in its LDS (row:
  // D / 4 pieces of 16 bytes, swizzled with the row), then all add the four up
  if (kg == 0) {
    s_m[wv][r16] = m[0];
    s_l[wv][r16] = bad ? NAN : l[0][0];
  }
  __syncthreads();
  float top = s_m[0][r16];
#pragma unroll
  for (int w = 1; w < AW; w++) top = fmaxf(top, s_m[w][r16]);
  const float f = m[0] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[0] - top);
#pragma unroll
  for (int dt = 0; dt < D / 16; dt++) {
    f32x4 x = o[0][dt];
#pragma unroll
    for (int e = 0; e < 4; e++) x[e] *= f;
    *(lds_f32x4*)(uintptr_t)(mine + r16 * (4 * D) + 16 * ((4 * dt + kg) ^ r16)) = x;
  }
  __syncthreads();
  constexpr int PPR = D / 4;  // 16-byte pieces a row
  const int n = min(16, rows - row0) * PPR;
  for (int i = tid; i < n; i += 64 * AW) {
    const int r = i / PPR, p = i % PPR;
    f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < AW; w++) x += *(lds_f32x4*)(uintptr_t)(lds + WAVE * w + r * (4 * D) + 16 * (p ^ r));
    float mx = s_m[0][r], sum = 0.f;
#pragma unroll
    for (int w = 1; w < AW; w++) mx = fmaxf(mx, s_m[w][r]);
#pragma unroll
    for (int w = 0; w < AW; w++) {
      const float mw = s_m[w][r], lw = s_l[w][r];
      sum += lw == 0.f ? 0.f : lw * __builtin_amdgcn_exp2f(mw - (mx == -INFINITY ? 0.f : mx));
    }
    store_o<F16, D, DEV>(A, slot, only, h, b0, row0 + r, 4 * p, x, mx, sum);
  }
}

// Keys [k_lo, k_hi) of the prefix for up to 64 RB query rows from row0 of all `rows`: wave w takes RB blocks
// of 16 rows from row0 + 16 RB w and all the keys, 64 at a time, from LDS that the workgroup fills together
// (two stages: the next one is on its way while this one is multiplied). One barrier a step: once every
// wave is there, the stage is complete and the other one has been read. Bound by the vector and matrix units: a
// step of 32 rows costs a wave 1088 cycles of products and about as many of exponentials (32 at a quarter of the
// rate) and the rest, and two waves share a SIMD; 16384 rows for 512 query rows keep the matrix units 37% busy.
// Without any K and V fetched the steps took 1.6 us where they take 2.35; asking for K and V half a step earlier,
// with a second barrier, or putting the exponentials of one half between the products of the other gained nothing.
template <bool F16, int D, int RB>
__device__ __forceinline__ void prefix_part(const AttnArgs& A, int h, int row0, int rows, int k_lo, int k_hi, int slot, bool only,
                                            uint32_t lds) {
  constexpr uint32_t HALF = TS * D * 2, STAGE = 2 * HALF;
  const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, kg = lane >> 4;
  const Lanes<D, false> lk(lane);
  const Lanes<D, true> lv(lane);
  Pages pages(A.prefix_pages, A.num_pages, k_lo >> A.lp, (k_hi - 1) >> A.lp, lane, true);
  // wave w brings keys 16 w .. + 15 of a step
  auto fetch = [&](int k0, uint32_t dst) {
    const Tile t(pages, A, h, D, k0 + 16 * wv, k_hi - 1, lane);
    lk.template fetch<false>(A.k + t.at, t.last, dst + HALF / 4 * wv, lane);
    lv.template fetch<false>(A.v + t.at, t.last, dst + HALF + HALF / 4 * wv, lane);
  };
  fetch(k_lo, lds);
  u32x4 qf[RB][D / 32];
  const int mine = row0 + 16 * RB * wv;
  load_q<D, RB>(A, h, 0, mine, rows, r16, kg, qf);
  float m[RB];
  f32x4 l[RB], o[RB][D / 16];
  clear(m, l, o);
  const uint32_t ka = k_frag<D>(r16, kg), va = v_frag<D>(r16, kg);
  uint32_t st = 0;
  for (int k0 = k_lo; k0 < k_hi; k0 += TS, st ^= STAGE) {
    PG_BARRIER();
    if (k0 + TS < k_hi) fetch(k0 + TS, lds + (st ^ STAGE));
    attend_step<F16, D, RB, TS / 16>(lds + st, lds + st + HALF, k_hi - k0, A.scale_log2, SLACK, kg, ka, va, qf, m, l, o, [] {});
  }
  // every wave has seen some of the page ids: a bad one anywhere reaches all rows of the tile
  const int bad = __syncthreads_or(pages.bad);
#pragma unroll
  for (int rb = 0; rb < RB; rb++) {
    const int r = mine + 16 * rb + r16;
    const float sum = bad ? NAN : l[rb][0];
    if (r < rows)
#pragma unroll
      for (int dt = 0; dt < D / 16; dt++)         store_o<F16, D, false>(A, slot, only, h, 0, r, 16 * dt + 4 * kg, o[rb][dt], m[rb], sum);
  }
}

// positions that a sequence has: lens[b] and what was appended since, within its table
__device__ __forceinline__ int own_rows(const int* lens, int b, int add, int width, int lp) {
  const int most = width << lp;
  return max(0, min(min(lens[b], most) + add, most));
}

// keys of one part of `parts` of `len` keys, in units of 128 (a step for each wave, two of the prefix)
constexpr int UNIT = KS * AW;
__host__ __device__ __forceinline__ int part_keys(int len, int parts) { return ((len + parts - 1) / parts + UNIT - 1) / UNIT * UNIT; }

// How the query rows of a prefix are tiled: for up to 16 rows, the keys are split among the waves (own_part); of more,
// the rows are (prefix_part; 32 rows behind 8192 14.8 us, 21.4 with the keys split). JOINED: no tiles of the prefix; each
// sequence's workgroup goes over the prefix and then over its own rows, so that nothing is left to join and the call is
// one launch. OWN: no prefix, and the last workgroup of a sequence's parts joins them (a launch before has cleared the
// tickets that tell which one is last): the GPU's time is that of a second launch (one sequence over 64 of 250 pages
// 15.8 us, 16.0 with it), the host's 4 us less.
enum : int { ROWS16, ROWS64, ROWS128, JOINED, OWN };
__host__ __device__ constexpr int tile_rows(int form) { return form == ROWS16 ? 16 : form == ROWS64 ? 64 : 128; }

// One row (query head, sequence), by one wave: the parts' outputs, scaled to their common maximum, over their sums. Rows
// without a key give zeros. Lane p takes part p's maximum and sum (and part p + 64's); LPR lanes hold
// a row's output, and the wave's 64 / LPR groups of them take the parts in turn, eight in flight, and are
// added in order, so that a result does not depend on timing. The first eight are asked for together with the maxima,
// which tell whether a part had a key (if not, its output was not written and is not used). DEV: the parts are of this
// launch.
constexpr int MAX_PARTS = 128;
template <bool F16, int D, bool DEV>
__device__ __forceinline__ void join_row(const AttnArgs& A, size_t row, int parts, int lane) {
  constexpr int LPR = D / 4, GROUPS = 64 / LPR, AHEAD = 8;
  const size_t rows = (size_t)A.batch * A.hq;
  const int grp = lane / LPR, c = lane % LPR;
  f32x4 y[AHEAD];
  auto fetch = [&](int p0) {
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
      const float* at = A.part_o + (row + rows * min(p0 + GROUPS * u + grp, parts - 1)) * D + 4 * c;
      if constexpr (DEV) {
        const u32x2 lo = get_dev(at), hi = get_dev(at + 2);
        y[u] = __builtin_bit_cast(f32x4, u32x4{lo.x, lo.y, hi.x, hi.y});
      } else {
        y[u] = *reinterpret_cast<const f32x4*>(at);
      }
    }
  };
  float2 ml[2] = {make_float2(-INFINITY, 0.f), make_float2(-INFINITY, 0.f)};
  if (parts > 0) {
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const float2* p = A.part_ml + row + rows * min(lane + 64 * i, parts - 1);
      ml[i] = DEV ? __builtin_bit_cast(float2, get_dev(p)) : *p;
    }
    fetch(0);
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
    if (lane + 64 * i >= parts) ml[i] = make_float2(-INFINITY, 0.f);
  float mx[1] = {fmaxf(ml[0].x, ml[1].x)};
  wave_max_n(mx);
  const float base = mx[0] == -INFINITY ? 0.f : mx[0];
  float w[2], l = 0.f;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const float f = __builtin_amdgcn_exp2f(ml[i].x - base);
    l += ml[i].y == 0.f ? 0.f : f * ml[i].y;
    w[i] = ml[i].y == 0.f ? -1.f : f;  // (no key: its output was not written)
  }
  l = wave_sum(l);
  f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int p0 = 0; p0 < parts; p0 += GROUPS * AHEAD) {
    if (p0 > 0) fetch(p0);
#pragma unroll
    for (int u = 0; u < AHEAD; u++) {
      const int p = p0 + GROUPS * u + grp;
      const float f = __shfl(p < 64 ? w[0] : w[1], p & 63, 64);
      if (p < parts && !(f < 0.f))
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] += f * y[u][e];
    }
  }
#pragma unroll
  for (int e = 0; e < 4; e++) {
    if (GROUPS == 4) x[e] += __shfl_xor(x[e], 16, 64);
    x[e] += __shfl_xor(x[e], 32, 64);
  }
  if (grp > 0) return;
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  *reinterpret_cast<u32x2*>(A.out + row / A.hq * A.o_sb + row % A.hq * A.o_sh + 4 * c) =
      u32x2{pack2<F16>(x[0] * inv, x[1] * inv), pack2<F16>(x[2] * inv, x[3] * inv)};
}

template <bool F16, int D, int FORM>
__global__ void __launch_bounds__(64 * AW, 2) attn_kernel(AttnArgs A) {
  __shared__ __align__(1024) uint8_t s_kv[4 * TS * D * 2];
  __shared__ float s_m[AW][16], s_l[AW][16];
  static_assert(sizeof(s_kv) == AW * 2 * KS * D * 2, "the forms take the same LDS");
  const uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)&s_kv[0];
  if constexpr (FORM == JOINED) {
    const int h = blockIdx.x % A.hkv, id = blockIdx.x / A.hkv, tile = id % A.own_tiles, b = id / A.own_tiles;
    const int len = own_rows(A.lens, b, A.len_add, A.width, A.lp);
    const Run runs[2] = {{A.prefix_pages, 0, A.prefix_len}, {A.tables + (size_t)b * A.t_sb + (size_t)h * A.t_sh, 0, len}};
    own_part<F16, D, 2, false>(A, runs, h, b, 16 * tile, A.g, 0, true, lds, s_m, s_l);
  } else if constexpr (FORM == OWN) {
    int id = blockIdx.x;
    const int h = id % A.hkv;
    id /= A.hkv;
    const int tile = id % A.own_tiles;
    id /= A.own_tiles;
    const int b = id % A.batch, part = id / A.batch, rows = min(16, A.g - 16 * tile), tid = threadIdx.x;
    const int len = own_rows(A.lens, b, A.len_add, A.width, A.lp);
    const int ch = part_keys(len, A.ns), lo = part * ch, hi = min(len, lo + ch);
    if (lo >= hi) {
      if (part > 0) return;  // (the parts that have a key are joined)
      for (int i = tid; i < rows * (D / 4); i += 64 * AW)
        store_o<F16, D, true>(A, 0, true, h, b, 16 * tile + i / (D / 4), 4 * (i % (D / 4)), f32x4{0.f, 0.f, 0.f, 0.f}, 0.f, 0.f);
      return;
    }
    const int parts = (len + ch - 1) / ch;
    const Run mine[1] = {{A.tables + (size_t)b * A.t_sb + (size_t)h * A.t_sh, lo, hi}};
    own_part<F16, D, 1, true>(A, mine, h, b, 16 * tile, A.g, part, parts == 1, lds, s_m, s_l);
    if (parts == 1) return;
    PG_AWAIT(0);  // the wave's stores have been written, and after the barrier every wave's
    __shared__ int s_last;
    __syncthreads();
    if (tid == 0)
      s_last = __hip_atomic_fetch_add(A.tickets + ((size_t)b * A.hkv + h) * A.own_tiles + tile, 1u, __ATOMIC_RELAXED,
                                      __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)parts - 1;
    __syncthreads();
    if (!s_last) return;
    for (int r = tid >> 6; r < rows; r += AW)
      join_row<F16, D, true>(A, (size_t)b * A.hq + h * A.g + 16 * tile + r, parts, tid & 63);
  } else {
    // parts of the prefix and of own rows alternate, a workgroup a CU of each, while there are both
    const bool only = A.np + A.ns == 1;
    const int n_prefix = A.hkv * A.prefix_tiles * A.np, n_own = A.hkv * A.own_tiles * A.groups * A.ns;
    const int runs = min(n_prefix, n_own) / NUM_CUS, bid = blockIdx.x, run = bid / NUM_CUS, rest = bid - runs * NUM_CUS;
    const bool prefix = run < 2 * runs ? run % 2 == 0 : rest < n_prefix;
    int id = run < 2 * runs ? run / 2 * NUM_CUS + bid % NUM_CUS : rest < n_prefix ? rest : bid - n_prefix;
    const int h = id % A.hkv;  // (fastest: with 8 kv heads each XCD reads one head's rows)
    id /= A.hkv;
    if (prefix) {
      const int rows = A.batch * A.g, row0 = tile_rows(FORM) * (id % A.prefix_tiles), part = id / A.prefix_tiles;
      const int ch = part_keys(A.prefix_len, A.np), lo = part * ch, hi = min(A.prefix_len, lo + ch);
      if constexpr (FORM == ROWS16) {
        const Run mine[1] = {{A.prefix_pages, lo, hi}};
        own_part<F16, D, 1, false>(A, mine, h, 0, row0, rows, part, only, lds, s_m, s_l);
      } else {
        prefix_part<F16, D, FORM == ROWS64 ? 1 : 2>(A, h, row0, rows, lo, hi, part, only, lds);
      }
      return;
    }
    const int tile = id % A.own_tiles;
    id /= A.own_tiles;
    if (A.groups < A.batch) {
      const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), b = AW * id + wv;
      if (b >= A.batch) return;
      const int len = own_rows(A.lens, b, A.len_add, A.width, A.lp);
      const Run mine = {A.tables + (size_t)b * A.t_sb + (size_t)h * A.t_sh, 0, len};
      wave_part<F16, D>(A, mine, h, b, 16 * tile, A.g, A.np, only, lds + 4 * KS * D * wv, lane);
      return;
    }
    const int b = id % A.batch, part = id / A.batch;
    const int len = own_rows(A.lens, b, A.len_add, A.width, A.lp);
    const int ch = part_keys(len, A.ns), lo = part * ch, hi = min(len, lo + ch);
    if (lo >= hi) {
      // no key: the part's sum says so, or, as the only part, the output is zero
      const int n = min(16, A.g - 16 * tile) * (D / 4);
      for (int i = threadIdx.x; i < n; i += 64 * AW)
        if (only || i % (D / 4) == 0)
          store_o<F16, D, false>(A, A.np + part, only, h, b, 16 * tile + i / (D / 4), 4 * (i % (D / 4)), f32x4{0.f, 0.f, 0.f, 0.f},
                                 -INFINITY, 0.f);
      return;
    }
    const Run mine[1] = {{A.tables + (size_t)b * A.t_sb + (size_t)h * A.t_sh, lo, hi}};
    own_part<F16, D, 1, false>(A, mine, h, b, 16 * tile, A.g, A.np + part, only, lds, s_m, s_l);
  }
}

// A wave a row.
template <bool F16, int D>
__global__ void __launch_bounds__(256) combine_kernel(AttnArgs A) {
  const size_t row = (size_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (size_t)A.batch * A.hq) return;
  join_row<F16, D, false>(A, row, A.np + A.ns, threadIdx.x & 63);
}

// ------------------------------------------------------------------ choosing pages
// The score of a page for the queries of one kv head is the most that their products with any of its
// keys can add up to, given the bounds lo <= key <= hi of each dim:
//   sum over queries and dims of max(q lo, q hi) = sum over dims of hi sum(max(q, 0)) + lo sum(min(q, 0)),
// two products a dim whatever the number of queries. It is summed in 64 bits, where these 16-bit
// values' products and sums are exact but for far smaller terms, so that the choice does not hang on
// the order of the additions. Chosen are the last page and the top - 1 best others, the lower
// of equals first; a score that is not a number counts as the greatest.
//
// One workgroup a (kv head, sequence), 7.5 us for 250 pages, of which 2.7 are the sums (128 64-bit conversions
// and products a lane on one CU) and 2.3 the choice: 16 lanes take a page (8 dims each at 128), the scores go to LDS
// as unsigned 64-bit keys in the order of the scores. Of up to 1024 of them one wave finds the last that is
// chosen, of more the workgroup, by a radix selection 8 bits at a time. The chosen pages are written in
// ascending order.
constexpr int ST = 1024;              // threads

__device__ __forceinline__ uint64_t order_key(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);  // (-0 counts as 0)
  if (x != x) return ~0ull;
  return u >> 63 ? ~u : u | 1ull << 63;
}

// (the lane orders of row16_sum)
template <int CTRL>
__device__ __forceinline__ double dpp64(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, 0xF, 0xF, true);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, 0xF, 0xF, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// Of n <= 64 R keys, one wave: the `want` greatest, the lower of equals first, in ascending order. The least
// chosen key is built from the top bit down, each bit by counting the keys that are at least as great,
// until the count fits (some 20 bits for scores that differ) or the key is complete.
template <int R>
__device__ __forceinline__ void choose(const uint64_t* key, const int* id, int n, int want, int* chosen, int* pages, int lane) {
  if (want == 0) return;
  uint64_t k[R], least = 0;
#pragma unroll
  for (int r = 0; r < R; r++) k[r] = 64 * r + lane < n ? key[64 * r + lane] : 0;  // (a key is never 0)
  bool fits = false;
  for (int bit = 63; bit >= 0 && !fits; bit--) {
    const uint64_t x = least | 1ull << bit;
    int count = 0;
#pragma unroll
    for (int r = 0; r < R; r++) count += (int)__popcll(__ballot(k[r] >= x));
    if (count >= want) least = x;
    fits = count == want;
  }
  int equals = 0;  // keys equal to `least` that are chosen
  if (!fits) {
    equals = want;
#pragma unroll
    for (int r = 0; r < R; r++) equals -= (int)__popcll(__ballot(k[r] > least));
  }
  const uint64_t below = (1ull << lane) - 1;
  int at = 0;
#pragma unroll
  for (int r = 0; r < R; r++) {
    const uint64_t eq = __ballot(k[r] == least);
    const bool take = k[r] > least || (k[r] == least && (fits || (int)__popcll(eq & below) < equals));
    const uint64_t all = __ballot(take);
    if (take) {
      const int to = at + (int)__popcll(all & below);
      chosen[to] = 64 * r + lane;
      pages[to] = id[64 * r + lane];
    }
    at += (int)__popcll(all);
    equals = max(0, equals - (int)__popcll(eq));
  }
}

template <bool F16, int D>
__global__ void __launch_bounds__(ST) select_kernel(SelectArgs A) {
  constexpr int LPP = D / 8, PPW = ST / LPP;  // lanes a page, pages at a time
  extern __shared__ __align__(16) uint64_t s_key[];  // [width]
  __shared__ double s_q[2][D];
  __shared__ uint32_t s_hist[256];
  __shared__ uint32_t s_sel[2];    // the digit chosen, keys still wanted in it
  __shared__ uint32_t s_cnt[2][ST / 64];
  __shared__ int s_id[ST];  // (of up to ST pages)
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int len = own_rows(A.lens, b, A.len_add, A.width, A.lp), used = (len + (1 << A.lp) - 1) >> A.lp;
  const int* table = A.tables + (size_t)b * A.t_sb;
  int* chosen = A.chosen + ((size_t)b * A.hkv + h) * A.top;
  int* pages = A.pages + ((size_t)b * A.hkv + h) * A.top;
  const int count = min(used, A.top), n = used - 1;  // n: pages with a score
  if (tid < A.own_tiles) A.tickets[((size_t)b * A.hkv + h) * A.own_tiles + tid] = 0;
  if (h == 0 && tid == 0) A.sub_lens[b] = count == 0 ? 0 : ((count - 1) << A.lp) + ((len - 1) & ((1 << A.lp) - 1)) + 1;
  for (int i = count + tid; i < A.top; i += ST) chosen[i] = -1, pages[i] = -1;
  if (used <= A.top) {
    for (int i = tid; i < used; i += ST) chosen[i] = i, pages[i] = table[i];
    return;
  }
  // (the first ids are asked for before the queries, whose sums need a barrier)
  int id[4];
#pragma unroll
  for (int u = 0; u < 4; u++) id[u] = *(gint*)(table + min(tid / LPP + PPW * u, n - 1));
  const int last = *(gint*)(table + n);
  if (tid < D) {
    double pos = 0.0, neg = 0.0;
    for (int g = 0; g < A.g; g++) {
      const float x = to_f32<F16>(*(gu16*)(A.q + (size_t)b * A.q_sb + (size_t)(h * A.g + g) * A.q_sh + tid));
      if (x > 0.f) pos += x; else neg += x;  // (not a number: in neg, and so in every score)
    }
    s_q[0][tid] = neg;
    s_q[1][tid] = pos;
  }
  __syncthreads();
  {
    const int c = tid % LPP;
    double ql[8], qh[8];
#pragma unroll
    for (int i = 0; i < 8; i++) ql[i] = s_q[0][8 * c + i], qh[i] = s_q[1][8 * c + i];
    // four pages at a time: their ids, then their bounds, are in flight together
    for (int p0 = tid / LPP; p0 < n; p0 += 4 * PPW) {
      if (p0 >= 4 * PPW)
#pragma unroll
        for (int u = 0; u < 4; u++) id[u] = *(gint*)(table + min(p0 + PPW * u, n - 1));
      u32x4 lo[4], hi[4];
#pragma unroll
      for (int u = 0; u < 4; u++) {
        const int at = id[u] >= 0 && id[u] < A.num_pages ? id[u] : 0;
        const uint16_t* bd = A.bounds + ((size_t)at * A.hkv + h) * 2 * D + 8 * c;
        lo[u] = *(gu32x4*)bd;
        hi[u] = *(gu32x4*)(bd + D);
      }
#pragma unroll
      for (int u = 0; u < 4; u++) {
        float lf[8], hf[8];
        to_f32x8<F16>(lo[u], lf);
        to_f32x8<F16>(hi[u], hf);
        double x = 0.0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          x = fma((double)lf[i], ql[i], x);
          x = fma((double)hf[i], qh[i], x);
        }
        x += dpp64<0xB1>(x);
        x += dpp64<0x4E>(x);
        x += dpp64<0x141>(x);
        if (LPP == 16) x += dpp64<0x140>(x);
        // (a page outside the pool is chosen: its sequence's outputs are then not numbers)
        if (id[u] < 0 || id[u] >= A.num_pages) x = INFINITY;
        if (c == 0 && p0 + PPW * u < n) {
          s_key[p0 + PPW * u] = order_key(x);
          if (n <= ST) s_id[p0 + PPW * u] = id[u];
        }
      }
    }
  }
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
  if (n <= ST) {
    if (wv > 0) return;
    if (n <= 256)
      choose<4>(s_key, s_id, n, A.top - 1, chosen, pages, lane);
    else
      choose<ST / 64>(s_key, s_id, n, A.top - 1, chosen, pages, lane);
    if (lane == 0) chosen[A.top - 1] = n, pages[A.top - 1] = last;
    return;
  }
  // ---- the want-th greatest of used - 1 keys, 8 bits at a time from the top
  uint32_t want = A.top - 1;
  uint64_t prefix = 0, mask = 0;
  if (want > 0) {
    for (int shift = 56; shift >= 0; shift -= 8) {
      if (tid < 256) s_hist[tid] = 0;
      __syncthreads();
      for (int i = tid; i < n; i += ST) {
        const uint64_t k = s_key[i];
        if ((k & mask) == prefix) atomicAdd(&s_hist[(k >> shift) & 255], 1u);
      }
      __syncthreads();
      if (wv == 0) {
        // lane: digits 255 - 4 lane .. 252 - 4 lane, from the greatest down
        uint32_t c4[4], sum = 0;
#pragma unroll
        for (int i = 0; i < 4; i++) sum += c4[i] = s_hist[255 - 4 * lane - i];
        uint32_t before = sum;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
          const uint32_t y = __shfl_up(before, off, 64);
          if (lane >= off) before += y;
        }
        before -= sum;  // keys with a greater digit than this lane's
        if (before < want && before + sum >= want) {
          uint32_t at = before;
          int i = 0;
          while (at + c4[i] < want) at += c4[i++];
          s_sel[0] = 255 - 4 * lane - i;
          s_sel[1] = want - at;
        }
      }
      __syncthreads();
      prefix |= (uint64_t)s_sel[0] << shift;
      mask |= 255ull << shift;
      want = s_sel[1];
    }
  }
  // ---- keys above the last chosen one, and the first `want` of its equals, in ascending order
  uint32_t eq0 = 0, out0 = 0;
  for (int i0 = 0; i0 < n && A.top > 1; i0 += ST) {
    const int i = i0 + tid;
    const uint64_t k = i < n ? s_key[i] : 0;
    const bool gt = i < n && k > prefix, eq = i < n && k == prefix;
    const uint64_t be = __ballot(eq), bg = __ballot(gt);
    if (lane == 0) s_cnt[0][wv] = __popcll(be), s_cnt[1][wv] = __popcll(bg);
    __syncthreads();
    uint32_t e = eq0, g = 0, all_e = 0, all_g = 0;
    for (int w = 0; w < ST / 64; w++) {
      if (w < wv) e += s_cnt[0][w], g += s_cnt[1][w];
      all_e += s_cnt[0][w];
      all_g += s_cnt[1][w];
    }
    e += __popcll(be & below);
    g += __popcll(bg & below);
    // of the equals before this one, at most `want` were chosen
    if (gt || (eq && e < want)) {
      const uint32_t at = out0 + g + (min(e, want) - min(eq0, want));
      chosen[at] = i;
      pages[at] = table[i];
    }
    out0 += all_g + min(eq0 + all_e, want) - min(eq0, want);
    eq0 += all_e;
    __syncthreads();
  }
  if (tid == 0) chosen[A.top - 1] = n, pages[A.top - 1] = last;
}

// ------------------------------------------------------------------ launches
static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static bool pool_ok(const MqPagePool* p, bool need_bounds) {
  if (!p || !p->k || !p->v || (need_bounds && !p->bounds)) return false;
  if (!aligned16(p->k) || !aligned16(p->v) || !aligned16(p->bounds)) return false;
  if (p->num_layers < 1 || p->num_layers > 65535 || p->num_pages < 1 || p->num_kv_heads < 1 || p->num_kv_heads > 1024)
    return false;
  if (p->page_size < 16 || p->page_size > 256 || (p->page_size & (p->page_size - 1))) return false;
  return (p->head_dim == 64 || p->head_dim == 128) && (p->dtype == MQ_BF16 || p->dtype == MQ_FP16);
}
static bool ids_ok(const int* ids, int n, int num_pages) {
  for (int i = 0; i < n; i++)
    if (ids[i] < 0 || ids[i] >= num_pages) return false;
  return true;
}
constexpr int MAX_KEYS = 1 << 30;  // (sums of lengths stay in 32 bits)
static int log2_of(int x) { return __builtin_ctz((unsigned)x); }

template <int N>
static void copy_launch(const MqPagePool& P, const int* src, const int* dst, int n, hipStream_t stream) {
  CopyArgs<N> A;
  A.base[0] = P.k; A.base[1] = P.v; A.base[2] = P.bounds;
  A.page_bytes = (uint32_t)P.num_kv_heads * P.page_size * P.head_dim * 2;
  A.bounds_bytes = (uint32_t)P.num_kv_heads * 2 * P.head_dim * 2;
  A.per_page = (A.page_bytes + CB - 1) / CB;
  A.num_pages = P.num_pages;
  for (int i = 0; i < n; i++) A.ids[i] = make_int2(src[i], dst[i]);
  const uint32_t parts = 2 * A.per_page + (P.bounds ? (A.bounds_bytes + CB - 1) / CB : 0);
  copy_kernel<N><<<dim3(parts, n, P.num_layers), CT, 0, stream>>>(A);
}

template <int N, bool IN>
static void move_launch(const MqPagePool& P, const int* pages, int n, int first, int length, const void* kc, const void* vc,
                        int max_seq, hipStream_t stream) {
  MoveArgs<N> A;
  A.k = static_cast<uint16_t*>(P.k); A.v = static_cast<uint16_t*>(P.v); A.bounds = static_cast<uint16_t*>(P.bounds);
  A.kc = static_cast<uint16_t*>(const_cast<void*>(kc)); A.vc = static_cast<uint16_t*>(const_cast<void*>(vc));
  A.num_pages = P.num_pages; A.hkv = P.num_kv_heads; A.page = P.page_size; A.d = P.head_dim;
  A.max_seq = max_seq; A.first = first; A.length = length;
  memcpy(A.ids, pages, sizeof(int) * n);
  const dim3 grid(P.num_kv_heads, n, P.num_layers);
  if (P.dtype == MQ_FP16)
    move_kernel<N, IN, true><<<grid, CT, 0, stream>>>(A);
  else
    move_kernel<N, IN, false><<<grid, CT, 0, stream>>>(A);
}

// Both directions between a contiguous cache and pages, LIST_LONG pages a launch.
template <bool IN>
static int move(const MqPagePool* P, const int* pages, int length, const void* kc, const void* vc, int max_seq,
                hipStream_t stream) {
  if (!pool_ok(P, false) || !pages || !kc || !vc || !aligned16(kc) || !aligned16(vc) || length < 1 ||
      length > MAX_KEYS || max_seq < length)
    return MQ_ERR_ARG;
  const int n = (length + P->page_size - 1) / P->page_size;
  if (!ids_ok(pages, n, P->num_pages)) return MQ_ERR_ARG;
  (void)hipGetLastError();  // clear an error left by an unrelated earlier call
  for (int i = 0; i < n; i += LIST_LONG) {
    const int m = n - i < LIST_LONG ? n - i : LIST_LONG, first = i * P->page_size;
    if (m <= LIST_SHORT)
      move_launch<LIST_SHORT, IN>(*P, pages + i, m, first, length, kc, vc, max_seq, stream);
    else
      move_launch<LIST_LONG, IN>(*P, pages + i, m, first, length, kc, vc, max_seq, stream);
    if (hipGetLastError() != hipSuccess) return MQ_ERR_HIP;
  }
  return MQ_OK;
}

int append_rows(const AppendArgs& A, bool f16, hipStream_t stream) {
  if (f16)
    append_kernel<true><<<A.batch, CT, 0, stream>>>(A);
  else
    append_kernel<false><<<A.batch, CT, 0, stream>>>(A);
  return hipGetLastError() == hipSuccess ? MQ_OK : MQ_ERR_HIP;
}

// How an attention call is split. Query rows of the prefix go in tiles of up to 128, so that its keys are read
// as few times as there are tiles; of 64 while there are at most 1024 steps of 128 rows by 64 keys, four a CU: a step
// then takes half as long, and what a workgroup does one behind the other is what bounds such calls (64 sequences behind
// 2000 rows with up to 64 own 14.5 us against 17.7, 23 behind 1117 with 5 queries a kv head 8.2 against 9.5; the other
// way from some 2000 steps on: 128 behind 8192 with up to 500 own 40.8 against 45.8 with tiles of 64, 256 behind 15001
// with up to 1024 110 against 130). A sequence's own rows are shared by its G query heads a kv head only, in
// tiles of 16. Keys are split until the launch has about two workgroups a CU, in parts of at least 128 keys, of 256 where
// there would be more than 32 (one sequence with 8192 own rows 12.3 us in 32 parts, 13.7 in 64; with 30000 15.9 in 64 and
// 17.9 in 32, at two kv heads).
// Each part's result is another 4 D + 8 bytes a query row written and read, so a prefix takes fewer parts where those
// cost nothing (us a captured call):
// - tiles of more than 16 rows beside own rows as many as end about when these do, at 1.8 us for 64 keys of a tile and
//   5.4 TB/s for half of the longest own length a sequence (64 sequences behind 8192 rows with up to 2000 own: 60 against
//   74 with no such limit; 256 behind 15001 with up to 1024: 113 against 138; at 1.45 us, an alone tile's time, 68 and 120);
// - of a prefix of few steps, at most 16 each, 192 workgroups, since what a part costs before and after its steps is
//   several of them (64 behind 8192 with up to 200 own: 24 against 28; 20 behind 15000 with up to 500: 22 against 26), and
//   so for tiles of 16 rows at any length (8 sequences behind 8192 13.5 against 18.3, behind 30000 26.8 against 28.3).
//
// Short contexts of few sequences take one launch instead (JOINED), whose workgroups go over prefix and own rows alike:
// up to 640 keys the two cost the GPU the same (4 sequences behind 512 rows 7.3 us in two launches, 7.6 in one; 32
// sequences 9.3 and 9.1), past them one workgroup's walk is the longer one (1000 keys 8.1 and 12.7), and a
// launch costs the host 3 us (that call 17.4 us, 14.1 in one launch).
constexpr int JOINED_KEYS = 640;
// Own rows of more than 512 (sequence, kv head)s do not fit the chip at once as a workgroup each: short ones, up to 256
// keys, then take a wave each, which also saves joining four (256 sequences with up to 30 own rows 7.2 us against 15.9,
// behind 1984 rows 25.9 against 31.2; up to 200 rows 36.4 and 40.2; up to 400 55.5 against 52.1, so no more).
constexpr int PACK_KEYS = 256, PACK_OVER = 512;
// Without a prefix, up to 512 own rows stay one part, and the call one launch: 4 sequences with up to 200 rows 6.0 us
// against 7.6 in two parts, 400 rows 7.9 and 7.7, 600 9.4 and 7.9; 40 with up to 400 11.7 and 14.1.
constexpr int WHOLE_KEYS = 512;
AttnPlan plan_attention(int batch, int hkv, int g, int d, int prefix_len, int max_len) {
  AttnPlan p{};
  constexpr int WANT = 512, MANY = 32;
  constexpr long long HALF_TILES = 1024;
  constexpr double STEP_US = 1.8, SHORT_WANT = 192., SHORT_STEPS = 16.;
  const int rows = batch * g;
  p.own_tiles = (g + 15) / 16;
  if (prefix_len > 0 && max_len > 0 && prefix_len + max_len <= JOINED_KEYS && (long long)batch * hkv * p.own_tiles <= NUM_CUS) {
    p.form = JOINED;
    p.groups = batch;
    p.ns = 1;
    return p;
  }
  const long long steps128 = (long long)hkv * ((rows + 127) / 128) * ((prefix_len + TS - 1) / TS);
  p.form = rows <= 16 ? ROWS16 : rows <= 64 || steps128 <= HALF_TILES ? ROWS64 : ROWS128;
  auto parts = [&](int len, long long tiles, double want) {
    const int units = (len + UNIT - 1) / UNIT, most = units <= MANY ? units : units / 2 > MANY ? units / 2 : MANY;
    double n = ceil(want / (double)tiles);
    n = fmax(1., fmin(n, fmin(most, MAX_PARTS / 2)));
    const int ch = part_keys(len, (int)n);
    return (len + ch - 1) / ch;  // (as many as have a key)
  };
  if (prefix_len > 0) {
    p.prefix_tiles = (rows + tile_rows(p.form) - 1) / tile_rows(p.form);
    const long long tiles = (long long)hkv * p.prefix_tiles;
    double want = WANT;
    const double steps = (double)tiles * ((prefix_len + TS - 1) / TS), own_us = (double)batch * hkv * max_len * d * 2 / 5.4e6;
    if (p.form != ROWS16 && own_us > 0.) want = fmin(want, steps * STEP_US / own_us);
    if (p.form == ROWS16 || steps <= SHORT_STEPS * SHORT_WANT) want = fmin(want, SHORT_WANT);
    p.np = parts(prefix_len, tiles, want);
  }
  p.groups = batch;
  const long long own = (long long)batch * hkv * p.own_tiles;
  if (max_len > 0 && max_len <= PACK_KEYS && own > PACK_OVER) {
    p.groups = (batch + AW - 1) / AW;
    p.ns = 1;
  } else if (max_len > 0) {
    p.ns = prefix_len == 0 && max_len <= WHOLE_KEYS ? 1 : parts(max_len, own, WANT);
  }
  const size_t rows_all = p.np + p.ns == 1 ? 0 : (size_t)(p.np + p.ns) * batch * hkv * g;
  p.out_bytes = (rows_all * d * 4 + 255) / 256 * 256;
  p.bytes = p.out_bytes + (rows_all * 8 + 255) / 256 * 256;
  return p;
}

template <bool F16, int D>
static void attn_launch(const AttnArgs& A, int form, unsigned blocks, hipStream_t stream) {
  if (blocks > 0) {
    switch (form) {
      case ROWS16: attn_kernel<F16, D, ROWS16><<<blocks, 64 * AW, 0, stream>>>(A); break;
      case ROWS64: attn_kernel<F16, D, ROWS64><<<blocks, 64 * AW, 0, stream>>>(A); break;
      case JOINED: attn_kernel<F16, D, JOINED><<<blocks, 64 * AW, 0, stream>>>(A); break;
      case OWN: attn_kernel<F16, D, OWN><<<blocks, 64 * AW, 0, stream>>>(A); return;
      default: attn_kernel<F16, D, ROWS128><<<blocks, 64 * AW, 0, stream>>>(A); break;
    }
  }
  if (A.np + A.ns != 1) combine_kernel<F16, D><<<((unsigned)A.batch * A.hq + 3) / 4, 256, 0, stream>>>(A);
}

// The launches of an attention; A without its split and partial results, which come from `p` and
// `ws` (plan_attention's bytes).
int run_attention(AttnArgs A, const AttnPlan& p, int d, bool f16, void* ws, hipStream_t stream) {
  A.prefix_tiles = p.prefix_tiles; A.np = p.np; A.own_tiles = p.own_tiles; A.ns = p.ns; A.groups = p.groups;
  A.part_o = static_cast<float*>(ws);
  A.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + p.out_bytes);
  const long long blocks = (long long)A.hkv * ((long long)p.prefix_tiles * p.np + (long long)p.own_tiles * p.groups * p.ns);
  if (blocks > 0x7fffffff) return MQ_ERR_ARG;
  if (d == 128)
    f16 ? attn_launch<true, 128>(A, p.form, (unsigned)blocks, stream) : attn_launch<false, 128>(A, p.form, (unsigned)blocks, stream);
  else
    f16 ? attn_launch<true, 64>(A, p.form, (unsigned)blocks, stream) : attn_launch<false, 64>(A, p.form, (unsigned)blocks, stream);
  return hipGetLastError() == hipSuccess ? MQ_OK : MQ_ERR_HIP;
}

// (a call that needs none takes NULL)
static bool workspace_ok(const void* ws, size_t has, size_t needs) { return needs == 0 || (ws && aligned16(ws) && has >= needs); }

static bool rows_ok(const void* p, int64_t sb, int64_t sh) { return p && aligned16(p) && sb % 8 == 0 && sh % 8 == 0; }

// What both attentions ask of their common arguments.
static bool attn_ok(const MqPagePool* P, bool sparse, const void* q, int64_t q_sb, int64_t q_sh, const void* out, int64_t o_sb,
                    int64_t o_sh, int num_q_heads, int batch, const int* tables, int64_t t_sb, int width, const int* lens,
                    float scale) {
  return pool_ok(P, sparse) && rows_ok(q, q_sb, q_sh) && rows_ok(out, o_sb, o_sh) && batch >= 1 && batch <= 65535 &&
         num_q_heads >= P->num_kv_heads && num_q_heads <= 16384 && num_q_heads % P->num_kv_heads == 0 && tables && lens &&
         width >= 1 && width <= MQ_MAX_TABLE_WIDTH && t_sb >= 0 && scale > 0.f && isfinite(scale);
}

static AttnArgs attn_args(const MqPagePool& P, const void* q, int64_t q_sb, int64_t q_sh, void* out, int64_t o_sb,
                          int64_t o_sh, int num_q_heads, int batch, float scale) {
  AttnArgs A{};
  A.k = static_cast<const uint16_t*>(P.k); A.v = static_cast<const uint16_t*>(P.v);
  A.q = static_cast<const uint16_t*>(q); A.out = static_cast<uint16_t*>(out);
  A.q_sb = q_sb; A.q_sh = q_sh; A.o_sb = o_sb; A.o_sh = o_sh;
  A.num_pages = P.num_pages; A.hkv = P.num_kv_heads; A.hq = num_q_heads; A.g = num_q_heads / P.num_kv_heads;
  A.lp = log2_of(P.page_size); A.batch = batch;
  A.scale_log2 = scale * 1.44269504088896341f;
  return A;
}

int shared_attention(const MqPagePool* P, const void* q, int64_t q_sb, int64_t q_sh, void* out, int64_t o_sb, int64_t o_sh,
                     int num_q_heads, int batch, const int* prefix_pages, int prefix_len, const int* tables, int64_t t_sb,
                     int width, const int* lens, int len_add, int max_len, float scale, void* ws, size_t ws_bytes,
                     hipStream_t stream) {
  if (!attn_ok(P, false, q, q_sb, q_sh, out, o_sb, o_sh, num_q_heads, batch, tables, t_sb, width, lens, scale) ||
      prefix_len < 0 || prefix_len > MAX_KEYS || (prefix_len > 0 && !prefix_pages) || max_len < 0 || max_len > MAX_KEYS)
    return MQ_ERR_ARG;
  const AttnPlan p = plan_attention(batch, P->num_kv_heads, num_q_heads / P->num_kv_heads, P->head_dim, prefix_len, max_len);
  if (!workspace_ok(ws, ws_bytes, p.bytes)) return MQ_ERR_ARG;
  AttnArgs A = attn_args(*P, q, q_sb, q_sh, out, o_sb, o_sh, num_q_heads, batch, scale);
  A.prefix_pages = prefix_pages; A.prefix_len = prefix_len;
  A.tables = tables; A.t_sb = t_sb; A.width = width; A.lens = lens; A.len_add = len_add;
  return run_attention(A, p, P->head_dim, P->dtype == MQ_FP16, ws, stream);
}

// The chosen pages, the rows in them and the tickets, ahead of the attention's partial results in the workspace.
static size_t chosen_bytes(int batch, int hkv, int g, int top) {
  return ((size_t)batch * (hkv * ((size_t)top + (g + 15) / 16) + 1) * 4 + 255) / 256 * 256;
}

size_t sparse_workspace(int batch, int hkv, int g, int d, int top, int width, int page_size) {
  return chosen_bytes(batch, hkv, g, top) + plan_attention(batch, hkv, g, d, 0, (top < width ? top : width) * page_size).bytes;
}

int sparse_attention(const MqPagePool* P, const void* q, int64_t q_sb, int64_t q_sh, void* out, int64_t o_sb, int64_t o_sh,
                     int* chosen, int num_q_heads, int batch, const int* tables, int64_t t_sb, int width, const int* lens,
                     int len_add, int top, float scale, void* ws, size_t ws_bytes, hipStream_t stream) {
  if (!attn_ok(P, true, q, q_sb, q_sh, out, o_sb, o_sh, num_q_heads, batch, tables, t_sb, width, lens, scale) || !chosen ||
      top < 1 || top > MQ_MAX_TABLE_WIDTH)
    return MQ_ERR_ARG;
  const int most = top < width ? top : width, hkv = P->num_kv_heads, g = num_q_heads / hkv;
  AttnPlan p = plan_attention(batch, hkv, g, P->head_dim, 0, most * P->page_size);
  if (p.groups == batch) p.form = OWN;  // (else there is one part)
  const size_t head = chosen_bytes(batch, hkv, g, top);
  if (!workspace_ok(ws, ws_bytes, head + p.bytes)) return MQ_ERR_ARG;
  AttnArgs A = attn_args(*P, q, q_sb, q_sh, out, o_sb, o_sh, num_q_heads, batch, scale);
  SelectArgs S{};
  S.q = A.q; S.bounds = static_cast<const uint16_t*>(P->bounds);
  S.q_sb = q_sb; S.q_sh = q_sh; S.t_sb = t_sb; S.tables = tables; S.lens = lens;
  S.chosen = chosen; S.pages = static_cast<int*>(ws); S.sub_lens = S.pages + (size_t)batch * hkv * top;
  S.tickets = reinterpret_cast<uint32_t*>(S.sub_lens + batch); S.own_tiles = p.own_tiles;
  S.num_pages = P->num_pages; S.hkv = hkv; S.g = g; S.lp = A.lp; S.width = width; S.top = top; S.len_add = len_add;
  const dim3 grid(hkv, batch);
  const size_t keys = (size_t)width * 8;
  const bool f16 = P->dtype == MQ_FP16;
  if (P->head_dim == 128)
    f16 ? select_kernel<true, 128><<<grid, ST, keys, stream>>>(S) : select_kernel<false, 128><<<grid, ST, keys, stream>>>(S);
  else
    f16 ? select_kernel<true, 64><<<grid, ST, keys, stream>>>(S) : select_kernel<false, 64><<<grid, ST, keys, stream>>>(S);
  if (hipGetLastError() != hipSuccess) return MQ_ERR_HIP;
  A.tables = S.pages; A.t_sb = (int64_t)hkv * top; A.t_sh = top; A.width = top; A.lens = S.sub_lens;
  A.tickets = S.tickets;
  return run_attention(A, p, P->head_dim, f16, static_cast<char*>(ws) + head, stream);
}

}  // namespace pg
}  // namespace mq

using namespace mq;
using namespace mq::pg;

extern "C" int mq_pages_copy(const MqPagePool* pool, const int* src, const int* dst, int n, hipStream_t stream) {
  if (!pool_ok(pool, false) || n < 0 || (n > 0 && (!src || !dst))) return MQ_ERR_ARG;
  if (!ids_ok(src, n, pool->num_pages) || !ids_ok(dst, n, pool->num_pages)) return MQ_ERR_ARG;
  (void)hipGetLastError();  // clear an error left by an unrelated earlier call
  for (int i = 0; i < n; i += LIST_LONG) {
    const int m = n - i < LIST_LONG ? n - i : LIST_LONG;
    if (m <= LIST_SHORT)
      copy_launch<LIST_SHORT>(*pool, src + i, dst + i, m, stream);
    else
      copy_launch<LIST_LONG>(*pool, src + i, dst + i, m, stream);
    if (hipGetLastError() != hipSuccess) return MQ_ERR_HIP;
  }
  return MQ_OK;
}

extern "C" int mq_pages_load(const MqPagePool* pool, const int* pages, int length, const void* k_cache, const void* v_cache,
                             int max_seq_len, hipStream_t stream) {
  return mq::pg::move<true>(pool, pages, length, k_cache, v_cache, max_seq_len, stream);
}

extern "C" int mq_pages_store(const MqPagePool* pool, const int* pages, int length, void* k_cache, void* v_cache,
                              int max_seq_len, hipStream_t stream) {
  return mq::pg::move<false>(pool, pages, length, k_cache, v_cache, max_seq_len, stream);
}

extern "C" int mq_pages_append(const MqPagePool* pool, const void* k, const void* v, long long k_sb, long long k_sh,
                               long long v_sb, long long v_sh, const int* tables, long long table_stride, int width,
                               const int* lens, int batch, hipStream_t stream) {
  if (!pool_ok(pool, false) || pool->num_layers != 1 || !rows_ok(k, k_sb, k_sh) || !rows_ok(v, v_sb, v_sh) || !tables ||
      table_stride < 0 || width < 1 || width > MQ_MAX_TABLE_WIDTH || !lens || batch < 1 || batch > 65535)
    return MQ_ERR_ARG;
  AppendArgs A{};
  A.k = static_cast<uint16_t*>(pool->k); A.v = static_cast<uint16_t*>(pool->v); A.bounds = static_cast<uint16_t*>(pool->bounds);
  A.kr = static_cast<const uint16_t*>(k); A.vr = static_cast<const uint16_t*>(v);
  A.k_sb = k_sb; A.k_sh = k_sh; A.v_sb = v_sb; A.v_sh = v_sh; A.tables = tables; A.lens = lens; A.t_sb = table_stride;
  A.num_pages = pool->num_pages; A.hkv = pool->num_kv_heads; A.lp = log2_of(pool->page_size); A.d = pool->head_dim;
  A.width = width; A.batch = batch;
  (void)hipGetLastError();  // clear an error left by an unrelated earlier call
  return append_rows(A, pool->dtype == MQ_FP16, stream);
}

extern "C" int mq_attention_workspace(const MqPagePool* pool, int num_q_heads, int batch, int prefix_len, int max_len, int top,
                                      size_t* bytes) {
  if (!pool || !bytes || pool->num_kv_heads < 1 || num_q_heads < pool->num_kv_heads || num_q_heads > 16384 ||
      num_q_heads % pool->num_kv_heads || batch < 1 || batch > 65535 || prefix_len < 0 || prefix_len > MAX_KEYS || max_len < 0 ||
      max_len > MAX_KEYS || top < 0 || top > MQ_MAX_TABLE_WIDTH)
    return MQ_ERR_ARG;
  *bytes = plan_attention(batch, pool->num_kv_heads, num_q_heads / pool->num_kv_heads, pool->head_dim, prefix_len, max_len).bytes +
           (top > 0 ? chosen_bytes(batch, pool->num_kv_heads, num_q_heads / pool->num_kv_heads, top) : 0);
  return MQ_OK;
}

extern "C" int mq_shared_prefix_attention(const MqPagePool* pool, const void* q, long long q_sb, long long q_sh, void* out,
                                          long long o_sb, long long o_sh, int num_q_heads, int batch, const int* prefix_pages,
                                          int prefix_len, const int* tables, long long table_stride, int width,
                                          const int* lens, int max_len, float scale, void* workspace,
                                          size_t workspace_bytes, hipStream_t stream) {
  (void)hipGetLastError();  // clear an error left by an unrelated earlier call
  return shared_attention(pool, q, q_sb, q_sh, out, o_sb, o_sh, num_q_heads, batch, prefix_pages, prefix_len, tables,
                          table_stride, width, lens, 0, max_len, scale, workspace, workspace_bytes, stream);
}

extern "C" int mq_sparse_attention(const MqPagePool* pool, const void* q, long long q_sb, long long q_sh, void* out,
                                   long long o_sb, long long o_sh, int* chosen, int num_q_heads, int batch,
                                   const int* tables, long long table_stride, int width, const int* lens, int top,
                                   float scale, void* workspace, size_t workspace_bytes, hipStream_t stream) {
  (void)hipGetLastError();  // clear an error left by an unrelated earlier call
  return sparse_attention(pool, q, q_sb, q_sh, out, o_sb, o_sh, chosen, num_q_heads, batch, tables, table_stride, width, lens, 0,
                          top, scale, workspace, workspace_bytes, stream);
}
