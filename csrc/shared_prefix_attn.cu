// Decode attention of rows that share a prefix (the samples of one prompt).
//
//   o[b,h] = sum_t softmax_t(scale * q[b,h] . k[t]) v[t]
//
// over row b's keys, of which the first P are the same for every row of its group.
// The keys [0, P) of a group are read once for all of its rows: their queries form
// the M side of a matrix product.  Keys [P, L_b) are read per row.  Both kinds of work
// are units of 64- or 128-key tiles:
//
//   prefix unit: MR query rows (row, head of one KV head) x the group's prefix
//   suffix unit: the G query heads of one KV head of one row x the row's own keys
//
// spread over the CTAs by a plan: the tiles of all (prefix unit, KV head) are laid on one
// line, those of all (suffix unit, KV head) on another, and each line is cut into equal
// runs, one per CTA.  So every CTA has the same share of both kinds, ragged lengths
// balance, and a long prefix is split over many CTAs.  Each CTA leaves, per unit it
// touched, the fp32 partial (max, sum, unnormalised output) of an online softmax in
// base 2; the combine kernel joins a row's partials in the order of its keys.  No
// atomics: the result does not depend on timing.
//
// shared_prefix_plan_kernel     group bounds, unit list, tile offsets, every CTA's first units
// shared_prefix_tc_kernel       bf16 cache, 128 dims, pages of a multiple of 8 keys: tcgen05
// shared_prefix_attn_kernel     32, 64 and 128 dims, bf16 and e4m3, any page: mma.sync
// shared_prefix_combine_kernel  one warp per (row, head)
//
// The plan depends on the lengths only: one plan serves all layers of a decode step.
#include "tc_common.cuh"

#include <cfloat>

namespace rlb {
namespace sp {

using namespace rlb::tc;
typedef __nv_bfloat16 bf16;

constexpr int BT = 64;        // a prefix is shared in multiples of these
constexpr int MR = 64;        // query rows of a prefix unit
constexpr int kMaxHeads = 64; // query heads per KV head
constexpr int kUnitInts = 8;  // first tile, tiles, first key, keys' end, table row, first row, first query row, query rows
constexpr int kRowInts = 4;   // group's first unit (-1: none), group's first row, whether the row has keys
constexpr int kStart = 1;     // what the start and end of a unit count for on the line, in tiles
constexpr int kHeader = 8;    // prefix: tiles per CTA, tiles in all; suffix: the same

__device__ int g_shared_prefix_error = 0;
constexpr int kErrLengths = 1, kErrPage = 2, kErrWait = 3;  // error words

// What differs between the plans of the two kernels: CTAs, keys per tile.
struct Shape {
  int ctas, tile;
};
// keys per tile of the general kernel; both sides measured there
__host__ __device__ constexpr int general_tile(int hd, bool f8) { return hd <= 64 && !f8 ? 128 : 64; }
// The rule between the two kernels; both sides measured beside shared_prefix_attn_kernel.
bool use_tc(int64_t hd, int64_t block, bool f8) { return hd == 128 && !f8 && block % 8 == 0; }
Shape shape_of(int64_t hd, int64_t block, bool f8) {
  return use_tc(hd, block, f8) ? Shape{num_sms(), 128} : Shape{2 * num_sms(), general_tile((int)hd, f8)};
}

// where the units start in a plan
__host__ __device__ inline int unit_offset(int ctas) { return kHeader + (2 * ctas + 3) / 4 * 4; }
__host__ __device__ inline int max_chunks(int B, int G, int Gq) { return G + (B * Gq + MR - 1) / MR; }

// ------------------------------------------------------------------------- plan
// One block, bound by latency: its loads, three scans and a search per CTA take 4.5 us (8 rows) to 6.0 us (256
// rows).  With 512 threads 4.6 and 6.1 us; up to 256 rows a scan is one pass either way.
constexpr int kPlanThreads = 256;

// inclusive scan of one value per thread, none below 0 (sum, or running maximum)
template <bool MAX, typename T>
__device__ __forceinline__ T block_scan(T v, T* s_warp) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const T u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = MAX ? max(v, u) : v + u;
  }
  __syncthreads();
  if (lane == 31) s_warp[w] = v;
  __syncthreads();
  // joined over the warps before, by every warp for itself
  constexpr int W = kPlanThreads / 32;
  T u = lane < w ? s_warp[lane] : (T)0;
#pragma unroll
  for (int o = 1; o < W; o <<= 1) {
    const T x = __shfl_xor_sync(0xffffffffu, u, o);
    u = MAX ? max(u, x) : u + x;
  }
  u = __shfl_sync(0xffffffffu, u, 0);
  return MAX ? max(u, v) : u + v;
}

// last entry of the ascending a[0..n) that is at most x
__device__ __forceinline__ int last_at_most(const int* a, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid + 1;
    else hi = mid;
  }
  return lo - 1;
}

// plan: [kHeader][first prefix unit of each CTA][first suffix unit of each CTA][units x kUnitInts][rows x kRowInts]
__global__ void __launch_bounds__(kPlanThreads)
shared_prefix_plan_kernel(const int* __restrict__ group_starts, const int* __restrict__ prefix_lens,
                          const int* __restrict__ seq_lens, int G, int B, int Gq, int nkv, int ctas, int tile,
                          int capacity, int* __restrict__ plan) {
  extern __shared__ int s_mem[];
  __shared__ int s_warp[32];
  __shared__ long long s_warp2[32];
  pdl_launch_dependents();
  int* s_len = s_mem;            // [B]
  int* s_start = s_len + B;      // [G + 1]
  int* s_share = s_start + G + 1;  // [G] prefix length, then shared keys
  int* s_leader = s_share + G;   // [G] a row whose table is read
  int* s_unit0 = s_leader + G;   // [G]
  int* s_first = s_unit0 + G;    // [units]
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nc_max = max_chunks(B, G, Gq), units = nc_max + B;
  int* cta_unit = plan + kHeader;
  int* unit = plan + unit_offset(ctas);
  int* rowinfo = unit + units * kUnitInts;
  // lengths are kept inside the block tables, and so short that no place on a line leaves 31 bits
  const int longest = (int)min((long long)capacity, (long long)max((1 << 30) / (nkv * units), 1) * BT);
  bool bad = false;
  // the first of each array at once: one wait for memory instead of three
  const int len0 = tid < B ? seq_lens[tid] : 0, share0 = tid < G ? prefix_lens[tid] : 0;
  const int start0 = tid <= G ? group_starts[tid] : 0;
  for (int b = tid; b < B; b += kPlanThreads) {
    const int len = max(b == tid ? len0 : seq_lens[b], 0);
    bad |= len > longest;
    s_len[b] = min(len, longest);
  }
  for (int g = tid; g < G; g += kPlanThreads) s_share[g] = max(g == tid ? share0 : prefix_lens[g], 0);
  // group starts, made ascending and kept inside [0, B]: groups never overlap
  int carry = 0;
  for (int g0 = 0; g0 <= G; g0 += kPlanThreads) {
    const int g = g0 + tid;
    const int raw = g0 == 0 ? start0 : g <= G ? group_starts[g] : 0;
    const int v = block_scan<true>(max(carry, min(max(raw, 0), B)), s_warp);
    if (g <= G) {
      s_start[g] = v;
      bad |= v != raw;
    }
    __syncthreads();
    carry = s_start[min(G, g0 + kPlanThreads - 1)];
  }
  if (bad) atomicExch(&g_shared_prefix_error, kErrLengths);
  // a group shares what every live row of it has, in multiples of BT; one live row shares nothing
  for (int g = warp; g < G; g += kPlanThreads / 32) {
    int len = s_share[g], live = 0, leader = B;
    for (int b = s_start[g] + lane; b < s_start[g + 1]; b += 32) {
      const int L = s_len[b];
      if (L > 0) {
        len = min(len, L);
        leader = min(leader, b);
        ++live;
      }
    }
    len = __reduce_min_sync(0xffffffffu, len);
    leader = __reduce_min_sync(0xffffffffu, leader);
    live = __reduce_add_sync(0xffffffffu, live);
    if (lane == 0) {
      s_share[g] = live > 1 ? len / BT * BT : 0;
      s_leader[g] = leader;
    }
  }
  __syncthreads();
  // prefix units: per group, ceil(rows * Gq / MR) chunks of its query rows
  int unit_carry = 0, prefix_places = 0;
  for (int g0 = 0; g0 < G; g0 += kPlanThreads) {
    const int g = g0 + tid;
    int chunks = 0, n = 0, start = 0, rows = 0;
    if (g < G) {
      start = s_start[g];
      rows = (s_start[g + 1] - start) * Gq;
      n = (s_share[g] + tile - 1) / tile;
      chunks = n > 0 ? (rows + MR - 1) / MR : 0;
    }
    // both sums in one scan: units in the high half, places on the line in the low one
    const int places = n + kStart;
    const long long end = block_scan<false>(((long long)chunks << 32) + chunks * places, s_warp2);
    const int u0 = unit_carry + (int)(end >> 32) - chunks, a0 = prefix_places + (int)end - chunks * places;
    if (g < G) s_unit0[g] = u0;
    for (int c = 0; c < chunks; ++c) {
      int4* m = reinterpret_cast<int4*>(unit + (u0 + c) * kUnitInts);
      s_first[u0 + c] = a0 + c * places;
      m[0] = make_int4(a0 + c * places, n, 0, s_share[g]);
      m[1] = make_int4(s_leader[g], start, c * MR, min(MR, rows - c * MR));
    }
    __syncthreads();
    if (tid == kPlanThreads - 1) s_warp2[0] = end;
    __syncthreads();
    unit_carry += (int)(s_warp2[0] >> 32);
    prefix_places += (int)s_warp2[0];
    __syncthreads();
  }
  for (int u = unit_carry + tid; u < nc_max; u += kPlanThreads) {  // unused prefix units
    s_first[u] = prefix_places;
    *reinterpret_cast<int4*>(unit + u * kUnitInts) = make_int4(prefix_places, 0, 0, 0);
  }
  // suffix units: row b's keys behind its group's shared ones
  int suffix_places = 0;
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int k0 = 0, k1 = 0, u0 = -1, start = 0;
    if (b < B) {
      k1 = s_len[b];
      const int g = last_at_most(s_start, G, b);
      if (g >= 0 && b < s_start[g + 1] && s_share[g] > 0) {
        k0 = min(s_share[g], k1);
        u0 = s_unit0[g];
        start = s_start[g];
      }
    }
    const int n = (k1 - k0 + tile - 1) / tile;
    const int places = n > 0 ? n + kStart : 0;
    const int end = block_scan<false>(places, s_warp);
    if (b < B) {
      int4* m = reinterpret_cast<int4*>(unit + (nc_max + b) * kUnitInts);
      const int a0 = suffix_places + end - places;
      s_first[nc_max + b] = a0;
      m[0] = make_int4(a0, n, k0, k1);
      m[1] = make_int4(b, b, 0, Gq);
      *reinterpret_cast<int4*>(rowinfo + b * kRowInts) = make_int4(u0, start, k1 > 0, 0);
    }
    __syncthreads();
    if (tid == kPlanThreads - 1) s_warp[0] = end;
    __syncthreads();
    suffix_places += s_warp[0];
    __syncthreads();
  }
  const long long total0 = (long long)prefix_places * nkv, total1 = (long long)suffix_places * nkv;
  const int per0 = max((int)((total0 + ctas - 1) / ctas), 1), per1 = max((int)((total1 + ctas - 1) / ctas), 1);
  if (tid == 0) *reinterpret_cast<int4*>(plan) = make_int4(per0, (int)total0, per1, (int)total1);
  // every CTA's first unit of each line: the last one that starts at or before its first tile
  // (units without tiles start where the next one does, so this one has tiles)
  for (int i = tid; i < 2 * ctas; i += kPlanThreads) {
    const bool suffix = i >= ctas;
    const long long x = (long long)(suffix ? i - ctas : i) * (suffix ? per1 : per0);
    int u = 0;
    if (x < (suffix ? total1 : total0))
      u = suffix ? nc_max + last_at_most(s_first + nc_max, B, (int)x / nkv) : last_at_most(s_first, nc_max, (int)x / nkv);
    cta_unit[i] = u;
  }
}

// --------------------------------------------------------------------- attention
// One lane of a converged warp.  The compiler knows this form: what the lane issues takes its operands
// from uniform registers, where a plain "lane == 0" costs a move of each through a per-lane loop (measured: 50
// to 75 cycles a matrix product of 16 to 64 columns, against 103).
__device__ __forceinline__ bool elect_one() {
  uint32_t x;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(x));
  return x != 0;
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const void* tmap, uint32_t mbar, int head, int key, int span) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n" ::"r"(
          dst),
      "l"(tmap), "r"(mbar), "r"(0), "r"(head), "r"(key), "r"(span)
      : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_arrive(uint32_t mbar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];\n" ::"r"(mbar) : "memory");
}
__device__ __forceinline__ void ldsm_x4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm_x4_t(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <bool F16>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// two e4m3 values (low 16 bits) as f16x2: exact
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t x) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(x & 0xffffu), __NV_E4M3);
  return (uint32_t)h.x | ((uint32_t)h.y << 16);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void consumers_sync() { asm volatile("bar.sync 1, 128;\n" ::: "memory"); }

// a stage of KT keys in shared memory
template <int HD, bool F8, int KT>
struct Tile {
  static constexpr int KEYS = KT;
  static constexpr int RB = HD * (F8 ? 1 : 2);              // bytes of a key
  static constexpr int BOXB = RB < 128 ? RB : 128;          // bytes of a key in one box = its swizzle span
  static constexpr int NBOX = RB / BOXB;
  static_assert(NBOX <= 2, "at most 256 bytes a key");
  static constexpr int CH = BOXB / 16;                      // 16-byte chunks of a box row
  static constexpr int BYTES = KT * RB;                     // of K (or V)
  // offset of chunk c of a key, as the TMA unit's swizzle (span BOXB) places it
  static __device__ __forceinline__ int at(int row, int c) {
    const int box = c / CH, cc = c % CH;
    const int x = CH == 8 ? (row & 7) : CH == 4 ? ((row >> 1) & 3) : ((row >> 2) & 1);
    return box * KT * BOXB + (row * CH + (cc ^ x)) * 16;
  }
};

template <int HD>
constexpr int kRedBytes = 2 * (HD / 4 + 2) * 32 * 4;  // merge buffer: two warps, half of their rows

struct Args {
  const bf16* q;
  long long q_row, q_head;  // strides
  const uint8_t *k, *v;     // caches (the path without TMA)
  const int* tables;
  int table_row, n_blocks, block, box;  // table width, pages, keys per page, keys per TMA box of a tile (0: no TMA)
  const int* plan;
  int ctas, units, B, nq, nkv, Gq;
  uint32_t inv_gq;  // ceil(2^32 / Gq): rr / Gq is the high word of rr * inv_gq for every query row rr of a group
  float scale_log2;
  float *part_o, *part_ml;
};

// a CTA's run on one of the two lines of tiles, and the position in it
struct Cursor {
  const int* unit;
  int u, u_end, kvh, j;               // unit, KV head, tile
  int n, k0, k1, trow, row0, r0, rn;  // of the unit
  int x, x1, nkv;                     // position, end of the run
  __device__ __forceinline__ void load() {
    const int4 a = *reinterpret_cast<const int4*>(unit + u * kUnitInts);
    const int4 b = *reinterpret_cast<const int4*>(unit + u * kUnitInts + 4);
    n = a.y, k0 = a.z, k1 = a.w, trow = b.x, row0 = b.y, r0 = b.z, rn = b.w;
  }
  // line 0: prefix units, line 1: suffix units; false when the CTA has no tile of it
  __device__ __forceinline__ bool begin(const Args& a, int line) {
    const int per = a.plan[2 * line], total = a.plan[2 * line + 1];
    nkv = a.nkv;
    x = (int)min((long long)total, (long long)blockIdx.x * per);
    x1 = min(total, x + per);
    if (x >= x1) return false;
    unit = a.plan + unit_offset(a.ctas);
    u_end = line ? a.units : a.units - a.B;
    u = a.plan[kHeader + line * a.ctas + blockIdx.x];
    load();
    const int y = x - unit[u * kUnitInts] * nkv;
    kvh = y / (n + kStart);
    j = y - kvh * (n + kStart) - kStart;
    if (j < 0) {  // the run begins in the unit's starting places: at its first tile, if that is in the run
      x -= j;
      j = 0;
    }
    return x < x1;
  }
  // to the next tile; true when it belongs to the same segment (unit, KV head and run)
  __device__ __forceinline__ bool next() {
    ++x;
    if (++j < n) return x < x1;
    j = 0;
    x += kStart;
    if (++kvh < nkv || x >= x1) return false;
    kvh = 0;
    do {
      if (++u >= u_end) return false;
      load();
    } while (n == 0);
    return false;
  }
  __device__ __forceinline__ bool done() const { return x >= x1; }
};

// Where the partial of local query row rl of a segment goes: a slot of the row when the segment is its
// unit's first, else a slot of the CTA.  sub: the tc kernel keeps two partials of a segment, of its
// even and of its odd tiles.
__device__ __forceinline__ long long partial_slot(const Args& a, const Cursor& s, int line, int sub, int rl) {
  const int nqt = a.B * a.nq, ls = 2 * line + sub;
  if (s.j > 0) return 4LL * nqt + ((long long)ls * a.ctas + blockIdx.x) * MR + rl;
  const int r = s.r0 + rl;
  return (long long)ls * nqt + (long long)(s.row0 + r / a.Gq) * a.nq + s.kvh * a.Gq + r % a.Gq;
}

// the pages of a unit, 32 table entries at a time, one per lane of the producer warp
struct Pages {
  int page0 = 0, ids = 0;
  bool fresh = true;
  // all lanes: the page of table entry p of row trow
  __device__ __forceinline__ int get(const Args& a, int trow, int p) {
    const int lane = threadIdx.x & 31;
    if (fresh || p < page0 || p >= page0 + 32) {
      page0 = p;
      fresh = false;
      ids = a.tables[(long long)trow * a.table_row + min(p + lane, a.table_row - 1)];
    }
    int b = __shfl_sync(0xffffffffu, ids, p - page0);
    if (b < 0 || b >= a.n_blocks || p >= a.table_row) {  // reported; a page of the cache is read instead
      if (lane == 0) atomicExch(&g_shared_prefix_error, kErrPage);
      b = 0;
    }
    return b;
  }
};

// The producer warp's walk over a line: the cursor, and the place of its next key in the cache.
// Divisions by the page size happen once a segment; boxes of `box` keys divide pages and stages.
struct Feed {
  Cursor s;
  Pages pages;
  int key, off, p, z;  // next key, its offset in its page, that page's table entry, its place in the cache
  int line;
  bool valid;
  __device__ __forceinline__ void seek(const Args& a, int tile) {
    key = s.k0 + s.j * tile;
    p = key / a.block;
    off = key - p * a.block;
    pages.fresh = true;
    z = pages.get(a, s.trow, p) * a.block + off;
  }
  // the prefix line's run, then the suffix line's
  __device__ __forceinline__ void begin(const Args& a, int tile, int from = 0) {
    valid = false;
    for (line = from; line < 2 && !valid; ++line) valid = s.begin(a, line);
    --line;
    if (valid) seek(a, tile);
  }
  // behind a tile's last key: to the next tile
  __device__ __forceinline__ void next(const Args& a, int tile) {
    if (s.next()) return;
    if (!s.done()) seek(a, tile);
    else begin(a, tile, line + 1);
  }
  // the next C::KEYS keys of one cache (whole boxes, none behind the last key).  All copies are issued by one
  // straight piece of code: entering it costs ten times what a further copy in it does.
  template <typename C, int BOX>
  __device__ __forceinline__ void load_boxes(const Args& a, const CUtensorMap* tm, uint32_t dst, uint32_t bar) {
    constexpr int NB = C::KEYS / BOX;
    int at[NB], n = 0;
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      at[b] = z;
      if (key < s.k1) {
        ++n;
        key += BOX;
        if (key < s.k1) {
          off += BOX;
          z += BOX;
          if (off == a.block) {
            off = 0;
            z = pages.get(a, s.trow, ++p) * a.block;
          }
        }
      }
    }
    if (elect_one()) {
      mbar_expect_tx(bar, n * BOX * C::RB);
#pragma unroll
      for (int b = 0; b < NB; ++b)
        if (b < n) {
          tma_4d(dst + b * BOX * C::BOXB, tm, bar, s.kvh, at[b], 0);
          if (C::NBOX > 1) tma_4d(dst + (C::KEYS + b * BOX) * C::BOXB, tm, bar, s.kvh, at[b], 1);
        }
    }
    __syncwarp();
  }
  template <typename C>
  __device__ __forceinline__ void load(const Args& a, const CUtensorMap* tm, uint32_t dst, uint32_t bar) {
    if (a.box == 64) load_boxes<C, 64>(a, tm, dst, bar);
    else if (a.box == 32) load_boxes<C, 32>(a, tm, dst, bar);
    else if (a.box == 16) load_boxes<C, 16>(a, tm, dst, bar);
    else load_boxes<C, 8>(a, tm, dst, bar);
  }
};

// waits, within a limit, for the copies of stages [k - stages, k) that are still in flight (after an abort)
__device__ __forceinline__ void drain(uint32_t bar_full, int stages, int k) {
  for (int i = max(0, k - stages); i < k; ++i) {
    const long long t0 = clock64();
    while (!mbar_test(bar_full + 8 * (i % stages), (i / stages) & 1) && clock64() - t0 < kWaitCycles) {
    }
  }
}

// factor 2^(13 - exponent) that brings a row of q of largest magnitude mx near 2^13, where f16 keeps bf16's
// 8-bit mantissas exact over 31 binades (down to 2^-17, in steps of 2^-24) and loses bits gradually below; tiny
// rows are scaled by 2^110, and one that holds an infinity or NaN not at all: what f16 cannot hold there becomes
// infinite (such a row's scores are infinite or NaN whatever the rest)
__device__ __forceinline__ int f16_row_exponent(float mx) {
  const int ex = (int)(__float_as_uint(mx) >> 23);
  return ex == 255 ? 140 : max(ex, 30);
}
__device__ __forceinline__ float f16_row_factor(int ex) { return __uint_as_float((uint32_t)(267 - ex) << 23); }
__device__ __forceinline__ float f16_row_inverse(int ex) { return __uint_as_float((uint32_t)(ex - 13) << 23); }

template <int HD, bool F8, int KT>
struct Warp {  // a consumer warp's state: 16 query rows, HD dims, stages of KT keys
  using C = Tile<HD, F8, KT>;
  uint32_t q[HD / 16][4];
  float o[HD / 8][4];
  float m[2], l[2], c[2];  // running reference score (log2), partial sum, score factor of rows g and g + 8
  int lane, g, t;

  __device__ __forceinline__ void start(const Args& a, const Cursor& s, int wm) {
    // Q fragments.  For an e4m3 cache the products run in f16 (an e4m3 value is exact there): each
    // query row is scaled by a power of two, and its dims are taken in the order in which a lane
    // holds four neighbouring bytes of a key.
    const bf16* p[2];
    bool ok[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int rl = wm * 16 + g + 8 * h;
      const int r = s.r0 + rl;
      ok[h] = rl < s.rn;
      p[h] = a.q + (long long)(s.row0 + (ok[h] ? r / a.Gq : 0)) * a.q_row +
             (long long)(s.kvh * a.Gq + (ok[h] ? r % a.Gq : 0)) * a.q_head;
      m[h] = -INFINITY;
      l[h] = 0.f;
      c[h] = a.scale_log2;
    }
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int h = e & 1;
        const int d = F8 ? kk * 16 + 4 * t + (e >> 1) * 2 : kk * 16 + 2 * t + (e >> 1) * 8;
        q[kk][e] = ok[h] ? *reinterpret_cast<const uint32_t*>(p[h] + d) : 0u;
      }
    if constexpr (F8) {
      float mx[2] = {0.f, 0.f}, f[2];
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&q[kk][e]));
          mx[e & 1] = fmaxf(mx[e & 1], fmaxf(fabsf(x.x), fabsf(x.y)));
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
        mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
        const int ex = f16_row_exponent(mx[h]);
        f[h] = f16_row_factor(ex);
        c[h] = a.scale_log2 * f16_row_inverse(ex);
      }
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 x = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&q[kk][e]));
          q[kk][e] = pack_f16(x.x * f[e & 1], x.y * f[e & 1]);
        }
    }
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  }

  // The score that P of a tile refers to, from the tile's largest one.  With an e4m3 cache P is an f16
  // operand, whose values end at 2^-24: referred to the largest score, weights below 2^-25 of it would be lost
  // (a thousand keys and more may lie there, next to one large score) though the sums count them.  Referred to
  // 2^14 less, P reaches 2^14 (f16 ends at 2^16) and keeps its 11 bits down to 2^-28 of the largest weight.
  // Above 2^20 the subtraction could round, past f16's end from 2^25 on; weights are 0 or 1 there anyway.
  static __device__ __forceinline__ float reference(float mx) { return F8 && fabsf(mx) < 1048576.f ? mx - 14.f : mx; }

  // keys [key0, key0 + NK) of a stage of which the first nvalid are the row's
  template <int NK, bool PART>
  __device__ __forceinline__ void tile(uint32_t sk, uint32_t sv, int key0, int nvalid) {
    constexpr int NT = NK / 8;
    float s[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
    if constexpr (F8) {
#pragma unroll
      for (int kk = 0; kk < HD / 16; kk += 2)
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
          uint32_t r[4];
          ldsm_x4(r, sk + C::at(key0 + j * 8 + (lane & 15), kk + (lane >> 4)));
#pragma unroll
          for (int e = 0; e < 4; ++e)
            mma16816<true>(s[j + (e & 1)], q[kk + (e >> 1)], e4m3x2_f16x2(r[e]), e4m3x2_f16x2(r[e] >> 16));
        }
    } else {
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
          uint32_t r[4];
          ldsm_x4(r, sk + C::at(key0 + j * 8 + ((lane >> 4) << 3) + (lane & 7), 2 * kk + ((lane >> 3) & 1)));
          mma16816<false>(s[j], q[kk], r[0], r[1]);
          mma16816<false>(s[j + 1], q[kk], r[2], r[3]);
        }
    }
    float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float x = s[j][e] * c[e >> 1];
        if (PART && key0 + 8 * j + 2 * t + (e & 1) >= nvalid) x = -INFINITY;
        s[j][e] = x;
        mx[e >> 1] = fmaxf(mx[e >> 1], x);
      }
    float mu[2];
    bool grew = false;
    float alpha[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 1));
      mx[h] = fmaxf(mx[h], __shfl_xor_sync(0xffffffffu, mx[h], 2));
      const float mn = fmaxf(m[h], reference(mx[h]));
      grew |= mn > m[h];
      mu[h] = mn == -INFINITY ? 0.f : mn;
      alpha[h] = ex2(m[h] - mu[h]);
      m[h] = mn;
    }
    if (__any_sync(0xffffffffu, grew)) {
      l[0] *= alpha[0];
      l[1] *= alpha[1];
#pragma unroll
      for (int j = 0; j < HD / 8; ++j) {
        o[j][0] *= alpha[0];
        o[j][1] *= alpha[0];
        o[j][2] *= alpha[1];
        o[j][3] *= alpha[1];
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[j][e] = ex2(s[j][e] - mu[e >> 1]);
        l[e >> 1] += s[j][e];
      }
    // O += P V; P is rounded to the type of V's product (values at most 1, or 2^14 in f16; sums kept in fp32)
#pragma unroll
    for (int ks = 0; ks < NT / 2; ++ks) {
      uint32_t a[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float lo = s[2 * ks + (e >> 1)][2 * (e & 1)], hi = s[2 * ks + (e >> 1)][2 * (e & 1) + 1];
        a[e] = F8 ? pack_f16(lo, hi) : pack_bf16(lo, hi);
      }
      uint32_t keep[2] = {0xffffffffu, 0xffffffffu};
      if (PART) {  // what lies behind the last key may be anything, NaN included
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int k = key0 + ks * 16 + 8 * e + 2 * t;
          keep[e] = (k < nvalid ? 0xffffu : 0u) | (k + 1 < nvalid ? 0xffff0000u : 0u);
        }
      }
      if constexpr (F8) {
#pragma unroll
        for (int d = 0; d < HD / 16; d += 2) {
          uint32_t r[4];
          ldsm_x4_t(r, sv + C::at(key0 + ks * 16 + (lane & 15), d + (lane >> 4)));
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] = __byte_perm(r[e], 0, 0x3120);  // dims 2g | 2g+1 of keys 2t, 2t+1
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            mma16816<true>(o[2 * (d + e)], a, e4m3x2_f16x2(r[2 * e]) & keep[0], e4m3x2_f16x2(r[2 * e + 1]) & keep[1]);
            mma16816<true>(o[2 * (d + e) + 1], a, e4m3x2_f16x2(r[2 * e] >> 16) & keep[0],
                           e4m3x2_f16x2(r[2 * e + 1] >> 16) & keep[1]);
          }
        }
      } else {
#pragma unroll
        for (int d = 0; d < HD / 16; ++d) {
          uint32_t r[4];
          ldsm_x4_t(r, sv + C::at(key0 + ks * 16 + (lane & 15), 2 * d + (lane >> 4)));
          if (PART) {
#pragma unroll
            for (int e = 0; e < 4; ++e) r[e] &= keep[e & 1];
          }
          mma16816<false>(o[2 * d], a, r[0], r[1]);
          mma16816<false>(o[2 * d + 1], a, r[2], r[3]);
        }
      }
    }
  }

  __device__ __forceinline__ void finish_sums() {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    }
  }

  // rows g + 8h: to / from another warp, each lane its own values
  __device__ __forceinline__ void put(float* buf, int h) const {
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
      buf[(2 * j) * 32 + lane] = o[j][2 * h];
      buf[(2 * j + 1) * 32 + lane] = o[j][2 * h + 1];
    }
    buf[(HD / 4) * 32 + lane] = m[h];
    buf[(HD / 4 + 1) * 32 + lane] = l[h];
  }
  __device__ __forceinline__ void join(const float* buf, int h) {
    const float mo = buf[(HD / 4) * 32 + lane];
    const float mn = fmaxf(m[h], mo);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float fa = ex2(m[h] - mu), fb = ex2(mo - mu);
    m[h] = mn;
    l[h] = l[h] * fa + buf[(HD / 4 + 1) * 32 + lane] * fb;
#pragma unroll
    for (int j = 0; j < HD / 8; ++j) {
      o[j][2 * h] = o[j][2 * h] * fa + buf[(2 * j) * 32 + lane] * fb;
      o[j][2 * h + 1] = o[j][2 * h + 1] * fa + buf[(2 * j + 1) * 32 + lane] * fb;
    }
  }

  __device__ __forceinline__ void store(float* po, float* pml, int h) const {
    if (F8) {
#pragma unroll
      for (int d = 0; d < HD / 16; ++d)
        *reinterpret_cast<float4*>(po + 16 * d + 4 * t) =
            make_float4(o[2 * d][2 * h], o[2 * d + 1][2 * h], o[2 * d][2 * h + 1], o[2 * d + 1][2 * h + 1]);
    } else {
#pragma unroll
      for (int j = 0; j < HD / 8; ++j)
        *reinterpret_cast<float2*>(po + 8 * j + 2 * t) = make_float2(o[j][2 * h], o[j][2 * h + 1]);
    }
    if (t == 0) *reinterpret_cast<float2*>(pml) = make_float2(m[h], l[h]);
  }
};

// joins the partials of the warps kq = 0 .. wk-1 that split the keys of the same rows into warp 0's;
// all four warps call it
template <typename W>
__device__ __forceinline__ void join_warps(W& w, float* red, int stride, int wk, int wm, int kq, int rows) {
  w.finish_sums();
  for (int step = wk / 2; step > 0; step /= 2)
    for (int h = 0; h < 2; ++h) {
      if (h == 1 && rows <= 8) break;
      float* buf = red + (wk == 4 ? kq % step : wm) * stride;
      if (kq >= step && kq < 2 * step) w.put(buf, h);
      consumers_sync();
      if (kq < step) w.join(buf, h);
      consumers_sync();
    }
}

template <int HD, bool F8>
struct Gen {  // shared memory of the general kernel: two CTAs on an SM
  static constexpr int KT = general_tile(HD, F8);
  using C = Tile<HD, F8, KT>;
  static constexpr int FIT = (112 * 1024 - kRedBytes<HD> - 1024 - 256) / (2 * C::BYTES);
  static constexpr int ST = FIT < 8 ? FIT : 8;
  static constexpr int SMEM = 1024 + ST * 2 * C::BYTES + kRedBytes<HD> + 256;
  static_assert(ST >= 2, "two stages at least");
};

// One producer warp and four mma.sync warps, for every head size, page size and head count.
//
// Bound by instructions and their latencies (e4m3: each scheduler issues 0.35 instructions a cycle for its two
// warps; DRAM at 1.4 TB/s).  A CTA takes 3.6 us for 64 keys x 64 query rows with an e4m3 cache of 128 dims (128
// products a warp, and 256 conversions, which each of the four warps repeats for its own 16 rows) and 1.6 us for
// 64 keys of a suffix unit, where the warps split the keys.
//
// A tile has 64 keys, or 128 for bf16 of 32 and 64 dims: longer tiles share a suffix warp's chain of products,
// maximum and exponentials among twice the keys, but the lines are cut less evenly, and with conversions (e4m3)
// or 128 dims there is no room in registers.  Kernel + plan + combine on a B200, 32 / 8 heads, in us, tiles of
// 64 against 128 (lengths are ragged, up to those stated):
//   (prompts x rows, prompt + own keys)    bf16 32 dims    bf16 64 dims    e4m3 64 dims    e4m3 128 dims
//   128 x 1, 1500 own keys                   48.0  40.6      62.7  54.3
//   2 x 8, 4096 + 256                        29.5  22.6      30.0  24.3      31.1  29.2      40.4  38.5
//   8 x 16, 2048 + 1024                      41.6  37.6      53.2  51.1      58.0  60.7     101.2 108.3
//   16 x 16, 2048 + 2048                     80.8  71.9     111.2 111.0     120.2 126.6     207.9 218.9
//   1 x 32, 32768 + 512                      50.2  47.9      59.8  60.7      80.7  82.0     143.7 144.5
//
// Against the tcgen05 kernel, the same sums, bf16 of 128 dims, which the rule between the two sends there:
//   (prompts x rows, prompt + own keys)         this     tc
//   4 x 16, 1024 + 1024                         56.2   44.0
//   8 x 16, 2048 + 1024                         88.7   74.2
//   16 x 16, 2048 + 2048                       203.1  169.9
//   1 x 32, 32768 + 512                        106.6   78.4
// Earlier forms of the tcgen05 kernel for e4m3 (its tiles converted to f16 in shared memory) and for 64 dims (half of
// its products' rows unused) took 63.2, 126.3, 259.2, 116.3 and 39.9, 61.2, 123.6, 68.2 us for the four cases, where
// this one takes 59.4, 101.1, 205.4, 142.1 and 32.5, 51.1, 111.0, 60.7.  Both were measured while L2 fetched 256 bytes
// for a key of 128, which has cost this kernel up to a fifth: the rule is settled for bf16 of 128 dims, and for the
// rest it says what is built.  One prompt with an e4m3 cache was faster there even so.  Here e4m3 needs no conversion
// pass: a lane's four bytes of a key are the operand words of an f16 product after one conversion each.
template <int HD, bool F8>
__global__ void __launch_bounds__(160, 2)
shared_prefix_attn_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                          const __grid_constant__ Args a) {
  constexpr int KT = Gen<HD, F8>::KT;
  using C = Tile<HD, F8, KT>;
  constexpr int ST = Gen<HD, F8>::ST;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  float* red = reinterpret_cast<float*>(smem_raw + (base - raw) + ST * 2 * C::BYTES);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(red) + kRedBytes<HD>);
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * ST;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * ST);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(bar_full + 8 * s, a.box ? 2 : 32);  // K and V, or every lane of the producer
      mbar_init(bar_empty + 8 * s, 4);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncthreads();
  pdl_wait();

  if (warp == 4) {
    int k = 0;
    Feed f;
    for (f.begin(a, KT); f.valid && !*abort_flag; ++k) {
      const int st = k % ST;
      if (!mbar_wait_err(bar_empty + 8 * st, ((k / ST) & 1) ^ 1, abort_flag, &g_shared_prefix_error, kErrWait)) break;
      const uint32_t sk = base + st * 2 * C::BYTES, sv = sk + C::BYTES;
      if (a.box) {
        Feed v = f;
        v.template load<C>(a, &tv, sv, bar_full + 8 * st);
        f.template load<C>(a, &tk, sk, bar_full + 8 * st);
      } else {
        const int key = f.s.k0 + f.s.j * KT;
        for (int r = 0; r < KT; ++r) {
          const int kr = min(key + r, f.s.k1 - 1);
          const long long slot = (long long)f.pages.get(a, f.s.trow, kr / a.block) * a.block + kr % a.block;
          const long long off = (slot * a.nkv + f.s.kvh) * C::RB;
          for (int c = lane; c < 2 * (C::RB / 16); c += 32) {
            const int cc = c % (C::RB / 16);
            const bool is_v = c >= C::RB / 16;
            cp_async16((is_v ? sv : sk) + C::at(r, cc), (is_v ? a.v : a.k) + off + cc * 16);
          }
        }
        cp_async_arrive(bar_full + 8 * st);
      }
      f.next(a, KT);
    }
    if (*abort_flag) drain(bar_full, ST, k);
    return;
  }

  Warp<HD, F8, KT> w;
  w.lane = lane;
  w.g = lane >> 2;
  w.t = lane & 3;
  int k = 0;
  for (int line = 0; line < 2; ++line) {
    Cursor s;
    if (!s.begin(a, line)) continue;
    while (!s.done()) {
      // 16 query rows a warp; with fewer rows than 64 the warps split the keys instead
      const Cursor e = s;
      const int wk = e.rn <= 16 ? 4 : e.rn <= 32 ? 2 : 1;
      const int wm = warp / wk, kq = warp % wk, key0 = kq * (KT / wk);
      w.start(a, e, wm);
      for (bool more = true; more; ++k) {
        const int st = k % ST;
        const uint32_t sk = base + st * 2 * C::BYTES, sv = sk + C::BYTES;
        const int nvalid = e.k1 - (e.k0 + s.j * KT);
        more = s.next();
        // a wait that ran out leaves the loops running on whatever is there: the error word tells
        mbar_wait_err(bar_full + 8 * st, (k / ST) & 1, abort_flag, &g_shared_prefix_error, kErrWait);
        if (wm * 16 < e.rn && key0 < nvalid) {
          if (wk == 1) {
#pragma unroll 1
            for (int at = 0; at < min(nvalid, KT); at += 64) {
              if (nvalid >= at + 64) w.template tile<64, false>(sk, sv, at, KT);
              else w.template tile<64, true>(sk, sv, at, nvalid);
            }
          } else if (wk == 2) {
            if (nvalid >= KT) w.template tile<KT / 2, false>(sk, sv, key0, KT);
            else w.template tile<KT / 2, true>(sk, sv, key0, nvalid);
          } else {
            if (nvalid >= KT) w.template tile<KT / 4, false>(sk, sv, key0, KT);
            else w.template tile<KT / 4, true>(sk, sv, key0, nvalid);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_empty + 8 * st);
      }
      join_warps(w, red, (HD / 4 + 2) * 32, wk, wm, kq, e.rn);
      if (kq == 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int rl = wm * 16 + w.g + 8 * h;
          if (rl < e.rn) {
            const long long slot = partial_slot(a, e, line, 0, rl);
            w.store(a.part_o + slot * HD, a.part_ml + slot * 2, h);
          }
        }
      }
    }
  }
}

// ------------------------------------------------------------------ tcgen05 variant
// One CTA per SM, 128 keys at a time, keys on the M side of both products:
//
//   S_j = K_j Q^T       M 128 keys, N query rows (16, 32 or 64), K 128 dims
//   O  += V_j^T P_j     M 128 dims, N query rows, K 128 keys
//
// so that a suffix unit with a handful of query rows costs a handful of columns, and a softmax thread
// owns a key: N exponentials per 128 keys.  Decode is bound by the cache's bytes, and this keeps the work
// per byte low on both kinds of units.
//
// The chain from S to P is latency, not work, so two groups of four softmax warps take turns: tile by
// tile, each with its own maxima, sums, P and O.  The even and the odd tiles of a segment are two
// partials for the combine kernel.
//
// P = 2^(S - m) needs no maximum for its precision, only a range: m is the score of a segment's first
// key (of the group's first tile), one per query row, so the largest P is at least 1.  bf16 has the exponents
// of fp32, so P may reach 2^60 (which leaves O room for values of V up to 2^50 over 2^17 keys).  A barrier's OR
// tells when a value exceeds that, or a reference is so large that scores round; only then are
// maxima taken (warp reductions, then across the four warps), O and the sums rescaled and P formed again.
//
// A segment's O is stored when the group's next tile waits for the same product anyway.
//
// warps 0, 3   load K tiles and V tiles (TMA), each into a ring of its own
// warp 1       issues the products, S up to three tiles ahead (of the next unit, too)
// warp 2       brings the query rows of the next segments to shared memory
// warps 4-11   softmax: thread r of a group owns key r of its tiles, and dim r of its output
//
// Measured on a B200 (kernel alone, 32 / 8 heads of 128 dims, pages of 256; the floor reads every key once at
// the rate of a plain copy):
//   16 prompts of up to 2048 keys x 8-16 rows with up to 2048 own keys   160 us, 5.7 TB/s (floor 139 us)
//   4 prompts of up to 1024 keys x 8-16 rows with up to 1024 own keys     34 us, 3.6 TB/s (floor 19 us)
//   1 prompt of 32768 keys x 32 rows                                      64 us, 2.7 TB/s (floor 26 us)
// The first is bound by HBM.  In the third a CTA has about 28 prefix and 4 suffix tiles: some 3700 cycles a tile,
// where HBM needs 1390 for its bytes (two units read the same keys), the exponentials of 64 columns about 512, and
// two softmax groups of some 3000 cycles a tile, in turns, 1500.  What fills the rest has not been found: the groups
// may not overlap, or the two units of a key drift apart (28 % L2 hits, of 50 % possible).  Short units add about a
// tile's time each for their query rows, first scores and output.
//
// Tried and not kept: the two products of a query row on the M side (128 rows a unit; a suffix then costs as
// much as a prefix), mma.sync for the suffix beside it (16-key steps are 300 instructions of latency), one
// ring for K and V (74 against 59 us on the second case), one producer warp for both (185 against 165 us on
// the first), issue by a plain lane 0 instead of an elected one (103 against 40 cycles a product).
struct Tc {
  using E = Tile<128, false, 128>;  // a K or V tile
  static constexpr int THREADS = 384;
  static constexpr int Q = (MR + 16) * 256;  // see QPlace
  static constexpr int P = 128 * MR * 2;
  // places for K and V tiles, in rings of their own: a K tile is free as soon as its S is complete, a V tile
  // only after P, and in one ring it would hold up the K tiles behind it
  static constexpr int KN = 2, VN = 3;
  static constexpr int QB = 5;  // places of query rows: one for the prefix line, up to 4 for the suffix line
  static constexpr int BARS = 2 * (KN + VN) + 2 * QB + 4 + 4;
  static constexpr int STAT = (2 + 4 + 2 + 1) * MR * 4;  // of a softmax group, see Stat
  static constexpr int SMEM = 1024 + Q + 2 * P + (KN + VN) * E::BYTES + 2 * STAT + BARS * 8 + 16;
  static constexpr uint32_t COLS = 512;  // tensor memory: S four times 64, O twice 64
  static constexpr uint32_t FMT = (1u << 4) | (1u << 7) | (1u << 10) | (8u << 24);  // M 128, bf16 operands
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

// Shared-memory matrix descriptors (128-byte swizzle, 8-row groups 1024 bytes apart) in two words: the low
// one is the address / 16, with the leading offset / 16 above it, and advances by plain additions; the high one
// is the same for all.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr, uint32_t leading) { return (saddr >> 4) | ((leading >> 4) << 16); }
template <bool ACC>
__device__ __forceinline__ void umma(uint32_t tmem_d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t acc = 1) {
  if constexpr (ACC)
    asm volatile(
        "{\n .reg .b64 x, y;\n .reg .pred p;\n mov.b64 x, {%1, %4};\n mov.b64 y, {%2, %4};\n setp.eq.u32 p, 0, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(tmem_d),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(kDescHi));
  else
    asm volatile(
        "{\n .reg .b64 x, y;\n .reg .pred p;\n mov.b64 x, {%1, %4};\n mov.b64 y, {%2, %4};\n setp.ne.u32 p, %5, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}\n" ::"r"(tmem_d),
        "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(kDescHi), "r"(acc));
}
// n columns of this thread's lane, complete on return (one statement: nothing can use them before)
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t taddr, float* r);
template <>
__device__ __forceinline__ void tmem_load<16>(uint32_t taddr, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      " tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(taddr)
      : "memory");
}
template <>
__device__ __forceinline__ void tmem_load<32>(uint32_t taddr, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
      " tcgen05.wait::ld.sync.aligned;\n"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]), "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]), "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float* r) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(r);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(
          taddr),
      "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
      "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
      : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }
// barriers of softmax group wg: 1 + 2 wg, and 2 + 2 wg for the OR of a predicate
__device__ __forceinline__ void group_sync(int wg) { asm volatile("bar.sync %0, 128;\n" ::"r"(1 + 2 * wg) : "memory"); }
__device__ __forceinline__ bool group_any(int wg, bool x) {
  int r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.b32 q, %1, 0;\n barrier.cta.red.or.pred p, %2, 128, q;\n selp.s32 %0, 1, 0, p;\n}\n"
      : "=r"(r)
      : "r"((int)x), "r"(2 + 2 * wg)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ bool mbar_poll(uint32_t addr, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(addr), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ float warp_max_f32(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;\n" : "=f"(r) : "f"(x));
  return r;
}

// A CTA's tiles in order: its run of the prefix line, then its run of the suffix line.
struct Walk {
  Cursor s;
  int line, seg, t;  // segments of the line so far, tiles of the segment so far
  bool valid;
  __device__ __forceinline__ void begin(const Args& a) {
    seg = t = line = 0;
    valid = s.begin(a, 0);
    if (!valid) {
      line = 1;
      valid = s.begin(a, 1);
    }
  }
  __device__ __forceinline__ bool last_of_segment() const { return s.j + 1 == s.n || s.x + 1 >= s.x1; }
  // to the next tile; true when it belongs to the same segment
  __device__ __forceinline__ bool next(const Args& a) {
    ++t;
    if (s.next()) return true;
    ++seg;
    t = 0;
    if (s.done()) {
      valid = line == 0 && s.begin(a, 1);
      line = 1;
      seg = 0;
    }
    return false;
  }
};
// columns of a segment with rn query rows
__device__ __forceinline__ int columns(int rn) { return rn <= 16 ? 16 : rn <= 32 ? 32 : 64; }

// The place of a segment's query rows: the first MR rows of the buffer for the prefix line; for the suffix
// line 1, 2 or 4 places, of which the first lies behind them where it fits (so the line's first rows need
// not wait for the prefix line's last product).  Each place has its own pair of barriers.
struct QPlace {
  int bar, row0, rows;  // barrier pair, first row in the buffer (a multiple of 8), rows of a span
  uint32_t parity;
  bool shared;  // lies in the prefix line's rows
  __device__ __forceinline__ QPlace(const Args& a, int line, int seg) {
    rows = line ? columns(a.Gq) : MR;
    const int lg = rows == 64 ? 0 : rows == 32 ? 1 : 2, i = seg & ((1 << lg) - 1);
    bar = line ? 1 + i : 0;
    shared = !(rows == 16 && i == 0);
    row0 = shared ? i * rows : MR;
    parity = (seg >> lg) & 1;
  }
};

constexpr float kNoMax = -FLT_MAX;  // where a row has no score yet (-inf - -inf would be NaN): no finite score is less
// References from this size on: score * scale - m in one rounding is off by the product's own rounding error, half a
// binade here and any number of them far beyond (2^31: P overflows, or is 0 for the largest score itself).
constexpr float kFar = 16777216.f;  // 2^24

// what the threads of a softmax group share
struct Stat {
  int* slot;        // [2][MR] where the partials go, of a segment and of the one before
  float* red;       // [4][MR] per warp: maxima, sums
  float* m;         // [2][MR] reference scores in use (log2)
  float* alpha;     // [MR]
};
__device__ __forceinline__ void load4(float* d, const float* s) {
  const float4 v = *reinterpret_cast<const float4*>(s);
  d[0] = v.x, d[1] = v.y, d[2] = v.z, d[3] = v.w;
}

template <int N>
struct Softmax {
  static constexpr int H = N < 32 ? N : 32;  // columns at a time
  static constexpr float kMost = 1152921504606846976.f;  // 2^60

  // 2^(S - m) of this thread's key, packed, and the largest of them; FAR: scores are rounded as m was, so that
  // equal ones cancel whatever their size
  template <bool FAR>
  static __device__ __forceinline__ float weights(uint32_t* p, uint32_t t_s, bool live, float scale, const float* sm) {
    float top = 0.f;
#pragma unroll
    for (int h = 0; h < N; h += H) {
      float y[H];
      tmem_load<H>(t_s + h, y);
#pragma unroll
      for (int i = 0; i < H; i += 4) {
        float m[4];
        load4(m, sm + h + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[i + e] = ex2(FAR ? __fadd_rn(__fmul_rn(y[i + e], scale), -m[e]) : y[i + e] * scale - m[e]);
          top = fmaxf(top, y[i + e]);
        }
      }
#pragma unroll
      for (int i = 0; i < H; i += 2) {
        const uint32_t v = pack_bf16(y[i], y[i + 1]);
        p[(h + i) / 2] = live ? v : 0u;
      }
    }
    return live ? top : 0.f;
  }

  // one tile up to P (packed in p) and the sums of the rounded P in l; wait_o() waits for the group's
  // product before; far: column r has a reference of kFar or more
  template <typename W>
  static __device__ __forceinline__ void tile(int wg, uint32_t t_s, uint32_t t_o, bool live, bool first, float scale,
                                              const Stat& st, float* sm, float* l, uint32_t* p, int r, bool& far,
                                              W wait_o) {
    const int warp4 = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
    const float top = weights<false>(p, t_s, live, scale, sm);
    if (group_any(wg, top > kMost || far)) {  // rare: by the maximum
#pragma unroll 1
      for (int h = 0; h < N; h += 16) {
        float y[16];
        tmem_load<16>(t_s + h, y);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float mx = warp_max_f32(live ? __fmul_rn(y[i], scale) : -INFINITY);
          if (lane == i) st.red[warp4 * MR + h + i] = mx;
        }
      }
      group_sync(wg);
      if (r < N) {
        const float old = sm[r];
        const float mx = fmaxf(fmaxf(st.red[r], st.red[MR + r]), fmaxf(st.red[2 * MR + r], st.red[3 * MR + r]));
        const float now = fmaxf(old, mx);
        st.alpha[r] = ex2(old - now);
        sm[r] = now;
        far = fabsf(now) >= kFar;
      }
      group_sync(wg);
      if (!first) {
        wait_o();
        tc_fence_after();
#pragma unroll 1
        for (int h = 0; h < N; h += 16) {
          float o[16];
          tmem_load<16>(t_o + h, o);
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] *= st.alpha[h + i];
          tmem_st16(t_o + h, o);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
#pragma unroll
        for (int i = 0; i < N; ++i) l[i] *= st.alpha[i];
      }
      weights<true>(p, t_s, live, scale, sm);  // at most 1
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      const float2 v = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&p[i]));
      l[2 * i] += v.x;
      l[2 * i + 1] += v.y;
    }
  }

  static __device__ __forceinline__ void write(const uint32_t* p, uint8_t* prow, int r) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i)
      *reinterpret_cast<uint4*>(prow + ((i ^ (r & 7)) << 4)) = make_uint4(p[4 * i], p[4 * i + 1], p[4 * i + 2], p[4 * i + 3]);
  }

  // sums of l over the warp's 32 keys, each column once: exchanges of ever smaller halves
  static __device__ __forceinline__ void reduce(float* l, float* red) {
    const int warp4 = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
    int n = N;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const bool up = lane & o;
      if (n > 1) {
        n /= 2;
#pragma unroll
        for (int i = 0; i < N / 2; ++i)
          if (i < n) {
            const float send = up ? l[i] : l[i + n], keep = up ? l[i + n] : l[i];
            l[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
          }
      } else {
        l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
      }
    }
    if constexpr (N == 64) {
      red[warp4 * MR + 2 * lane] = l[0];
      red[warp4 * MR + 2 * lane + 1] = l[1];
    } else {
      red[warp4 * MR + lane / (32 / N)] = l[0];
    }
  }
};

// the scores of a segment's first key (of the group), by the warp that has it
__device__ __forceinline__ void refer(uint32_t t_s, int cols, float scale, float* sm) {
  for (int h = 0; h < cols; h += 16) {
    float y[16];
    tmem_load<16>(t_s + h, y);
    if ((threadIdx.x & 31) == 0)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = y[i] * scale;
        sm[h + i] = x == -INFINITY ? kNoMax : x;
      }
  }
}
// a segment's outputs: thread r has dim r
__device__ __forceinline__ void store_o(uint32_t t_o, const int* slot, float* part_o, int rn, int r) {
  for (int h = 0; h < rn; h += 16) {
    int4 at[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) at[i] = reinterpret_cast<const int4*>(slot + h)[i];
    float o[16];
    tmem_load<16>(t_o + h, o);
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (h + i < rn) part_o[(long long)reinterpret_cast<const int*>(at)[i] * 128 + r] = o[i];
  }
}

__global__ void __launch_bounds__(Tc::THREADS, 1)
shared_prefix_tc_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                        const __grid_constant__ Args a) {
  using T = Tc;
  using E = T::E;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  const uint32_t s_q = base;                           // query rows
  const uint32_t s_p = s_q + T::Q;                     // [2] P of the softmax groups
  const uint32_t s_k = s_p + 2 * T::P;                 // [KN]
  const uint32_t s_v = s_k + T::KN * E::BYTES;         // [VN]
  uint8_t* g_stat = gbase + (s_v - base) + T::VN * E::BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(g_stat + 2 * T::STAT);
  const uint32_t bar_k = smem_u32(bars);               // [KN] K ready for the products
  const uint32_t bar_kfree = bar_k + 8 * T::KN;        // [KN] K read
  const uint32_t bar_v = bar_kfree + 8 * T::KN;        // [VN] V ready
  const uint32_t bar_vfree = bar_v + 8 * T::VN;        // [VN] V read
  const uint32_t bar_q = bar_vfree + 8 * T::VN;        // [QB] query rows ready
  const uint32_t bar_qfree = bar_q + 8 * T::QB;        // [QB] query rows read
  const uint32_t bar_s = bar_qfree + 8 * T::QB;        // [4] S complete
  const uint32_t bar_p = bar_s + 32;                   // [2] S read, P written, O rescaled
  const uint32_t bar_o = bar_p + 16;                   // [2] O complete up to the tile
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + T::BARS);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto wait = [&](uint32_t bar, uint32_t parity) {
    return mbar_wait_err(bar, parity, abort_flag, &g_shared_prefix_error, kErrWait);
  };
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int i = 0; i < T::KN; ++i) {
      mbar_init(bar_k + 8 * i, 1);
      mbar_init(bar_kfree + 8 * i, 1);
    }
    for (int i = 0; i < T::VN; ++i) {
      mbar_init(bar_v + 8 * i, 1);
      mbar_init(bar_vfree + 8 * i, 1);
    }
    for (int i = 0; i < T::QB; ++i) {
      mbar_init(bar_q + 8 * i, 1);
      mbar_init(bar_qfree + 8 * i, 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(bar_s + 8 * i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar_p + 8 * i, 4);
      mbar_init(bar_o + 8 * i, 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_u32(tmem_slot)),
                 "r"(T::COLS));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, t_o = tmem + 4 * MR;
  pdl_wait();
  // the walk is the same in every role: tile k belongs to softmax group k & 1
  if (warp == 0 || warp == 3) {  // K tiles, V tiles
    const bool v = warp == 3;
    const int n = v ? T::VN : T::KN;
    const uint32_t full = v ? bar_v : bar_k, free = v ? bar_vfree : bar_kfree, dst = v ? s_v : s_k;
    Feed f;
    int k = 0, i = 0;
    uint32_t parity = 1;
    for (f.begin(a, 128); f.valid && wait(free + 8 * i, parity); ++k) {
      f.load<E>(a, v ? &tv : &tk, dst + i * E::BYTES, full + 8 * i);
      f.next(a, 128);
      if (++i == n) i = 0, parity ^= 1;
    }
    if (__any_sync(0xffffffffu, *abort_flag)) drain(full, n, k);
  } else if (warp == 1) {
    Walk w;
    w.begin(a);
    int ka = 0;                      // tiles whose S is issued
    int ki = 0, vi = 0;              // places of the next K and V
    uint32_t kph = 0, vph = 0;
    uint32_t info = 0;               // of tile i, at bits 8 (i & 3): columns / 8, and 16 when O is added to
    QPlace q(a, w.line, w.seg);
    bool q_ready = false;
    auto ready = [&](uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_poll(bar, parity)); };
    auto issue_s = [&] {  // S of the walk's tile; its buffer is free: P of tile ka - 4 was awaited
      tc_fence_after();
      const int sb = ka & 3;
      const uint32_t n8 = columns(w.s.rn) >> 3, id = T::FMT | (n8 << 17);
      const uint32_t kd = desc_lo(s_k + ki * E::BYTES, 0), qd = desc_lo(s_q + q.row0 * 256, 0);
      const uint32_t span = (uint32_t)q.rows * 8;  // 128 bytes a row, in units of 16
      const bool last = w.last_of_segment();
      if (elect_one()) {
        umma<false>(tmem + sb * MR, kd, qd, id, 0);
#pragma unroll
        for (int kk = 1; kk < 8; ++kk)
          umma<true>(tmem + sb * MR, kd + (kk >> 2) * 1024 + (kk & 3) * 2, qd + (kk >> 2) * span + (kk & 3) * 2, id);
        umma_commit(bar_s + 8 * sb);
        umma_commit(bar_kfree + 8 * ki);
        if (last) umma_commit(bar_qfree + 8 * q.bar);
      }
      __syncwarp();
      info = (info & ~(0xffu << (8 * sb))) | ((n8 | (w.t >= 2 ? 16u : 0u)) << (8 * sb));
      if (!w.next(a) && w.valid) {
        q = QPlace(a, w.line, w.seg);
        q_ready = false;
      }
      ++ka;
      if (++ki == T::KN) ki = 0, kph ^= 1;
    };
    auto issue_o = [&](int k) {  // O += V P of tile k
      tc_fence_after();
      const int wg = k & 1;
      const uint32_t i = info >> (8 * (k & 3)), id = T::FMT | (1u << 15) | (1u << 16) | ((i & 15u) << 17);
      const uint32_t vd = desc_lo(s_v + vi * E::BYTES, 128 * 128), pd = desc_lo(s_p + wg * T::P, 0);
      if (elect_one()) {
        umma<false>(t_o + wg * MR, vd, pd, id, i & 16u);
#pragma unroll
        for (int kk = 1; kk < 8; ++kk) umma<true>(t_o + wg * MR, vd + kk * 128, pd + kk * 128, id);
        umma_commit(bar_o + 8 * wg);
        umma_commit(bar_vfree + 8 * vi);
      }
      __syncwarp();
      if (++vi == T::VN) vi = 0, vph ^= 1;
    };
    // whichever of the two products has its operands is issued: S up to three tiles ahead of O
    int idle = 0;
    long long since = 0;
    for (int k = 0; k < ka || w.valid;) {
      bool progress = false;
      if (w.valid && ka <= k + 3) {
        if (!q_ready) q_ready = ready(bar_q + 8 * q.bar, q.parity);
        if (q_ready && ready(bar_k + 8 * ki, kph)) {
          issue_s();
          progress = true;
        }
      }
      if (k < ka && ready(bar_p + 8 * (k & 1), (k >> 1) & 1) && ready(bar_v + 8 * vi, vph)) {
        issue_o(k);
        ++k;
        progress = true;
      }
      if (progress) {
        idle = 0;
      } else if ((++idle & 63) == 0) {  // bounded: look at the clock now and then
        if (__any_sync(0xffffffffu, *abort_flag)) break;
        const long long now = clock64();
        if (idle == 64) {
          since = now;
        } else if (now - since > kWaitCycles) {
          atomicExch(&g_shared_prefix_error, kErrWait);
          *abort_flag = 1;
        }
      }
    }
  } else if (warp == 2) {
    // query rows: 16 lanes a row, 16 bytes each; rows up to the segment's columns are zero
    const int ch = lane & 15, first_row = lane >> 4;
    Walk w;
    int prefix_segs = 0;
    for (w.begin(a); w.valid;) {
      const QPlace q(a, w.line, w.seg);
      if (!wait(bar_qfree + 8 * q.bar, q.parity ^ 1)) break;
      if (w.line == 0) {
        ++prefix_segs;
      } else if (prefix_segs > 0 && q.shared) {  // the prefix line's products have read its rows
        if (!wait(bar_qfree, (prefix_segs - 1) & 1)) break;
        prefix_segs = 0;
      }
      const int rows = columns(w.s.rn);
      auto src = [&](int r) {
        const uint32_t rr = w.s.r0 + r, b = a.Gq == 1 ? rr : __umulhi(rr, a.inv_gq), h = rr - b * a.Gq;
        return a.q + (long long)(w.s.row0 + b) * a.q_row + (long long)(w.s.kvh * a.Gq + h) * a.q_head + ch * 8;
      };
      const uint32_t at = q.row0 * 256 + (ch >> 3) * (q.rows * 128);
      auto place = [&](int r) { return at + r * 128 + (((ch & 7) ^ (r & 7)) << 4); };
      for (int r = first_row; r < rows; r += 2)
        cp_async16_or_zero(s_q + place(r), r < w.s.rn ? src(r) : a.q, r < w.s.rn);
      asm volatile("cp.async.wait_all;\n" ::: "memory");
      fence_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar_q + 8 * q.bar);
      while (w.next(a)) {
      }
    }
  } else {
    // every thread takes every step whatever its waits say (the error word tells): the barriers stay in step
    const int wg = (warp >> 2) - 1, r = threadIdx.x & 127;  // key of a tile, dim of the output
    const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16, t_og = t_o + lane_off + wg * MR;
    uint8_t* prow = gbase + (s_p - base) + wg * T::P + r * 128;
    Stat st;
    st.slot = reinterpret_cast<int*>(g_stat + wg * T::STAT);
    st.red = reinterpret_cast<float*>(st.slot + 2 * MR);
    st.m = st.red + 4 * MR;
    st.alpha = st.m + 2 * MR;
    Walk w;
    int k = 0, mine = 0, buf = 0, left = 0;  // the group's tiles, segments mod 2, query rows whose O is not stored yet
    auto wait_o = [&] {  // the group's product before
      if (mine > 0) wait(bar_o + 8 * wg, (mine - 1) & 1);
    };
    auto flush = [&] {  // the O of the segment before
      if (left > 0) store_o(t_og, st.slot + (buf ^ 1) * MR, a.part_o, left, r);
      left = 0;
    };
    for (w.begin(a); w.valid;) {
      const Cursor s = w.s;
      const bool mine0 = (k & 1) == wg;               // the segment's first tile is this group's
      const bool part = mine0 || !w.last_of_segment();  // the segment has a tile of this group
      if (part && r < s.rn) st.slot[buf * MR + r] = (int)partial_slot(a, s, w.line, mine0 ? 0 : 1, r);
      float l[MR];
#pragma unroll
      for (int i = 0; i < MR; ++i) l[i] = 0.f;
      float* sm = st.m + buf * MR;
      bool first = true, far = false;  // far: this thread's column has a reference of kFar or more
      for (bool same = true; same; ++k) {
        const int nvalid = s.k1 - (s.k0 + w.s.j * 128);
        same = w.next(a);
        if ((k & 1) != wg) continue;
        const bool live = r < nvalid;
        const int sb = k & 3;
        wait(bar_s + 8 * sb, (k >> 2) & 1);
        tc_fence_after();
        const uint32_t t_s = tmem + lane_off + sb * MR;
        if (first) {
          if ((warp & 3) == 0) refer(t_s, columns(s.rn), a.scale_log2, sm);
          group_sync(wg);
          far = r < columns(s.rn) && fabsf(sm[r]) >= kFar;
        }
        uint32_t p[MR / 2];
        if (s.rn <= 16) Softmax<16>::tile(wg, t_s, t_og, live, first, a.scale_log2, st, sm, l, p, r, far, wait_o);
        else if (s.rn <= 32) Softmax<32>::tile(wg, t_s, t_og, live, first, a.scale_log2, st, sm, l, p, r, far, wait_o);
        else Softmax<64>::tile(wg, t_s, t_og, live, first, a.scale_log2, st, sm, l, p, r, far, wait_o);
        wait_o();  // it reads P's place
        tc_fence_after();
        if (first) flush();
        first = false;
        if (s.rn <= 16) Softmax<16>::write(p, prow, r);
        else if (s.rn <= 32) Softmax<32>::write(p, prow, r);
        else Softmax<64>::write(p, prow, r);
        if (nvalid < 128) {  // what lies behind the last key may be anything: P is 0 there, and V must be finite
          const int e = k % T::VN;
          wait(bar_v + 8 * e, (k / T::VN) & 1);
          if (!live)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              *reinterpret_cast<uint4*>(gbase + (s_v - base) + e * E::BYTES + E::at(r, i)) = make_uint4(0u, 0u, 0u, 0u);
        }
        fence_async();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p + 8 * wg);
        ++mine;
      }
      if (part) {
        if (s.rn <= 16) Softmax<16>::reduce(l, st.red);
        else if (s.rn <= 32) Softmax<32>::reduce(l, st.red);
        else Softmax<64>::reduce(l, st.red);
        group_sync(wg);
        if (r < s.rn) {
          const float sum = (st.red[r] + st.red[MR + r]) + (st.red[2 * MR + r] + st.red[3 * MR + r]);
          const float m = sum == 0.f ? -INFINITY : sm[r];  // the reference counts 1 at least, unless there was no score
          *reinterpret_cast<float2*>(a.part_ml + (long long)st.slot[buf * MR + r] * 2) = make_float2(m, sum);
        }
        left = s.rn;
        buf ^= 1;
      }
    }
    wait_o();
    tc_fence_after();
    flush();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(T::COLS));
}

// ----------------------------------------------------------------------- combine
// One warp per (row, head): the partials of its prefix unit, then of its suffix unit, in the
// order of the keys.  Bound by latency: its launch overlaps the attention, behind which it takes 2 to 4 us.
template <int HD>
__global__ void __launch_bounds__(128)
shared_prefix_combine_kernel(const int* __restrict__ plan, int ctas, int subs, int units, int B, int nq, int nkv, int Gq,
                             const float* __restrict__ part_o, const float* __restrict__ part_ml, float v_scale,
                             bf16* __restrict__ out) {
  constexpr int V = HD / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= B * nq) return;
  const int b = i / nq, h = i - b * nq, kvh = h / Gq, hl = h - kvh * Gq;
  const int* unit = plan + unit_offset(ctas);
  const int* row = unit + units * kUnitInts + b * kRowInts;
  const int nqt = B * nq;
  float M = -INFINITY, L = 0.f, o[V];
#pragma unroll
  for (int d = 0; d < V; ++d) o[d] = 0.f;
  auto add = [&](long long slot) {
    const float2 ml = *reinterpret_cast<const float2*>(part_ml + slot * 2);
    float p[V];
#pragma unroll
    for (int d = 0; d < V; ++d) p[d] = part_o[slot * HD + lane * V + d];
    const float mn = fmaxf(M, ml.x);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float fa = ex2(M - mu), fb = ex2(ml.x - mu);
    M = mn;
    L = L * fa + ml.y * fb;
#pragma unroll
    for (int d = 0; d < V; ++d) o[d] = o[d] * fa + p[d] * fb;
  };
  auto add_unit = [&](int line, int u, int local) {
    const int n = unit[u * kUnitInts + 1], per = plan[2 * line];
    if (n == 0) return;
    const int x = unit[u * kUnitInts] * nkv + kvh * (n + kStart) + kStart;
    for (int c = x / per; c <= (x + n - 1) / per; ++c) {
      const int tiles = min(x + n, (c + 1) * per) - max(x, c * per);
      for (int sub = 0; sub < min(subs, tiles); ++sub) {
        const int ls = 2 * line + sub;
        add(c * per <= x ? (long long)ls * nqt + i : 4LL * nqt + ((long long)ls * ctas + c) * MR + local);
      }
    }
  };
  if (row[2]) {  // a row without keys stays zero
    if (row[0] >= 0) {
      const int r = (b - row[1]) * Gq + hl;
      add_unit(0, row[0] + r / MR, r % MR);
    }
    add_unit(1, units - B + b, hl);
  }
  const float inv = L == 0.f ? 0.f : v_scale / L;
  bf16* po = out + (long long)i * HD + lane * V;
#pragma unroll
  for (int d = 0; d < V; ++d) po[d] = __float2bfloat16_rn(o[d] * inv);
}

// 4-D map of a cache: [128-byte spans of a key][pages * block keys][KV heads][dims of a span], boxes of one
// span of `box` keys of one head
CUtensorMap cache_tmap(const at::Tensor& c, int box, bool f8) {
  CUtensorMap m;
  const int hd = c.size(3), nkv = c.size(2), elt = f8 ? 1 : 2;
  const int inner = std::min(hd * elt, 128), spans = hd * elt / inner;
  cuuint64_t dims[4] = {(cuuint64_t)(inner / elt), (cuuint64_t)nkv, (cuuint64_t)(c.size(0) * c.size(1)), (cuuint64_t)spans};
  cuuint64_t strides[3] = {(cuuint64_t)hd * elt, (cuuint64_t)nkv * hd * elt, (cuuint64_t)inner};
  cuuint32_t bx[4] = {(cuuint32_t)(inner / elt), 1u, (cuuint32_t)box, 1u};
  cuuint32_t estr[4] = {1u, 1u, 1u, 1u};
  const CUtensorMapSwizzle sw = inner == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                : inner == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                              : CU_TENSOR_MAP_SWIZZLE_32B;
  // what L2 fetches at once: the bytes of a key of this head and no more, since the next head's turn comes long
  // after (128 rows of 1500 keys of their own, 64 dims: 91 us, against 110 with 256 bytes)
  const CUtensorMapL2promotion l2 = inner * spans >= 256  ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B
                                    : inner * spans >= 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_128B
                                    : inner * spans >= 64 ? CU_TENSOR_MAP_L2_PROMOTION_L2_64B
                                                          : CU_TENSOR_MAP_L2_PROMOTION_NONE;
  CUresult r = tma_encode_fn()(&m, f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                               c.data_ptr(), dims, strides, bx, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                               l2, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, std::string("rl_b200: cuTensorMapEncodeTiled failed (") + std::to_string((int)r) + ")");
  return m;
}

int plan_ints(Shape p, int units, int B) { return unit_offset(p.ctas) + units * kUnitInts + B * kRowInts; }

// keys of a TMA box, at most `most`: a power of two that divides the page, so a box never leaves its
// page and an aligned stage is whole boxes; 0 below 8 keys (a period of the swizzle)
int box_keys(int64_t block, int most) {
  while (block % most) most /= 2;
  return most < 8 ? 0 : most;
}

template <typename K, typename... A>
void launch_pdl(K kern, int grid, int block, int smem, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream();
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  RLB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kern, args...));
}

}  // namespace sp
}  // namespace rlb

using namespace rlb;

// int32 plan of the work of one decode step (see the kernel): group g's rows are
// [group_starts[g], group_starts[g+1]), of whose keys the first prefix_lens[g] are the same
at::Tensor shared_prefix_plan(at::Tensor group_starts, at::Tensor prefix_lens, at::Tensor seq_lens, int64_t nq,
                              int64_t nkv, int64_t hd, int64_t block, int64_t max_blocks, bool f8) {
  for (at::Tensor* t : {&group_starts, &prefix_lens, &seq_lens}) {
    RLB_CHECK(t->is_cuda() && t->dim() == 1 && t->device() == seq_lens.device(),
              "shared_prefix_plan: integer vectors on one CUDA device expected");
    if (t->scalar_type() != at::kInt || !t->is_contiguous()) *t = t->to(at::kInt).contiguous();
  }
  const int64_t G = prefix_lens.size(0), B = seq_lens.size(0);
  RLB_CHECK(group_starts.size(0) == G + 1, "shared_prefix_plan: group_starts needs one entry more than prefix_lens");
  RLB_CHECK(nkv >= 1 && nq >= nkv && nq % nkv == 0 && nq / nkv <= sp::kMaxHeads,
            "shared_prefix_plan: query heads must be a multiple of the KV heads, at most 64 per KV head");
  RLB_CHECK(B <= 8192 && G <= 8192 && block >= 1 && max_blocks >= 0, "shared_prefix_plan: at most 8192 rows and groups");
  const int capacity = (int)std::min<int64_t>(block * std::min<int64_t>(max_blocks, 1LL << 31), (1LL << 31) - 256);
  const c10::cuda::CUDAGuard guard(seq_lens.device());
  const int Gq = nq / nkv;
  const sp::Shape p = sp::shape_of(hd, block, f8);
  const int units = sp::max_chunks(B, G, Gq) + B;
  auto plan = at::empty({sp::plan_ints(p, units, B)}, seq_lens.options());
  const int smem = ((int)B + 4 * (int)G + 1 + units) * 4;
  RLB_CHECK(smem <= 200 * 1024, "shared_prefix_plan: too many rows and groups");
  if (smem > 48 * 1024)
    RLB_CUDA_CHECK(cudaFuncSetAttribute(sp::shared_prefix_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  sp::shared_prefix_plan_kernel<<<1, sp::kPlanThreads, smem, stream()>>>(
      group_starts.data_ptr<int>(), prefix_lens.data_ptr<int>(), seq_lens.data_ptr<int>(), G, B, Gq, nkv, p.ctas, p.tile,
      capacity, plan.data_ptr<int>());
  RLB_CUDA_CHECK(cudaGetLastError());
  return plan;
}

// planned here unless `given` holds the plan of these lengths
at::Tensor shared_prefix_attn(at::Tensor q, at::Tensor k_cache, at::Tensor v_cache, at::Tensor block_tables,
                              at::Tensor seq_lens, at::Tensor group_starts, at::Tensor prefix_lens,
                              c10::optional<at::Tensor> given, double scale, double k_scale, double v_scale) {
  RLB_CHECK(q.is_cuda() && q.dim() == 3 && q.scalar_type() == at::kBFloat16,
            "shared_prefix_attn: q must be bf16 [rows, heads, dims]");
  const c10::cuda::CUDAGuard guard(q.device());
  const bool f8 = k_cache.scalar_type() == at::kFloat8_e4m3fn;
  RLB_CHECK(f8 || k_cache.scalar_type() == at::kBFloat16, "shared_prefix_attn: the cache must be bf16 or e4m3");
  RLB_CHECK(k_cache.dim() == 4 && k_cache.is_contiguous() && v_cache.is_contiguous() &&
                v_cache.sizes() == k_cache.sizes() && v_cache.scalar_type() == k_cache.scalar_type(),
            "shared_prefix_attn: contiguous caches [pages, block, KV heads, dims] of one shape and type expected");
  const int64_t B = q.size(0), nq = q.size(1), hd = q.size(2), nb = k_cache.size(0), bs = k_cache.size(1),
                nkv = k_cache.size(2);
  RLB_CHECK(hd == 32 || hd == 64 || hd == 128, "shared_prefix_attn: head_dim must be 32, 64 or 128");
  RLB_CHECK(k_cache.size(3) == hd && nkv >= 1 && nq >= nkv && nq % nkv == 0 && nq / nkv <= sp::kMaxHeads,
            "shared_prefix_attn: heads of q and cache do not match");
  RLB_CHECK(nb >= 1 && bs >= 1 && nb * bs < (1LL << 31), "shared_prefix_attn: the cache needs 1 to 2^31 - 1 keys");
  RLB_CHECK(block_tables.is_cuda() && block_tables.dim() == 2 && block_tables.size(0) == B &&
                (B == 0 || block_tables.size(1) >= 1),
            "shared_prefix_attn: block tables [rows, pages] expected");
  RLB_CHECK(seq_lens.dim() == 1 && seq_lens.size(0) == B, "shared_prefix_attn: a length for every row expected");
  if (block_tables.scalar_type() != at::kInt || !block_tables.is_contiguous())
    block_tables = block_tables.to(at::kInt).contiguous();
  const int64_t groups = prefix_lens.size(0);
  const int Gq = nq / nkv;
  const bool tc = sp::use_tc(hd, bs, f8);
  const sp::Shape p = sp::shape_of(hd, bs, f8);
  const int units = sp::max_chunks(B, groups, Gq) + B;
  for (const at::Tensor& t : {k_cache, v_cache, block_tables, seq_lens})
    RLB_CHECK(t.device() == q.device(), "shared_prefix_attn: all tensors must be on one device");
  for (const at::Tensor& t : {k_cache, v_cache})
    RLB_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, "shared_prefix_attn: caches must be 16-byte aligned");
  auto out = at::empty({B, nq, hd}, q.options());
  if (B == 0) return out;
  const bool planned = given.has_value() && given->defined();
  at::Tensor plan = planned ? *given : shared_prefix_plan(group_starts, prefix_lens, seq_lens, nq, nkv, hd, bs,
                                                           block_tables.size(1), f8);
  RLB_CHECK(plan.is_cuda() && plan.scalar_type() == at::kInt && plan.is_contiguous() && plan.device() == q.device() &&
                plan.numel() == sp::plan_ints(p, units, B),
            "shared_prefix_attn: the plan is of another batch");
  if (q.stride(2) != 1 || q.stride(1) % 8 || q.stride(0) % 8) q = q.contiguous();
  if (reinterpret_cast<uintptr_t>(q.data_ptr()) % 16) q = q.clone(at::MemoryFormat::Contiguous);
  const long long slots = 4 * B * nq + 4LL * p.ctas * sp::MR;
  RLB_CHECK(slots < (1LL << 31), "shared_prefix_attn: too many rows");
  auto part = at::empty({slots * (hd + 2)}, q.options().dtype(at::kFloat));
  sp::Args a;
  a.q = (const sp::bf16*)q.data_ptr();
  a.q_row = q.stride(0);
  a.q_head = q.stride(1);
  a.k = (const uint8_t*)k_cache.data_ptr();
  a.v = (const uint8_t*)v_cache.data_ptr();
  a.tables = block_tables.data_ptr<int>();
  a.table_row = block_tables.size(1);
  a.n_blocks = nb;
  a.block = bs;
  a.box = sp::box_keys(bs, sp::BT);
  a.plan = plan.data_ptr<int>();
  a.ctas = p.ctas;
  a.units = units;
  a.B = B;
  a.nq = nq;
  a.nkv = nkv;
  a.Gq = Gq;
  a.inv_gq = Gq == 1 ? 0 : (uint32_t)(((1ull << 32) + Gq - 1) / Gq);
  a.scale_log2 = (float)(scale * (f8 ? k_scale : 1.0) * 1.4426950408889634);
  a.part_o = part.data_ptr<float>();
  a.part_ml = a.part_o + slots * hd;
  CUtensorMap tk = {}, tv = {};
  if (a.box) {
    tk = sp::cache_tmap(k_cache, a.box, f8);
    tv = sp::cache_tmap(v_cache, a.box, f8);
  }
  auto launch = [&](auto hdv, auto f8v) {
    constexpr int HD = decltype(hdv)::value;
    constexpr bool F8 = decltype(f8v)::value;
    if constexpr (HD == 128 && !F8) {
      if (tc) {
        auto kern = sp::shared_prefix_tc_kernel;
        RLB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, sp::Tc::SMEM));
        sp::launch_pdl(kern, p.ctas, sp::Tc::THREADS, sp::Tc::SMEM, tk, tv, a);
      }
    }
    if (!tc) {
      auto kern = sp::shared_prefix_attn_kernel<HD, F8>;
      constexpr int smem = sp::Gen<HD, F8>::SMEM;
      RLB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      sp::launch_pdl(kern, p.ctas, 160, smem, tk, tv, a);
    }
    sp::launch_pdl(sp::shared_prefix_combine_kernel<HD>, (int)((B * nq + 3) / 4), 128, 0, (const int*)a.plan, p.ctas,
                   tc ? 2 : 1, units, (int)B, (int)nq, (int)nkv, Gq, (const float*)a.part_o, (const float*)a.part_ml,
                   f8 ? (float)v_scale : 1.f, (sp::bf16*)out.data_ptr());
  };
  auto by_type = [&](auto hdv) {
    if (f8) launch(hdv, std::true_type{});
    else launch(hdv, std::false_type{});
  };
  if (hd == 128) by_type(std::integral_constant<int, 128>{});
  else if (hd == 64) by_type(std::integral_constant<int, 64>{});
  else by_type(std::integral_constant<int, 32>{});
  return out;
}

int64_t shared_prefix_error_flag(bool reset) {
  int v = 0;
  RLB_CUDA_CHECK(cudaMemcpyFromSymbol(&v, rlb::sp::g_shared_prefix_error, sizeof(int)));
  if (reset) {
    const int z = 0;
    RLB_CUDA_CHECK(cudaMemcpyToSymbol(rlb::sp::g_shared_prefix_error, &z, sizeof(int)));
  }
  return v;
}
