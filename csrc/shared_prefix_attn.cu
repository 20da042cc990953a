// Decode attention of rows that share a prefix (the samples of one prompt).
//
//   o[b,h] = sum_t softmax_t(scale * q[b,h] . k[t]) v[t]
//
// over row b's keys, of which the first P are the same for every row of its group.
// The keys [0, P) of a group are read once for all of its rows: their queries form
// the M side of a matrix product.  Keys [P, L_b) are read per row.  Both kinds of work
// are units of 64-key tiles:
//
//   prefix unit: 64 query rows (row, head of one KV head) x the group's prefix
//   suffix unit: the G query heads of one KV head of one row x the row's own keys
//
// spread over the CTAs by a plan: the tiles of all (unit, KV head) are laid on one
// line and cut into equal runs, one per CTA, so ragged lengths balance and a long
// prefix is split over many CTAs.  Each CTA leaves, per unit it touched, the fp32
// partial (max, sum, unnormalised output) of an online softmax in base 2; the
// combine kernel joins a row's partials in the order of its keys.  No atomics: the
// result does not depend on timing.
//
// shared_prefix_plan_kernel   group bounds, unit list, tile offsets, every CTA's first unit
// shared_prefix_attn_kernel   one producer warp (TMA) and four mma.sync warps
// shared_prefix_combine_kernel  one warp per (row, head)
//
// The plan depends on the lengths only: one plan serves all layers of a decode step.
#include "tc_common.cuh"

namespace rlb {
namespace sp {

using namespace rlb::tc;
typedef __nv_bfloat16 bf16;

constexpr int BT = 64;        // keys per tile; a prefix is shared in whole tiles
constexpr int MR = 64;        // query rows of a prefix unit
constexpr int kUnitInts = 8;  // first tile, tiles, first key, keys' end, table row, first row, first query row, query rows
constexpr int kRowInts = 4;   // group's first unit (-1: none), group's first row
constexpr int kHeader = 8;    // tiles per CTA, tiles in all

__device__ int g_shared_prefix_error = 0;
constexpr int kErrGroups = 1, kErrPage = 2, kErrWait = 3;  // error words

__host__ __device__ inline int max_chunks(int B, int G, int Gq) { return G + (B * Gq + MR - 1) / MR; }

// ------------------------------------------------------------------------- plan
constexpr int kPlanThreads = 1024;

// inclusive scan of one value per thread (sum, or running maximum)
template <bool MAX>
__device__ __forceinline__ int block_scan(int v, int* s_warp) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v = MAX ? max(v, u) : v + u;
  }
  __syncthreads();
  if (lane == 31) s_warp[w] = v;
  __syncthreads();
  if (w == 0) {
    int x = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x = MAX ? max(x, u) : x + u;
    }
    s_warp[lane] = x;
  }
  __syncthreads();
  if (w > 0) v = MAX ? max(v, s_warp[w - 1]) : v + s_warp[w - 1];
  return v;
}

// plan: [kHeader][first unit of each CTA: ctas][units x kUnitInts][rows x kRowInts]
__global__ void __launch_bounds__(kPlanThreads)
shared_prefix_plan_kernel(const int* __restrict__ group_starts, const int* __restrict__ prefix_lens,
                          const int* __restrict__ seq_lens, int G, int B, int Gq, int nkv, int ctas,
                          int* __restrict__ plan) {
  extern __shared__ int s_mem[];  // [G+1] group starts, [G] prefix tiles, [G] leader, [units] first tile
  __shared__ int s_warp[32];
  pdl_launch_dependents();
  int* s_start = s_mem;
  int* s_tiles = s_start + G + 1;
  int* s_leader = s_tiles + G;
  int* s_first = s_leader + G;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int nc_max = max_chunks(B, G, Gq), units = nc_max + B;
  int* cta_unit = plan + kHeader;
  int* unit = cta_unit + ctas;
  int* rowinfo = unit + units * kUnitInts;
  // group starts, made ascending and kept inside [0, B]: groups never overlap
  int carry = 0;
  bool bad = false;
  for (int g0 = 0; g0 <= G; g0 += kPlanThreads) {
    const int g = g0 + tid;
    const int raw = g <= G ? group_starts[g] : 0;
    int v = block_scan<true>(max(carry, min(max(raw, 0), B)), s_warp);
    if (g <= G) {
      s_start[g] = v;
      bad |= v != raw;
    }
    __syncthreads();
    carry = s_start[min(G, g0 + kPlanThreads - 1)];
  }
  if (bad) atomicExch(&g_shared_prefix_error, kErrGroups);
  for (int b = tid; b < B; b += kPlanThreads) {
    rowinfo[b * kRowInts] = -1;
    rowinfo[b * kRowInts + 1] = 0;
  }
  __syncthreads();
  // a group shares the whole tiles that every live row of it has; one live row shares nothing
  for (int g = warp; g < G; g += kPlanThreads / 32) {
    int len = max(prefix_lens[g], 0), live = 0, leader = B;
    for (int b = s_start[g] + lane; b < s_start[g + 1]; b += 32) {
      const int L = seq_lens[b];
      if (L > 0) {
        len = min(len, L);
        leader = min(leader, b);
        ++live;
      }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      len = min(len, __shfl_xor_sync(0xffffffffu, len, o));
      leader = min(leader, __shfl_xor_sync(0xffffffffu, leader, o));
      live += __shfl_xor_sync(0xffffffffu, live, o);
    }
    if (lane == 0) {
      s_tiles[g] = live > 1 ? len / BT : 0;
      s_leader[g] = leader;
    }
  }
  __syncthreads();
  // prefix units: per group, ceil(rows * Gq / MR) chunks of its query rows
  int unit_carry = 0, tile_carry = 0;
  for (int g0 = 0; g0 < G; g0 += kPlanThreads) {
    const int g = g0 + tid;
    int chunks = 0, n = 0, start = 0, rows = 0;
    if (g < G) {
      start = s_start[g];
      rows = (s_start[g + 1] - start) * Gq;
      n = s_tiles[g];
      chunks = n > 0 ? (rows + MR - 1) / MR : 0;
    }
    const int uend = block_scan<false>(chunks, s_warp);
    const int tend = block_scan<false>(chunks * n, s_warp);
    const int u0 = unit_carry + uend - chunks, a0 = tile_carry + tend - chunks * n;
    for (int c = 0; c < chunks; ++c) {
      int* m = unit + (u0 + c) * kUnitInts;
      s_first[u0 + c] = m[0] = a0 + c * n;
      m[1] = n;
      m[2] = 0;
      m[3] = n * BT;
      m[4] = s_leader[g];
      m[5] = start;
      m[6] = c * MR;
      m[7] = min(MR, rows - c * MR);
    }
    if (chunks > 0)
      for (int b = start; b < s_start[g + 1]; ++b) {
        rowinfo[b * kRowInts] = u0;
        rowinfo[b * kRowInts + 1] = start;
      }
    __syncthreads();
    if (tid == kPlanThreads - 1) {
      s_warp[0] = unit_carry + uend;
      s_warp[1] = tile_carry + tend;
    }
    __syncthreads();
    unit_carry = s_warp[0];
    tile_carry = s_warp[1];
    __syncthreads();
  }
  for (int u = unit_carry + tid; u < nc_max; u += kPlanThreads) {  // unused prefix units
    int* m = unit + u * kUnitInts;
    s_first[u] = m[0] = tile_carry;
    m[1] = 0;
  }
  // suffix units: row b's keys behind its group's shared tiles
  for (int b0 = 0; b0 < B; b0 += kPlanThreads) {
    const int b = b0 + tid;
    int k0 = 0, k1 = 0;
    if (b < B) {
      k1 = max(seq_lens[b], 0);
      // the group of row b: the last one that starts at or before it
      int lo = 0, hi = G;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_start[mid] <= b) lo = mid + 1;
        else hi = mid;
      }
      if (lo > 0 && b < s_start[lo]) k0 = min(s_tiles[lo - 1] * BT, k1);
    }
    const int n = (k1 - k0 + BT - 1) / BT;
    const int tend = block_scan<false>(n, s_warp);
    if (b < B) {
      int* m = unit + (nc_max + b) * kUnitInts;
      s_first[nc_max + b] = m[0] = tile_carry + tend - n;
      m[1] = n;
      m[2] = k0;
      m[3] = k1;
      m[4] = b;
      m[5] = b;
      m[6] = 0;
      m[7] = Gq;
      rowinfo[b * kRowInts + 2] = k1 > 0;
    }
    __syncthreads();
    if (tid == kPlanThreads - 1) s_warp[0] = tile_carry + tend;
    __syncthreads();
    tile_carry = s_warp[0];
    __syncthreads();
  }
  const long long total = (long long)tile_carry * nkv;
  const int per = (int)((total + ctas - 1) / ctas);
  if (tid == 0) {
    plan[0] = max(per, 1);
    plan[1] = (int)total;
  }
  // every CTA's first unit: the last one that starts at or before its first tile
  for (int i = tid; i < ctas; i += kPlanThreads) {
    const long long x = (long long)i * max(per, 1);
    int u = 0;
    if (x < total) {
      const int a = (int)(x / nkv);
      int lo = 0, hi = units;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (s_first[mid] <= a) lo = mid + 1;
        else hi = mid;
      }
      u = lo - 1;
    }
    cta_unit[i] = u;
  }
}

// --------------------------------------------------------------------- attention
__device__ __forceinline__ void tma_3d(uint32_t dst, const void* tmap, uint32_t mbar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n" ::"r"(
          dst),
      "l"(tmap), "r"(mbar), "r"(x), "r"(y), "r"(z)
      : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
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

template <int HD, bool F8>
struct Cfg {
  static constexpr int RB = HD * (F8 ? 1 : 2);              // bytes of a key
  static constexpr int BOXB = RB < 128 ? RB : 128;          // bytes of a key in one box = its swizzle span
  static constexpr int NBOX = RB / BOXB;
  static constexpr int CH = BOXB / 16;                      // 16-byte chunks of a box row
  static constexpr int TILE = BT * RB;                      // bytes of K (or V) of a tile
  // stages: as many as leave room for two CTAs on an SM, at most 8
  static constexpr int RED = 2 * (HD / 4 + 2) * 32 * 4;     // merge buffer: two warps, half of the rows
  static constexpr int FIT = (112 * 1024 - RED - 1024 - 256) / (2 * TILE);
  static constexpr int ST = FIT < 8 ? FIT : 8;
  static constexpr int SMEM = 1024 + ST * 2 * TILE + RED + 256;
  static_assert(ST >= 2, "two stages at least");
  // offset of chunk c of a key, as the TMA unit's swizzle (span BOXB) places it
  static __device__ __forceinline__ int at(int row, int c) {
    const int box = c / CH, cc = c % CH;
    const int x = CH == 8 ? (row & 7) : CH == 4 ? ((row >> 1) & 3) : ((row >> 2) & 1);
    return box * BT * BOXB + (row * CH + (cc ^ x)) * 16;
  }
};

struct Args {
  const bf16* q;
  long long q_row, q_head;  // strides
  const uint8_t *k, *v;     // caches (the path without TMA)
  const int* tables;
  int table_row, n_blocks, block, box;  // table width, pages, keys per page, keys per TMA box (0: no TMA)
  const int* plan;
  int ctas, units, B, nq, nkv, Gq;
  float scale_log2;
  float *part_o, *part_ml;
};

// a position on the line of tiles
struct Cursor {
  int u, kvh, j;                    // unit, KV head, tile
  int n, k0, k1, trow, row0, r0, rn;  // of the unit
  __device__ __forceinline__ void load(const int* unit) {
    const int4 a = *reinterpret_cast<const int4*>(unit + u * kUnitInts);
    const int4 b = *reinterpret_cast<const int4*>(unit + u * kUnitInts + 4);
    n = a.y, k0 = a.z, k1 = a.w, trow = b.x, row0 = b.y, r0 = b.z, rn = b.w;
  }
  __device__ __forceinline__ void seek(const int* unit, int first_unit, int x, int nkv) {
    u = first_unit;
    load(unit);
    const int y = x - unit[u * kUnitInts] * nkv;
    kvh = y / n;
    j = y - kvh * n;
  }
  // the next tile; false when it belongs to another segment (unit or KV head)
  __device__ __forceinline__ bool next(const int* unit, int units, int nkv) {
    if (++j < n) return true;
    j = 0;
    if (++kvh < nkv) return false;
    kvh = 0;
    do {
      if (++u >= units) return false;
      load(unit);
    } while (n == 0);
    return false;
  }
};

template <int HD, bool F8>
struct Warp {  // a consumer warp's state: 16 query rows, HD dims
  using C = Cfg<HD, F8>;
  uint32_t q[HD / 16][4];
  float o[HD / 8][4];
  float m[2], l[2], c[2];  // running maximum (log2), partial sum, score factor of rows g and g + 8
  int lane, g, t;

  __device__ __forceinline__ void start(const Args& a, const Cursor& s, int wm) {
    // Q fragments.  For an e4m3 cache the products run in f16 (an e4m3 value is exact there):
    // each query row is scaled by a power of two to a maximum near 2^13, which keeps 8-bit
    // mantissas exact over 37 binades, and its dims are taken in the order in which a lane holds
    // four neighbouring bytes of a key.
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
        int ex = (int)(__float_as_uint(mx[h]) >> 23);  // biased exponent
        ex = ex == 255 ? 140 : max(ex, 30);            // infinities stay; tiny rows are scaled by 2^110
        f[h] = __uint_as_float((uint32_t)(127 + 140 - ex) << 23);   // 2^(13 - (ex - 127))
        c[h] = a.scale_log2 * __uint_as_float((uint32_t)(127 - 140 + ex) << 23);
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

  // keys [key0, key0 + BT / WK) of a tile of which the first nvalid are the row's
  template <int WK, bool PART>
  __device__ __forceinline__ void tile(uint32_t sk, uint32_t sv, int key0, int nvalid) {
    constexpr int NT = BT / WK / 8;
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
      const float mn = fmaxf(m[h], mx[h]);
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
    // O += P V; P is rounded to the type of V's product (values at most 1, sums kept in fp32)
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

template <int HD, bool F8>
__global__ void __launch_bounds__(160, 2)
shared_prefix_attn_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                          const __grid_constant__ Args a) {
  using C = Cfg<HD, F8>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  float* red = reinterpret_cast<float*>(smem_raw + (base - raw) + C::ST * 2 * C::TILE);
  uint64_t* bars = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(red) + C::RED);
  const uint32_t bar_full = smem_u32(bars), bar_empty = bar_full + 8 * C::ST;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * C::ST);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::ST; ++s) {
      mbar_init(bar_full + 8 * s, a.box ? 1 : 32);
      mbar_init(bar_empty + 8 * s, 4);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
  }
  __syncthreads();
  pdl_wait();
  const int per = a.plan[0], total = a.plan[1];
  const int x0 = (int)min((long long)total, (long long)blockIdx.x * per), x1 = min(total, x0 + per);
  if (x0 >= x1) return;
  const int* unit = a.plan + kHeader + a.ctas;
  Cursor s;
  s.seek(unit, a.plan[kHeader + blockIdx.x], x0, a.nkv);

  if (warp == 4) {
    // producer: the pages of a unit come 32 table entries at a time, one per lane
    int page0 = -1, pages = 0;
    bool fresh = true;
    int k = 0;
    for (int x = x0; x < x1 && !*abort_flag; ++x, ++k) {
      const int st = k % C::ST;
      const int key = s.k0 + s.j * BT;
      const int last = (min(key + BT, s.k1) - 1) / a.block;  // last page with keys of the tile
      if (!mbar_wait_err(bar_empty + 8 * st, ((k / C::ST) & 1) ^ 1, abort_flag, &g_shared_prefix_error, kErrWait)) break;
      const uint32_t sk = base + st * 2 * C::TILE, sv = sk + C::TILE;
      auto page = [&](int p) {  // all lanes: the page of table entry p
        if (fresh || p < page0 || p >= page0 + 32) {
          page0 = p;
          fresh = false;
          const int e = min(p + lane, a.table_row - 1);
          pages = a.tables[(long long)s.trow * a.table_row + e];
        }
        int b = __shfl_sync(0xffffffffu, pages, p - page0);
        if (b < 0 || b >= a.n_blocks || p >= a.table_row) {  // reported; a page of the cache is read instead
          if (lane == 0) atomicExch(&g_shared_prefix_error, kErrPage);
          b = 0;
        }
        return b;
      };
      if (a.box) {
        if (lane == 0) mbar_expect_tx(bar_full + 8 * st, 2 * C::TILE);
        for (int r = 0; r < BT; r += a.box) {
          // boxes behind the last key re-read its page: they are masked
          const int p = min((key + r) / a.block, last);
          const int z = page(p) * a.block + (key + r) % a.block;
          if (lane == 0)
#pragma unroll
            for (int b = 0; b < C::NBOX; ++b) {
              const uint32_t off = b * BT * C::BOXB + r * C::BOXB;
              tma_3d(sk + off, &tk, bar_full + 8 * st, b * (HD / C::NBOX), s.kvh, z);
              tma_3d(sv + off, &tv, bar_full + 8 * st, b * (HD / C::NBOX), s.kvh, z);
            }
        }
      } else {
        for (int r = 0; r < BT; ++r) {
          const int kr = min(key + r, s.k1 - 1);
          const long long slot = (long long)page(kr / a.block) * a.block + kr % a.block;
          const long long off = (slot * a.nkv + s.kvh) * C::RB;
          for (int c = lane; c < 2 * (C::RB / 16); c += 32) {
            const int cc = c % (C::RB / 16);
            const bool is_v = c >= C::RB / 16;
            cp_async16((is_v ? sv : sk) + C::at(r, cc), (is_v ? a.v : a.k) + off + cc * 16);
          }
        }
        cp_async_arrive(bar_full + 8 * st);
      }
      if (!s.next(unit, a.units, a.nkv)) fresh = true;
    }
    if (*abort_flag)  // let the copies in flight land before the block leaves
      for (int i = max(0, k - C::ST); i < k; ++i) {
        const long long t0 = clock64();
        while (!mbar_test(bar_full + 8 * (i % C::ST), (i / C::ST) & 1) && clock64() - t0 < kWaitCycles) {
        }
      }
    return;
  }

  Warp<HD, F8> w;
  w.lane = lane;
  w.g = lane >> 2;
  w.t = lane & 3;
  const int nqt = a.B * a.nq;
  bool first = true;
  int wk = 1, wm = 0, kq = 0, j0 = 0;
  for (int x = x0, k = 0; x < x1; ++x, ++k) {
    const int st = k % C::ST;
    if (first) {
      // 16 query rows a warp; with fewer rows than 64 the warps split the keys instead
      wk = s.rn <= 16 ? 4 : s.rn <= 32 ? 2 : 1;
      wm = warp / wk;
      kq = warp % wk;
      j0 = s.j;
      w.start(a, s, wm);
      first = false;
    }
    const uint32_t sk = base + st * 2 * C::TILE, sv = sk + C::TILE;
    const int nvalid = s.k1 - (s.k0 + s.j * BT);
    // a wait that ran out leaves the loops running on whatever is there: the error word tells
    mbar_wait_err(bar_full + 8 * st, (k / C::ST) & 1, abort_flag, &g_shared_prefix_error, kErrWait);
    const int key0 = kq * (BT / wk);
    if (wm * 16 < s.rn && key0 < nvalid) {
      if (wk == 1) {
        if (nvalid >= BT) w.template tile<1, false>(sk, sv, 0, BT);
        else w.template tile<1, true>(sk, sv, 0, nvalid);
      } else if (wk == 2) {
        if (nvalid >= BT) w.template tile<2, false>(sk, sv, key0, BT);
        else w.template tile<2, true>(sk, sv, key0, nvalid);
      } else {
        if (nvalid >= BT) w.template tile<4, false>(sk, sv, key0, BT);
        else w.template tile<4, true>(sk, sv, key0, nvalid);
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(bar_empty + 8 * st);
    Cursor e = s;
    const bool more = s.next(unit, a.units, a.nkv);
    if (more && x + 1 < x1) continue;
    // end of the segment e: join the warps that split its keys, then leave the partial
    w.finish_sums();
    for (int step = wk / 2; step > 0; step /= 2)
      for (int h = 0; h < 2; ++h) {
        if (h == 1 && e.rn <= 8) break;
        float* buf = red + (wk == 4 ? kq % step : wm) * (HD / 4 + 2) * 32;
        if (kq >= step && kq < 2 * step) w.put(buf, h);
        consumers_sync();
        if (kq < step) w.join(buf, h);
        consumers_sync();
      }
    if (kq == 0) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int rl = wm * 16 + w.g + 8 * h;
        if (rl < e.rn) {
          long long slot;
          if (j0 == 0) {  // the unit's first segment: a slot of the row; another one: a slot of the CTA
            const int r = e.r0 + rl;
            slot = (long long)(e.row0 + r / a.Gq) * a.nq + e.kvh * a.Gq + r % a.Gq;
            if (e.u >= a.units - a.B) slot += nqt;
          } else {
            slot = 2LL * nqt + (long long)blockIdx.x * MR + rl;
          }
          w.store(a.part_o + slot * HD, a.part_ml + slot * 2, h);
        }
      }
    }
    first = true;
  }
}

// ----------------------------------------------------------------------- combine
// One warp per (row, head): the partials of its prefix unit, then of its suffix unit, in the
// order of the keys.
template <int HD>
__global__ void __launch_bounds__(128)
shared_prefix_combine_kernel(const int* __restrict__ plan, int ctas, int units, int B, int nq, int nkv, int Gq,
                             const float* __restrict__ part_o, const float* __restrict__ part_ml, float v_scale,
                             bf16* __restrict__ out) {
  constexpr int V = HD / 32;
  pdl_launch_dependents();
  pdl_wait();
  const int i = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (i >= B * nq) return;
  const int b = i / nq, h = i - b * nq, kvh = h / Gq, hl = h - kvh * Gq;
  const int per = plan[0];
  const int* unit = plan + kHeader + ctas;
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
  auto add_unit = [&](int u, int local, long long first_slot) {
    const int n = unit[u * kUnitInts + 1];
    if (n == 0) return;
    const int x = unit[u * kUnitInts] * nkv + kvh * n;
    add(first_slot);
    for (int c = x / per + 1; c <= (x + n - 1) / per; ++c) add(2LL * nqt + (long long)c * MR + local);
  };
  if (row[2]) {  // a row without keys stays zero
    if (row[0] >= 0) {
      const int r = (b - row[1]) * Gq + hl;
      add_unit(row[0] + r / MR, r % MR, i);
    }
    add_unit(units - B + b, hl, (long long)nqt + i);
  }
  const float inv = L == 0.f ? 0.f : v_scale / L;
  bf16* po = out + (long long)i * HD + lane * V;
#pragma unroll
  for (int d = 0; d < V; ++d) po[d] = __float2bfloat16_rn(o[d] * inv);
}

// 3-D map of a cache: [pages * block keys][KV heads][dims], boxes of `box` keys of one head
CUtensorMap cache_tmap(const at::Tensor& c, int box, bool f8) {
  CUtensorMap m;
  const int hd = c.size(3), nkv = c.size(2), elt = f8 ? 1 : 2;
  const int inner = std::min(hd * elt, 128);
  cuuint64_t dims[3] = {(cuuint64_t)hd, (cuuint64_t)nkv, (cuuint64_t)(c.size(0) * c.size(1))};
  cuuint64_t strides[2] = {(cuuint64_t)hd * elt, (cuuint64_t)nkv * hd * elt};
  cuuint32_t bx[3] = {(cuuint32_t)(inner / elt), 1u, (cuuint32_t)box};
  cuuint32_t estr[3] = {1u, 1u, 1u};
  const CUtensorMapSwizzle sw = inner == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                : inner == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                              : CU_TENSOR_MAP_SWIZZLE_32B;
  CUresult r = tma_encode_fn()(&m, f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
                               c.data_ptr(), dims, strides, bx, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, sw,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "rl_b200: cuTensorMapEncodeTiled failed (", (int)r, ")");
  return m;
}

int plan_ints(int ctas, int units, int B) { return kHeader + ctas + units * kUnitInts + B * kRowInts; }
int grid_ctas() { return 2 * num_sms(); }

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
                              int64_t nkv) {
  for (const at::Tensor& t : {group_starts, prefix_lens, seq_lens})
    RLB_CHECK(t.is_cuda() && t.dim() == 1 && t.scalar_type() == at::kInt && t.is_contiguous() &&
                  t.device() == seq_lens.device(),
              "shared_prefix_plan: contiguous int32 vectors on one CUDA device expected");
  const int64_t G = prefix_lens.size(0), B = seq_lens.size(0);
  RLB_CHECK(group_starts.size(0) == G + 1, "shared_prefix_plan: group_starts needs one entry more than prefix_lens");
  RLB_CHECK(nkv >= 1 && nq >= nkv && nq % nkv == 0 && nq / nkv <= sp::MR,
            "shared_prefix_plan: query heads must be a multiple of the KV heads, at most 64 per KV head");
  RLB_CHECK(B <= 8192 && G <= 8192, "shared_prefix_plan: at most 8192 rows and groups");
  const c10::cuda::CUDAGuard guard(seq_lens.device());
  const int Gq = nq / nkv, ctas = sp::grid_ctas(), units = sp::max_chunks(B, G, Gq) + B;
  auto plan = at::empty({sp::plan_ints(ctas, units, B)}, seq_lens.options());
  const int smem = (3 * (int)G + 1 + units) * 4;
  RLB_CHECK(smem <= 200 * 1024, "shared_prefix_plan: too many rows and groups");
  cudaFuncSetAttribute(sp::shared_prefix_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  sp::shared_prefix_plan_kernel<<<1, sp::kPlanThreads, smem, stream()>>>(
      group_starts.data_ptr<int>(), prefix_lens.data_ptr<int>(), seq_lens.data_ptr<int>(), G, B, Gq, nkv, ctas,
      plan.data_ptr<int>());
  RLB_CUDA_CHECK(cudaGetLastError());
  return plan;
}

at::Tensor shared_prefix_attn(at::Tensor q, at::Tensor k_cache, at::Tensor v_cache, at::Tensor block_tables,
                              at::Tensor plan, int64_t groups, double scale, double k_scale, double v_scale) {
  RLB_CHECK(q.is_cuda() && q.dim() == 3 && q.scalar_type() == at::kBFloat16 && q.stride(2) == 1 &&
                q.stride(1) % 2 == 0 && q.stride(0) % 2 == 0 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 4 == 0,
            "shared_prefix_attn: q must be bf16 [rows, heads, dims] with even strides");
  const bool f8 = k_cache.scalar_type() == at::kFloat8_e4m3fn;
  RLB_CHECK(f8 || k_cache.scalar_type() == at::kBFloat16, "shared_prefix_attn: the cache must be bf16 or e4m3");
  RLB_CHECK(k_cache.dim() == 4 && k_cache.is_contiguous() && v_cache.is_contiguous() &&
                v_cache.sizes() == k_cache.sizes() && v_cache.scalar_type() == k_cache.scalar_type(),
            "shared_prefix_attn: contiguous caches [pages, block, KV heads, dims] of one shape and type expected");
  const int64_t B = q.size(0), nq = q.size(1), hd = q.size(2), nb = k_cache.size(0), bs = k_cache.size(1),
                nkv = k_cache.size(2);
  RLB_CHECK(hd == 32 || hd == 64 || hd == 128, "shared_prefix_attn: head_dim must be 32, 64 or 128");
  RLB_CHECK(k_cache.size(3) == hd && nkv >= 1 && nq >= nkv && nq % nkv == 0 && nq / nkv <= sp::MR,
            "shared_prefix_attn: heads of q and cache do not match");
  RLB_CHECK(nb >= 1 && bs >= 1 && nb * bs < (1LL << 31), "shared_prefix_attn: the cache needs 1 to 2^31 - 1 keys");
  RLB_CHECK(block_tables.is_cuda() && block_tables.dim() == 2 && block_tables.scalar_type() == at::kInt &&
                block_tables.is_contiguous() && block_tables.size(0) == B && (B == 0 || block_tables.size(1) >= 1),
            "shared_prefix_attn: int32 block tables [rows, pages] expected");
  const int Gq = nq / nkv, ctas = sp::grid_ctas();
  const int units = sp::max_chunks(B, groups, Gq) + B;
  RLB_CHECK(plan.is_cuda() && plan.scalar_type() == at::kInt && plan.is_contiguous() && groups >= 0 &&
                plan.numel() == sp::plan_ints(ctas, units, B),
            "shared_prefix_attn: the plan is of another batch");
  for (const at::Tensor& t : {k_cache, v_cache, block_tables, plan})
    RLB_CHECK(t.device() == q.device(), "shared_prefix_attn: all tensors must be on one device");
  for (const at::Tensor& t : {k_cache, v_cache})
    RLB_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, "shared_prefix_attn: caches must be 16-byte aligned");
  const c10::cuda::CUDAGuard guard(q.device());
  auto out = at::empty({B, nq, hd}, q.options());
  if (B == 0) return out;
  // keys of a TMA box: a power of two that divides the page, so a box never leaves its page and an
  // aligned tile is whole boxes.  Below 8 keys (a swizzle period) rows are copied one by one instead.
  int box = sp::BT;
  while (bs % box) box /= 2;
  if (box < 8) box = 0;
  const long long slots = 2 * B * nq + (long long)ctas * sp::MR;
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
  a.box = box;
  a.plan = plan.data_ptr<int>();
  a.ctas = ctas;
  a.units = units;
  a.B = B;
  a.nq = nq;
  a.nkv = nkv;
  a.Gq = Gq;
  a.scale_log2 = (float)(scale * (f8 ? k_scale : 1.0) * 1.4426950408889634);
  a.part_o = part.data_ptr<float>();
  a.part_ml = a.part_o + slots * hd;
  CUtensorMap tk = {}, tv = {};
  if (box) {
    tk = sp::cache_tmap(k_cache, box, f8);
    tv = sp::cache_tmap(v_cache, box, f8);
  }
  auto launch = [&](auto hdv, auto f8v) {
    constexpr int HD = decltype(hdv)::value;
    constexpr bool F8 = decltype(f8v)::value;
    using C = sp::Cfg<HD, F8>;
    auto kern = sp::shared_prefix_attn_kernel<HD, F8>;
    RLB_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM));
    sp::launch_pdl(kern, ctas, 160, C::SMEM, tk, tv, a);
    sp::launch_pdl(sp::shared_prefix_combine_kernel<HD>, (int)((B * nq + 3) / 4), 128, 0, (const int*)a.plan, ctas,
                   units, (int)B, (int)nq, (int)nkv, Gq, (const float*)a.part_o, (const float*)a.part_ml,
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
