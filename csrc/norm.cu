// RMSNorm forward / backward and the fused residual-add + RMSNorm.
//
// One warp per row (rows are hidden vectors of a packed token batch).  The
// forward makes two passes over the row (sum of squares, then normalise); the
// second pass re-reads from L1, so DRAM sees one read of x (and delta) and
// one write of y (and the residual sum).  bf16 rows with H % 8 == 0 use 16-byte
// vector accesses.  The backward accumulates the weight gradient per warp in
// shared memory and writes one fp32 partial row per CTA; a second kernel sums
// the partials (deterministic, no atomics).
//
// rmsnorm_fp8 is the forward whose output goes to a block-scaled fp8 projection:
// it leaves the normalised row as e4m3 with one scale per 128 values (see the
// kernel's comment).
#include "fp8_scale.cuh"

#include <cstdlib>

namespace rlb {

constexpr int kNormWarps = 4;

template <typename T>
__global__ void __launch_bounds__(kNormWarps * 32)
rmsnorm_fwd_kernel(const T* __restrict__ x, const T* __restrict__ delta, const T* __restrict__ w,
                   T* __restrict__ y, T* __restrict__ s_out, float* __restrict__ rstd, int rows, int H,
                   float eps) {
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x * kNormWarps + (threadIdx.x >> 5);
  pdl_launch_dependents();
  if (row >= rows) return;
  const T* xr = x + (size_t)row * H;
  const T* dr = delta ? delta + (size_t)row * H : nullptr;
  T* sr = s_out ? s_out + (size_t)row * H : nullptr;
  float ss = 0.f;
  const bool vec = (sizeof(T) == 2) && (H % 8 == 0);
  if (vec) {
    const int nv = H / 8;
    for (int j = lane; j < nv; j += 32) {
      float f[8];
      unpack8(reinterpret_cast<const bf16x8*>(xr)[j], f);
      if (dr) {
        float g[8];
        unpack8(reinterpret_cast<const bf16x8*>(dr)[j], g);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] += g[i];
        bf16x8 p = pack8(f);
        reinterpret_cast<bf16x8*>(sr)[j] = p;
        unpack8(p, f);  // normalise the rounded sum that is stored
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += f[i] * f[i];
    }
  } else {
    for (int j = lane; j < H; j += 32) {
      float v = to_f(xr[j]);
      if (dr) {
        T s = from_f<T>(v + to_f(dr[j]));
        sr[j] = s;
        v = to_f(s);
      }
      ss += v * v;
    }
  }
  ss = warp_sum(ss);
  const float r = rsqrtf(ss / H + eps);
  if (lane == 0) rstd[row] = r;
  const T* src = dr ? sr : xr;
  __syncwarp();
  T* yr = y + (size_t)row * H;
  if (vec) {
    const int nv = H / 8;
    for (int j = lane; j < nv; j += 32) {
      float f[8], g[8];
      unpack8(reinterpret_cast<const bf16x8*>(src)[j], f);
      unpack8(reinterpret_cast<const bf16x8*>(w)[j], g);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = f[i] * r * g[i];
      reinterpret_cast<bf16x8*>(yr)[j] = pack8(f);
    }
  } else {
    for (int j = lane; j < H; j += 32) yr[j] = from_f<T>(to_f(src[j]) * r * to_f(w[j]));
  }
}

// Few-row variant (decode batches): one 128-thread CTA per row so that a batch of
// tens of rows still spreads over many SMs.  bf16 rows with H % 8 == 0 only.
__global__ void __launch_bounds__(128)
rmsnorm_fwd_rowcta_kernel(const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ delta,
                          const __nv_bfloat16* __restrict__ w, __nv_bfloat16* __restrict__ y,
                          __nv_bfloat16* __restrict__ s_out, float* __restrict__ rstd, int H, float eps) {
  pdl_launch_dependents();
  __shared__ float red[32];
  const int row = blockIdx.x;
  const int nv = H / 8;
  const bf16x8* xr = reinterpret_cast<const bf16x8*>(x + (size_t)row * H);
  const bf16x8* dr = delta ? reinterpret_cast<const bf16x8*>(delta + (size_t)row * H) : nullptr;
  bf16x8* sr = s_out ? reinterpret_cast<bf16x8*>(s_out + (size_t)row * H) : nullptr;
  constexpr int kMaxV = 8;  // vectors per thread kept in registers (H <= 8192)
  float v[kMaxV][8];
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < kMaxV; ++k) {
    const int j = threadIdx.x + k * 128;
    if (j < nv) {
      unpack8(xr[j], v[k]);
      if (dr) {
        float d[8];
        unpack8(dr[j], d);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[k][i] += d[i];
        bf16x8 p = pack8(v[k]);
        sr[j] = p;
        unpack8(p, v[k]);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += v[k][i] * v[k][i];
    }
  }
  ss = block_sum(ss, red);
  const float r = rsqrtf(ss / H + eps);
  if (threadIdx.x == 0) rstd[row] = r;
  bf16x8* yr = reinterpret_cast<bf16x8*>(y + (size_t)row * H);
  const bf16x8* wv = reinterpret_cast<const bf16x8*>(w);
#pragma unroll
  for (int k = 0; k < kMaxV; ++k) {
    const int j = threadIdx.x + k * 128;
    if (j < nv) {
      float g[8];
      unpack8(wv[j], g);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = v[k][i] * r * g[i];
      yr[j] = pack8(v[k]);
    }
  }
}

// RMSNorm (of x + delta) with an e4m3 output, one scale per 128 values of a row:
//
//   s = x + delta (rounded to T, stored);  y = s * rsqrt(mean(s^2) + eps) * w (rounded to T)
//   scale = max|y| / 448 over 128 values (or the next power of two);  q = e4m3(y / scale)
//
// One pass over memory: 2 B of x, 2 of delta, 2 of s and 1 of q per value (bf16),
// where the separate norm and quantisation move 11.  The row stays in
// registers (packed, NV vectors of 8 per thread) between the sum of squares and
// the output, so its loads are all in flight at once; 16 neighbouring lanes hold
// the 128 values of a scale, so the maximum is a half-warp shuffle.
//
// y is rounded to T before it is quantised, and TPR threads take a row's vectors
// in the order of the unquantised kernels above: the result equals rmsnorm_fwd /
// add_rmsnorm_fwd followed by quant_fp8_group(_t) bit for bit (a NaN stays one).
// TPR = 128 is the few-row (decode) kernel, TPR = 32 the many-row one, by the same
// rule.
//
// On a B200 (bf16, with delta; the norm and the quantisation as two kernels in brackets): 16384 x 4096 in
// 93 us (237), 5.1 TB/s, bound by the latency of its loads at four blocks of 128 threads an SM, whose
// registers hold the rows; 64 x 4096 in 2.8 us (7.3), a launch and one chain of load, sum and store.
//
// Scales are row-major [rows, H/128], or (mn_major) [H/128, ld] with the padding
// rows up to ld set to 1, the layout that the hardware-scaled GEMM reads.
template <typename T>
struct alignas(8 * sizeof(T)) Vec8 {
  T v[8];
  // keeps the values packed: without it the compiler holds a second, unpacked copy of the row
  // in registers from one phase to the next
  __device__ __forceinline__ void keep() {
    uint32_t* p = reinterpret_cast<uint32_t*>(v);
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(T) / 4); ++i) asm volatile("" : "+r"(p[i]));
  }
};

// Sums and magnitudes on packed pairs (a sum of two 8- or 11-bit mantissas is rounded once either way, as in
// fp32 and then to T); scalars for fp32.
template <typename T>
__device__ __forceinline__ void add8(Vec8<T>& a, const Vec8<T>& b) {
  if constexpr (sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      reinterpret_cast<T2*>(a.v)[i] = __hadd2_rn(reinterpret_cast<T2*>(a.v)[i], reinterpret_cast<const T2*>(b.v)[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) a.v[i] += b.v[i];
  }
}
template <typename T>
__device__ __forceinline__ float amax8(const Vec8<T>& a) {
  if constexpr (sizeof(T) == 2) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    const T2* p = reinterpret_cast<const T2*>(a.v);
    const T2 m = __hmax2(__hmax2(__habs2(p[0]), __habs2(p[1])), __hmax2(__habs2(p[2]), __habs2(p[3])));
    const float r = fmaxf(to_f(m.x), to_f(m.y));
    return r == r ? r : 0.f;  // as fmaxf: a NaN counts for nothing
  } else {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(a.v[i]));
    return m;
  }
}

template <typename T, int NV, int TPR>
__global__ void __launch_bounds__(128, sizeof(T) == 2 && NV <= 16 ? 4 : 1)
rmsnorm_fp8_kernel(const T* __restrict__ x, const T* __restrict__ delta, const T* __restrict__ w,
                   T* __restrict__ s_out, __nv_fp8_e4m3* __restrict__ q, float* __restrict__ scales, int rows, int H,
                   float eps, bool pow2, int ld) {
  pdl_launch_dependents();
  __shared__ float red[32];
  const int t = TPR == 128 ? threadIdx.x : (threadIdx.x & 31);
  const int row = TPR == 128 ? blockIdx.x : blockIdx.x * 4 + (threadIdx.x >> 5);
  const int ngroups = H / 128;
  if (row >= rows) {  // padding rows of the mn-major scales (ld is 0 otherwise); uniform over a row's threads
    if (row < ld)
      for (int g = t; g < ngroups; g += TPR) scales[(size_t)g * ld + row] = 1.f;
    return;
  }
  const int nv = H / 8;
  const Vec8<T>* xr = reinterpret_cast<const Vec8<T>*>(x + (size_t)row * H);
  const Vec8<T>* dr = delta ? reinterpret_cast<const Vec8<T>*>(delta + (size_t)row * H) : nullptr;
  Vec8<T>* sr = s_out ? reinterpret_cast<Vec8<T>*>(s_out + (size_t)row * H) : nullptr;
  const Vec8<T>* wr = reinterpret_cast<const Vec8<T>*>(w);
  Vec8<T> f[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int j = t + k * TPR;
    if (j < nv) f[k] = xr[j];
  }
  float ss = 0.f;
  // loads of delta (and below of w) go LB at a time: one by one, each would wait for memory
  constexpr int LB = 4;
#pragma unroll
  for (int k0 = 0; k0 < NV; k0 += LB) {
    Vec8<T> d[LB];
    if (dr)
#pragma unroll
      for (int k = 0; k < LB; ++k)
        if (t + (k0 + k) * TPR < nv) d[k] = dr[t + (k0 + k) * TPR];
#pragma unroll
    for (int k = 0; k < LB; ++k) {
      const int j = t + (k0 + k) * TPR;
      if (j < nv) {
        if (dr) {
          add8(f[k0 + k], d[k]);
          sr[j] = f[k0 + k];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float v = to_f(f[k0 + k].v[i]);
          ss += v * v;
        }
        f[k0 + k].keep();
      }
    }
  }
  ss = TPR == 128 ? block_sum(ss, red) : warp_sum(ss);
  const float r = rsqrtf(ss / H + eps);
  // y takes the row's place; its largest magnitudes, one per vector, then per 16 lanes.
  // H % 128 == 0: a half-warp's 16 vectors are all inside the row or all outside.
  float amax[NV];
#pragma unroll
  for (int k0 = 0; k0 < NV; k0 += LB) {
    Vec8<T> g[LB];
#pragma unroll
    for (int k = 0; k < LB; ++k)
      if (t + (k0 + k) * TPR < nv) g[k] = wr[t + (k0 + k) * TPR];
#pragma unroll
    for (int k = 0; k < LB; ++k) {
      amax[k0 + k] = 0.f;
      if (t + (k0 + k) * TPR < nv) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          f[k0 + k].v[i] = from_f<T>(to_f(f[k0 + k].v[i]) * r * to_f(g[k].v[i]));
        amax[k0 + k] = amax8(f[k0 + k]);
        f[k0 + k].keep();
      }
    }
  }
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) amax[k] = fmaxf(amax[k], __shfl_xor_sync(0xffffffffu, amax[k], o));
  // lane k of a half-warp does the two divisions of its k-th scale and hands the inverse round
  const int lane16 = t & 15;
  float inv[(NV + 15) / 16];
#pragma unroll
  for (int c = 0; c < (NV + 15) / 16; ++c) {
    float m = 0.f;
#pragma unroll
    for (int k = 16 * c; k < NV && k < 16 * c + 16; ++k) m = lane16 == k - 16 * c ? amax[k] : m;
    const float sc = fp8_scale(m, pow2);
    inv[c] = 1.f / sc;
    const int g = ((t & ~15) + (16 * c + lane16) * TPR) >> 4;
    if (16 * c + lane16 < NV && g < ngroups) scales[ld ? (size_t)g * ld + row : (size_t)row * ngroups + g] = sc;
  }
  uint2* qr = reinterpret_cast<uint2*>(q + (size_t)row * H);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int j = t + k * TPR;
    const float iv = __shfl_sync(0xffffffffu, inv[k / 16], k % 16, 16);
    if (j < nv) {
      uint32_t p[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const T* y = f[k].v + 4 * h;
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(to_f(y[0]) * iv, to_f(y[1]) * iv), __NV_SATFINITE,
                                                     __NV_E4M3);
        const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(to_f(y[2]) * iv, to_f(y[3]) * iv), __NV_SATFINITE,
                                                     __NV_E4M3);
        p[h] = lo | (hi << 16);
      }
      qr[j] = make_uint2(p[0], p[1]);
    }
  }
}

// dx = r * dy * w - x * r^3 * sum(dy * w * x) / H   (+ ds)
// dw_partial[cta][h] = sum over this CTA's rows of dy * x * r
template <typename T>
__global__ void __launch_bounds__(kNormWarps * 32)
rmsnorm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x, const T* __restrict__ w,
                   const float* __restrict__ rstd, const T* __restrict__ ds, T* __restrict__ dx,
                   float* __restrict__ dw_partial, int rows, int H) {
  extern __shared__ float acc[];  // [kNormWarps][H]
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  float* my = acc + (size_t)wid * H;
  for (int j = lane; j < H; j += 32) my[j] = 0.f;
  __syncwarp();
  const bool vec = (sizeof(T) == 2) && (H % 8 == 0);
  for (int row = blockIdx.x * kNormWarps + wid; row < rows; row += gridDim.x * kNormWarps) {
    const T* dyr = dy + (size_t)row * H;
    const T* xr = x + (size_t)row * H;
    const float r = rstd[row];
    float dot = 0.f;
    if (vec) {
      for (int j = lane; j < H / 8; j += 32) {
        float a[8], b[8], c[8];
        unpack8(reinterpret_cast<const bf16x8*>(dyr)[j], a);
        unpack8(reinterpret_cast<const bf16x8*>(xr)[j], b);
        unpack8(reinterpret_cast<const bf16x8*>(w)[j], c);
#pragma unroll
        for (int i = 0; i < 8; ++i) dot += a[i] * c[i] * b[i];
      }
    } else {
      for (int j = lane; j < H; j += 32) dot += to_f(dyr[j]) * to_f(w[j]) * to_f(xr[j]);
    }
    dot = warp_sum(dot);
    const float c3 = dot * r * r * r / H;
    T* dxr = dx + (size_t)row * H;
    const T* dsr = ds ? ds + (size_t)row * H : nullptr;
    if (vec) {
      for (int j = lane; j < H / 8; j += 32) {
        float a[8], b[8], c[8], o[8];
        unpack8(reinterpret_cast<const bf16x8*>(dyr)[j], a);
        unpack8(reinterpret_cast<const bf16x8*>(xr)[j], b);
        unpack8(reinterpret_cast<const bf16x8*>(w)[j], c);
        float e[8] = {0, 0, 0, 0, 0, 0, 0, 0};
        if (dsr) unpack8(reinterpret_cast<const bf16x8*>(dsr)[j], e);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          o[i] = r * a[i] * c[i] - b[i] * c3 + e[i];
          my[j * 8 + i] += a[i] * b[i] * r;
        }
        reinterpret_cast<bf16x8*>(dxr)[j] = pack8(o);
      }
    } else {
      for (int j = lane; j < H; j += 32) {
        float a = to_f(dyr[j]), b = to_f(xr[j]);
        float o = r * a * to_f(w[j]) - b * c3 + (dsr ? to_f(dsr[j]) : 0.f);
        dxr[j] = from_f<T>(o);
        my[j] += a * b * r;
      }
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < H; j += blockDim.x) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < kNormWarps; ++k) s += acc[(size_t)k * H + j];
    dw_partial[(size_t)blockIdx.x * H + j] = s;
  }
}

__global__ void reduce_rows_kernel(const float* __restrict__ part, float* __restrict__ out, int n_rows, int H) {
  int j = blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= H) return;
  float s = 0.f;
  for (int i = 0; i < n_rows; ++i) s += part[(size_t)i * H + j];
  out[j] = s;
}

}  // namespace rlb

using namespace rlb;

// Few-row (decode) batches take the one-CTA-per-row kernel unless RLB_NORM_ROWCTA=0.
static bool use_rowcta(const at::Tensor& x, int H, int rows) {
  static int on = -1;
  if (on < 0) {
    const char* e = std::getenv("RLB_NORM_ROWCTA");
    on = (e == nullptr || e[0] != '0') ? 1 : 0;
  }
  return on == 1 && x.scalar_type() == at::kBFloat16 && H % 8 == 0 && H <= 8192 && rows < 4 * num_sms();
}

static void check_rows(const at::Tensor& x, const at::Tensor& w) {
  RLB_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(), "norm input must be a contiguous 2-D CUDA tensor");
  RLB_CHECK(w.dim() == 1 && w.size(0) == x.size(1) && w.scalar_type() == x.scalar_type(), "norm weight mismatch");
}

std::vector<at::Tensor> rmsnorm_fwd(at::Tensor x, at::Tensor w, double eps) {
  check_rows(x, w);
  const c10::cuda::CUDAGuard g(x.device());
  const int rows = x.size(0), H = x.size(1);
  auto y = at::empty_like(x);
  auto rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  if (rows == 0) return {y, rstd};
  if (use_rowcta(x, H, rows)) {
    rmsnorm_fwd_rowcta_kernel<<<rows, 128, 0, stream()>>>(
        (const __nv_bfloat16*)x.data_ptr(), nullptr, (const __nv_bfloat16*)w.data_ptr(), (__nv_bfloat16*)y.data_ptr(),
        nullptr, rstd.data_ptr<float>(), H, (float)eps);
    RLB_CUDA_CHECK(cudaGetLastError());
    return {y, rstd};
  }
  dim3 grid((rows + kNormWarps - 1) / kNormWarps);
  RLB_DISPATCH_FLOAT(x.scalar_type(), "rmsnorm_fwd", [&] {
    rmsnorm_fwd_kernel<scalar_t><<<grid, kNormWarps * 32, 0, stream()>>>(
        (const scalar_t*)x.data_ptr(), nullptr, (const scalar_t*)w.data_ptr(), (scalar_t*)y.data_ptr(), nullptr,
        rstd.data_ptr<float>(), rows, H, (float)eps);
  });
  RLB_CUDA_CHECK(cudaGetLastError());
  return {y, rstd};
}

std::vector<at::Tensor> add_rmsnorm_fwd(at::Tensor x, at::Tensor delta, at::Tensor w, double eps) {
  check_rows(x, w);
  RLB_CHECK(delta.sizes() == x.sizes() && delta.is_contiguous(), "delta shape mismatch");
  const c10::cuda::CUDAGuard g(x.device());
  const int rows = x.size(0), H = x.size(1);
  auto y = at::empty_like(x);
  auto s = at::empty_like(x);
  auto rstd = at::empty({rows}, x.options().dtype(at::kFloat));
  if (rows == 0) return {y, s, rstd};
  if (use_rowcta(x, H, rows)) {
    rmsnorm_fwd_rowcta_kernel<<<rows, 128, 0, stream()>>>(
        (const __nv_bfloat16*)x.data_ptr(), (const __nv_bfloat16*)delta.data_ptr(), (const __nv_bfloat16*)w.data_ptr(),
        (__nv_bfloat16*)y.data_ptr(), (__nv_bfloat16*)s.data_ptr(), rstd.data_ptr<float>(), H, (float)eps);
    RLB_CUDA_CHECK(cudaGetLastError());
    return {y, s, rstd};
  }
  dim3 grid((rows + kNormWarps - 1) / kNormWarps);
  RLB_DISPATCH_FLOAT(x.scalar_type(), "add_rmsnorm_fwd", [&] {
    rmsnorm_fwd_kernel<scalar_t><<<grid, kNormWarps * 32, 0, stream()>>>(
        (const scalar_t*)x.data_ptr(), (const scalar_t*)delta.data_ptr(), (const scalar_t*)w.data_ptr(),
        (scalar_t*)y.data_ptr(), (scalar_t*)s.data_ptr(), rstd.data_ptr<float>(), rows, H, (float)eps);
  });
  RLB_CUDA_CHECK(cudaGetLastError());
  return {y, s, rstd};
}

// x [.., H] -> (q like x in e4m3, scales fp32 [rows, H/128] or, mn_major, [H/128, rows rounded up to
// 128], s = x + delta when delta is given)
std::vector<at::Tensor> rmsnorm_fp8(at::Tensor x, c10::optional<at::Tensor> delta, at::Tensor w, double eps, bool pow2,
                                    bool mn_major) {
  const bool add = delta.has_value() && delta->defined();
  const int64_t H = x.dim() > 0 ? x.size(-1) : 0;
  RLB_CHECK(H >= 128 && H % 128 == 0 && H <= 16384, "rmsnorm_fp8: hidden size must be a multiple of 128, at most 16384");
  RLB_CHECK(x.is_cuda() && w.dim() == 1 && w.size(0) == H && w.scalar_type() == x.scalar_type() && w.device() == x.device(),
            "rmsnorm_fp8: weight mismatch");
  if (add)
    RLB_CHECK(delta->sizes() == x.sizes() && delta->scalar_type() == x.scalar_type() && delta->device() == x.device(),
              "rmsnorm_fp8: delta must match the input");
  const int64_t n_rows = x.numel() / H;
  RLB_CHECK(n_rows <= 0x7fffff00LL, "rmsnorm_fp8: too many rows");
  const c10::cuda::CUDAGuard g(x.device());
  const uintptr_t align = 8 * x.element_size();
  auto rows_of = [&](const at::Tensor& t) {  // contiguous, aligned to 8 values
    at::Tensor c = t.contiguous();
    return reinterpret_cast<uintptr_t>(c.data_ptr()) % align ? c.clone() : c;
  };
  x = rows_of(x);
  w = rows_of(w);
  const at::Tensor d = add ? rows_of(*delta) : at::Tensor();
  const int rows = (int)n_rows;
  const int ld = mn_major ? std::max(128, (rows + 127) / 128 * 128) : 0;
  auto f32 = x.options().dtype(at::kFloat);
  auto q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  auto scales = mn_major ? at::empty({H / 128, ld}, f32) : at::empty({rows, H / 128}, f32);
  at::Tensor s;
  std::vector<at::Tensor> out{q, scales};
  if (add) out.push_back(s = at::empty_like(x));
  const int out_rows = std::max(rows, ld);
  if (out_rows == 0) return out;
  // 128 threads a row while the rows are few, a warp a row when there are enough of them: the
  // rule of rmsnorm_fwd, whose sums it repeats.  Rows beyond 8192 values always take 128 threads.
  const bool cta = H > 8192 || use_rowcta(x, H, rows);
  RLB_DISPATCH_FLOAT(x.scalar_type(), "rmsnorm_fp8", [&] {
    auto launch = [&](auto nv, auto tpr) {
      constexpr int NV = decltype(nv)::value, TPR = decltype(tpr)::value;
      rmsnorm_fp8_kernel<scalar_t, NV, TPR><<<TPR == 128 ? out_rows : (out_rows + 3) / 4, 128, 0, stream()>>>(
          (const scalar_t*)x.data_ptr(), add ? (const scalar_t*)d.data_ptr() : nullptr,
          (const scalar_t*)w.data_ptr(), add ? (scalar_t*)s.data_ptr() : nullptr, (__nv_fp8_e4m3*)q.data_ptr(),
          scales.data_ptr<float>(), rows, (int)H, (float)eps, pow2, ld);
    };
    using std::integral_constant;
    if (cta) {
      integral_constant<int, 128> tpr;
      if (H <= 4096) launch(integral_constant<int, 4>{}, tpr);
      else if (H <= 8192) launch(integral_constant<int, 8>{}, tpr);
      else launch(integral_constant<int, 16>{}, tpr);
    } else {
      integral_constant<int, 32> tpr;
      if (H <= 2048) launch(integral_constant<int, 8>{}, tpr);
      else if (H <= 4096) launch(integral_constant<int, 16>{}, tpr);
      else launch(integral_constant<int, 32>{}, tpr);
    }
  });
  RLB_CUDA_CHECK(cudaGetLastError());
  return out;
}

static std::vector<at::Tensor> rmsnorm_bwd_impl(at::Tensor dy, at::Tensor x, at::Tensor w, at::Tensor rstd,
                                                c10::optional<at::Tensor> ds) {
  check_rows(x, w);
  RLB_CHECK(dy.sizes() == x.sizes() && dy.is_contiguous(), "dy shape mismatch");
  const c10::cuda::CUDAGuard g(x.device());
  const int rows = x.size(0), H = x.size(1);
  auto dx = at::empty_like(x);
  auto dw = at::zeros({H}, x.options().dtype(at::kFloat));
  if (rows == 0) return {dx, dw};
  int ctas = std::min((rows + kNormWarps - 1) / kNormWarps, 2 * num_sms());
  size_t smem = (size_t)kNormWarps * H * sizeof(float);
  RLB_CHECK(smem <= 200 * 1024, "hidden size too large for rmsnorm_bwd shared accumulator");
  auto part = at::empty({ctas, H}, x.options().dtype(at::kFloat));
  const void* dsp = (ds.has_value() && ds->defined()) ? ds->data_ptr() : nullptr;
  RLB_DISPATCH_FLOAT(x.scalar_type(), "rmsnorm_bwd", [&] {
    auto kern = rmsnorm_bwd_kernel<scalar_t>;
    if (smem > 48 * 1024) cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    kern<<<ctas, kNormWarps * 32, smem, stream()>>>(
        (const scalar_t*)dy.data_ptr(), (const scalar_t*)x.data_ptr(), (const scalar_t*)w.data_ptr(),
        rstd.data_ptr<float>(), (const scalar_t*)dsp, (scalar_t*)dx.data_ptr(), part.data_ptr<float>(), rows, H);
  });
  reduce_rows_kernel<<<(H + 255) / 256, 256, 0, stream()>>>(part.data_ptr<float>(), dw.data_ptr<float>(), ctas, H);
  RLB_CUDA_CHECK(cudaGetLastError());
  return {dx, dw};
}

std::vector<at::Tensor> rmsnorm_bwd(at::Tensor dy, at::Tensor x, at::Tensor w, at::Tensor rstd) {
  return rmsnorm_bwd_impl(dy, x, w, rstd, c10::nullopt);
}

std::vector<at::Tensor> rmsnorm_bwd_add(at::Tensor dy, at::Tensor x, at::Tensor w, at::Tensor rstd,
                                        c10::optional<at::Tensor> ds) {
  return rmsnorm_bwd_impl(dy, x, w, rstd, ds);
}

// ---------------------------------------------------------------------------
// Allocation-free C entry point (declared in noalloc.h, where its contract is
// described; it has no counterpart in the reference).  It launches the same
// backward kernels as rmsnorm_bwd above, with the per-CTA dw partials placed in
// a static device array instead of a freshly allocated tensor.
#include <cstdio>
#include <mutex>

#include "noalloc.h"

namespace rlb {
static __device__ __align__(256) float g_noalloc_rmsnorm_partials[RLB_NOALLOC_MAX_CTAS * RLB_NOALLOC_MAX_HIDDEN];
}  // namespace rlb

namespace {
constexpr int kNoallocMaxDevices = 64;
float* g_noalloc_scratch[kNoallocMaxDevices] = {nullptr};
std::mutex g_noalloc_mu;
thread_local char g_noalloc_err[256] = "";

int noalloc_fail(int code, const char* msg) {
  std::snprintf(g_noalloc_err, sizeof(g_noalloc_err), "%s", msg);
  return code;
}

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }
}  // namespace

extern "C" __attribute__((visibility("default"))) const char* rlb_noalloc_last_error(void) { return g_noalloc_err; }

extern "C" __attribute__((visibility("default"))) int rlb_rmsnorm_bwd_noalloc(const void* dy, const void* x,
                                                                            const void* w, const float* rstd,
                                                                            void* dx, float* dw, int rows,
                                                                            int hidden, cudaStream_t stream) {
  if (!dy || !x || !w || !rstd || !dx || !dw) return noalloc_fail(1, "rlb_rmsnorm_bwd_noalloc: null pointer");
  if (rows < 0 || hidden <= 0) return noalloc_fail(1, "rlb_rmsnorm_bwd_noalloc: rows must be >= 0 and hidden > 0");
  if (hidden > RLB_NOALLOC_MAX_HIDDEN) {
    std::snprintf(g_noalloc_err, sizeof(g_noalloc_err),
                  "rlb_rmsnorm_bwd_noalloc: hidden=%d exceeds the static scratch maximum of %d", hidden,
                  RLB_NOALLOC_MAX_HIDDEN);
    return 2;
  }
  if (hidden % 8 == 0 && !(aligned(dy, 16) && aligned(x, 16) && aligned(w, 16) && aligned(dx, 16)))
    return noalloc_fail(3, "rlb_rmsnorm_bwd_noalloc: dy, x, w and dx must be 16-byte aligned");
  if (!aligned(rstd, 4) || !aligned(dw, 4)) return noalloc_fail(3, "rlb_rmsnorm_bwd_noalloc: rstd/dw misaligned");
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return noalloc_fail(4, cudaGetErrorString(e));
  if (dev < 0 || dev >= kNoallocMaxDevices) return noalloc_fail(4, "rlb_rmsnorm_bwd_noalloc: device index too large");
  float* scratch = nullptr;
  {
    std::lock_guard<std::mutex> lock(g_noalloc_mu);
    if (g_noalloc_scratch[dev] == nullptr) {
      void* p = nullptr;
      e = cudaGetSymbolAddress(&p, rlb::g_noalloc_rmsnorm_partials);
      if (e != cudaSuccess || p == nullptr) return noalloc_fail(5, cudaGetErrorString(e));
      g_noalloc_scratch[dev] = static_cast<float*>(p);
    }
    scratch = g_noalloc_scratch[dev];
  }
  if (rows == 0) {
    e = cudaMemsetAsync(dw, 0, sizeof(float) * hidden, stream);
    return e == cudaSuccess ? 0 : noalloc_fail(6, cudaGetErrorString(e));
  }
  const int ctas = std::min((rows + kNormWarps - 1) / kNormWarps, RLB_NOALLOC_MAX_CTAS);
  const size_t smem = (size_t)kNormWarps * hidden * sizeof(float);
  auto kern = rmsnorm_bwd_kernel<__nv_bfloat16>;
  if (smem > 48 * 1024) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return noalloc_fail(6, cudaGetErrorString(e));
  }
  kern<<<ctas, kNormWarps * 32, smem, stream>>>(
      static_cast<const __nv_bfloat16*>(dy), static_cast<const __nv_bfloat16*>(x),
      static_cast<const __nv_bfloat16*>(w), rstd, nullptr, static_cast<__nv_bfloat16*>(dx), scratch, rows, hidden);
  reduce_rows_kernel<<<(hidden + 255) / 256, 256, 0, stream>>>(scratch, dw, ctas, hidden);
  e = cudaGetLastError();
  if (e != cudaSuccess) return noalloc_fail(6, cudaGetErrorString(e));
  return 0;
}
