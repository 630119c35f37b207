// irx_optim.hip — fused Adam over ONE flat fp32 parameter buffer (all parameters / gradients / moments are views
// of four flat arrays, instancerefer_amd/optim.py). Replaces torch.optim.Adam's ~10 multi-tensor launches and
// 160 per-parameter host-side scalar reads per step with a single HBM-bound launch: 16 B/lane, 4 streams in,
// 3 streams out = 28 B/element. Semantics = torch.optim.Adam(lr, betas, eps, weight_decay) (L2 added to the
// gradient; reference scripts/train.py:121: Adam(lr=1e-3, weight_decay=1e-5)).
#include "irx_common.h"
#include <stdlib.h>

__global__ __launch_bounds__(256) void k_adam(float* __restrict__ p, const float* __restrict__ g,
                                              float* __restrict__ m, float* __restrict__ v, size_t n, float lr,
                                              float b1, float b2, float eps, float wd, float bc1, float bc2_sqrt,
                                              float grad_scale) {
  size_t i = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) * 4;
  const size_t stride = (size_t)gridDim.x * blockDim.x * 4;
  const float step_size = lr / bc1;
  for (; i + 3 < n; i += stride) {
    float4 pp = *reinterpret_cast<float4*>(p + i);
    const float4 gg = *reinterpret_cast<const float4*>(g + i);
    float4 mm = *reinterpret_cast<float4*>(m + i);
    float4 vv = *reinterpret_cast<float4*>(v + i);
    float* pa = reinterpret_cast<float*>(&pp);
    const float* ga = reinterpret_cast<const float*>(&gg);
    float* ma = reinterpret_cast<float*>(&mm);
    float* va = reinterpret_cast<float*>(&vv);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float gr = ga[j] * grad_scale + wd * pa[j];
      ma[j] = b1 * ma[j] + (1.f - b1) * gr;
      va[j] = b2 * va[j] + (1.f - b2) * gr * gr;
      const float denom = sqrtf(va[j]) / bc2_sqrt + eps;
      pa[j] -= step_size * (ma[j] / denom);
    }
    *reinterpret_cast<float4*>(p + i) = pp;
    *reinterpret_cast<float4*>(m + i) = mm;
    *reinterpret_cast<float4*>(v + i) = vv;
  }
  // tail (n not a multiple of 4): handled by the first threads of block 0
  if (blockIdx.x == 0 && threadIdx.x < (n & 3)) {
    const size_t t = (n & ~(size_t)3) + threadIdx.x;
    const float gr = g[t] * grad_scale + wd * p[t];
    m[t] = b1 * m[t] + (1.f - b1) * gr;
    v[t] = b2 * v[t] + (1.f - b2) * gr * gr;
    p[t] -= step_size * (m[t] / (sqrtf(v[t]) / bc2_sqrt + eps));
  }
}

extern "C" int irx_adam_step(float* params, const float* grads, float* exp_avg, float* exp_avg_sq, size_t n,
                             float lr, float beta1, float beta2, float eps, float weight_decay, int step,
                             float grad_scale, void* stream) {
  IRX_REQUIRE(step >= 1, "irx_adam_step: step must be >= 1");
  if (n == 0) return IRX_OK;
  IRX_REQUIRE(params && grads && exp_avg && exp_avg_sq, "irx_adam_step: null pointer");
  IRX_REQUIRE((((uintptr_t)params | (uintptr_t)grads | (uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 15) == 0,
              "irx_adam_step: buffers must be 16-byte aligned");
  const double bc1 = 1.0 - pow((double)beta1, (double)step);
  const double bc2 = 1.0 - pow((double)beta2, (double)step);
  long long blocks = (long long)((n / 4 + 255) / 256);
  if (blocks > 2048) blocks = 2048;
  if (blocks < 1) blocks = 1;
  k_adam<<<(int)blocks, 256, 0, (hipStream_t)stream>>>(params, grads, exp_avg, exp_avg_sq, n, lr, beta1, beta2, eps,
                                                        weight_decay, (float)bc1, (float)sqrt(bc2), grad_scale);
  IRX_CHECK_LAUNCH("irx_adam_step");
  return IRX_OK;
}

// ---- global gradient norm over many tensors, and clipping --------------------------------------------------------------------------
// norm = sqrt(sum g^2) (or max |g|) over all tensors, factor = min(1, max_norm / (norm + 1e-6)); a NaN norm gives a NaN factor. Bound by
// memory: one read of the gradients for the norm; the factor is applied in the Adam launch (no pass of its own) or, for a list of
// tensors, in one more read and write that is left out when the factor is 1. Squares are summed in 64 bits (no overflow at 1.8e19, and the
// double rate is far above what memory delivers): a sum per workgroup, and every workgroup that needs the norm adds those sums itself,
// in the same order — no atomics, no launch in between.
// Measured: 60 M values of mixed types (180 MB): sums 35 us (5.1 TB/s; with one load at a time 51), scaling 56 us (6.4 TB/s); 8 M values in
// 167 tensors: gathered and summed in 20 us (two launches; torch's multi-tensor copy alone 86), Adam with the factor 36 us (6.2 TB/s).

#define IRX_CLIP_TENSORS 160                 // tensors of one launch: the table travels in the kernel's arguments (3.4 of 4 KB)
#define IRX_CLIP_PARTS 1024                  // wanted number of workgroups

struct ClipTable {
  void* p[IRX_CLIP_TENSORS];
  unsigned long long n[IRX_CLIP_TENSORS];
  int first[IRX_CLIP_TENSORS + 1];           // first chunk of each tensor
  unsigned char type[IRX_CLIP_TENSORS];      // 0 float32, 1 bfloat16, 2 float16; + 4: starts on 16 bytes
  int count;
};

template <int ID> __device__ __forceinline__ float clip_get(const void* p, size_t i) {
  if constexpr (ID == 0) return static_cast<const float*>(p)[i];
  else if constexpr (ID == 1) return __uint_as_float((unsigned)static_cast<const unsigned short*>(p)[i] << 16);
  else return (float)static_cast<const _Float16*>(p)[i];
}
template <int ID> __device__ __forceinline__ void clip_scale(void* p, size_t i, float f) {
  if constexpr (ID == 0) static_cast<float*>(p)[i] *= f;
  else if constexpr (ID == 1) static_cast<unsigned short*>(p)[i] = (unsigned short)irx_pk_bf16(clip_get<1>(p, i) * f, 0.f);
  else static_cast<_Float16*>(p)[i] = (_Float16)((float)static_cast<const _Float16*>(p)[i] * f);
}

// running sum of squares or running maximum (a NaN stays)
__device__ __forceinline__ void clip_take(double& a, float x, int inf) {
  if (inf) {
    const double v = fabs((double)x);
    if (v > a || v != v) a = v;
  } else {
    a = fma((double)x, (double)x, a);
  }
}
__device__ __forceinline__ double clip_join(double a, double b, int inf) {
  if (!inf) return a + b;
  return (a != a) ? a : (b != b) ? b : (a > b ? a : b);
}
// over the workgroup of 256; every thread gets the result
__device__ __forceinline__ double clip_block(double a, int inf, double* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) a = clip_join(a, __shfl_xor(a, o, 64), inf);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
  __syncthreads();
  return clip_join(clip_join(red[0], red[1], inf), clip_join(red[2], red[3], inf), inf);
}

template <int ID> __device__ __forceinline__ double clip_range(const void* p, size_t lo, size_t hi, bool wide, int inf) {
  double a[4] = {0, 0, 0, 0};
  size_t i = lo;
  if (wide) {                                // lo is a multiple of 8
    constexpr int N = ID == 0 ? 4 : 8;
    const size_t end = lo + (hi - lo) / N * N;
    auto at = [&](size_t k) __attribute__((always_inline)) { return *reinterpret_cast<const uint4*>(static_cast<const char*>(p) + k * (ID == 0 ? 4 : 2)); };
    auto take = [&](const uint4& u) __attribute__((always_inline)) {
      const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (ID == 0) clip_take(a[e], __uint_as_float(w[e]), inf);
        else {
          unsigned short s[2] = {(unsigned short)(w[e] & 0xffffu), (unsigned short)(w[e] >> 16)};
          clip_take(a[e], clip_get<ID>(s, 0), inf);
          clip_take(a[e], clip_get<ID>(s, 1), inf);
        }
      }
    };
    constexpr size_t ONE = 256 * N;
    i = lo + (size_t)threadIdx.x * N;
    for (; i + 3 * ONE < end; i += 4 * ONE) {                            // four loads on their way at a time
      const uint4 u0 = at(i), u1 = at(i + ONE), u2 = at(i + 2 * ONE), u3 = at(i + 3 * ONE);
      take(u0);
      take(u1);
      take(u2);
      take(u3);
    }
    for (; i < end; i += ONE) take(at(i));
    i = end;
  }
  for (i += threadIdx.x; i < hi; i += 256) clip_take(a[0], clip_get<ID>(p, i), inf);
  return clip_join(clip_join(a[0], a[1], inf), clip_join(a[2], a[3], inf), inf);
}

__device__ __forceinline__ int clip_find(const ClipTable& T, int chunk) {
  int lo = 0, hi = T.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (T.first[mid] <= chunk) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

__global__ __launch_bounds__(256) void k_clip_norm(ClipTable T, unsigned long long chunk, int inf, double* parts) {
  __shared__ double red[4];
  const int t = clip_find(T, blockIdx.x);
  const size_t lo = (size_t)(blockIdx.x - T.first[t]) * chunk;
  const size_t hi = lo + chunk < T.n[t] ? lo + chunk : T.n[t];
  const bool wide = T.type[t] & 4;
  const int ty = T.type[t] & 3;
  double a = ty == 0 ? clip_range<0>(T.p[t], lo, hi, wide, inf) : ty == 1 ? clip_range<1>(T.p[t], lo, hi, wide, inf) : clip_range<2>(T.p[t], lo, hi, wide, inf);
  a = clip_block(a, inf, red);
  if (threadIdx.x == 0) parts[blockIdx.x] = a;
}

// many sums -> one, so that the workgroups that need the norm do not each add thousands
__global__ __launch_bounds__(256) void k_clip_fold(const double* parts, int n, int inf, double* out) {
  __shared__ double red[4];
  double a = 0;
  for (int i = threadIdx.x; i < n; i += 256) a = clip_join(a, parts[i], inf);
  a = clip_block(a, inf, red);
  if (threadIdx.x == 0) *out = a;
}

// the norm and the factor from the workgroups' sums (every thread; `scale`: what the gradients still have to be multiplied by)
__device__ __forceinline__ float clip_factor(const double* parts, int n, int inf, double scale, float max_norm, float* norm_out, double* red) {
  double a = 0;
  for (int i = threadIdx.x; i < n; i += 256) a = clip_join(a, parts[i], inf);
  a = clip_block(a, inf, red);
  const double norm = (inf ? a : sqrt(a)) * scale;
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  const double f = (double)max_norm / (norm + 1e-6);
  return f > 1.0 ? 1.f : (float)f;           // (NaN stays)
}

template <int ID> __device__ __forceinline__ void clip_apply(void* p, size_t lo, size_t hi, bool wide, float f) {
  size_t i = lo;
  if (wide) {
    constexpr int N = ID == 0 ? 4 : 8;
    const size_t end = lo + (hi - lo) / N * N;
    for (i = lo + (size_t)threadIdx.x * N; i < end; i += 256 * N) {
      uint4* at = reinterpret_cast<uint4*>(static_cast<char*>(p) + i * (ID == 0 ? 4 : 2));
      uint4 u = *at;
      unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (ID == 0) w[e] = __float_as_uint(__uint_as_float(w[e]) * f);
        else if constexpr (ID == 1) w[e] = irx_pk_bf16(__uint_as_float(w[e] << 16) * f, __uint_as_float(w[e] & 0xffff0000u) * f);
        else {
          typedef _Float16 h2 __attribute__((ext_vector_type(2)));
          h2 x = __builtin_bit_cast(h2, w[e]);
          x = (h2){(_Float16)((float)x[0] * f), (_Float16)((float)x[1] * f)};
          w[e] = __builtin_bit_cast(unsigned, x);
        }
      }
      *at = make_uint4(w[0], w[1], w[2], w[3]);
    }
    i = end;
  }
  for (i += threadIdx.x; i < hi; i += 256) clip_scale<ID>(p, i, f);
}

__global__ __launch_bounds__(256) void k_clip_scale(ClipTable T, unsigned long long chunk, int inf, const double* parts, int n, float max_norm,
                                                    float* norm_out) {
  __shared__ double red[4];
  const float f = clip_factor(parts, n, inf, 1.0, max_norm, norm_out, red);
  if (f == 1.f || T.count == 0) return;
  const int t = clip_find(T, blockIdx.x);
  const size_t lo = (size_t)(blockIdx.x - T.first[t]) * chunk;
  const size_t hi = lo + chunk < T.n[t] ? lo + chunk : T.n[t];
  const bool wide = T.type[t] & 4;
  const int ty = T.type[t] & 3;
  if (ty == 0) clip_apply<0>(T.p[t], lo, hi, wide, f);
  else if (ty == 1) clip_apply<1>(T.p[t], lo, hi, wide, f);
  else clip_apply<2>(T.p[t], lo, hi, wide, f);
}

// elements of a workgroup: about IRX_CLIP_PARTS workgroups in all, at least 4096 elements each, a multiple of 8
static unsigned long long clip_chunk(unsigned long long total) {
  unsigned long long c = (total + IRX_CLIP_PARTS - 1) / IRX_CLIP_PARTS;
  if (c < 4096) c = 4096;
  return (c + 7) / 8 * 8;
}

extern "C" size_t irx_clip_grads_workspace_bytes(const unsigned long long* counts_host, int n_tensors) {
  if (!counts_host || n_tensors <= 0) return 16;
  unsigned long long total = 0, parts = 0;
  for (int i = 0; i < n_tensors; ++i) total += counts_host[i];
  const unsigned long long c = clip_chunk(total);
  for (int i = 0; i < n_tensors; ++i) parts += (counts_host[i] + c - 1) / c;
  return (size_t)(parts + 2) * sizeof(double);
}

struct ClipRange { uintptr_t lo, hi; };
static int clip_cmp(const void* a, const void* b) {
  const uintptr_t x = static_cast<const ClipRange*>(a)->lo, y = static_cast<const ClipRange*>(b)->lo;
  return x < y ? -1 : x > y;
}

extern "C" int irx_clip_grads(void* const* grads_host, const int* types_host, const unsigned long long* counts_host, int n_tensors, int inf_norm,
                              float max_norm, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  IRX_REQUIRE(n_tensors >= 0 && norm, "irx_clip_grads: %d tensors, norm %p", n_tensors, (void*)norm);
  IRX_REQUIRE(max_norm >= 0.f, "irx_clip_grads: the largest norm must be >= 0");
  IRX_REQUIRE(n_tensors == 0 || (grads_host && types_host && counts_host), "irx_clip_grads: null table");
  unsigned long long total = 0;
  for (int i = 0; i < n_tensors; ++i) {
    IRX_REQUIRE(types_host[i] >= 0 && types_host[i] <= 2, "irx_clip_grads: tensor %d has type %d (0 float32, 1 bfloat16, 2 float16)", i, types_host[i]);
    IRX_REQUIRE(counts_host[i] == 0 || grads_host[i], "irx_clip_grads: tensor %d is null", i);
    IRX_REQUIRE(((uintptr_t)grads_host[i] & (types_host[i] == 0 ? 3 : 1)) == 0, "irx_clip_grads: tensor %d is not aligned to its type", i);
    IRX_REQUIRE(counts_host[i] < (1ull << 48) && (total += counts_host[i]) < (1ull << 48), "irx_clip_grads: too many values");
  }
  if (n_tensors > 1) {                       // two workgroups must not scale the same values
    ClipRange* r = static_cast<ClipRange*>(malloc(sizeof(ClipRange) * n_tensors));
    IRX_REQUIRE(r, "irx_clip_grads: out of host memory");
    int m = 0;
    for (int i = 0; i < n_tensors; ++i)
      if (counts_host[i]) r[m++] = {(uintptr_t)grads_host[i], (uintptr_t)grads_host[i] + counts_host[i] * (types_host[i] == 0 ? 4 : 2)};
    qsort(r, m, sizeof(ClipRange), clip_cmp);
    bool twice = false;
    for (int i = 1; i < m; ++i) twice |= r[i].lo < r[i - 1].hi;
    free(r);
    IRX_REQUIRE(!twice, "irx_clip_grads: two tensors share memory");
  }
  const size_t need = irx_clip_grads_workspace_bytes(counts_host, n_tensors);
  if (!workspace || workspace_bytes < need) {
    irx_set_error("irx_clip_grads: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return IRX_ERR_WORKSPACE;
  }
  IRX_REQUIRE(((uintptr_t)workspace & 7) == 0, "irx_clip_grads: workspace must start on 8 bytes");
  hipStream_t st = (hipStream_t)stream;
  double* parts = static_cast<double*>(workspace);
  const unsigned long long c = clip_chunk(total);
  ClipTable T;
  int n_parts = 0;
  // the same walk twice: the sums of every chunk, then the scaling of every chunk
  for (int pass = 0; pass < 2; ++pass) {
    double* from = parts;
    int n = n_parts;
    if (pass == 1 && n_parts > 2 * IRX_CLIP_PARTS) {
      k_clip_fold<<<1, 256, 0, st>>>(parts, n_parts, inf_norm, parts + n_parts);
      IRX_CHECK_LAUNCH("irx_clip_grads(fold)");
      from = parts + n_parts;
      n = 1;
    }
    bool said = false;
    int i = 0;
    while (i < n_tensors) {
      T.count = 0;
      int chunks = 0;
      for (; i < n_tensors && T.count < IRX_CLIP_TENSORS; ++i) {
        if (!counts_host[i]) continue;
        const int k = T.count++;
        T.p[k] = grads_host[i];
        T.n[k] = counts_host[i];
        T.first[k] = chunks;
        T.type[k] = (unsigned char)(types_host[i] | ((((uintptr_t)grads_host[i]) & 15) == 0 ? 4 : 0));
        chunks += (int)((counts_host[i] + c - 1) / c);
      }
      if (!T.count) break;
      T.first[T.count] = chunks;
      if (pass == 0) {
        k_clip_norm<<<chunks, 256, 0, st>>>(T, c, inf_norm, parts + n_parts);
        n_parts += chunks;
      } else {
        k_clip_scale<<<chunks, 256, 0, st>>>(T, c, inf_norm, from, n, max_norm, said ? nullptr : norm);
        said = true;
      }
      IRX_CHECK_LAUNCH("irx_clip_grads");
    }
    if (pass == 1 && !said) {                // nothing to clip: the norm is 0
      T.count = 0;
      k_clip_scale<<<1, 256, 0, st>>>(T, c, inf_norm, parts, 0, max_norm, norm);
      IRX_CHECK_LAUNCH("irx_clip_grads");
    }
  }
  return IRX_OK;
}

// ---- Adam with the clipping's factor ----
// k_adam with the gradients multiplied by the factor as they are read: the clipped gradients are never written. Everything else is
// k_adam's arithmetic, so a factor of 1 gives k_adam's bits.
__global__ __launch_bounds__(256) void k_adam_clip(float* __restrict__ p, const float* __restrict__ g, float* __restrict__ m,
                                                   float* __restrict__ v, size_t n, float lr, float b1, float b2, float eps, float wd,
                                                   float bc1, float bc2_sqrt, float grad_scale, const double* parts, int n_parts, int inf,
                                                   float max_norm, float* norm_out) {
  __shared__ double red[4];
  const float f = clip_factor(parts, n_parts, inf, (double)grad_scale, max_norm, norm_out, red);
  const float gs = grad_scale * f;
  const float step_size = lr / bc1;
  auto one = [&](float& pp, float gg, float& mm, float& vv) __attribute__((always_inline)) {
    // (the multiply-adds that the compiler makes of k_adam's expressions, written out)
    const float gr = __builtin_fmaf(gs, gg, wd * pp);
    mm = __builtin_fmaf(b1, mm, (1.f - b1) * gr);
    vv = __builtin_fmaf(b2, vv, gr * ((1.f - b2) * gr));
    const float denom = sqrtf(vv) / bc2_sqrt + eps;
    pp = __builtin_fmaf(-step_size, mm / denom, pp);
  };
  size_t i = ((size_t)blockIdx.x * blockDim.x + threadIdx.x) * 4;
  const size_t stride = (size_t)gridDim.x * blockDim.x * 4;
  for (; i + 3 < n; i += stride) {
    float4 pp = *reinterpret_cast<float4*>(p + i);
    const float4 gg = *reinterpret_cast<const float4*>(g + i);
    float4 mm = *reinterpret_cast<float4*>(m + i);
    float4 vv = *reinterpret_cast<float4*>(v + i);
    one(pp.x, gg.x, mm.x, vv.x);
    one(pp.y, gg.y, mm.y, vv.y);
    one(pp.z, gg.z, mm.z, vv.z);
    one(pp.w, gg.w, mm.w, vv.w);
    *reinterpret_cast<float4*>(p + i) = pp;
    *reinterpret_cast<float4*>(m + i) = mm;
    *reinterpret_cast<float4*>(v + i) = vv;
  }
  if (blockIdx.x == 0 && threadIdx.x < (n & 3)) {
    const size_t t = (n & ~(size_t)3) + threadIdx.x;
    one(p[t], g[t], m[t], v[t]);
  }
}

// ---- gathering the gradients into the flat buffer, with their norm ----
// The copy that the optimizer's gather is, and the sum of squares on the way: one read and one write, no second pass for the norm. A
// tensor that already lies in its place (src == dst) is only read.
#define IRX_GATHER_TENSORS 128               // 3.6 KB of kernel arguments
struct GatherTable {
  const float* src[IRX_GATHER_TENSORS];
  float* dst[IRX_GATHER_TENSORS];
  unsigned long long n[IRX_GATHER_TENSORS];
  int first[IRX_GATHER_TENSORS + 1];
  int count;
};

__global__ __launch_bounds__(256) void k_gather_norm(GatherTable T, unsigned long long chunk, int inf, double* parts) {
  __shared__ double red[4];
  int t = 0, top = T.count - 1;
  while (t < top) {
    const int mid = (t + top + 1) >> 1;
    if (T.first[mid] <= (int)blockIdx.x) t = mid;
    else top = mid - 1;
  }
  const size_t lo = (size_t)(blockIdx.x - T.first[t]) * chunk;
  const size_t hi = lo + chunk < T.n[t] ? lo + chunk : T.n[t];
  const float* src = T.src[t];
  float* dst = T.dst[t];
  const bool copy = src != dst;
  double a[4] = {0, 0, 0, 0};
  size_t i = lo;
  if (((((uintptr_t)src) | ((uintptr_t)dst)) & 15) == 0) {
    const size_t end = lo + (hi - lo) / 4 * 4;
    auto take = [&](size_t k, const float4& v) __attribute__((always_inline)) {
      if (copy) *reinterpret_cast<float4*>(dst + k) = v;
      clip_take(a[0], v.x, inf);
      clip_take(a[1], v.y, inf);
      clip_take(a[2], v.z, inf);
      clip_take(a[3], v.w, inf);
    };
    auto at = [&](size_t k) __attribute__((always_inline)) { return *reinterpret_cast<const float4*>(src + k); };
    i = lo + (size_t)threadIdx.x * 4;
    for (; i + 3 * 1024 < end; i += 4 * 1024) {                                  // four loads on their way at a time
      const float4 v0 = at(i), v1 = at(i + 1024), v2 = at(i + 2 * 1024), v3 = at(i + 3 * 1024);
      take(i, v0);
      take(i + 1024, v1);
      take(i + 2 * 1024, v2);
      take(i + 3 * 1024, v3);
    }
    for (; i < end; i += 1024) take(i, at(i));
    i = end;
  }
  for (i += threadIdx.x; i < hi; i += 256) {
    const float v = src[i];
    if (copy) dst[i] = v;
    clip_take(a[0], v, inf);
  }
  const double s = clip_block(clip_join(clip_join(a[0], a[1], inf), clip_join(a[2], a[3], inf), inf), inf, red);
  if (threadIdx.x == 0) parts[blockIdx.x] = s;
}

static unsigned long long gather_chunk(const unsigned long long* counts, int n, unsigned long long* parts) {
  unsigned long long total = 0, k = 0;
  for (int i = 0; i < n; ++i) total += counts[i];
  const unsigned long long c = clip_chunk(total);
  for (int i = 0; i < n; ++i) k += (counts[i] + c - 1) / c;
  *parts = k;
  return c;
}

extern "C" size_t irx_grad_gather_parts(const unsigned long long* counts_host, int n_tensors) {
  if (!counts_host || n_tensors <= 0) return 0;
  unsigned long long k;
  gather_chunk(counts_host, n_tensors, &k);
  return (size_t)k;
}

extern "C" int irx_grad_gather_norm(const float* const* src_host, float* const* dst_host, const unsigned long long* counts_host, int n_tensors,
                                    int inf_norm, void* workspace, size_t workspace_bytes, void* stream) {
  IRX_REQUIRE(n_tensors >= 0 && (n_tensors == 0 || (src_host && dst_host && counts_host)), "irx_grad_gather_norm: null table");
  for (int i = 0; i < n_tensors; ++i) {
    IRX_REQUIRE(counts_host[i] < (1ull << 40), "irx_grad_gather_norm: tensor %d has too many values", i);
    IRX_REQUIRE(counts_host[i] == 0 || (src_host[i] && dst_host[i]), "irx_grad_gather_norm: tensor %d is null", i);
    IRX_REQUIRE((((uintptr_t)src_host[i] | (uintptr_t)dst_host[i]) & 3) == 0, "irx_grad_gather_norm: tensor %d is not aligned to 4 bytes", i);
  }
  if (n_tensors == 0) return IRX_OK;
  unsigned long long k;
  const unsigned long long c = gather_chunk(counts_host, n_tensors, &k);
  if (!workspace || workspace_bytes < (k + 1) * sizeof(double)) {
    irx_set_error("irx_grad_gather_norm: workspace of %zu bytes, %llu needed", workspace_bytes, (k + 1) * 8);
    return IRX_ERR_WORKSPACE;
  }
  IRX_REQUIRE(((uintptr_t)workspace & 7) == 0, "irx_grad_gather_norm: workspace must start on 8 bytes");
  double* parts = static_cast<double*>(workspace);
  hipStream_t st = (hipStream_t)stream;
  GatherTable T;
  int done = 0;
  for (int i = 0; i < n_tensors;) {
    T.count = 0;
    int chunks = 0;
    for (; i < n_tensors && T.count < IRX_GATHER_TENSORS; ++i) {
      if (!counts_host[i]) continue;
      const int t = T.count++;
      T.src[t] = src_host[i];
      T.dst[t] = dst_host[i];
      T.n[t] = counts_host[i];
      T.first[t] = chunks;
      chunks += (int)((counts_host[i] + c - 1) / c);
    }
    if (!T.count) break;
    T.first[T.count] = chunks;
    k_gather_norm<<<chunks, 256, 0, st>>>(T, c, inf_norm, parts + done);
    IRX_CHECK_LAUNCH("irx_grad_gather_norm");
    done += chunks;
  }
  if (done > 2 * IRX_CLIP_PARTS) {
    k_clip_fold<<<1, 256, 0, st>>>(parts, done, inf_norm, parts + done);
    IRX_CHECK_LAUNCH("irx_grad_gather_norm(fold)");
  }
  return IRX_OK;
}

extern "C" int irx_adam_step_clip(float* params, const float* grads, float* exp_avg, float* exp_avg_sq, size_t n, float lr, float beta1,
                                  float beta2, float eps, float weight_decay, int step, float grad_scale, const void* norm_parts,
                                  size_t n_parts, int inf_norm, float max_norm, float* norm, void* stream) {
  IRX_REQUIRE(step >= 1, "irx_adam_step_clip: step must be >= 1");
  IRX_REQUIRE(max_norm >= 0.f, "irx_adam_step_clip: the largest norm must be >= 0");
  if (n == 0) return IRX_OK;
  IRX_REQUIRE(params && grads && exp_avg && exp_avg_sq && norm_parts, "irx_adam_step_clip: null pointer");
  IRX_REQUIRE((((uintptr_t)params | (uintptr_t)grads | (uintptr_t)exp_avg | (uintptr_t)exp_avg_sq) & 15) == 0,
              "irx_adam_step_clip: buffers must be 16-byte aligned");
  const double bc1 = 1.0 - pow((double)beta1, (double)step);
  const double bc2 = 1.0 - pow((double)beta2, (double)step);
  const double* parts = static_cast<const double*>(norm_parts);
  const bool folded = n_parts > 2 * IRX_CLIP_PARTS;                      // their sum lies behind them
  long long blocks = (long long)((n / 4 + 255) / 256);
  if (blocks > 2048) blocks = 2048;
  if (blocks < 1) blocks = 1;
  k_adam_clip<<<(int)blocks, 256, 0, (hipStream_t)stream>>>(params, grads, exp_avg, exp_avg_sq, n, lr, beta1, beta2, eps, weight_decay, (float)bc1,
                                                             (float)sqrt(bc2), grad_scale, folded ? parts + n_parts : parts, folded ? 1 : (int)n_parts,
                                                             inf_norm, max_norm, norm);
  IRX_CHECK_LAUNCH("irx_adam_step_clip");
  return IRX_OK;
}
