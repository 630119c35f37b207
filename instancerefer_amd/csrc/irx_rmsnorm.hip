// irx_rmsnorm.hip — root-mean-square norm with the residual's addition, forward and backward.
//
//   h = x + r (rounded to the storage type: the norm reads what the residual stream holds), rstd = 1 / sqrt(mean(h^2) + eps), y = h rstd w
//   dx = dr = dh + rstd (w dy - h rstd mean(w dy h rstd)),   dw = sum over rows of dy h rstd
// Both directions are bound by memory: every tensor is read or written once, 16 bytes per lane, a row stays in registers between its sum and
// its use. Arithmetic and sums are 32 bits. dw: each workgroup walks rows and keeps its columns' sums in registers, the sums of all
// workgroups are then added in a fixed order (no atomics). Rows too wide for the registers, odd widths and unaligned rows take a form that
// reads the row twice, one element per lane.
// Measured: 8190 x 4096 bf16, float32 weights: forward 52 us (268 MB, 5.2 TB/s), backward 52 us (268 MB) + 4.5 us for the join of 1024
// workgroups' sums (512 workgroups: 81 us); 480 x 256 float32: 3.1, 3.4 and 3.1 us (one launch for both parts of the backward: 5.8 us).
#include "irx_common.h"

#define RMS_MAX_PARTS 1024

template <int ID> struct RmsT;
template <> struct RmsT<0> { typedef float S; };
template <> struct RmsT<1> { typedef unsigned short S; };
template <> struct RmsT<2> { typedef _Float16 S; };

template <int ID> __device__ __forceinline__ float rms_get(const void* p, long long i) {
  if constexpr (ID == 0) return static_cast<const float*>(p)[i];
  else if constexpr (ID == 1) return __uint_as_float((unsigned)static_cast<const unsigned short*>(p)[i] << 16);
  else return (float)static_cast<const _Float16*>(p)[i];
}
template <int ID> __device__ __forceinline__ float rms_round(float x) {
  if constexpr (ID == 0) return x;
  else if constexpr (ID == 1) return __uint_as_float(irx_pk_bf16(x, 0.f) << 16);
  else return (float)(_Float16)x;
}
template <int ID> __device__ __forceinline__ void rms_put(void* p, long long i, float x) {
  if constexpr (ID == 0) static_cast<float*>(p)[i] = x;
  else if constexpr (ID == 1) static_cast<unsigned short*>(p)[i] = (unsigned short)irx_pk_bf16(x, 0.f);
  else static_cast<_Float16*>(p)[i] = (_Float16)x;
}
// N consecutive elements (16 bytes of the storage type; weights may be float32 beside 16-bit tensors)
template <int ID, int N> __device__ __forceinline__ void rms_load(const void* p, long long i, float* o) {
  typedef typename RmsT<ID>::S S;
  if constexpr (N == 1) { o[0] = rms_get<ID>(p, i); return; }
  else if constexpr (ID == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      const float4 v = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + i + e);
      o[e] = v.x; o[e + 1] = v.y; o[e + 2] = v.z; o[e + 3] = v.w;
    }
  } else {
    struct alignas(16) V { S v[8]; };
    const V u = *reinterpret_cast<const V*>(static_cast<const S*>(p) + i);
#pragma unroll
    for (int e = 0; e < N; ++e) {
      if constexpr (ID == 1) o[e] = __uint_as_float((unsigned)u.v[e] << 16);
      else o[e] = (float)u.v[e];
    }
  }
}
template <int ID, int N> __device__ __forceinline__ void rms_store(void* p, long long i, const float* x) {
  typedef typename RmsT<ID>::S S;
  if constexpr (N == 1) { rms_put<ID>(p, i, x[0]); return; }
  else if constexpr (ID == 0) {
    *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(x[0], x[1], x[2], x[3]);
  } else if constexpr (ID == 1) {
    *reinterpret_cast<uint4*>(static_cast<S*>(p) + i) = make_uint4(irx_pk_bf16(x[0], x[1]), irx_pk_bf16(x[2], x[3]), irx_pk_bf16(x[4], x[5]), irx_pk_bf16(x[6], x[7]));
  } else {
    struct alignas(16) V { S v[8]; } u;
#pragma unroll
    for (int e = 0; e < N; ++e) u.v[e] = (S)x[e];
    *reinterpret_cast<V*>(static_cast<S*>(p) + i) = u;
  }
}
template <int ID, int N> __device__ __forceinline__ void rms_weight(const void* w, int w_f32, long long i, float* o) {
  if (w_f32) rms_load<0, N>(w, i, o);
  else rms_load<ID, N>(w, i, o);
}

// sum over the G threads of a row's group (a wave, or the whole workgroup of 256)
template <int G> __device__ __forceinline__ float rms_sum(float x, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, 64);
  if constexpr (G == 256) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
    __syncthreads();
    x = (red[0] + red[1]) + (red[2] + red[3]);
  }
  return x;
}

// G threads per row, N elements per load, NV loads per thread held in registers (0: the row is read again)
template <int ID, int N, int G, int NV>
__global__ __launch_bounds__(256) void k_rms_fwd(const void* x, const void* r, const void* w, int w_f32, long long rows, int cols, float eps,
                                                 void* y, void* h, float* rstd) {
  __shared__ float red[4];
  const int t = threadIdx.x % G;
  const long long row = (long long)blockIdx.x * (256 / G) + threadIdx.x / G;
  if (row >= rows) return;                                               // G = 256: the whole workgroup; G = 64: a whole wave
  const long long base = row * cols;
  const int nv = cols / N;
  float v[NV ? NV : 1][N];
  float ss = 0.f;
  auto fetch = [&](int c, float* o) __attribute__((always_inline)) {
    rms_load<ID, N>(x, base + (long long)c * N, o);
    if (r) {
      float b[N];
      rms_load<ID, N>(r, base + (long long)c * N, b);
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = rms_round<ID>(o[e] + b[e]);
    }
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = t + i * G;
      if (c < nv) {
        fetch(c, v[i]);
#pragma unroll
        for (int e = 0; e < N; ++e) ss = __builtin_fmaf(v[i][e], v[i][e], ss);
      }
    }
  } else {
    for (int c = t; c < nv; c += G) {
      fetch(c, v[0]);
#pragma unroll
      for (int e = 0; e < N; ++e) ss = __builtin_fmaf(v[0][e], v[0][e], ss);
    }
  }
  const float rs = 1.f / sqrtf(rms_sum<G>(ss, red) / (float)cols + eps);
  if (t == 0 && rstd) rstd[row] = rs;
  auto emit = [&](int c, const float* a) __attribute__((always_inline)) {
    float b[N];
    rms_weight<ID, N>(w, w_f32, (long long)c * N, b);
#pragma unroll
    for (int e = 0; e < N; ++e) b[e] = a[e] * rs * b[e];
    rms_store<ID, N>(y, base + (long long)c * N, b);
    if (h) rms_store<ID, N>(h, base + (long long)c * N, a);
  };
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * G < nv) emit(t + i * G, v[i]);
  } else {
    for (int c = t; c < nv; c += G) {
      fetch(c, v[0]);
      emit(c, v[0]);
    }
  }
}

template <int ID, int N, int G, int NV>
__global__ __launch_bounds__(256) void k_rms_bwd(const void* dy, const void* dh, const void* h, const void* w, int w_f32, const float* rstd,
                                                 long long rows, int cols, void* dx, float* part) {
  __shared__ float red[4];
  const int t = threadIdx.x % G;
  const int grp = blockIdx.x * (256 / G) + threadIdx.x / G, groups = gridDim.x * (256 / G);
  const int nv = cols / N;
  float dw[NV ? NV : 1][N], wv[NV ? NV : 1][N];
#pragma unroll
  for (int i = 0; i < (NV ? NV : 1); ++i)
#pragma unroll
    for (int e = 0; e < N; ++e) dw[i][e] = wv[i][e] = 0.f;
  if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * G < nv) rms_weight<ID, N>(w, w_f32, (long long)(t + i * G) * N, wv[i]);
  }
  for (long long row = grp; row < rows; row += groups) {                 // (the same number of turns for every thread of a group)
    const long long base = row * cols;
    const float rs = rstd[row];
    float a[NV ? NV : 1][N], g[NV ? NV : 1][N], s = 0.f;
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = t + i * G;
        if (c < nv) {
          rms_load<ID, N>(h, base + (long long)c * N, a[i]);
          rms_load<ID, N>(dy, base + (long long)c * N, g[i]);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            a[i][e] *= rs;
            dw[i][e] = __builtin_fmaf(g[i][e], a[i][e], dw[i][e]);
            g[i][e] *= wv[i][e];
            s = __builtin_fmaf(g[i][e], a[i][e], s);
          }
        }
      }
    } else {
      for (int c = t; c < nv; c += G) {
        float b[N];
        rms_load<ID, N>(h, base + (long long)c * N, a[0]);
        rms_load<ID, N>(dy, base + (long long)c * N, g[0]);
        rms_weight<ID, N>(w, w_f32, (long long)c * N, b);
#pragma unroll
        for (int e = 0; e < N; ++e) s = __builtin_fmaf(g[0][e] * b[e], a[0][e] * rs, s);
      }
    }
    const float mean = rms_sum<G>(s, red) / (float)cols;
    auto emit = [&](int c, const float* xh, const float* gw) __attribute__((always_inline)) {
      float o[N];
#pragma unroll
      for (int e = 0; e < N; ++e) o[e] = rs * (gw[e] - xh[e] * mean);
      if (dh) {
        float b[N];
        rms_load<ID, N>(dh, base + (long long)c * N, b);
#pragma unroll
        for (int e = 0; e < N; ++e) o[e] += b[e];
      }
      rms_store<ID, N>(dx, base + (long long)c * N, o);
    };
    if constexpr (NV > 0) {
#pragma unroll
      for (int i = 0; i < NV; ++i)
        if (t + i * G < nv) emit(t + i * G, a[i], g[i]);
    } else {
      for (int c = t; c < nv; c += G) {
        float b[N];
        rms_load<ID, N>(h, base + (long long)c * N, a[0]);
        rms_load<ID, N>(dy, base + (long long)c * N, g[0]);
        rms_weight<ID, N>(w, w_f32, (long long)c * N, b);
#pragma unroll
        for (int e = 0; e < N; ++e) {
          a[0][e] *= rs;
          g[0][e] *= b[e];
        }
        emit(c, a[0], g[0]);
      }
    }
  }
  if constexpr (NV > 0 && G == 64) {                                     // the four waves' sums of a column, in their order
    __shared__ float s[4][64 * NV * N];
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < N; ++e) s[wave][(t + i * 64) * N + e] = dw[i][e];
    __syncthreads();
    for (int c = threadIdx.x; c < cols; c += 256) part[(size_t)blockIdx.x * cols + c] = ((s[0][c] + s[1][c]) + s[2][c]) + s[3][c];
  } else if constexpr (NV > 0) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (t + i * G < nv)
#pragma unroll
        for (int e = 0; e < N; ++e) part[(size_t)blockIdx.x * cols + (size_t)(t + i * G) * N + e] = dw[i][e];
  }
}

// dw of the rows that do not fit the registers: one thread per column, blockIdx.y a share of the rows
template <int ID>
__global__ __launch_bounds__(256) void k_rms_dw(const void* dy, const void* h, const float* rstd, long long rows, int cols, float* part) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  const long long r0 = rows * blockIdx.y / gridDim.y, r1 = rows * (blockIdx.y + 1) / gridDim.y;
  float s = 0.f;
  for (long long r = r0; r < r1; ++r) s = __builtin_fmaf(rms_get<ID>(dy, r * cols + c), rms_get<ID>(h, r * cols + c) * rstd[r], s);
  part[(size_t)blockIdx.y * cols + c] = s;
}

// dw[c] = sum of the workgroups' sums, 32 interleaved runs per column, joined in their order
template <int ID>
__global__ __launch_bounds__(1024) void k_rms_dw_join(const float* part, int parts, int cols, void* dw, int w_f32) {
  __shared__ float s[32][33];
  const int cx = threadIdx.x & 31, ry = threadIdx.x >> 5, c = blockIdx.x * 32 + cx;
  float a = 0.f;
  if (c < cols)
#pragma unroll 4
    for (int p = ry; p < parts; p += 32) a += part[(size_t)p * cols + c];
  s[ry][cx] = a;
  __syncthreads();
  if (ry == 0 && c < cols) {
    float t = s[0][cx];
#pragma unroll
    for (int i = 1; i < 32; ++i) t += s[i][cx];
    if (w_f32) rms_put<0>(dw, c, t);
    else rms_put<ID>(dw, c, t);
  }
}

// which form a width takes: a wave per row while the row fits two loads per lane, a workgroup per row up to four, else two reads
struct RmsForm { int n, g, nv; };
static RmsForm rms_form(int cols, int dtype, bool aligned) {
  const int n = dtype == 0 ? 4 : 8;
  if (!aligned || cols % n) return {1, 256, 0};
  const int v = cols / n;
  if (v <= 64) return {n, 64, 1};
  if (v <= 128) return {n, 64, 2};
  if (v <= 256) return {n, 256, 1};
  if (v <= 512) return {n, 256, 2};
  if (v <= 1024) return {n, 256, 4};
  return {n, 256, 0};
}
// workgroups of the backward; each walks rows and leaves one sum per column
static int rms_groups(long long rows, const RmsForm& f) {
  const long long most = f.nv == 0 ? 256 : RMS_MAX_PARTS;
  const long long wgs = f.nv == 0 ? rows : (rows + 256 / f.g - 1) / (256 / f.g);
  return (int)(wgs < 1 ? 1 : wgs > most ? most : wgs);
}

extern "C" size_t irx_rms_norm_bwd_workspace_bytes(long long rows, int cols, int dtype) {
  if (rows <= 0 || cols <= 0) return 0;
  const int a = rms_groups(rows, rms_form(cols, dtype, true)), b = rms_groups(rows, rms_form(cols, dtype, false));
  return (size_t)(a > b ? a : b) * cols * sizeof(float);
}

template <int ID, int N> static void rms_launch_fwd(const RmsForm& f, const void* x, const void* r, const void* w, int wf, long long rows, int cols, float eps,
                                                    void* y, void* h, float* rstd, hipStream_t st) {
  // (a launch holds fewer than 2^32 threads: the wrapper below hands over at most 2^22 workgroups' rows at a time)
  const unsigned grid = (unsigned)((rows + 256 / f.g - 1) / (256 / f.g));
#define IRX_RMS(G_, NV_) k_rms_fwd<ID, N, G_, NV_><<<grid, 256, 0, st>>>(x, r, w, wf, rows, cols, eps, y, h, rstd)
  if constexpr (N == 1) IRX_RMS(256, 0);
  else if (f.g == 64) { if (f.nv == 1) IRX_RMS(64, 1); else IRX_RMS(64, 2); }
  else if (f.nv == 1) IRX_RMS(256, 1);
  else if (f.nv == 2) IRX_RMS(256, 2);
  else if (f.nv == 4) IRX_RMS(256, 4);
  else IRX_RMS(256, 0);
#undef IRX_RMS
}
template <int ID, int N> static void rms_launch_bwd(const RmsForm& f, int groups, const void* dy, const void* dh, const void* h, const void* w, int wf,
                                                    const float* rstd, long long rows, int cols, void* dx, float* part, hipStream_t st) {
  const long long all = (rows + 256 / f.g - 1) / (256 / f.g);
  const unsigned grid = f.nv ? (unsigned)groups : (unsigned)(all < 4096 ? all : 4096);
#define IRX_RMS(G_, NV_) k_rms_bwd<ID, N, G_, NV_><<<grid, 256, 0, st>>>(dy, dh, h, w, wf, rstd, rows, cols, dx, part)
  if constexpr (N == 1) IRX_RMS(256, 0);
  else if (f.g == 64) { if (f.nv == 1) IRX_RMS(64, 1); else IRX_RMS(64, 2); }
  else if (f.nv == 1) IRX_RMS(256, 1);
  else if (f.nv == 2) IRX_RMS(256, 2);
  else if (f.nv == 4) IRX_RMS(256, 4);
  else IRX_RMS(256, 0);
#undef IRX_RMS
}

static int rms_check(const char* who, long long rows, int cols, int dtype, const void* a, const void* b, const void* c, const void* d) {
  IRX_REQUIRE(dtype >= 0 && dtype <= 2, "%s: type %d (0 float32, 1 bfloat16, 2 float16)", who, dtype);
  IRX_REQUIRE(rows >= 0 && rows < (1ll << 31) && cols >= 1 && cols < (1 << 26), "%s: %lld rows of %d", who, rows, cols);
  IRX_REQUIRE(rows == 0 || (a && b && c && d), "%s: null tensor", who);
  return IRX_OK;
}
static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

extern "C" int irx_rms_norm_fwd(const void* x, const void* residual, const void* weight, int weight_f32, long long rows, int cols, int dtype,
                                float eps, void* y, void* h, float* rstd, void* stream) {
  if (int rc = rms_check("irx_rms_norm_fwd", rows, cols, dtype, x, weight, y, y)) return rc;
  IRX_REQUIRE(!residual || h || rows == 0, "irx_rms_norm_fwd: the sum with a residual needs an output");
  if (rows == 0) return IRX_OK;
  const RmsForm f = rms_form(cols, dtype, al16(x) && al16(residual) && al16(weight) && al16(y) && al16(h));
  hipStream_t st = (hipStream_t)stream;
  const long long step = (long long)(256 / f.g) << 22;
  const size_t elem = dtype == 0 ? 4 : 2;
  for (long long r0 = 0; r0 < rows; r0 += step) {
    const long long n = rows - r0 < step ? rows - r0 : step;
    auto from = [&](const void* p) { return p ? static_cast<const char*>(p) + (size_t)r0 * cols * elem : nullptr; };
    const void *xs = from(x), *rs = from(residual);
    void *ys = const_cast<char*>(from(y)), *hs = const_cast<char*>(from(h));
    float* sd = rstd ? rstd + r0 : nullptr;
    if (dtype == 0) f.n == 1 ? rms_launch_fwd<0, 1>(f, xs, rs, weight, 1, n, cols, eps, ys, hs, sd, st) : rms_launch_fwd<0, 4>(f, xs, rs, weight, 1, n, cols, eps, ys, hs, sd, st);
    else if (dtype == 1) f.n == 1 ? rms_launch_fwd<1, 1>(f, xs, rs, weight, weight_f32, n, cols, eps, ys, hs, sd, st) : rms_launch_fwd<1, 8>(f, xs, rs, weight, weight_f32, n, cols, eps, ys, hs, sd, st);
    else f.n == 1 ? rms_launch_fwd<2, 1>(f, xs, rs, weight, weight_f32, n, cols, eps, ys, hs, sd, st) : rms_launch_fwd<2, 8>(f, xs, rs, weight, weight_f32, n, cols, eps, ys, hs, sd, st);
  }
  IRX_CHECK_LAUNCH("irx_rms_norm_fwd");
  return IRX_OK;
}

extern "C" int irx_rms_norm_bwd(const void* dy, const void* dh, const void* h, const void* weight, int weight_f32, const float* rstd, long long rows,
                                int cols, int dtype, void* dx, void* dweight, void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = rms_check("irx_rms_norm_bwd", rows, cols, dtype, dy, h, weight, dx)) return rc;
  IRX_REQUIRE(dweight && (rstd || rows == 0), "irx_rms_norm_bwd: null tensor");
  const size_t need = irx_rms_norm_bwd_workspace_bytes(rows, cols, dtype);
  if (need && (!workspace || workspace_bytes < need)) {
    irx_set_error("irx_rms_norm_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return IRX_ERR_WORKSPACE;
  }
  hipStream_t st = (hipStream_t)stream;
  float* part = static_cast<float*>(workspace);
  int groups = 0;
  if (rows > 0) {
    const RmsForm f = rms_form(cols, dtype, al16(dy) && al16(dh) && al16(h) && al16(weight) && al16(dx));
    groups = rms_groups(rows, f);
    if (dtype == 0) f.n == 1 ? rms_launch_bwd<0, 1>(f, groups, dy, dh, h, weight, 1, rstd, rows, cols, dx, part, st) : rms_launch_bwd<0, 4>(f, groups, dy, dh, h, weight, 1, rstd, rows, cols, dx, part, st);
    else if (dtype == 1) f.n == 1 ? rms_launch_bwd<1, 1>(f, groups, dy, dh, h, weight, weight_f32, rstd, rows, cols, dx, part, st) : rms_launch_bwd<1, 8>(f, groups, dy, dh, h, weight, weight_f32, rstd, rows, cols, dx, part, st);
    else f.n == 1 ? rms_launch_bwd<2, 1>(f, groups, dy, dh, h, weight, weight_f32, rstd, rows, cols, dx, part, st) : rms_launch_bwd<2, 8>(f, groups, dy, dh, h, weight, weight_f32, rstd, rows, cols, dx, part, st);
    IRX_CHECK_LAUNCH("irx_rms_norm_bwd");
    if (f.nv == 0) {
      const dim3 grid((cols + 255) / 256, groups);
      if (dtype == 0) k_rms_dw<0><<<grid, 256, 0, st>>>(dy, h, rstd, rows, cols, part);
      else if (dtype == 1) k_rms_dw<1><<<grid, 256, 0, st>>>(dy, h, rstd, rows, cols, part);
      else k_rms_dw<2><<<grid, 256, 0, st>>>(dy, h, rstd, rows, cols, part);
      IRX_CHECK_LAUNCH("irx_rms_norm_bwd(dw)");
    }
  }
  const unsigned grid = (unsigned)((cols + 31) / 32);
  if (dtype == 0) k_rms_dw_join<0><<<grid, 1024, 0, st>>>(part, groups, cols, dweight, 1);
  else if (dtype == 1) k_rms_dw_join<1><<<grid, 1024, 0, st>>>(part, groups, cols, dweight, weight_f32);
  else k_rms_dw_join<2><<<grid, 1024, 0, st>>>(part, groups, cols, dweight, weight_f32);
  IRX_CHECK_LAUNCH("irx_rms_norm_bwd(join)");
  return IRX_OK;
}
