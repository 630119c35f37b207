// irx_attn_bwd.hip — attention over packed sequences, backward: dq, dk, dv and the gradient of the bias table.
//
// With P_ij = 2^(s_ij - m_i) / l_i from the saved row maximum and sum, D_i = out_i . dout_i and dS_ij = P_ij (dout_i . v_j - D_i):
//   dq_i = scale sum_j dS_ij k_j,   dk_j = scale sum_i dS_ij q_i,   dv_j = sum_i P_ij dout_i   (dk, dv over every query head of the group).
// Two kernels, so that every sum stays in one workgroup's registers and the order of addition never changes (no atomics on memory): one
// owns queries and walks the keys (D, dq, bias gradient), the other owns keys and walks the group's queries (dk, dv). Scores and dout . v
// are computed in both: 7 products in place of 5. Both use the transposed layouts of irx_attn.h: P and dS are operands as they come.
// P and dS are rounded to the operand type for the second products; row statistics, D, dS itself and all sums are 32 bits. D is formed
// from the stored output and what its rounding left over, where the forward kept that.
// Measured: 12289 causal rows, 8 / 2 heads of 64, float16: dq 290 us in two parts (800 TFLOP/s of its three products) and 10 for their
// join, dk / dv 382 us (810 of its four) and 16. Six causal sequences of 130 to 2719 rows, 16 / 4 heads of 128, bf16: 160 us (620), 277 us
// (480: its accumulators leave one wave per SIMD; with values in LDS and two waves 314 us, the registers spill). Bound there as the
// forward is: matrix and vector instructions take turns.
#include "irx_attn.h"

#include <type_traits>

int at_check(const char* who, const AtParams& P, int dim, int dtype, int elem);

// Sums of a 32 x 32 result block (keys down: register 4 g + r of lane half h is key 8 g + 4 h + r; queries across the 32 lanes of a half)
// along its diagonals: lane p gets the sum over key - query = 31 - p (lane 63: nothing). Key by key the running sums move one lane up and
// the key's row is added (v_mov wave_shr:1), so the row of key n ends 31 - n lanes above its queries; two chains of 16 keys at once.
// (An LDS sum per value, ds_add_f32, takes 190 clocks here, one wave at a time: 3 us for such a block and four waves.)
__device__ __forceinline__ float at_up(float x) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), 0x138, 0xf, 0xf, true)); }
__device__ __forceinline__ float at_diagonals(const float* x) {
  float a = 0.f, b = 0.f;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    at_u32x2 lo[4], hi[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {                                        // both halves' rows into lanes 0..31, zeros above
      lo[r] = __builtin_bit_cast(at_u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x[4 * g + r]), 0u, false, false));
      hi[r] = __builtin_bit_cast(at_u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x[8 + 4 * g + r]), 0u, false, false));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        a = at_up(a) + __uint_as_float(lo[r][h]);
        b = at_up(b) + __uint_as_float(hi[r][h]);
      }
  }
  const int lane = threadIdx.x & 63;                                     // the first chain's rows still lack 16 lanes
  const float up = __int_as_float(__builtin_amdgcn_ds_bpermute(((lane - 16) & 63) * 4, __float_as_int(a)));
  return b + (lane < 16 ? 0.f : up);
}

// ---- dq, D and the bias gradient by distance ----------------------------------------------------------------------------------
// Bias gradient: sum of dS over all pairs of one distance. Each wave owns an LDS array by distance and adds a block's 63 diagonals to it
// at once, one lane each (no atomics, a fixed order); distances at or beyond the clip are summed in registers.
template <class T, int D, bool BIAS>
__global__ __launch_bounds__(256, T::ESZ == 2 ? 2 : 1) void k_attn_dq(AtParams P, int total) {
  typedef AtTile<T, D> Tile;
  typedef typename T::F F;
  typedef typename T::S S;
  constexpr int STEPS = D / 16, BLOCKS = D / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  // two buffers of (keys, values); one where two and the bias arrays do not fit the 160 KB
  constexpr int BUFS = (T::ESZ == 4 && D == 128 && BIAS) ? 1 : 2;
  float* sb = reinterpret_cast<float*>(smem + 2 * BUFS * Tile::BYTES);
  const int W = 2 * P.far + 1;
  float* sd = sb + W;                                                    // [wave][W]

  const int per = gridDim.x >> 3;
  const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (id >= total) return;
  const int slot = P.slots - 1 - id % P.slots, hs = id / P.slots, head = hs % P.heads, part = hs / P.heads;

  int first;
  const AtSpan sp = at_span(P.cu_q, P.batch, P.tq, IRX_ATTN_BM, slot, &first);
  if (sp.begin >= sp.end) {
    if constexpr (BIAS)
      for (int d = threadIdx.x; d < W; d += 256) P.part[(((size_t)part * P.slots + slot) * P.heads + head) * W + d] = 0.f;
    return;
  }
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kb = 0, ke = 0;
  if (sp.seq >= 0) {
    kb = __builtin_amdgcn_readfirstlane(at_edge(P.cu_k, P.batch, P.tk, sp.seq + 1));
    ke = __builtin_amdgcn_readfirstlane(at_edge(P.cu_k, P.batch, P.tk, sp.seq + 2));
  }
  const int lk = ke > kb ? ke - kb : 0, off = lk - (sp.end - first);
  const int row0 = sp.begin + wave * 32;
  const int q = row0 + (lane & 31);
  const bool mine = q < sp.end;
  const int i0 = row0 - first;
  const int lim = !mine ? 0 : (P.causal ? min(lk, i0 + (lane & 31) + 1 + off) : lk);
  const int wave_full = row0 + 32 > sp.end ? 0 : (P.causal ? min(lk, i0 + 1 + off) : lk);
  const int wave_any = row0 >= sp.end ? 0 : (P.causal ? min(lk, min(i0 + 32, sp.end - first) + off) : lk);
  const int block_any = P.causal ? min(lk, min(sp.begin + IRX_ATTN_BM, sp.end) - first + off) : lk;
  int t0 = 0, t1 = (max(block_any, 0) + IRX_ATTN_BN - 1) / IRX_ATTN_BN;
  if (P.splits > 1) {
    const int n = t1;
    t0 = (int)((long long)n * part / P.splits);
    t1 = (int)((long long)n * (part + 1) / P.splits);
  }
  const int kvh = head / (P.heads / P.kv_heads);
  const S* kp = reinterpret_cast<const S*>(P.k.p) + kb * P.k.st + kvh * P.k.sh;
  const S* vp = reinterpret_cast<const S*>(P.v.p) + kb * P.v.st + kvh * P.v.sh;
  const float c1 = P.scale * IRX_LOG2E;

  F qf[STEPS], df[STEPS];
  float delta = 0.f, m = 0.f, inv = 0.f;
  {
    const S* qp = reinterpret_cast<const S*>(P.q.p) + q * P.q.st + head * P.q.sh + 8 * half;
    const S* dp = reinterpret_cast<const S*>(P.dout.p) + q * P.dout.st + head * P.dout.sh + 8 * half;
    const S* op = reinterpret_cast<const S*>(P.out) + ((size_t)q * P.heads + head) * D + 8 * half;
    const S* rp = reinterpret_cast<const S*>(P.rest) + ((size_t)q * P.heads + head) * D + 8 * half;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      qf[s] = mine ? at_ldg<T>(qp + 16 * s) : at_zero<T>();
      df[s] = mine ? at_ldg<T>(dp + 16 * s) : at_zero<T>();
      const F of = mine ? at_ldg<T>(op + 16 * s) : at_zero<T>();
      const F rf = mine && P.rest ? at_ldg<T>(rp + 16 * s) : at_zero<T>();
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(at_get<T>(of, e) + at_get<T>(rf, e), at_get<T>(df[s], e), delta);
    }
    delta = at_pair_sum(delta);
    if (mine) {
      const float* st = P.stats + ((size_t)head * P.tq + q) * 2;
      m = st[0];
      inv = st[1];
      if (half == 0 && part == 0) P.delta[(size_t)head * P.tq + q] = delta;
    }
  }
  if constexpr (BIAS) {
    at_load_bias<T>(sb, P, head);
    for (int d = threadIdx.x; d < 4 * W; d += 256) sd[d] = 0.f;
  }
  float* mysd = sd + wave * W + P.far;                                   // indexed by distance
  float below = 0.f, above = 0.f;

  at_f32x16 acc[BLOCKS];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[b][i] = 0.f;

  const unsigned lds0 = at_lds_addr(smem);
  const long long ks = P.k.st * T::ESZ, vs = P.v.st * T::ESZ;
  unsigned ko[Tile::CHUNKS], vo[Tile::CHUNKS];
  Tile::dma_offsets(ko, ks);
  Tile::dma_offsets(vo, vs);
  auto fetch = [&](int t) __attribute__((always_inline)) {
    const unsigned to = lds0 + ((t - t0) % BUFS) * 2 * Tile::BYTES;
    const int k0 = t * IRX_ATTN_BN;
    Tile::dma(to, kp + k0 * P.k.st, ks, lk - k0, ko);
    Tile::dma(to + Tile::BYTES, vp + k0 * P.v.st, vs, lk - k0, vo);
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    const int k0 = t * IRX_ATTN_BN;
    at_landed();
    __syncthreads();
    if (BUFS == 2 && t + 1 < t1) fetch(t + 1);
    const unsigned char* lk_ = smem + ((t - t0) % BUFS) * 2 * Tile::BYTES;
    const unsigned char* lv_ = lk_ + Tile::BYTES;
#pragma unroll
    for (int kb2 = 0; kb2 < 2; ++kb2) {
      const int k1 = k0 + 32 * kb2;
      if (k1 >= wave_any) break;
      at_f32x16 x, y;
      __builtin_amdgcn_iglp_opt(1);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = y[i] = 0.f;
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        x = at_mma(Tile::row_frag(lk_, 32 * kb2, st), qf[st], x);
        y = at_mma(Tile::row_frag(lv_, 32 * kb2, st), df[st], y);
      }
      float p[16];
      bool near = false, inside = false;
      const int d0 = k1 + 4 * half - (i0 + (lane & 31) + off);
      if constexpr (BIAS) {
        const int lo = k1 - (i0 + 31 + off), hi = k1 + 31 - (i0 + off);
        near = !(hi <= -P.far || lo >= P.far);
        inside = lo > -P.far && hi < P.far;
        if (!near) {                                                     // (never bias - m first: the forward rounds score + bias)
          const float b = sb[hi <= -P.far ? 0 : 2 * P.far];
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = at_exp2(__builtin_fmaf(x[i], c1, b) - m) * inv;
        } else if (inside) {
          const float* b = sb + d0 + P.far;
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = at_exp2(__builtin_fmaf(x[i], c1, b[8 * (i >> 2) + (i & 3)]) - m) * inv;
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int d = d0 + 8 * (i >> 2) + (i & 3);
            p[i] = at_exp2(__builtin_fmaf(x[i], c1, sb[min(max(d, -P.far), P.far) + P.far]) - m) * inv;
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = at_exp2(__builtin_fmaf(x[i], c1, -m)) * inv;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] *= y[i] - delta;                 // dS
      if (k1 + 32 > wave_full) {
        const int left = lim - k1 - 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = 8 * (i >> 2) + (i & 3) < left ? p[i] : 0.f;
      }
      if constexpr (BIAS) {
        if (near) {
          const float z = at_diagonals(p);
          const int d = k1 - (i0 + off) + 31 - lane;
          if (lane < 63) {
            if (d <= -P.far) below += z;
            else if (d >= P.far) above += z;
            else mysd[d] += z;
          }
        } else {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) s += p[i];
          if (k1 - (i0 + off) <= -P.far) below += s;
          else above += s;
        }
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const F f = at_pack<T>(p + 8 * ks);
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) acc[b] = at_mma(Tile::col_frag(lk_, 32 * kb2 + 16 * ks, b), f, acc[b]);
      }
    }
    if (BUFS == 1) {
      __syncthreads();
      if (t + 1 < t1) fetch(t + 1);
    }
  }
  if constexpr (BIAS) {
    __syncthreads();                                                     // (no tile at all: the zeros above are another thread's)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      below += __shfl_xor(below, o, 64);
      above += __shfl_xor(above, o, 64);
    }
    if (lane == 0) {                                                     // nobody else adds to the clipped distances
      if (P.far == 0) mysd[0] = below + above;
      else {
        mysd[-P.far] = below;
        mysd[P.far] = above;
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < W; d += 256) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) s += sd[w * W + d];
      P.part[(((size_t)part * P.slots + slot) * P.heads + head) * W + d] = s;
    }
  }
  if (!mine) return;
  const size_t at = ((size_t)q * P.heads + head) * D + 4 * half;
  if (P.splits > 1) {
    float* o = P.so + (size_t)part * P.tq * P.heads * D + at;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        at_st4<AtF32>(o + 32 * b + 8 * g, acc[b][4 * g], acc[b][4 * g + 1], acc[b][4 * g + 2], acc[b][4 * g + 3]);
    return;
  }
  S* o = reinterpret_cast<S*>(P.dst) + at;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      at_st4<T>(o + 32 * b + 8 * g, acc[b][4 * g] * P.scale, acc[b][4 * g + 1] * P.scale, acc[b][4 * g + 2] * P.scale, acc[b][4 * g + 3] * P.scale);
}

// adds the parts of dq in their order and rounds
template <class T>
__global__ __launch_bounds__(256) void k_attn_dq_join(AtParams P, size_t n) {
  const size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  at_f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < P.splits; ++p) s += *reinterpret_cast<const at_f32x4*>(P.so + p * n + at);
  at_st4<T>(reinterpret_cast<typename T::S*>(P.dst) + at, s[0] * P.scale, s[1] * P.scale, s[2] * P.scale, s[3] * P.scale);
}

// ---- bias gradient: distances -> buckets, over all tiles -----------------------------------------------------------------------
// One workgroup per (bucket, head): lists the bucket's distances in order, then adds their partial sums of every tile (64 bits, fixed order).
// These workgroups are the last ones of the dk / dv launch, where they fill its tail; a launch of their own took 5 to 9 us (32 sequences
// of 61 to 700 rows, 8 heads of 64, bf16, forward and backward: 184 -> 178 us).
template <class T> __device__ __forceinline__ void at_dbias(const AtParams& P, int slots, int bucket, int head, unsigned char* smem) {
  int* list = reinterpret_cast<int*>(smem);
  int* kind = list + 2 * IRX_ATTN_MAX_FAR + 1;
  double* red = reinterpret_cast<double*>(smem + (2 * (2 * IRX_ATTN_MAX_FAR + 1) * sizeof(int) + 15) / 16 * 16);
  int* count = reinterpret_cast<int*>(red + 4);
  const int heads = P.heads, far = P.far, buckets = P.buckets, W = 2 * far + 1;
  const int32_t* map = P.map;
  const float* part = P.part;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int d = threadIdx.x; d < W; d += 256) {
    const int b = map[d];
    kind[d] = b < 0 ? 0 : (b >= buckets ? buckets - 1 : b);
  }
  __syncthreads();
  if (wave == 0) {
    int n = 0;
    for (int base = 0; base < W; base += 64) {
      const int d = base + lane;
      const bool in = d < W && kind[d < W ? d : 0] == bucket;
      const unsigned long long hit = __ballot(in);
      if (in) list[n + __popcll(hit & ((1ull << lane) - 1))] = d;
      n += __popcll(hit);
    }
    if (lane == 0) *count = n;
  }
  __syncthreads();
  const int c = *count;
  double s = 0;
  if (c) {
    const long long n = (long long)slots * c;
    const long long step = (1 << 30) / c * (long long)c;                 // whole tiles at a time, so that the divisions below are 32 bits
    for (long long from = 0; from < n; from += step) {
      const float* p0 = part + (size_t)(from / c) * heads * W;
      const int m = (int)(n - from < step ? n - from : step);
#pragma unroll 4
      for (int i = threadIdx.x; i < m; i += 256) s += (double)p0[((size_t)(i / c) * heads + head) * W + list[i % c]];
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    const float x = (float)(((red[0] + red[1]) + red[2]) + red[3]);
    const size_t at = (size_t)bucket * heads + head;
    if (P.table_f32 || T::ID == IRX_ATTN_F32) reinterpret_cast<float*>(P.dtable)[at] = x;
    else if constexpr (T::ID == IRX_ATTN_BF16) reinterpret_cast<unsigned short*>(P.dtable)[at] = (unsigned short)irx_pk_bf16(x, 0.f);
    else reinterpret_cast<_Float16*>(P.dtable)[at] = (_Float16)x;
  }
}

// ---- dk, dv -----------------------------------------------------------------------------------------------------------------------
template <class T, int D, bool BIAS>
__global__ __launch_bounds__(256, (T::ESZ == 2 && D <= 64) ? 2 : 1) void k_attn_dkv(AtParams P, int total, int q_slots) {
  typedef AtTile<T, D> Tile;
  typedef typename T::F F;
  typedef typename T::S S;
  constexpr int STEPS = D / 16, BLOCKS = D / 32;
  // float16 keeps 10 bits below 2^-14: weights of long rows are that small, so they go through the product times 2^10
  constexpr float UP = T::ID == IRX_ATTN_F16 ? 1024.f : 1.f;
  static_assert(4 * Tile::BYTES >= 16384, "the bias gradient's lists lie in the tiles' place");
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  float* srow = reinterpret_cast<float*>(smem + 4 * Tile::BYTES);        // [buffer][row maxima | 1 / row sums | D][64 queries]
  float* sb = srow + 6 * IRX_ATTN_BN;

  const int per = (total + 7) >> 3;
  if constexpr (BIAS) {
    const int extra = (int)blockIdx.x - 8 * per;
    if (extra >= 0) {
      at_dbias<T>(P, q_slots, extra % P.buckets, extra / P.buckets, smem);
      return;
    }
  }
  const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (id >= total) return;
  const int slot = id % P.slots, rest = id / P.slots, kvh = rest % P.kv_heads, part = rest / P.kv_heads;

  int first;
  const AtSpan sp = at_span(P.cu_k, P.batch, P.tk, IRX_ATTN_BM, slot, &first);
  if (sp.begin >= sp.end) return;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int qb = 0, qe = 0;
  if (sp.seq >= 0) {
    qb = __builtin_amdgcn_readfirstlane(at_edge(P.cu_q, P.batch, P.tq, sp.seq + 1));
    qe = __builtin_amdgcn_readfirstlane(at_edge(P.cu_q, P.batch, P.tq, sp.seq + 2));
  }
  const int lq = qe > qb ? qe - qb : 0, off = (sp.end - first) - lq;
  const int row0 = sp.begin + wave * 32;
  const int key = row0 + (lane & 31);
  const bool mine = key < sp.end;
  const int j0 = row0 - first, j = j0 + (lane & 31);                     // index in the sequence
  const int from = P.causal ? j - off : 0;                               // queries [from, lq) see this lane's key
  const int wave_full = P.causal ? j0 + 31 - off : 0;                    // ... every key of the wave
  const int wave_any = P.causal ? j0 - off : 0;
  const int block_any = P.causal ? max(sp.begin - first - off, 0) : 0;
  const int group = P.heads / P.kv_heads;
  const float c1 = P.scale * IRX_LOG2E;

  F kf[STEPS], vf[STEPS];
  {
    const S* kp = reinterpret_cast<const S*>(P.k.p) + key * P.k.st + kvh * P.k.sh + 8 * half;
    const S* vp = reinterpret_cast<const S*>(P.v.p) + key * P.v.st + kvh * P.v.sh + 8 * half;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      kf[s] = mine ? at_ldg<T>(kp + 16 * s) : at_zero<T>();
      vf[s] = mine ? at_ldg<T>(vp + 16 * s) : at_zero<T>();
    }
  }
  at_f32x16 dk[BLOCKS], dv[BLOCKS];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) dk[b][i] = dv[b][i] = 0.f;

  // items (query head of the group, tile of 64 queries), in order; a launch with few workgroups gives each a part of them
  const int tile0 = block_any / IRX_ATTN_BN, tiles = max((lq + IRX_ATTN_BN - 1) / IRX_ATTN_BN - tile0, 0);
  const int it0 = (int)((long long)group * tiles * part / P.splits), it1 = (int)((long long)group * tiles * (part + 1) / P.splits);
  const unsigned lds0 = at_lds_addr(smem);
  const long long qs = P.q.st * T::ESZ, os = P.dout.st * T::ESZ;
  unsigned qo[Tile::CHUNKS], oo[Tile::CHUNKS];
  Tile::dma_offsets(qo, qs);
  Tile::dma_offsets(oo, os);
  float rm = 0.f, ri = 0.f, rd = 0.f;                                    // row statistics on their way (threads 0..63)
  // head of the group and tile of the item that is fetched next / worked on
  int fg = tiles ? it0 / tiles : 0, ft = it0 - fg * tiles, g = fg, tl = ft;
  auto fetch = [&](int it) __attribute__((always_inline)) {
    const int head = kvh * group + fg, q0 = (tile0 + ft) * IRX_ATTN_BN;
    if (++ft == tiles) {
      ft = 0;
      ++fg;
    }
    if (threadIdx.x < IRX_ATTN_BN) {
      const int r = q0 + (int)threadIdx.x;
      rm = ri = rd = 0.f;
      if (r < lq) {
        const size_t at = (size_t)head * P.tq + qb + r;
        rm = P.stats[2 * at];
        ri = P.stats[2 * at + 1];
        rd = P.delta[at];
      }
    }
    const unsigned to = lds0 + ((it - it0) & 1) * 2 * Tile::BYTES;
    Tile::dma(to, reinterpret_cast<const S*>(P.q.p) + (qb + q0) * P.q.st + head * P.q.sh, qs, lq - q0, qo);
    Tile::dma(to + Tile::BYTES, reinterpret_cast<const S*>(P.dout.p) + (qb + q0) * P.dout.st + head * P.dout.sh, os, lq - q0, oo);
  };
  if (it0 < it1) fetch(it0);
  int bias_head = -1;
  for (int it = it0; it < it1; ++it) {
    const int q0 = (tile0 + tl) * IRX_ATTN_BN;
    const unsigned char* lq_ = smem + ((it - it0) & 1) * 2 * Tile::BYTES;
    const unsigned char* ld_ = lq_ + Tile::BYTES;
    float* sm = srow + ((it - it0) & 1) * 3 * IRX_ATTN_BN;
    float* si = sm + IRX_ATTN_BN;
    float* se = si + IRX_ATTN_BN;
    at_landed();
    if (threadIdx.x < IRX_ATTN_BN) {
      sm[threadIdx.x] = rm;
      si[threadIdx.x] = ri * UP;
      se[threadIdx.x] = rd * (1.f / UP);
    }
    __syncthreads();
    if (it + 1 < it1) fetch(it + 1);
    if constexpr (BIAS) {
      if (bias_head != g) {                                              // (nobody reads the old one any more: the barrier above)
        bias_head = g;
        at_load_bias<T>(sb, P, kvh * group + g);
        __syncthreads();
      }
    }
    if (++tl == tiles) {
      tl = 0;
      ++g;
    }
    auto scores = [&](int qb2, at_f32x16& x, at_f32x16& y) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = y[i] = 0.f;
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        x = at_mma(Tile::row_frag(lq_, 32 * qb2, st), kf[st], x);
        y = at_mma(Tile::row_frag(ld_, 32 * qb2, st), vf[st], y);
      }
    };
    auto weights = [&](auto edge, int qb2, const at_f32x16& x, const at_f32x16& y, F (&pf)[2], F (&sf)[2]) __attribute__((always_inline)) {
      const int q1 = q0 + 32 * qb2;
      float bias[16];
      if constexpr (BIAS) {
        const int lo = j0 - (q1 + 31 + off), hi = j0 + 31 - (q1 + off);  // distances key - query in this block
        const int d0 = j - (q1 + 4 * half + off);                        // of register i: d0 - 8 (i / 4) - i % 4
        if (hi <= -P.far || lo >= P.far) {
          const float b = sb[hi <= -P.far ? 0 : 2 * P.far];
#pragma unroll
          for (int i = 0; i < 16; ++i) bias[i] = b;
        } else if (lo >= -P.far && hi <= P.far) {
          const float* b = sb + d0 + P.far;
#pragma unroll
          for (int i = 0; i < 16; ++i) bias[i] = b[-(8 * (i >> 2) + (i & 3))];
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) bias[i] = sb[min(max(d0 - 8 * (i >> 2) - (i & 3), -P.far), P.far) + P.far];
        }
      }
      float p[16], ds[16];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int at = 32 * qb2 + 8 * r + 4 * half;
        const at_f32x4 m4 = *reinterpret_cast<const at_f32x4*>(sm + at);
        const at_f32x4 i4 = *reinterpret_cast<const at_f32x4*>(si + at);
        const at_f32x4 e4 = *reinterpret_cast<const at_f32x4*>(se + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * r + e;
          p[i] = at_exp2(BIAS ? __builtin_fmaf(x[i], c1, bias[i]) - m4[e] : __builtin_fmaf(x[i], c1, -m4[e])) * i4[e];
          ds[i] = p[i] * __builtin_fmaf(y[i], 1.f / UP, -e4[e]);
          if constexpr (edge) {
            const int qi = q0 + at + e;
            const bool see = qi >= from && qi < lq;
            p[i] = see ? p[i] : 0.f;
            ds[i] = see ? ds[i] : 0.f;
          }
        }
      }
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        pf[ks] = at_pack<T>(p + 8 * ks);
        sf[ks] = at_pack<T>(ds + 8 * ks);
      }
    };
    auto sums = [&](int qb2, const F (&pf)[2], const F (&sf)[2]) __attribute__((always_inline)) {
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
          dv[b] = at_mma(Tile::col_frag(ld_, 32 * qb2 + 16 * ks, b), pf[ks], dv[b]);
          dk[b] = at_mma(Tile::col_frag(lq_, 32 * qb2 + 16 * ks, b), sf[ks], dk[b]);
        }
    };
    if (row0 >= sp.end) continue;
#pragma unroll
    for (int qb2 = 0; qb2 < 2; ++qb2) {
      const int q1 = q0 + 32 * qb2;
      if (q1 + 31 < wave_any || q1 >= lq) continue;
      at_f32x16 x, y;
      F pf[2], sf[2];
      __builtin_amdgcn_iglp_opt(1);                                      // LDS reads between the matrix instructions: 3 % at dimension 128
      scores(qb2, x, y);
      if (q1 < wave_full || q1 + 32 > lq) weights(std::true_type{}, qb2, x, y, pf, sf);
      else weights(std::false_type{}, qb2, x, y, pf, sf);
      sums(qb2, pf, sf);
    }
  }
  if (!mine) return;
  const size_t at = ((size_t)key * P.kv_heads + kvh) * D + 4 * half;
  if (P.splits > 1) {
    const size_t one = (size_t)P.tk * P.kv_heads * D;
    float* ok = P.so + 2 * part * one + at;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        at_st4<AtF32>(ok + 32 * b + 8 * r, dk[b][4 * r], dk[b][4 * r + 1], dk[b][4 * r + 2], dk[b][4 * r + 3]);
        at_st4<AtF32>(ok + one + 32 * b + 8 * r, dv[b][4 * r], dv[b][4 * r + 1], dv[b][4 * r + 2], dv[b][4 * r + 3]);
      }
    return;
  }
  S* ok = reinterpret_cast<S*>(P.dst) + at;
  S* ov = reinterpret_cast<S*>(P.dst2) + at;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      at_st4<T>(ok + 32 * b + 8 * r, dk[b][4 * r] * P.scale, dk[b][4 * r + 1] * P.scale, dk[b][4 * r + 2] * P.scale, dk[b][4 * r + 3] * P.scale);
      at_st4<T>(ov + 32 * b + 8 * r, dv[b][4 * r] * (1.f / UP), dv[b][4 * r + 1] * (1.f / UP), dv[b][4 * r + 2] * (1.f / UP), dv[b][4 * r + 3] * (1.f / UP));
    }
}

// adds the parts of dk and dv in their order and rounds
template <class T>
__global__ __launch_bounds__(256) void k_attn_dkv_join(AtParams P, size_t one) {
  const size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= 2 * one) return;
  const bool is_v = at >= one;
  at_f32x4 s = {0.f, 0.f, 0.f, 0.f};
  for (int p = 0; p < P.splits; ++p) s += *reinterpret_cast<const at_f32x4*>(P.so + 2 * p * one + at);
  const float f = is_v ? (T::ID == IRX_ATTN_F16 ? 1.f / 1024.f : 1.f) : P.scale;
  typename T::S* to = reinterpret_cast<typename T::S*>(is_v ? P.dst2 : P.dst) + (is_v ? at - one : at);
  at_st4<T>(to, s[0] * f, s[1] * f, s[2] * f, s[3] * f);
}

// Parts of the query axis for dk / dv, by sizes alone: about four workgroups (128 keys of one key head each) per place on the chip, so
// that the longest ones, the first keys of a long causal sequence, do not end alone. Two places per compute unit up to dimension 64 in 16
// bits, else one (registers). Measured, us for the whole backward pass and forward: 12289 causal, 8 / 2 heads of 64: 1085 with 1024
// workgroups, 966 with 2048; six ragged prompts, 16 / 4 heads of 128: 534 with 1024, 552 with 2048 (the parts are written and read again).
static int dkv_splits(long long tq, long long tk, int batch, int heads, int kv_heads, int dim, int elem) {
  if (batch <= 0 || tk <= 0 || tq <= 0) return 1;
  const long long wgs = (tk / IRX_ATTN_BM + (batch < tk ? batch : tk)) * kv_heads;
  const long long items = heads / kv_heads * ((tq / batch + IRX_ATTN_BN - 1) / IRX_ATTN_BN);
  long long s = (elem == 2 && dim <= 64 ? 2048 : 1024) / (wgs > 0 ? wgs : 1);
  if (s > items / 4) s = items / 4;
  return s < 1 ? 1 : s > 8 ? 8 : (int)s;
}

// Parts of the key axis for dq, by sizes alone, as for the forward. Measured, backward pass, us without and with:
// 4096 causal rows, 8 heads of 64, bf16: 163, 144; 6000 rows, 12 heads: 340, 290; 3000 rows, 4 heads of 64, float32: 445, 242; 12289 rows,
// 8 heads, fp16: 697, 692; 1024 rows, 16 heads: 66, 69.
static int dq_splits(long long tq, long long tk, int batch, int heads, int elem, bool causal) {
  if (batch <= 0 || tk <= 0 || tq <= 0) return 1;
  return at_key_parts((tq / IRX_ATTN_BM + (batch < tq ? batch : tq)) * heads, tk / batch, elem, causal);
}

template <class T, int D, bool BIAS> static int launch_bwd(AtParams P, void* dq, void* dk, void* dv, void* dtable, hipStream_t st) {
  const size_t tiles = 4 * AtTile<T, D>::BYTES, w = BIAS ? sizeof(float) * (2 * P.far + 1) : 0;
  if (P.tq > 0) {
    P.slots = at_slots(P.tq, P.batch, IRX_ATTN_BM);
    P.dst = dq;
    const size_t lds = (BIAS && T::ESZ == 4 && D == 128 ? tiles / 2 : tiles) + 5 * w;
    P.splits = dq_splits(P.tq, P.tk, P.batch, P.heads, T::ESZ, P.causal);
    const long long total = (long long)P.slots * P.heads * P.splits;
    if (int rc = at_want_lds(reinterpret_cast<const void*>(&k_attn_dq<T, D, BIAS>), lds, "irx_attn_packed_bwd")) return rc;
    k_attn_dq<T, D, BIAS><<<(unsigned)((total + 7) / 8 * 8), 256, lds, st>>>(P, (int)total);
    IRX_CHECK_LAUNCH("irx_attn_packed_bwd(dq)");
    if (P.splits > 1) {
      const size_t n = (size_t)P.tq * P.heads * D;
      k_attn_dq_join<T><<<(unsigned)((n / 4 + 255) / 256), 256, 0, st>>>(P, n);
      IRX_CHECK_LAUNCH("irx_attn_packed_bwd(dq join)");
    }
  }
  const int q_slots = P.slots * P.splits;                                // tiles and parts that hold bias sums
  if (P.tk > 0 || (BIAS && P.tq > 0)) {                                  // (no keys: the bias gradient is zero, and written)
    const long long extra = BIAS && P.tq > 0 ? (long long)P.buckets * P.heads : 0;
    P.dtable = dtable;
    P.slots = at_slots(P.tk, P.batch, IRX_ATTN_BM);
    P.dst = dk;
    P.dst2 = dv;
    P.splits = dkv_splits(P.tq, P.tk, P.batch, P.heads, P.kv_heads, D, T::ESZ);
    const size_t lds = tiles + 6 * IRX_ATTN_BN * sizeof(float) + w;
    const long long total = (long long)P.slots * P.kv_heads * P.splits;
    if (int rc = at_want_lds(reinterpret_cast<const void*>(&k_attn_dkv<T, D, BIAS>), lds, "irx_attn_packed_bwd")) return rc;
    k_attn_dkv<T, D, BIAS><<<(unsigned)((total + 7) / 8 * 8 + extra), 256, lds, st>>>(P, (int)total, q_slots);
    IRX_CHECK_LAUNCH("irx_attn_packed_bwd(dkv)");
    if (P.splits > 1) {
      const size_t one = (size_t)P.tk * P.kv_heads * D;
      k_attn_dkv_join<T><<<(unsigned)((one / 2 + 255) / 256), 256, 0, st>>>(P, one);
      IRX_CHECK_LAUNCH("irx_attn_packed_bwd(join)");
    }
  }
  return IRX_OK;
}
template <class T, int D> static int launch_bwd_b(const AtParams& P, void* dq, void* dk, void* dv, void* dt, hipStream_t st) {
  return P.table ? launch_bwd<T, D, true>(P, dq, dk, dv, dt, st) : launch_bwd<T, D, false>(P, dq, dk, dv, dt, st);
}
template <class T> static int launch_bwd_d(const AtParams& P, int dim, void* dq, void* dk, void* dv, void* dt, hipStream_t st) {
  return dim == 32 ? launch_bwd_b<T, 32>(P, dq, dk, dv, dt, st) : dim == 64 ? launch_bwd_b<T, 64>(P, dq, dk, dv, dt, st) : launch_bwd_b<T, 128>(P, dq, dk, dv, dt, st);
}

// D, then (aligned) the parts of dq or, later, of dk and dv, then the bias gradient by distance (counted as if causal: the most there is)
static size_t bwd_delta(int tq, int heads) { return ((size_t)heads * tq + 3) / 4 * 4; }
static size_t bwd_parts(int tq, int tk, int batch, int heads, int kv_heads, int dim, int elem) {
  const int s = dkv_splits(tq, tk, batch, heads, kv_heads, dim, elem), r = dq_splits(tq, tk, batch, heads, elem, true);
  const size_t kv = s > 1 ? (size_t)s * 2 * tk * kv_heads * dim : 0, q = r > 1 ? (size_t)r * tq * heads * dim : 0;
  return kv > q ? kv : q;
}
extern "C" size_t irx_attn_packed_bwd_workspace_bytes(int tq, int tk, int batch, int heads, int kv_heads, int dim, int dtype, int far) {
  if (tq <= 0 || tk < 0 || batch < 0 || heads <= 0 || kv_heads <= 0 || dim <= 0) return 0;
  const size_t part = far < 0 ? 0 : (size_t)at_slots(tq, batch, IRX_ATTN_BM) * dq_splits(tq, tk, batch, heads, dtype == IRX_ATTN_F32 ? 4 : 2, true) * heads * (2 * (size_t)far + 1);
  return (bwd_delta(tq, heads) + bwd_parts(tq, tk, batch, heads, kv_heads, dim, dtype == IRX_ATTN_F32 ? 4 : 2) + part) * sizeof(float);
}

extern "C" int irx_attn_packed_bwd(const void* q, long long q_row, long long q_head, const void* k, long long k_row, long long k_head,
                                   const void* v, long long v_row, long long v_head, const void* dout, long long do_row, long long do_head,
                                   const void* out, const void* rest, const float* stats, const int32_t* cu_q, const int32_t* cu_k, int batch, int tq, int tk,
                                   int heads, int kv_heads, int dim, int dtype, float scale, int causal, const void* table, int table_f32,
                                   const int32_t* map, int buckets, int far, void* dq, void* dk, void* dv, void* dtable, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  AtParams P = {};
  P.q = {q, q_row, q_head};
  P.k = {k, k_row, k_head};
  P.v = {v, v_row, v_head};
  P.dout = {dout, do_row, do_head};
  P.cu_q = cu_q; P.cu_k = cu_k;
  P.batch = batch; P.tq = tq; P.tk = tk; P.heads = heads; P.kv_heads = kv_heads; P.causal = causal != 0; P.scale = scale;
  P.table = table; P.table_f32 = table_f32; P.map = map; P.buckets = buckets; P.far = far;
  P.out = out; P.rest = dtype == IRX_ATTN_F32 ? nullptr : rest; P.stats = stats;
  if (int rc = at_check("irx_attn_packed_bwd", P, dim, dtype, dtype == IRX_ATTN_F32 ? 4 : 2)) return rc;
  IRX_REQUIRE(tq == 0 || (dout && out && stats && dq), "irx_attn_packed_bwd: null tensor");
  IRX_REQUIRE(tk == 0 || (dk && dv), "irx_attn_packed_bwd: null gradient");
  IRX_REQUIRE(!table || dtable, "irx_attn_packed_bwd: null bias gradient");
  IRX_REQUIRE((((uintptr_t)out | (uintptr_t)rest | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) == 0, "irx_attn_packed_bwd: rows must start on 16 bytes");
  const size_t need = irx_attn_packed_bwd_workspace_bytes(tq, tk, batch, heads, kv_heads, dim, dtype, table ? far : -1);
  if (need && (!workspace || workspace_bytes < need)) {
    irx_set_error("irx_attn_packed_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return IRX_ERR_WORKSPACE;
  }
  IRX_REQUIRE(((uintptr_t)workspace & 15) == 0, "irx_attn_packed_bwd: workspace must start on 16 bytes");
  P.delta = static_cast<float*>(workspace);
  P.so = P.delta + bwd_delta(tq, heads);
  P.part = P.so + bwd_parts(tq, tk, batch, heads, kv_heads, dim, dtype == IRX_ATTN_F32 ? 4 : 2);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == IRX_ATTN_F32) return launch_bwd_d<AtF32>(P, dim, dq, dk, dv, dtable, st);
  if (dtype == IRX_ATTN_BF16) return launch_bwd_d<AtBf16>(P, dim, dq, dk, dv, dtable, st);
  return launch_bwd_d<AtF16>(P, dim, dq, dk, dv, dtable, st);
}
