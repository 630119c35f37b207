// irx_attn_bwd.hip — attention over packed sequences, backward: dq, dk, dv and the gradient of the bias table.
//
// With P_ij = 2^(s_ij - m_i) / l_i from the saved row maximum and sum, D_i = out_i . dout_i and dS_ij = P_ij (dout_i . v_j - D_i):
//   dq_i = scale sum_j dS_ij k_j,   dk_j = scale sum_i dS_ij q_i,   dv_j = sum_i P_ij dout_i   (dk, dv over every query head of the group).
// Two kernels, so that every sum stays in one workgroup's registers and the order of addition never changes (no atomics on memory): one
// owns queries and walks the keys (D, dq, bias gradient), the other owns keys and walks the group's queries (dk, dv). Scores and dout . v
// are computed in both: 7 products in place of 5. Both use the transposed layouts of irx_attn.h: P and dS are operands as they come.
// P and dS are rounded to the operand type for the second products; row statistics, D, dS itself and all sums are 32 bits. D is formed
// from the stored (rounded) output, as the formula's own terms are no more exact than that.
#include "irx_attn.h"

int at_check(const char* who, const AtParams& P, int dim, int dtype, int elem);

// LDS sum without a returned value (ds_add_f32)
__device__ __forceinline__ void at_lds_add(float* p, float v) { __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP); }

// ---- dq, D and the bias gradient by distance ----------------------------------------------------------------------------------
// Bias gradient: sum of dS over all pairs of one distance. Each wave half owns an LDS array by distance and adds its registers one by
// one: within one instruction the 32 lanes (consecutive queries, one key) hit 32 different distances, so no two lanes meet and the order
// of additions is fixed; distances at or beyond the clip are summed in registers.
template <class T, int D, bool BIAS>
__global__ __launch_bounds__(256, T::ESZ == 2 ? 2 : 1) void k_attn_dq(AtParams P, int total) {
  typedef AtTile<T, D> Tile;
  typedef typename T::F F;
  typedef typename T::S S;
  constexpr int STEPS = D / 16, BLOCKS = D / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* lk_ = smem;
  unsigned char* lv_ = smem + Tile::BYTES;
  float* sb = reinterpret_cast<float*>(smem + 2 * Tile::BYTES);
  const int W = 2 * P.far + 1;
  float* sd = sb + W;                                                    // [wave][half][W]

  const int per = gridDim.x >> 3;
  const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (id >= total) return;
  const int slot = P.slots - 1 - id % P.slots, head = id / P.slots;

  int first;
  const AtSpan sp = at_span(P.cu_q, P.batch, P.tq, IRX_ATTN_BM, slot, &first);
  if (sp.begin >= sp.end) {
    if constexpr (BIAS)
      for (int d = threadIdx.x; d < W; d += 256) P.part[((size_t)slot * P.heads + head) * W + d] = 0.f;
    return;
  }
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kb = 0, ke = 0;
  if (sp.seq >= 0) {
    kb = at_edge(P.cu_k, P.batch, P.tk, sp.seq + 1);
    ke = at_edge(P.cu_k, P.batch, P.tk, sp.seq + 2);
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
  const int t1 = (max(block_any, 0) + IRX_ATTN_BN - 1) / IRX_ATTN_BN;
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
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      qf[s] = mine ? at_ldg<T>(qp + 16 * s) : at_zero<T>();
      df[s] = mine ? at_ldg<T>(dp + 16 * s) : at_zero<T>();
      const F of = mine ? at_ldg<T>(op + 16 * s) : at_zero<T>();
#pragma unroll
      for (int e = 0; e < 8; ++e) delta = __builtin_fmaf(at_get<T>(of, e), at_get<T>(df[s], e), delta);
    }
    delta += at_other_half(delta);
    if (mine) {
      const float* st = P.stats + ((size_t)head * P.tq + q) * 2;
      m = st[0];
      inv = st[1];
      if (half == 0) P.delta[(size_t)head * P.tq + q] = delta;
    }
  }
  if constexpr (BIAS) {
    at_load_bias<T>(sb, P, head);
    for (int d = threadIdx.x; d < 8 * W; d += 256) sd[d] = 0.f;
  }
  float* mysd = sd + (wave * 2 + half) * W;
  float below = 0.f, above = 0.f;

  at_f32x16 acc[BLOCKS];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[b][i] = 0.f;

  for (int t = 0; t < t1; ++t) {
    const int k0 = t * IRX_ATTN_BN;
    __syncthreads();
    Tile::template copy_in<256>(lk_, kp + k0 * P.k.st, P.k.st, lk - k0);
    Tile::template copy_in<256>(lv_, vp + k0 * P.v.st, P.v.st, lk - k0);
    __syncthreads();
#pragma unroll
    for (int kb2 = 0; kb2 < 2; ++kb2) {
      const int k1 = k0 + 32 * kb2;
      if (k1 >= wave_any) break;
      at_f32x16 x, y;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = y[i] = 0.f;
#pragma unroll
      for (int st = 0; st < STEPS; ++st) {
        x = at_mma(Tile::row_frag(lk_, 32 * kb2, st), qf[st], x);
        y = at_mma(Tile::row_frag(lv_, 32 * kb2, st), df[st], y);
      }
      float p[16];
      bool near = false;
      const int d0 = k1 + 4 * half - (i0 + (lane & 31) + off);
      if constexpr (BIAS) {
        const int lo = k1 - (i0 + 31 + off), hi = k1 + 31 - (i0 + off);
        near = !(hi <= -P.far || lo >= P.far);
        if (!near) {
          const float b = sb[hi <= -P.far ? 0 : 2 * P.far] - m;
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = at_exp2(__builtin_fmaf(x[i], c1, b)) * inv;
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
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int d = d0 + 8 * (i >> 2) + (i & 3);
            if (d > -P.far && d < P.far) at_lds_add(mysd + d + P.far, p[i]);
            else if (d <= -P.far) below += p[i];
            else above += p[i];
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
  }
  if constexpr (BIAS) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      below += __shfl_xor(below, o, 64);
      above += __shfl_xor(above, o, 64);
    }
    if ((lane & 31) == 0) {                                              // nobody else adds to the clipped distances
      if (P.far == 0) mysd[0] = below + above;
      else {
        mysd[0] = below;
        mysd[2 * P.far] = above;
      }
    }
    __syncthreads();
    for (int d = threadIdx.x; d < W; d += 256) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) s += sd[w * W + d];
      P.part[((size_t)slot * P.heads + head) * W + d] = s;
    }
  }
  if (!mine) return;
  S* o = reinterpret_cast<S*>(P.dst) + ((size_t)q * P.heads + head) * D + 4 * half;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      at_st4<T>(o + 32 * b + 8 * g, acc[b][4 * g] * P.scale, acc[b][4 * g + 1] * P.scale, acc[b][4 * g + 2] * P.scale, acc[b][4 * g + 3] * P.scale);
}

// ---- dk, dv -----------------------------------------------------------------------------------------------------------------------
template <class T, int D, bool BIAS>
__global__ __launch_bounds__(256, 1) void k_attn_dkv(AtParams P, int total) {
  typedef AtTile<T, D> Tile;
  typedef typename T::F F;
  typedef typename T::S S;
  constexpr int STEPS = D / 16, BLOCKS = D / 32;
  // float16 keeps 10 bits below 2^-14: weights of long rows are that small, so they go through the product times 2^10
  constexpr float UP = T::ID == IRX_ATTN_F16 ? 1024.f : 1.f;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  unsigned char* lq_ = smem;
  unsigned char* ld_ = smem + Tile::BYTES;
  float* sm = reinterpret_cast<float*>(smem + 2 * Tile::BYTES);          // row maxima, 1 / row sums, D of the tile's 64 queries
  float* si = sm + IRX_ATTN_BN;
  float* se = si + IRX_ATTN_BN;
  float* sb = se + IRX_ATTN_BN;

  const int per = gridDim.x >> 3;
  const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (id >= total) return;
  const int slot = id % P.slots, kvh = id / P.slots;

  int first;
  const AtSpan sp = at_span(P.cu_k, P.batch, P.tk, IRX_ATTN_BM, slot, &first);
  if (sp.begin >= sp.end) return;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int qb = 0, qe = 0;
  if (sp.seq >= 0) {
    qb = at_edge(P.cu_q, P.batch, P.tq, sp.seq + 1);
    qe = at_edge(P.cu_q, P.batch, P.tq, sp.seq + 2);
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

  for (int g = 0; g < group; ++g) {
    const int head = kvh * group + g;
    if constexpr (BIAS) {
      __syncthreads();
      at_load_bias<T>(sb, P, head);
    }
    const S* qp = reinterpret_cast<const S*>(P.q.p) + qb * P.q.st + head * P.q.sh;
    const S* dp = reinterpret_cast<const S*>(P.dout.p) + qb * P.dout.st + head * P.dout.sh;
    const float* st = P.stats + ((size_t)head * P.tq + qb) * 2;
    const float* de = P.delta + (size_t)head * P.tq + qb;
    for (int q0 = block_any / IRX_ATTN_BN * IRX_ATTN_BN; q0 < lq; q0 += IRX_ATTN_BN) {
      __syncthreads();
      Tile::template copy_in<256>(lq_, qp + q0 * P.q.st, P.q.st, lq - q0);
      Tile::template copy_in<256>(ld_, dp + q0 * P.dout.st, P.dout.st, lq - q0);
      if (threadIdx.x < IRX_ATTN_BN) {
        const int r = q0 + (int)threadIdx.x;
        const bool in = r < lq;
        sm[threadIdx.x] = in ? st[2 * (size_t)r] : 0.f;
        si[threadIdx.x] = in ? st[2 * (size_t)r + 1] : 0.f;
        se[threadIdx.x] = in ? de[r] : 0.f;
      }
      __syncthreads();
#pragma unroll
      for (int qb2 = 0; qb2 < 2; ++qb2) {
        const int q1 = q0 + 32 * qb2;
        if (q1 + 31 < wave_any || q1 >= lq || row0 >= sp.end) continue;
        at_f32x16 x, y;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = y[i] = 0.f;
#pragma unroll
        for (int s = 0; s < STEPS; ++s) {
          x = at_mma(Tile::row_frag(lq_, 32 * qb2, s), kf[s], x);
          y = at_mma(Tile::row_frag(ld_, 32 * qb2, s), vf[s], y);
        }
        float p[16], ds[16];
        const int lo = j0 - (q1 + 31 + off), hi = j0 + 31 - (q1 + off);  // distances key - query in this block
        const bool near = BIAS && !(hi <= -P.far || lo >= P.far);
        float far_bias = 0.f;
        if constexpr (BIAS) far_bias = sb[hi <= -P.far ? 0 : 2 * P.far];
        const bool edge = q1 < wave_full || q1 + 32 > lq;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int at = 32 * qb2 + 8 * r + 4 * half;
          const at_f32x4 m4 = *reinterpret_cast<const at_f32x4*>(sm + at);
          const at_f32x4 i4 = *reinterpret_cast<const at_f32x4*>(si + at);
          const at_f32x4 e4 = *reinterpret_cast<const at_f32x4*>(se + at);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int i = 4 * r + e;
            float b = -m4[e];
            if constexpr (BIAS) {
              if (near) {
                const int d = j - (q0 + at + e + off);
                p[i] = at_exp2(__builtin_fmaf(x[i], c1, sb[min(max(d, -P.far), P.far) + P.far]) - m4[e]) * i4[e];
              } else {
                p[i] = at_exp2(__builtin_fmaf(x[i], c1, far_bias + b)) * i4[e];
              }
            } else {
              p[i] = at_exp2(__builtin_fmaf(x[i], c1, b)) * i4[e];
            }
            ds[i] = p[i] * (y[i] - e4[e]);
            if (edge) {
              const int qi = q0 + at + e;
              const bool see = qi >= from && qi < lq;
              p[i] = see ? p[i] : 0.f;
              ds[i] = see ? ds[i] : 0.f;
            }
            p[i] *= UP;
          }
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const F pf = at_pack<T>(p + 8 * ks), sf = at_pack<T>(ds + 8 * ks);
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b) {
            dv[b] = at_mma(Tile::col_frag(ld_, 32 * qb2 + 16 * ks, b), pf, dv[b]);
            dk[b] = at_mma(Tile::col_frag(lq_, 32 * qb2 + 16 * ks, b), sf, dk[b]);
          }
        }
      }
    }
  }
  if (!mine) return;
  const size_t at = ((size_t)key * P.kv_heads + kvh) * D + 4 * half;
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

// ---- bias gradient: distances -> buckets, over all tiles -----------------------------------------------------------------------
// One workgroup per (bucket, head): lists the bucket's distances in order, then adds their partial sums of every tile (64 bits, fixed order).
template <class T>
__global__ __launch_bounds__(256) void k_attn_dbias(const float* part, int slots, int heads, int far, const int32_t* map, int buckets,
                                                    void* dtable, int table_f32) {
  __shared__ int list[2 * IRX_ATTN_MAX_FAR + 1];
  __shared__ int count;
  __shared__ double red[4];
  const int bucket = blockIdx.x, head = blockIdx.y, W = 2 * far + 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (wave == 0) {
    int n = 0;
    for (int base = 0; base < W; base += 64) {
      const int d = base + lane;
      int b = d < W ? map[d] : -1;
      if (d < W) b = b < 0 ? 0 : (b >= buckets ? buckets - 1 : b);
      const unsigned long long hit = __ballot(d < W && b == bucket);
      if (d < W && b == bucket) list[n + __popcll(hit & ((1ull << lane) - 1))] = d;
      n += __popcll(hit);
    }
    if (lane == 0) count = n;
  }
  __syncthreads();
  const int c = count;
  double s = 0;
  if (c) {
    const long long n = (long long)slots * c;
    for (long long i = threadIdx.x; i < n; i += 256) s += (double)part[((size_t)(i / c) * heads + head) * W + list[i % c]];
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if (lane == 0) red[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    const float x = (float)(((red[0] + red[1]) + red[2]) + red[3]);
    const size_t at = (size_t)bucket * heads + head;
    if (table_f32 || T::ID == IRX_ATTN_F32) reinterpret_cast<float*>(dtable)[at] = x;
    else if constexpr (T::ID == IRX_ATTN_BF16) reinterpret_cast<unsigned short*>(dtable)[at] = (unsigned short)irx_pk_bf16(x, 0.f);
    else reinterpret_cast<_Float16*>(dtable)[at] = (_Float16)x;
  }
}

template <class T, int D, bool BIAS> static int launch_bwd(AtParams P, void* dq, void* dk, void* dv, void* dtable, hipStream_t st) {
  const size_t tiles = 2 * AtTile<T, D>::BYTES, w = BIAS ? sizeof(float) * (2 * P.far + 1) : 0;
  if (P.tq > 0) {
    P.slots = at_slots(P.tq, P.batch, IRX_ATTN_BM);
    P.dst = dq;
    const size_t lds = tiles + 9 * w;
    const long long total = (long long)P.slots * P.heads;
    if (int rc = at_want_lds(reinterpret_cast<const void*>(&k_attn_dq<T, D, BIAS>), lds, "irx_attn_packed_bwd")) return rc;
    k_attn_dq<T, D, BIAS><<<(unsigned)((total + 7) / 8 * 8), 256, lds, st>>>(P, (int)total);
    IRX_CHECK_LAUNCH("irx_attn_packed_bwd(dq)");
    if constexpr (BIAS) {
      k_attn_dbias<T><<<dim3(P.buckets, P.heads), 256, 0, st>>>(P.part, P.slots, P.heads, P.far, P.map, P.buckets, dtable, P.table_f32);
      IRX_CHECK_LAUNCH("irx_attn_packed_bwd(bias)");
    }
  }
  if (P.tk > 0) {
    P.slots = at_slots(P.tk, P.batch, IRX_ATTN_BM);
    P.dst = dk;
    P.dst2 = dv;
    const size_t lds = tiles + 3 * IRX_ATTN_BN * sizeof(float) + w;
    const long long total = (long long)P.slots * P.kv_heads;
    if (int rc = at_want_lds(reinterpret_cast<const void*>(&k_attn_dkv<T, D, BIAS>), lds, "irx_attn_packed_bwd")) return rc;
    k_attn_dkv<T, D, BIAS><<<(unsigned)((total + 7) / 8 * 8), 256, lds, st>>>(P, (int)total);
    IRX_CHECK_LAUNCH("irx_attn_packed_bwd(dkv)");
  }
  return IRX_OK;
}
template <class T, int D> static int launch_bwd_b(const AtParams& P, void* dq, void* dk, void* dv, void* dt, hipStream_t st) {
  return P.table ? launch_bwd<T, D, true>(P, dq, dk, dv, dt, st) : launch_bwd<T, D, false>(P, dq, dk, dv, dt, st);
}
template <class T> static int launch_bwd_d(const AtParams& P, int dim, void* dq, void* dk, void* dv, void* dt, hipStream_t st) {
  return dim == 32 ? launch_bwd_b<T, 32>(P, dq, dk, dv, dt, st) : dim == 64 ? launch_bwd_b<T, 64>(P, dq, dk, dv, dt, st) : launch_bwd_b<T, 128>(P, dq, dk, dv, dt, st);
}

extern "C" size_t irx_attn_packed_bwd_workspace_bytes(int tq, int batch, int heads, int far_or_minus1) {
  if (tq <= 0 || batch < 0 || heads <= 0) return 0;
  const size_t delta = (size_t)heads * tq;
  const size_t part = far_or_minus1 < 0 ? 0 : (size_t)at_slots(tq, batch, IRX_ATTN_BM) * heads * (2 * (size_t)far_or_minus1 + 1);
  return (delta + part) * sizeof(float);
}

extern "C" int irx_attn_packed_bwd(const void* q, long long q_row, long long q_head, const void* k, long long k_row, long long k_head,
                                   const void* v, long long v_row, long long v_head, const void* dout, long long do_row, long long do_head,
                                   const void* out, const float* stats, const int32_t* cu_q, const int32_t* cu_k, int batch, int tq, int tk,
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
  P.out = out; P.stats = stats;
  if (int rc = at_check("irx_attn_packed_bwd", P, dim, dtype, dtype == IRX_ATTN_F32 ? 4 : 2)) return rc;
  IRX_REQUIRE(tq == 0 || (dout && out && stats && dq), "irx_attn_packed_bwd: null tensor");
  IRX_REQUIRE(tk == 0 || (dk && dv), "irx_attn_packed_bwd: null gradient");
  IRX_REQUIRE(!table || dtable, "irx_attn_packed_bwd: null bias gradient");
  IRX_REQUIRE((((uintptr_t)out | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) == 0, "irx_attn_packed_bwd: rows must start on 16 bytes");
  const size_t need = irx_attn_packed_bwd_workspace_bytes(tq, batch, heads, table ? far : -1);
  if (need && (!workspace || workspace_bytes < need)) {
    irx_set_error("irx_attn_packed_bwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
    return IRX_ERR_WORKSPACE;
  }
  P.delta = static_cast<float*>(workspace);
  P.part = P.delta + (size_t)heads * tq;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == IRX_ATTN_F32) return launch_bwd_d<AtF32>(P, dim, dq, dk, dv, dtable, st);
  if (dtype == IRX_ATTN_BF16) return launch_bwd_d<AtBf16>(P, dim, dq, dk, dv, dtable, st);
  return launch_bwd_d<AtF16>(P, dim, dq, dk, dv, dtable, st);
}
