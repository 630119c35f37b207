// irx_attn.h — shared parts of the packed-attention kernels (irx_attn.hip: forward, irx_attn_bwd.hip: backward), gfx950 only.
//
// Matrix-core layouts used throughout (v_mfma_f32_32x32x16 for 16-bit types, eight v_mfma_f32_32x32x2 for float32):
//   A operand: lane l holds row l % 32 and eight values of the summed axis, B operand: column l % 32 and eight values,
//   result:    lane l holds column l % 32 and rows 8 g + 4 (l / 32) + r in register 4 g + r  (g, r = 0..3).
// The summed axis may be taken in any order as long as both operands take the same one. So a result (scores: keys down, one query
// per lane) goes straight into the next product as its B operand, registers 8 s .. 8 s + 7 being the eight values of step s, when the
// A operand takes its rows in that order too: 16 s + 4 (l / 32) + {0..3} and 16 s + 8 + 4 (l / 32) + {0..3}. In 16 bits that is what two
// transposing LDS reads (ds_read_b64_tr_b16, four rows of one column each) deliver; in 32 bits eight ds_read_b32. No value crosses lanes
// between the two products, and a softmax row is one lane pair (l, l + 32).
#pragma once
#include "irx_common.h"

#define IRX_ATTN_F32 0
#define IRX_ATTN_BF16 1
#define IRX_ATTN_F16 2
#define IRX_ATTN_WAVES 4                     // waves of a workgroup; each owns 32 rows (queries or keys) of the workgroup's tile
#define IRX_ATTN_BM (32 * IRX_ATTN_WAVES)    // rows of a workgroup's own tile
#define IRX_ATTN_BN 64                       // rows of the tile that passes through LDS
#define IRX_ATTN_MAX_FAR 512                 // largest clipped distance of the bucket map (LDS: 5 (2 far + 1) floats in the backward)

typedef float at_f32x16 __attribute__((ext_vector_type(16)));
typedef float at_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 at_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 at_f16x8 __attribute__((ext_vector_type(8)));
typedef short at_s16x4 __attribute__((ext_vector_type(4)));
typedef short at_s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned at_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned at_u32x2 __attribute__((ext_vector_type(2)));

struct at_f32x8 { float v[8]; };

struct AtBf16 { typedef unsigned short S; typedef at_bf16x8 F; enum { ESZ = 2, ID = IRX_ATTN_BF16 }; };
struct AtF16  { typedef unsigned short S; typedef at_f16x8 F;  enum { ESZ = 2, ID = IRX_ATTN_F16 }; };
struct AtF32  { typedef float S;          typedef at_f32x8 F;  enum { ESZ = 4, ID = IRX_ATTN_F32 }; };

// Strides in elements. Every tensor is [rows][heads][dim] with contiguous dim; row and head strides are multiples of 16 bytes.
struct AtTensor { const void* p; long long st, sh; };

// `rest`: D = out . dout with the output as it was before its rounding. Taken from the rounded one, bf16 gradients are 6 % further off
// (1024 causal rows of 64, relative to 64 bits: dq 2.55e-3 instead of 2.44e-3; 1.66e-3 is the rounding of dq itself).
struct AtParams {
  AtTensor q, k, v, dout;                    // dout: backward only
  const void* out; const void* rest;         // backward: the output and, in 16 bits, what its rounding left (or NULL), laid out alike
  const float* stats;                        // out [tq][heads][dim] contiguous; stats [heads][tq][2] = (exponent of weight 1, 1 / sum of weights)
  void* dst; void* dst2;                     // fwd: out, its rounding's rest (may be NULL); dq kernel: dq; dk/dv kernel: dk, dv
  float* wstats;                             // fwd: stats (may be NULL)
  float* delta;                              // [heads][tq]: sum_d out * dout, written by the dq kernel, read by the dk/dv kernel
  const int32_t* cu_q; const int32_t* cu_k;
  int batch, tq, tk, heads, kv_heads, causal;
  float scale;
  const void* table; const int32_t* map;     // bias table [buckets][heads] (float32 or the tensors' type), map [2 far + 1]
  int table_f32, buckets, far;
  float* part;                               // backward: bias gradient by distance, [slots][heads][2 far + 1]
  void* dtable;                              // ... and by bucket, the result
  int slots;
  int splits; float* so; float* sst;         // a long axis in parts: partial results and, forward, (max, sum)
};

// ---- which rows a workgroup owns ------------------------------------------------------------------------------------------
// cu cuts [0, total) into batch + 2 pieces: before cu[0], the sequences, behind cu[batch] (the outer two are padding: no partner rows, so
// zeros are written there). Piece s owns the slots from floor(start_s / BM) + s on: at least as many as it has tiles, with no
// knowledge of the lengths on the host. Every value read from cu is clamped to [0, total]: whatever cu holds, all addresses stay inside.
struct AtSpan { int begin, end, seq; };      // rows [begin, end) of sequence seq (-1: padding); begin >= end: nothing to do

__device__ __forceinline__ int at_edge(const int32_t* cu, int batch, int total, int s) {
  if (s <= 0) return 0;
  if (s > batch + 1) return total;
  const int c = cu[s - 1];
  return c < 0 ? 0 : (c > total ? total : c);
}

__device__ __forceinline__ AtSpan at_span(const int32_t* cu, int batch, int total, int bm, int slot, int* first) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int base = 0; base < batch + 2; base += 64) {
    const int s = base + lane;
    const bool le = s < batch + 2 && at_edge(cu, batch, total, s) / bm + s <= slot;
    const int c = __popcll(__ballot(le));
    n += c;
    if (c < 64) break;
  }
  const int s = __builtin_amdgcn_readfirstlane(n - 1);
  const int lo = at_edge(cu, batch, total, s);
  int hi = at_edge(cu, batch, total, s + 1);
  if (hi < lo) hi = lo;
  int t = slot - (lo / bm + s);
  if (t < 0) t = 0;
  AtSpan r;
  const long long b = (long long)lo + (long long)t * bm;
  r.begin = (int)(b < hi ? b : hi);
  r.end = hi;
  r.seq = (s >= 1 && s <= batch) ? s - 1 : -1;
  *first = lo;
  return r;
}

static inline int at_slots(int total, int batch, int bm) { return total / bm + batch + 2; }

// Parts of the key axis for a kernel that owns queries, `wgs` workgroups of 128 rows over about `keys` keys each. Measured: irx_attn.hip's
// and irx_attn_bwd.hip's launches.
static inline int at_key_parts(long long wgs, long long keys, int elem, bool causal) {
  if (keys < 1024) return 1;
  if (wgs >= 512) {
    // one round and a half of workgroups: under a causal mask the longest tiles end last, two parts even it out for a join of 8 bytes per value
    return causal && wgs < 1024 && keys * (1024 - wgs) * (elem == 4 ? 4 : 1) >= 1 << 21 ? 2 : 1;
  }
  long long s = wgs > 266 ? 2 : 800 / wgs;
  if (s > keys / 256) s = keys / 256;
  return s > 32 ? 32 : (int)s;
}

// ---- fragments ------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ at_f32x16 at_mma(at_bf16x8 a, at_bf16x8 b, at_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ at_f32x16 at_mma(at_f16x8 a, at_f16x8 b, at_f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ at_f32x16 at_mma(const at_f32x8& a, const at_f32x8& b, at_f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[j], b.v[j], c, 0, 0, 0);
  return c;
}

// eight consecutive results, rounded to the operand type (to nearest even; float32: as they are)
template <class T> __device__ __forceinline__ typename T::F at_pack(const float* x);
template <> __device__ __forceinline__ at_bf16x8 at_pack<AtBf16>(const float* x) {
  at_u32x4 u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = irx_pk_bf16(x[2 * i], x[2 * i + 1]);
  return __builtin_bit_cast(at_bf16x8, u);
}
template <> __device__ __forceinline__ at_f16x8 at_pack<AtF16>(const float* x) {
  at_f16x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (_Float16)x[i];
  return r;
}
template <> __device__ __forceinline__ at_f32x8 at_pack<AtF32>(const float* x) {
  at_f32x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = x[i];
  return r;
}

template <class T> __device__ __forceinline__ float at_get(typename T::F f, int i);
template <> __device__ __forceinline__ float at_get<AtBf16>(at_bf16x8 f, int i) { return (float)f[i]; }
template <> __device__ __forceinline__ float at_get<AtF16>(at_f16x8 f, int i) { return (float)f[i]; }
template <> __device__ __forceinline__ float at_get<AtF32>(at_f32x8 f, int i) { return f.v[i]; }

// 8 consecutive elements from global memory (16-byte aligned)
template <class T> __device__ __forceinline__ typename T::F at_ldg(const typename T::S* p) {
  if constexpr (T::ESZ == 2) {
    return __builtin_bit_cast(typename T::F, *reinterpret_cast<const at_u32x4*>(p));
  } else {
    at_f32x8 r;
    const at_f32x4 a = *reinterpret_cast<const at_f32x4*>(p), b = *reinterpret_cast<const at_f32x4*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) { r.v[i] = a[i]; r.v[4 + i] = b[i]; }
    return r;
  }
}
template <class T> __device__ __forceinline__ typename T::F at_zero() {
  if constexpr (T::ESZ == 2) {
    return __builtin_bit_cast(typename T::F, (at_u32x4){0u, 0u, 0u, 0u});
  } else {
    at_f32x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = 0.f;
    return r;
  }
}

// four consecutive elements (one register group of a result) to global memory
template <class T> __device__ __forceinline__ void at_st4(typename T::S* p, float a, float b, float c, float d) {
  if constexpr (T::ID == IRX_ATTN_F32) {
    *reinterpret_cast<at_f32x4*>(p) = (at_f32x4){a, b, c, d};
  } else if constexpr (T::ID == IRX_ATTN_BF16) {
    *reinterpret_cast<at_u32x2*>(p) = (at_u32x2){irx_pk_bf16(a, b), irx_pk_bf16(c, d)};
  } else {
    typedef _Float16 h4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<h4*>(p) = (h4){(_Float16)a, (_Float16)b, (_Float16)c, (_Float16)d};
  }
}

// the same, and what the rounding left over, rounded in its turn (rest == NULL: not wanted). The values are products: float16 has an instruction
// that multiplies and rounds at once, and where the compiler takes it for one of the two uses only, output and rest belong to different neighbours
// of a value in the middle. So a value is a float register before either use.
template <class T> __device__ __forceinline__ void at_st4_rest(typename T::S* p, typename T::S* rest, float a, float b, float c, float d) {
  if constexpr (T::ID == IRX_ATTN_F16) asm("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
  at_st4<T>(p, a, b, c, d);
  if constexpr (T::ID == IRX_ATTN_BF16) {
    if (rest) {
      const at_u32x2 u = (at_u32x2){irx_pk_bf16(a, b), irx_pk_bf16(c, d)};
      at_st4<T>(rest, a - __uint_as_float(u[0] << 16), b - __uint_as_float(u[0] & 0xffff0000u), c - __uint_as_float(u[1] << 16),
                d - __uint_as_float(u[1] & 0xffff0000u));
    }
  } else if constexpr (T::ID == IRX_ATTN_F16) {
    if (rest) at_st4<T>(rest, a - (float)(_Float16)a, b - (float)(_Float16)b, c - (float)(_Float16)c, d - (float)(_Float16)d);
  }
}

// ---- direct loads into LDS ----------------------------------------------------------------------------------------------------
// In asm: with the builtin the compiler takes every later LDS read to depend on the load and waits where it was issued. The only wait is
// at_landed() before the barrier that hands the tile over.
typedef int at_i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ at_i32x4 at_rsrc(const void* base, unsigned bytes) {
  const unsigned long long b = (unsigned long long)base;
  return (at_i32x4){__builtin_amdgcn_readfirstlane((int)(unsigned)b), __builtin_amdgcn_readfirstlane((int)((unsigned)(b >> 32) & 0xffffu)),
                    __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
__device__ __forceinline__ unsigned at_lds_addr(const void* p) {
  return (unsigned)(unsigned long long)(__attribute__((address_space(3))) const void*)p;
}
__device__ __forceinline__ void at_dma(at_i32x4 rs, unsigned lds, unsigned off) {
  unsigned keep;
  asm volatile(
      "s_mov_b32 %0, m0\n\t"
      "s_mov_b32 m0, %1\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %2, %3, 0 offen lds\n\t"
      "s_mov_b32 m0, %0"
      : "=&s"(keep)
      : "s"(lds), "v"(off), "s"(rs)
      : "memory");
}
__device__ __forceinline__ void at_landed() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// ---- LDS images -----------------------------------------------------------------------------------------------------------
// A tile is BN rows (a multiple of 32, at least 4 KB) of D elements, as they are in memory; the 16-byte pieces of a row are XOR-swizzled by the row so that neither reads
// of one piece from 16 rows (ds_read_b128) nor transposing reads of 64 bytes from four rows meet in a bank (64 banks, 256 bytes a turn).
template <class T, int D, int BN = IRX_ATTN_BN, int WAVES = IRX_ATTN_WAVES> struct AtTile {
  enum { RB = D * T::ESZ, PIECES = RB / 16, BYTES = BN * RB };
  __device__ static __forceinline__ int swz(int row) {
    if constexpr (T::ESZ == 2) {
      if constexpr (PIECES == 16) return ((row & 3) << 2) | ((row >> 2) & 3);
      else if constexpr (PIECES == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
      else return (row >> 2) & 3;
    } else {
      if constexpr (PIECES >= 16) return (((row >> 2) & 1) << 3) | (((row >> 3) & 1) << 2) | (row & 3);
      else return (row >> 1) & 7;
    }
  }
  __device__ static __forceinline__ int at(int row, int piece) { return row * RB + ((piece ^ swz(row)) << 4); }

  // A tile's way into LDS: direct loads (16 bytes per lane, 1 KB per instruction, no registers in between). The LDS side is linear, so the
  // swizzle is in the addresses: lane l of chunk c fills piece p of row r and asks for piece p ^ swz(r). Rows from `count` on lie behind
  // the descriptor's end and arrive as zeros. The waves take the chunks in turn (WAVES = 1: a wave's own tile).
  enum { CHUNKS = BYTES / 1024 / WAVES };
  static_assert(BYTES % (1024 * WAVES) == 0, "whole chunks");
  __device__ static __forceinline__ void dma_offsets(unsigned (&off)[CHUNKS], long long stride_bytes) {
    const int wave = WAVES == 1 ? 0 : threadIdx.x >> 6, lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int byte = (WAVES * i + wave) * 1024 + lane * 16, row = byte / RB, piece = (byte % RB) / 16;
      off[i] = (unsigned)row * (unsigned)stride_bytes + (unsigned)((piece ^ swz(row)) * 16);
    }
  }
  __device__ static __forceinline__ void dma(unsigned lds, const void* src, long long stride_bytes, int count, const unsigned (&off)[CHUNKS]) {
    const unsigned n = count < BN ? (unsigned)(count < 0 ? 0 : count) : BN;
    const at_i32x4 rs = at_rsrc(src, n ? (n - 1) * (unsigned)stride_bytes + RB : 0);
    const unsigned at = lds + (WAVES == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * 1024;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) at_dma(rs, at + i * WAVES * 1024, off[i]);
  }
  // A operand, rows row0 + l % 32, values 16 step + 8 (l / 32) .. + 7 of the row
  __device__ static __forceinline__ typename T::F row_frag(const unsigned char* lds, int row0, int step) {
    const int lane = threadIdx.x & 63, row = row0 + (lane & 31), half = lane >> 5;
    if constexpr (T::ESZ == 2) {
      return __builtin_bit_cast(typename T::F, *reinterpret_cast<const at_u32x4*>(lds + at(row, 2 * step + half)));
    } else {
      at_f32x8 r;
      const at_f32x4 a = *reinterpret_cast<const at_f32x4*>(lds + at(row, 4 * step + 2 * half));
      const at_f32x4 b = *reinterpret_cast<const at_f32x4*>(lds + at(row, 4 * step + 2 * half + 1));
#pragma unroll
      for (int i = 0; i < 4; ++i) { r.v[i] = a[i]; r.v[4 + i] = b[i]; }
      return r;
    }
  }
  // A operand of the transposed tile: row = column 32 block + l % 32 of the tile, values = its rows row0 + {4 h + 0..3, 8 + 4 h + 0..3}
  __device__ static __forceinline__ typename T::F col_frag(const unsigned char* lds, int row0, int block) {
    const int lane = threadIdx.x & 63, half = lane >> 5;
    if constexpr (T::ESZ == 2) {
      // a group of 16 lanes reads four rows of 16 columns (8 bytes per lane) and each lane gets one column of the four
      const int li = lane & 15, g16 = (lane >> 4) & 1, col = 32 * block + 16 * g16 + 4 * (li & 3), row = row0 + 4 * half + (li >> 2);
      typedef __attribute__((address_space(3))) at_s16x4* lp;
      const at_s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + at(row, col >> 3) + (col & 7) * 2));
      const at_s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + at(row + 8, col >> 3) + (col & 7) * 2));
      const at_s16x8 v = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      return __builtin_bit_cast(typename T::F, v);
    } else {
      at_f32x8 r;
      const int col = 32 * block + (lane & 31);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int row = row0 + (i & 4) * 2 + 4 * half + (i & 3);
        r.v[i] = *reinterpret_cast<const float*>(lds + at(row, col >> 2) + (col & 3) * 4);
      }
      return r;
    }
  }
};

// the value of lane l ^ 32 joined with this lane's, without LDS (v_permlane32_swap)
__device__ __forceinline__ float at_pair_max(float x) {
  const at_u32x2 r = __builtin_bit_cast(at_u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float at_pair_sum(float x) {
  const at_u32x2 r = __builtin_bit_cast(at_u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// dynamic LDS above the runtime's default of 64 KB has to be asked for
static inline int at_want_lds(const void* fn, size_t bytes, const char* who) {
  if (bytes > 65536) IRX_CHECK_HIP(hipFuncSetAttribute(fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), who);
  return IRX_OK;
}

#define IRX_LOG2E 1.44269504088896340736f

// The forward's weights are 2^(s - m), m the exponent of weight 1: the running maximum less LIFT, moved only when a row's maximum outgrows it by
// SLACK, so weights stay below 2^(LIFT + SLACK). float16 has 10 bits down to 2^-14, steps of 2^-24 below, and ends at 65504: with the row's
// largest weight at 2^7 or more a weight is off by 2^-11 of itself or 2^-32 of the largest (unlifted 2^-25: where the heaviest key's value is
// zero and 1000 keys at 2^-25 of it make the result, that was all of it). bf16 and float32 have the range.
template <class T> struct AtLift { static constexpr float LIFT = T::ID == IRX_ATTN_F16 ? 7.f : 0.f, SLACK = T::ID == IRX_ATTN_F16 ? 4.f : 8.f; };

// bias of one head by clipped distance, times log2 e, into LDS. A finite bias stays finite (the type's lowest value times log2 e would not).
template <class T> __device__ __forceinline__ void at_load_bias(float* sb, const AtParams& P, int head) {
  for (int i = threadIdx.x; i < 2 * P.far + 1; i += blockDim.x) {
    int b = P.map[i];
    b = b < 0 ? 0 : (b >= P.buckets ? P.buckets - 1 : b);
    float x;
    const size_t at = (size_t)b * P.heads + head;
    if (P.table_f32 || T::ID == IRX_ATTN_F32) x = reinterpret_cast<const float*>(P.table)[at];
    else if constexpr (T::ID == IRX_ATTN_BF16) x = __uint_as_float((unsigned)reinterpret_cast<const unsigned short*>(P.table)[at] << 16);
    else x = (float)reinterpret_cast<const _Float16*>(P.table)[at];
    float y = x * IRX_LOG2E;
    if (fabsf(x) <= 3.402823466e38f) y = fminf(fmaxf(y, -3.402823466e38f), 3.402823466e38f);
    sb[i] = y;
  }
}
