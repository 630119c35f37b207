// irx_attn.hip — attention over packed sequences, forward (grouped heads, causal or full, learned relative position bias by buckets).
//
// One pass over the keys with the running maximum and sum of each row: o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m). A workgroup owns 128
// query rows of one head (four waves, 32 rows each); tiles of 64 keys and their values pass through LDS. The scores are computed transposed
// (keys down, queries across), so that a row of the softmax is one lane pair and the weights are the next product's operand as they are
// (irx_attn.h); the output is accumulated transposed as well and its rescaling is one factor per lane.
// Tiles come by direct loads into the LDS buffer that is not being read, one barrier per tile.
// Measured (six causal sequences of 130 to 2719 rows, 32 / 8 heads of 128, bf16): 184 us, 710 TFLOP/s of visible pairs. Counters there: the
// matrix units are busy 41 % of the time, vector instructions take another 41 % (half of it the exponentials), LDS 20 % without a bank
// conflict: the two waves per SIMD that the registers allow take turns more than they overlap. Tried there and slower: 32-key tiles with
// three waves per SIMD (207), the scores of the next tile beside the weights of this one (275; at dimension 64 without bias 10 % faster),
// wave priorities around the matrix instructions (191), a zigzag order of the tiles (the same).
// Exponents are base 2 (scale * log2 e is folded into one multiply-add per score); scores, weights' sums and the output are 32 bits, the
// weights are rounded to the operand type for the second product, by at most a relative 2^-8 (bf16) or 2^-11 (float16; AtLift has the end of
// its range) each, which is the output's own rounding's size; in short launches they go through it in two terms (fwd_two).
#include "irx_attn.h"

// keys of a tile and workgroups per compute unit that the registers have to allow. 32 keys in float32: half the work where descriptions
// end in the first half of a tile (16 of up to 30 words, dimension 64: 9.7 -> 7.5 us), the same speed on long ones; 16 bits: 64 (long
// causal prompts, dimension 128: 186 us, with 32 and one more workgroup per unit 207).
template <class T, int D> constexpr int fwd_bn() { return T::ESZ == 4 ? 32 : 64; }
template <class T, int D> constexpr int fwd_waves() { return T::ESZ == 4 && D == 128 ? 1 : 2; }

// TWO: a weight enters the second product in two terms, its rounding to 16 bits and the rounding of what that left over (fwd_two).
template <class T, int D, bool BIAS, bool TWO>
__global__ __launch_bounds__(256, (fwd_waves<T, D>())) void k_attn_fwd(AtParams P, int total) {
  constexpr int BN = fwd_bn<T, D>(), N = BN / 2;                        // keys of a tile, scores per lane
  typedef AtTile<T, D, BN> Tile;
  typedef typename T::F F;
  typedef typename T::S S;
  constexpr int STEPS = D / 16, BLOCKS = D / 32;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  float* sb = reinterpret_cast<float*>(smem + 4 * Tile::BYTES);           // two buffers of (keys, values) before it

  // consecutive workgroups go to the 8 XCDs in turn: give each XCD a contiguous run of (head, slot), so that a head's keys and values are
  // read through one L2; the last slots of a sequence, the longest ones under a causal mask, first
  const int per = gridDim.x >> 3;
  const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (id >= total) return;
  const int slot = P.slots - 1 - id % P.slots;
  const int hs = id / P.slots, head = hs % P.heads, part = hs / P.heads;

  int first;
  const AtSpan sp = at_span(P.cu_q, P.batch, P.tq, IRX_ATTN_BM, slot, &first);
  if (sp.begin >= sp.end) return;
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
  const int i0 = row0 - first;                                           // index in the sequence of this wave's first row
  const int lim = P.causal ? min(lk, i0 + (lane & 31) + 1 + off) : lk;   // keys [0, lim) are visible to this lane's row
  const int wave_full = P.causal ? min(lk, i0 + 1 + off) : lk;           // ... to every row of the wave
  const int wave_any = row0 >= sp.end ? 0 : (P.causal ? min(lk, min(i0 + 32, sp.end - first) + off) : lk);
  const int block_any = P.causal ? min(lk, min(sp.begin + IRX_ATTN_BM, sp.end) - first + off) : lk;
  int t0 = 0, t1 = (max(block_any, 0) + BN - 1) / BN;
  if (P.splits > 1) {
    const int n = t1;
    t0 = (int)((long long)n * part / P.splits);
    t1 = (int)((long long)n * (part + 1) / P.splits);
  }
  const int kvh = head / (P.heads / P.kv_heads);
  const S* kp = reinterpret_cast<const S*>(P.k.p) + kb * P.k.st + kvh * P.k.sh;
  const S* vp = reinterpret_cast<const S*>(P.v.p) + kb * P.v.st + kvh * P.v.sh;
  const float c1 = P.scale * IRX_LOG2E;

  F qf[STEPS];
  {
    const S* qp = reinterpret_cast<const S*>(P.q.p) + q * P.q.st + head * P.q.sh + 8 * half;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) qf[s] = mine ? at_ldg<T>(qp + 16 * s) : at_zero<T>();
  }
  if constexpr (BIAS) at_load_bias<T>(sb, P, head);

  at_f32x16 acc[BLOCKS];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[b][i] = 0.f;
  float m = -INFINITY, l = 0.f;               // l: this lane's half of the row only

  // while a tile is worked on, the next one is on its way into the other buffer: one barrier per tile
  const unsigned lds0 = at_lds_addr(smem);
  const long long ks = P.k.st * T::ESZ, vs = P.v.st * T::ESZ;
  unsigned ko[Tile::CHUNKS], vo[Tile::CHUNKS];
  Tile::dma_offsets(ko, ks);
  Tile::dma_offsets(vo, vs);
  auto fetch = [&](int t) __attribute__((always_inline)) {
    const unsigned to = lds0 + ((t - t0) & 1) * 2 * Tile::BYTES;
    const int k0 = t * BN;
    Tile::dma(to, kp + k0 * P.k.st, ks, lk - k0, ko);
    Tile::dma(to + Tile::BYTES, vp + k0 * P.v.st, vs, lk - k0, vo);
  };
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    const int k0 = t * BN;
    at_landed();
    __syncthreads();
    if (t + 1 < t1) fetch(t + 1);
    const unsigned char* lk_ = smem + ((t - t0) & 1) * 2 * Tile::BYTES;
    const unsigned char* lv_ = lk_ + Tile::BYTES;
    if (k0 >= wave_any) continue;
    __builtin_amdgcn_iglp_opt(1);                                        // LDS reads between the matrix instructions: 4 % at dimension 128
    float s[N];
#pragma unroll
    for (int kb2 = 0; kb2 < BN / 32; ++kb2) {
      at_f32x16 x;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = 0.f;
#pragma unroll
      for (int st = 0; st < STEPS; ++st) x = at_mma(Tile::row_frag(lk_, 32 * kb2, st), qf[st], x);
#pragma unroll
      for (int i = 0; i < 16; ++i) s[16 * kb2 + i] = x[i];
    }
    // key of register i: k0 + 8 (i / 4) + 4 half + i % 4
    if constexpr (BIAS) {
#pragma unroll
      for (int kb2 = 0; kb2 < BN / 32; ++kb2) {                                // distances key - query of a 32 x 32 block: lo .. hi
        const int k1 = k0 + 32 * kb2, lo = k1 - (i0 + 31 + off), hi = k1 + 31 - (i0 + off);
        const int d0 = k1 + 4 * half - (i0 + (lane & 31) + off);
        if (hi <= -P.far || lo >= P.far) {
          const float b = sb[hi <= -P.far ? 0 : 2 * P.far];
#pragma unroll
          for (int i = 0; i < 16; ++i) s[16 * kb2 + i] = __builtin_fmaf(s[16 * kb2 + i], c1, b);
        } else if (lo >= -P.far && hi <= P.far) {
          const float* b = sb + d0 + P.far;
#pragma unroll
          for (int i = 0; i < 16; ++i) s[16 * kb2 + i] = __builtin_fmaf(s[16 * kb2 + i], c1, b[8 * (i >> 2) + (i & 3)]);
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[16 * kb2 + i] = __builtin_fmaf(s[16 * kb2 + i], c1, sb[min(max(d0 + 8 * (i >> 2) + (i & 3), -P.far), P.far) + P.far]);
        }
      }
    }
    if (k0 + BN > wave_full) {
      const int left = lim - k0 - 4 * half;
#pragma unroll
      for (int i = 0; i < N; ++i) s[i] = 8 * (i >> 2) + (i & 3) < left ? s[i] : -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < N; ++i) mx = fmaxf(mx, s[i]);
    mx = at_pair_max(mx);
    if constexpr (!BIAS) mx *= c1;                                       // c1 > 0
    mx -= AtLift<T>::LIFT;
    // m moves only when a row outgrows it by SLACK: most tiles rescale nothing
    if (__any(mx > m + AtLift<T>::SLACK || m == -INFINITY)) {
      const float mn = fmaxf(m, mx);
      const float a = mn == -INFINITY ? 1.f : at_exp2(m - mn);
      m = mn;
      l *= a;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][i] *= a;
    }
    const float ms = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      s[i] = at_exp2(BIAS ? s[i] - ms : __builtin_fmaf(s[i], c1, -ms));
      sum += s[i];
    }
    l += sum;
#pragma unroll
    for (int ks = 0; ks < BN / 16; ++ks) {
      const F p = at_pack<T>(s + 8 * ks);
      F rest = p;
      if constexpr (TWO) {
        float r[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = s[8 * ks + e] - at_get<T>(p, e);
        rest = at_pack<T>(r);
      }
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        const F v = Tile::col_frag(lv_, 16 * ks, b);
        acc[b] = at_mma(v, p, acc[b]);
        if constexpr (TWO) acc[b] = at_mma(v, rest, acc[b]);
      }
    }
  }
  l = at_pair_sum(l);
  if (!mine) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;                            // a row that sees nothing: zeros
  if (P.splits > 1) {
    const size_t r = ((size_t)part * P.heads + head) * P.tq + q;
    float* o = P.so + r * D + 4 * half;
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        at_st4<AtF32>(o + 32 * b + 8 * g, acc[b][4 * g] * inv, acc[b][4 * g + 1] * inv, acc[b][4 * g + 2] * inv, acc[b][4 * g + 3] * inv);
    if (half == 0) {
      P.sst[2 * r] = m;
      P.sst[2 * r + 1] = l;
    }
    return;
  }
  const size_t at = ((size_t)q * P.heads + head) * D + 4 * half;
  S* o = reinterpret_cast<S*>(P.dst) + at;
  S* rest = P.dst2 ? reinterpret_cast<S*>(P.dst2) + at : nullptr;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      at_st4_rest<T>(o + 32 * b + 8 * g, rest ? rest + 32 * b + 8 * g : nullptr, acc[b][4 * g] * inv, acc[b][4 * g + 1] * inv, acc[b][4 * g + 2] * inv, acc[b][4 * g + 3] * inv);
  if (P.wstats && half == 0) {
    float* st = P.wstats + ((size_t)head * P.tq + q) * 2;
    st[0] = m == -INFINITY ? 0.f : m;
    st[1] = inv;
  }
}

// Few queries over many keys (single tokens, a handful of instances): the queries of ALL heads that share a key head are one tile of 32
// rows (row = token * group + head of the group), so keys and values are read once per key head, and every wave walks keys of its own:
// tiles of 32 keys through a buffer that only this wave uses, two in turn, no barrier. Bound by reading keys and values (16 tokens over
// 500 to 8100 keys, 16 / 4 heads of 128, bf16: 31 us for 124 MB, 4.0 TB/s, and 4 us for the join); each wave leaves a partial result.
template <class T, int D> constexpr int few_waves() { return T::ESZ == 4 && D == 128 ? 2 : 4; }   // LDS: 64 KB per wave there, 32 KB at most else

template <class T, int D>
__global__ __launch_bounds__((64 * few_waves<T, D>())) void k_attn_few(AtParams P, int total, int tokens) {
  constexpr int WV = few_waves<T, D>(), STEPS = D / 16, BLOCKS = D / 32;
  typedef AtTile<T, D, 32, 1> Tile;
  typedef typename T::F F;
  typedef typename T::S S;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int per = gridDim.x >> 3;
  const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
  if (id >= total) return;
  const int shares = P.splits / WV;                                      // workgroups of one (tile, key head)
  const int share = id % shares, rest = id / shares, kvh = rest % P.kv_heads, slot = rest / P.kv_heads;
  int first;
  const AtSpan sp = at_span(P.cu_q, P.batch, P.tq, tokens, slot, &first);
  if (sp.begin >= sp.end) return;
  const int lane = threadIdx.x & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  int kb = 0, ke = 0;
  if (sp.seq >= 0) {
    kb = __builtin_amdgcn_readfirstlane(at_edge(P.cu_k, P.batch, P.tk, sp.seq + 1));
    ke = __builtin_amdgcn_readfirstlane(at_edge(P.cu_k, P.batch, P.tk, sp.seq + 2));
  }
  const int lk = ke > kb ? ke - kb : 0, off = lk - (sp.end - first);
  const int group = P.heads / P.kv_heads;
  const int row = lane & 31, token = row / group, head = kvh * group + row % group;
  const int q = sp.begin + token;
  const bool mine = token < tokens && q < sp.end;
  const int lim = !mine ? 0 : P.causal ? max(0, min(lk, q - first + 1 + off)) : lk;
  const int full = P.causal ? min(lk, sp.begin - first + 1 + off) : lk;  // keys that every row sees
  const int any = P.causal ? max(0, min(lk, min(sp.begin + tokens, sp.end) - first + off)) : lk;
  const int part = share * WV + wave, n = (any + 31) / 32;
  const int t0 = (int)((long long)n * part / P.splits), t1 = (int)((long long)n * (part + 1) / P.splits);
  const S* kp = reinterpret_cast<const S*>(P.k.p) + kb * P.k.st + kvh * P.k.sh;
  const S* vp = reinterpret_cast<const S*>(P.v.p) + kb * P.v.st + kvh * P.v.sh;
  const float c1 = P.scale * IRX_LOG2E;
  const long long ks = P.k.st * T::ESZ, vs = P.v.st * T::ESZ;
  unsigned ko[Tile::CHUNKS], vo[Tile::CHUNKS];
  Tile::dma_offsets(ko, ks);
  Tile::dma_offsets(vo, vs);
  unsigned char* buf = smem + wave * 4 * Tile::BYTES;
  const unsigned lds0 = at_lds_addr(buf);

  F qf[STEPS];
  {
    const S* qp = reinterpret_cast<const S*>(P.q.p) + q * P.q.st + head * P.q.sh + 8 * half;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) qf[s] = mine ? at_ldg<T>(qp + 16 * s) : at_zero<T>();
  }
  at_f32x16 acc[BLOCKS];
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[b][i] = 0.f;
  float m = -INFINITY, l = 0.f;

  auto fetch = [&](int t) __attribute__((always_inline)) {
    const unsigned to = lds0 + ((t - t0) & 1) * 2 * Tile::BYTES;
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");                   // the buffer's last readers are back
    Tile::dma(to, kp + (long long)t * 32 * P.k.st, ks, lk - t * 32, ko);
    Tile::dma(to + Tile::BYTES, vp + (long long)t * 32 * P.v.st, vs, lk - t * 32, vo);
  };
  at_landed();                                                           // (the queries: from here on only tiles are on their way)
  if (t0 < t1) fetch(t0);
  for (int t = t0; t < t1; ++t) {
    if (t + 1 < t1) {
      fetch(t + 1);
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * Tile::CHUNKS) : "memory");      // everything but that tile
    } else {
      at_landed();
    }
    const unsigned char* lk_ = buf + ((t - t0) & 1) * 2 * Tile::BYTES;
    const unsigned char* lv_ = lk_ + Tile::BYTES;
    at_f32x16 x;
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 0.f;
#pragma unroll
    for (int st = 0; st < STEPS; ++st) x = at_mma(Tile::row_frag(lk_, 0, st), qf[st], x);
    float s[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = x[i];
    if (t * 32 + 32 > full) {
      const int left = lim - t * 32 - 4 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[i] = 8 * (i >> 2) + (i & 3) < left ? s[i] : -INFINITY;
    }
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
    mx = at_pair_max(mx) * c1 - AtLift<T>::LIFT;
    if (__any(mx > m + AtLift<T>::SLACK || m == -INFINITY)) {
      const float mn = fmaxf(m, mx);
      const float a = mn == -INFINITY ? 1.f : at_exp2(m - mn);
      m = mn;
      l *= a;
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][i] *= a;
    }
    const float ms = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      s[i] = at_exp2(__builtin_fmaf(s[i], c1, -ms));
      l += s[i];
    }
#pragma unroll
    for (int k2 = 0; k2 < 2; ++k2) {
      const F p = at_pack<T>(s + 8 * k2);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) acc[b] = at_mma(Tile::col_frag(lv_, 16 * k2, b), p, acc[b]);
    }
  }
  l = at_pair_sum(l);
  if (!mine) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const size_t r = ((size_t)part * P.heads + head) * P.tq + q;
  float* o = P.so + r * D + 4 * half;
#pragma unroll
  for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      at_st4<AtF32>(o + 32 * b + 8 * g, acc[b][4 * g] * inv, acc[b][4 * g + 1] * inv, acc[b][4 * g + 2] * inv, acc[b][4 * g + 3] * inv);
  if (half == 0) {
    P.sst[2 * r] = m;
    P.sst[2 * r + 1] = l;
  }
}

// Joins the parts of a row: o = sum_p w_p o_p / sum_p w_p, w_p = l_p 2^(m_p - max m), by groups of D / 4 threads. Many rows (MANY): a group
// per row, parts in order. Few: a workgroup per row, group g takes every G-th part, the groups' sums are joined in their order. Always the
// same result. 98 312 rows of 64 in two parts: 15 us by groups, 112 by workgroups (idle groups); 256 rows of 128 in 64 parts: 9 and 4.
template <class T, int D, bool MANY>
__global__ __launch_bounds__(256) void k_attn_join(AtParams P) {
  constexpr int PER = D / 4, G = 256 / PER;
  __shared__ at_f32x4 so[G][PER];
  __shared__ float sl[G];
  const int c = threadIdx.x % PER, g = threadIdx.x / PER, d = 4 * c;
  const size_t row = MANY ? (size_t)blockIdx.x * G + g : blockIdx.x, rows = (size_t)P.heads * P.tq;          // head * tq + q
  if (MANY && row >= rows) return;
  float M = -INFINITY;
#pragma unroll 4
  for (int p = 0; p < P.splits; ++p) M = fmaxf(M, P.sst[2 * (p * rows + row)]);
  const float Ms = M == -INFINITY ? 0.f : M;
  float L = 0.f;
  at_f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int p = MANY ? 0 : g; p < P.splits; p += MANY ? 1 : G) {
    const float l = P.sst[2 * (p * rows + row) + 1];
    const at_f32x4 x = *reinterpret_cast<const at_f32x4*>(P.so + (p * rows + row) * D + d);
    const float w = l == 0.f ? 0.f : l * at_exp2(P.sst[2 * (p * rows + row)] - Ms);
    L += w;
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = __builtin_fmaf(w, x[i], o[i]);
  }
  if constexpr (!MANY) {
    so[g][c] = o;
    if (c == 0) sl[g] = L;
    __syncthreads();
    if (g) return;
    L = sl[0];
#pragma unroll
    for (int i = 1; i < G; ++i) {
      L += sl[i];
      o += so[i][c];
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const size_t head = row / P.tq, q = row % P.tq;
  typedef typename T::S S;
  const size_t at = (q * P.heads + head) * D + d;
  at_st4_rest<T>(reinterpret_cast<S*>(P.dst) + at, P.dst2 ? reinterpret_cast<S*>(P.dst2) + at : nullptr, o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv);
  if (P.wstats && c == 0) {
    P.wstats[2 * row] = Ms;
    P.wstats[2 * row + 1] = inv;
  }
}

// (512 workgroups of rows: two per compute unit, from there on the parts are read at memory speed)
template <class T, int D> static int launch_join(const AtParams& P, hipStream_t st) {
  constexpr int G = 256 / (D / 4);
  const size_t rows = (size_t)P.heads * P.tq;
  if (rows >= 512 * G) k_attn_join<T, D, true><<<(unsigned)((rows + G - 1) / G), 256, 0, st>>>(P);
  else k_attn_join<T, D, false><<<(unsigned)rows, 256, 0, st>>>(P);
  IRX_CHECK_LAUNCH("irx_attn_packed_fwd(join)");
  return IRX_OK;
}

template <class T, int D> static int launch_few(AtParams P, int tokens, hipStream_t st) {
  const size_t lds = (size_t)few_waves<T, D>() * 4 * AtTile<T, D, 32, 1>::BYTES;
  P.slots = at_slots(P.tq, P.batch, tokens);
  const long long total = (long long)P.slots * P.kv_heads * (P.splits / few_waves<T, D>());
  if (int rc = at_want_lds(reinterpret_cast<const void*>(&k_attn_few<T, D>), lds, "irx_attn_packed_fwd")) return rc;
  k_attn_few<T, D><<<(unsigned)((total + 7) / 8 * 8), 64 * few_waves<T, D>(), lds, st>>>(P, (int)total, tokens);
  IRX_CHECK_LAUNCH("irx_attn_packed_fwd(few)");
  return launch_join<T, D>(P, st);
}

template <class T, int D, bool BIAS, bool TWO> static int launch_fwd(const AtParams& P, hipStream_t st) {
  const size_t lds = 4 * AtTile<T, D, fwd_bn<T, D>()>::BYTES + (BIAS ? sizeof(float) * (2 * P.far + 1) : 0);
  const long long total = (long long)P.slots * P.heads * P.splits;
  const unsigned grid = (unsigned)((total + 7) / 8 * 8);
  if (int rc = at_want_lds(reinterpret_cast<const void*>(&k_attn_fwd<T, D, BIAS, TWO>), lds, "irx_attn_packed_fwd")) return rc;
  k_attn_fwd<T, D, BIAS, TWO><<<grid, 256, lds, st>>>(P, (int)total);
  IRX_CHECK_LAUNCH("irx_attn_packed_fwd");
  return P.splits > 1 ? launch_join<T, D>(P, st) : IRX_OK;
}

// Two terms per weight where a 16-bit launch is short and leaves compute units without a workgroup: the output is then the exact one rounded once,
// and the gradients' D = out . dout does not carry the weights' rounding into every dS, which shows most in short sequences (57 rows, dimension 128, bf16:
// dq's error 1.51 times its own rounding, 1.41 with two terms). It costs nothing there but at the limit (256 rows, 64 heads, forward: dimension 64 9.4 us
// both ways, dimension 128 10.4 and 11.4). Everywhere it would cost the matrix-bound launches 4 to 8 % of both passes (12289 causal rows, 8 heads of
// 64, fp16: 900 and 972 us), and long rows average the weights' rounding out (dq 1.44 to 1.46, at dimension 32 1.49).
static bool fwd_two(const AtParams& P) {
  if (P.batch <= 0) return false;
  const long long busy = P.batch < P.tq ? P.batch : P.tq;
  return (P.tq / IRX_ATTN_BM + busy) * P.heads <= 256 && P.tk / P.batch <= 256;
}
template <class T, int D, bool BIAS> static int launch_fwd_t(const AtParams& P, hipStream_t st) {
  if constexpr (T::ESZ == 2)
    if (fwd_two(P)) return launch_fwd<T, D, BIAS, true>(P, st);
  return launch_fwd<T, D, BIAS, false>(P, st);
}
template <class T, int D> static int launch_fwd_b(const AtParams& P, int tokens, hipStream_t st) {
  if (tokens) return launch_few<T, D>(P, tokens, st);
  return P.table ? launch_fwd_t<T, D, true>(P, st) : launch_fwd_t<T, D, false>(P, st);
}
template <class T> static int launch_fwd_d(const AtParams& P, int dim, int tokens, hipStream_t st) {
  return dim == 32 ? launch_fwd_b<T, 32>(P, tokens, st) : dim == 64 ? launch_fwd_b<T, 64>(P, tokens, st) : launch_fwd_b<T, 128>(P, tokens, st);
}

int at_check(const char* who, const AtParams& P, int dim, int dtype, int elem) {
  IRX_REQUIRE(dtype >= IRX_ATTN_F32 && dtype <= IRX_ATTN_F16, "%s: type %d (0 float32, 1 bfloat16, 2 float16)", who, dtype);
  IRX_REQUIRE(dim == 32 || dim == 64 || dim == 128, "%s: head dimension %d (32, 64 or 128)", who, dim);
  IRX_REQUIRE(P.batch >= 0 && P.tq >= 0 && P.tk >= 0, "%s: negative size", who);
  IRX_REQUIRE(P.heads >= 1 && P.kv_heads >= 1 && P.heads % P.kv_heads == 0, "%s: %d heads over %d key / value heads", who, P.heads, P.kv_heads);
  IRX_REQUIRE(P.scale > 0.f && P.scale <= 3.402823466e38f, "%s: the scale must be positive and finite", who);
  IRX_REQUIRE(P.cu_q && P.cu_k, "%s: null offsets", who);
  const AtTensor* ts[4] = {&P.q, &P.k, &P.v, &P.dout};
  for (int i = 0; i < 4; ++i) {
    const AtTensor& t = *ts[i];
    if (i == 3 && !t.p) continue;
    const int rows = (i == 0 || i == 3) ? P.tq : P.tk;
    IRX_REQUIRE(t.p || rows == 0, "%s: null tensor", who);
    IRX_REQUIRE(((uintptr_t)t.p & 15) == 0 && (t.st * elem) % 16 == 0 && (t.sh * elem) % 16 == 0, "%s: rows and heads must start on 16 bytes", who);
    IRX_REQUIRE(t.st >= 0 && t.sh >= 0, "%s: negative stride", who);
    IRX_REQUIRE(t.st * elem < (1ll << 24), "%s: rows more than 16 MB apart", who);      // 64 rows of a tile: 32-bit byte offsets
  }
  if (P.table) {
    IRX_REQUIRE(P.map && P.buckets >= 1, "%s: a bias table needs its bucket map", who);
    IRX_REQUIRE(P.far >= 0 && P.far <= IRX_ATTN_MAX_FAR, "%s: clipped distance %d (at most %d)", who, P.far, IRX_ATTN_MAX_FAR);
  }
  const long long rows = P.tq > P.tk ? P.tq : P.tk;
  IRX_REQUIRE(rows + P.batch + 2 < (1ll << 30), "%s: too many rows", who);
  // (256 threads each, fewer than 2^32 in a launch; the backward's holds a workgroup per value of the bias table besides)
  IRX_REQUIRE((rows / IRX_ATTN_BM + P.batch + 2) * P.heads < 3ll << 22, "%s: too many tiles", who);
  IRX_REQUIRE(!P.table || (long long)P.buckets * P.heads < 1ll << 22, "%s: a bias table of %d buckets", who, P.buckets);
  return IRX_OK;
}

// How the forward is launched, by sizes alone. Few: the average sequence's queries, times the heads that share a key head, fit one tile
// of 32 rows, and there are many keys (16 single tokens over 500 to 8100 keys, 16 / 4 heads of 128: 35 us with the join, without it 83;
// about 256 workgroups: 512 41, 1024 51). Else parts of the key axis only where the whole launch is below a round of two workgroups per
// compute unit (4096 causal rows, 8 heads of 64, bf16: 67 us whole, 54 in three parts; 2048 rows, 16 heads of 128, full: 67 whole, 57 in two, 66 in
// three; 16000 causal, 4 heads of 128: 389 whole, 285 in two) or, causal, not far above it (12289 rows, 8 heads of 64,
// fp16: 245 and 222; 6000 rows, 12 heads of 64: 136 and 104; but 6000 rows, 16 heads of 128: 168 and 186, so the rule weighs the keys, which
// make the join cheap, against how full the second round is). tokens: queries of a few-row tile, 0: no.
struct FwdPlan { int tokens, splits; };
static FwdPlan fwd_plan(long long tq, long long tk, int batch, int heads, int kv_heads, int dim, int elem, bool bias, bool causal) {
  if (batch <= 0 || tk <= 0 || tq <= 0) return {0, 1};
  const long long keys = tk / batch, busy = batch < tq ? batch : tq;
  const int group = heads / kv_heads;
  if (!bias && group <= 32 && tq <= (long long)batch * (32 / group) && keys >= 512) {
    const int tokens = 32 / group, waves = elem == 4 && dim == 128 ? 2 : 4;
    long long s = (256 + busy * kv_heads - 1) / (busy * kv_heads);
    if (s > keys / 256) s = keys / 256;
    if (s < 1) s = 1;
    if (s > 16) s = 16;
    return {tokens, (int)s * waves};
  }
  const long long wgs = (tq / IRX_ATTN_BM + busy) * heads;
  return {0, at_key_parts(wgs, keys, elem, causal)};
}

extern "C" size_t irx_attn_packed_fwd_workspace_bytes(int tq, int tk, int batch, int heads, int kv_heads, int dim, int dtype, int mask) {
  if (tq <= 0 || tk < 0 || batch < 0 || heads <= 0 || kv_heads <= 0 || dim <= 0) return 0;
  const int s = fwd_plan(tq, tk, batch, heads, kv_heads, dim, dtype == IRX_ATTN_F32 ? 4 : 2, mask & 1, mask & 2).splits;
  return s <= 1 ? 0 : (size_t)s * heads * tq * (dim + 2) * sizeof(float);
}

extern "C" int irx_attn_packed_fwd(const void* q, long long q_row, long long q_head, const void* k, long long k_row, long long k_head,
                                   const void* v, long long v_row, long long v_head, const int32_t* cu_q, const int32_t* cu_k, int batch,
                                   int tq, int tk, int heads, int kv_heads, int dim, int dtype, float scale, int causal, const void* table,
                                   int table_f32, const int32_t* map, int buckets, int far, void* out, void* rest, float* stats, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  AtParams P = {};
  P.q = {q, q_row, q_head};
  P.k = {k, k_row, k_head};
  P.v = {v, v_row, v_head};
  P.cu_q = cu_q; P.cu_k = cu_k;
  P.batch = batch; P.tq = tq; P.tk = tk; P.heads = heads; P.kv_heads = kv_heads; P.causal = causal != 0; P.scale = scale;
  P.table = table; P.table_f32 = table_f32; P.map = map; P.buckets = buckets; P.far = far;
  P.dst = out; P.dst2 = dtype == IRX_ATTN_F32 ? nullptr : rest; P.wstats = stats;
  if (int rc = at_check("irx_attn_packed_fwd", P, dim, dtype, dtype == IRX_ATTN_F32 ? 4 : 2)) return rc;
  if (tq == 0) return IRX_OK;
  IRX_REQUIRE(out && (((uintptr_t)out | (uintptr_t)rest) & 15) == 0, "irx_attn_packed_fwd: out must be given and start on 16 bytes");
  P.slots = at_slots(tq, batch, IRX_ATTN_BM);
  const FwdPlan plan = fwd_plan(tq, tk, batch, heads, kv_heads, dim, dtype == IRX_ATTN_F32 ? 4 : 2, table != nullptr, causal != 0);
  P.splits = plan.splits;
  if (P.splits > 1) {
    const size_t need = irx_attn_packed_fwd_workspace_bytes(tq, tk, batch, heads, kv_heads, dim, dtype, (table != nullptr) + 2 * (causal != 0));
    if (!workspace || workspace_bytes < need) {
      irx_set_error("irx_attn_packed_fwd: workspace of %zu bytes, %zu needed", workspace_bytes, need);
      return IRX_ERR_WORKSPACE;
    }
    IRX_REQUIRE(((uintptr_t)workspace & 15) == 0, "irx_attn_packed_fwd: workspace must start on 16 bytes");
    P.so = static_cast<float*>(workspace);
    P.sst = P.so + (size_t)P.splits * heads * tq * dim;
  }
  hipStream_t st = (hipStream_t)stream;
  if (dtype == IRX_ATTN_F32) return launch_fwd_d<AtF32>(P, dim, plan.tokens, st);
  if (dtype == IRX_ATTN_BF16) return launch_fwd_d<AtBf16>(P, dim, plan.tokens, st);
  return launch_fwd_d<AtF16>(P, dim, plan.tokens, st);
}

extern "C" int irx_stream_capturing(void* stream) {
  if (!stream) return 0;
  hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing((hipStream_t)stream, &s) != hipSuccess) {
    (void)hipGetLastError();
    return 0;
  }
  return s != hipStreamCaptureStatusNone;
}
