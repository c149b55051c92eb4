// Linear attention with a decay for each head and, optionally, the delta
// rule, over packed sequences and a state S [Dk, Dv] of each (sequence, head):
//
//   S_t = a_t S_{t-1} + k_t u_t^T,   o_t = scale S_t^T q_t,   a_t = exp(g_t)
//   u_t = v_t,  or with beta  u_t = beta_t (v_t - a_t S_{t-1}^T k_t)
//
// Two forms, both right for sequences of any lengths: token by token with
// the state in registers, and in chunks of 64 tokens on the matrix cores.
// With G the running sum of g in a chunk that starts from S0:
//
//   (I + A) U = B (V - e^G K S0),  A_tj = beta_t e^{G_t - G_j} k_t.k_j  (j < t)
//   O = scale (e^G Q S0 + P U),    P_tj = e^{G_t - G_j} q_t.k_j         (j <= t)
//   S = e^{G_C} S0 + K^T (e^{G_C - G} U)
//
// T = (I + A)^-1 B and P depend on no state: one kernel makes them for all
// chunks at once, a second takes each (sequence, head, 16 columns of the
// state) through its chunks.
//
// The state and everything that goes into it keep fp32's precision on the
// bf16 matrix instructions: k is bf16 as it comes, an fp32 factor goes in as
// the three bf16 pieces whose sum it is (its 24 bits cut into 8 + 8 + 8),
// and of the products of two such factors those below 2^-24 are left out.
// The outputs, rounded to bf16 in the end, take two pieces (2^-16).  The sums
// G are made in 64 bits: a strong decay early in a chunk would otherwise cost
// the later differences their last places.
#include "common.h"
#include "kernels.h"

namespace rmoe {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kLinThreads = 256;
constexpr float kLeastLogDecay = -1.0e4f;  // exp of it is 0; keeps sums of -inf apart

struct Seq {
  int64_t begin;
  int len;
};

// Rows of sequence r, inside [0, tokens) whatever cu holds.
__device__ __forceinline__ Seq seq_of(const LinearArgs& a, int r) {
  const int b = min(max(a.cu[r], 0), a.tokens);
  const int e = min(max(a.cu[r + 1], b), a.tokens);
  return {b, e - b};
}

__device__ __forceinline__ float log_decay(const LinearArgs& a, int64_t row, int h) {
  const float g = a.decay[row * a.decay_row + h * a.decay_head];
  return g < kLeastLogDecay ? kLeastLogDecay : g;
}

__device__ __forceinline__ int64_t slot_of(const LinearArgs& a, int r) {
  const int64_t s = a.index ? a.index[r] : r;
  return s >= 0 && s < a.slots ? s : -1;
}

// Rows of `out` in front of the first sequence and behind the last one.
__device__ void clear_uncovered(const LinearArgs& a, int part, int parts) {
  const int64_t w = (int64_t)a.v_heads * a.dv / 8;  // 16-byte pieces of a row
  const int64_t lo = min(max(a.cu[0], 0), a.tokens) * w;
  const int64_t hi = (int64_t)min(max(a.cu[a.requests], 0), a.tokens) * w;
  const int64_t end = (int64_t)a.tokens * w;
  const uint4 z = make_uint4(0, 0, 0, 0);
  uint4* o = reinterpret_cast<uint4*>(a.out);
  const int64_t step = (int64_t)parts * kLinThreads;
  const int64_t at = (int64_t)part * kLinThreads + threadIdx.x;
  for (int64_t i = at; i < lo; i += step) o[i] = z;
  for (int64_t i = hi + at; i < end; i += step) o[i] = z;
}

constexpr int kClearParts = 16;  // workgroups that look for uncovered rows

// ------------------------------------------------------------ token by token
// A wave holds 16 columns of a state: lane (rg, c) the rows rg DK/16 .. of
// columns 4 c .. 4 c + 3.  Both sums over the rows, S^T k and S^T q, are of
// the state before the token, so a token costs one round of exchanges:
// o = a S^T q + (q.k) u.
template <int DK, bool DELTA>
__global__ __launch_bounds__(kLinThreads) void linear_step_kernel(const LinearArgs a) {
  constexpr int RW = DK / 16;  // rows of a lane
  const int tiles = a.dv / 16;
  const int64_t waves = (int64_t)a.requests * a.v_heads * tiles;
  const int64_t groups = (waves + 3) / 4;
  if (blockIdx.x >= groups) {
    clear_uncovered(a, (int)(blockIdx.x - groups), kClearParts);
    return;
  }
  const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (id >= waves) return;
  const int lane = threadIdx.x & 63, c = lane & 3, rg = lane >> 2;
  const int tile = (int)(id % tiles);
  const int hv = (int)(id / tiles % a.v_heads);
  const int r = (int)(id / tiles / a.v_heads);
  const int hk = hv / (a.v_heads / a.k_heads);
  const int col = tile * 16 + c * 4;
  const int64_t slot = slot_of(a, r);
  const int64_t at = ((slot * a.v_heads + hv) * DK + rg * RW) * a.dv + col;
  f32x4 s[RW];
#pragma unroll
  for (int i = 0; i < RW; ++i)
    s[i] = slot >= 0 ? *reinterpret_cast<const f32x4*>(a.state + at + (int64_t)i * a.dv)
                     : (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  const Seq q = seq_of(a, r);
  for (int t = 0; t < q.len; ++t) {
    const int64_t row = q.begin + t;
    const uint16_t* kp = a.k + row * a.k_row + hk * a.k_head + rg * RW;
    const uint16_t* qp = a.q + row * a.q_row + hk * a.q_head + rg * RW;
    float kv[RW], qv[RW];
#pragma unroll
    for (int i = 0; i < RW; i += 4) {
      const uint2 ku = *reinterpret_cast<const uint2*>(kp + i);
      const uint2 qu = *reinterpret_cast<const uint2*>(qp + i);
      kv[i] = bf16_lo(ku.x), kv[i + 1] = bf16_hi(ku.x);
      kv[i + 2] = bf16_lo(ku.y), kv[i + 3] = bf16_hi(ku.y);
      qv[i] = bf16_lo(qu.x), qv[i + 1] = bf16_hi(qu.x);
      qv[i + 2] = bf16_lo(qu.y), qv[i + 3] = bf16_hi(qu.y);
    }
    const uint16_t* vp = a.v + row * a.v_row + hv * a.v_head + col;
    float u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = bf16_to_f32(vp[j]);
    const float g = log_decay(a, row, hv);
    const float decay = expf(g);
    float beta = 1.0f;
    if constexpr (DELTA) beta = a.beta[row * a.beta_row + hv * a.beta_head];

    float sk[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sq[4] = {0.0f, 0.0f, 0.0f, 0.0f}, qk = 0.0f;
#pragma unroll
    for (int i = 0; i < RW; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (DELTA) sk[j] = fmaf(s[i][j], kv[i], sk[j]);
        sq[j] = fmaf(s[i][j], qv[i], sq[j]);
      }
      qk = fmaf(qv[i], kv[i], qk);
    }
#pragma unroll
    for (int d = 4; d < kWave; d <<= 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (DELTA) sk[j] += __shfl_xor(sk[j], d, kWave);
        sq[j] += __shfl_xor(sq[j], d, kWave);
      }
      qk += __shfl_xor(qk, d, kWave);
    }
    if constexpr (DELTA) {
#pragma unroll
      for (int j = 0; j < 4; ++j) u[j] = beta * (u[j] - decay * sk[j]);
    }
#pragma unroll
    for (int i = 0; i < RW; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) s[i][j] = fmaf(kv[i], u[j], decay * s[i][j]);
    if (rg == 0) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = f32_to_bf16(a.scale * fmaf(qk, u[j], decay * sq[j]));
      *reinterpret_cast<uint2*>(a.out + (row * a.v_heads + hv) * a.dv + col) =
          make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
    }
  }
  if (slot < 0) return;
#pragma unroll
  for (int i = 0; i < RW; ++i)
    *reinterpret_cast<f32x4*>(a.state_out + at + (int64_t)i * a.dv) = s[i];
}

// ------------------------------------------------------------------ in chunks
constexpr int kChunk = 64;
constexpr int kStep = 1024;  // bytes of one operand A of 16 x 32 values, in lane order

// Operand blocks of a wave's 16 rows: columns 0..31 for all four waves, then
// 32..63 for waves 2 and 3 (the others' are above the diagonal).
__device__ __forceinline__ int block_of(int wave, int ks) { return ks ? 2 + wave : wave; }
constexpr int kBlocks = 6;

// Workspace of one (chunk, value head): T's blocks in three pieces, P's in
// two, then e^G and e^{G_C - G} of its 64 tokens and e^{G_C}.
template <bool DELTA>
struct ChunkData {
  static constexpr int t = 0;
  static constexpr int p = DELTA ? kBlocks * 3 * kStep : 0;
  static constexpr int scal = p + kBlocks * 2 * kStep;
  static constexpr int bytes = scal + (2 * kChunk + 4) * 4;
};

// The chunks of sequence r start at number cu[r] / 64 + r, which leaves room
// for the part chunk that each sequence may end in, and needs no sums.
__device__ __forceinline__ int64_t chunk_base(const LinearArgs& a, int r) {
  return min(max(a.cu[r], 0), a.tokens) / kChunk + r;
}

__device__ __forceinline__ bf16x8 frag(const uint32_t (&w)[4]) {
  union {
    uint32_t w[4];
    bf16x8 v;
  } u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u.w[i] = w[i];
  return u.v;
}
__device__ __forceinline__ bf16x8 frag(const uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  return frag(w);
}
__device__ __forceinline__ f32x4 mfma(const bf16x8 a, const bf16x8 b, const f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// The upper halves of two words, the first one's below.
__device__ __forceinline__ uint32_t uppers(uint32_t a, uint32_t b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302);
}
// v[i] = sum of N pieces of 8 bits, each cut off the rest (the last of two is
// rounded by the cut, 2^-16; three are v itself): packed pairs of bf16.
template <int N>
__device__ __forceinline__ void pieces(const f32x4 v, uint32_t (&w)[N][2]) {
  float x[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int p = 0; p < N; ++p) {
    w[p][0] = uppers(__float_as_uint(x[0]), __float_as_uint(x[1]));
    w[p][1] = uppers(__float_as_uint(x[2]), __float_as_uint(x[3]));
    if (p + 1 < N) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        x[i] -= __uint_as_float(__float_as_uint(x[i]) & 0xFFFF0000u);
    }
  }
}

// LDS traffic of this wave done, then the barrier; loads from memory stay in
// flight across it.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

template <int DK, bool DELTA>
__global__ __launch_bounds__(kLinThreads) void linear_prepare_kernel(const LinearArgs a) {
  constexpr int KS = DK / 32;
  constexpr int MT = DK / 64;  // 16-row tiles of the state that a wave keeps
  constexpr int LD = kChunk + 4;
  __shared__ double Gs[kChunk];
  __shared__ float bs[kChunk];
  __shared__ float As[DELTA ? kChunk * LD : 1];
  __shared__ float Ts[DELTA ? kChunk * LD : 1];

  const int64_t blocks = a.chunks * a.v_heads;
  if (blockIdx.x >= blocks) {
    clear_uncovered(a, (int)(blockIdx.x - blocks), kClearParts);
    return;
  }
  const int64_t c = blockIdx.x / a.v_heads;
  const int hv = (int)(blockIdx.x - c * a.v_heads);
  const int each = a.v_heads / a.k_heads;
  const int hk = hv / each;
  int r = 0, hi = a.requests;  // the last r whose chunks start at or before c
  while (hi - r > 1) {
    const int mid = (r + hi) >> 1;
    if (chunk_base(a, mid) <= c)
      r = mid;
    else
      hi = mid;
  }
  const Seq sq = seq_of(a, r);
  const int64_t first = (c - chunk_base(a, r)) * kChunk;
  if (first < 0 || first >= sq.len) return;
  const int64_t row0 = sq.begin + first;
  const int len = (int)(sq.len - first < kChunk ? sq.len - first : kChunk);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;

  // running sums of the log decays, one token a lane
  double G = lane < len ? (double)log_decay(a, row0 + lane, hv) : 0.0;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const double up = __shfl_up(G, d, kWave);
    if (lane >= d) G += up;
  }
  const double Gc = __shfl(G, 63, kWave);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace) +
                (c * a.v_heads + hv) * (int64_t)ChunkData<DELTA>::bytes;
  if (wave == 0) {
    Gs[lane] = G;
    if constexpr (DELTA)
      bs[lane] = lane < len ? a.beta[(row0 + lane) * a.beta_row + hv * a.beta_head] : 0.0f;
    float* scal = reinterpret_cast<float*>(ws + ChunkData<DELTA>::scal);
    scal[lane] = expf((float)G);
    scal[kChunk + lane] = lane < len ? expf((float)(Gc - G)) : 0.0f;
    if (lane == 0) scal[2 * kChunk] = expf((float)Gc);
  }

  // 16 rows of q or k as an operand; rows past the end repeat the last one
  auto rows16 = [&](const uint16_t* x, int64_t row_stride, int64_t head_stride, int tile,
                    bf16x8(&f)[KS]) {
    const int i = 16 * tile + n;
    const uint16_t* p = x + (row0 + (i < len ? i : len - 1)) * row_stride + hk * head_stride + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) f[s] = frag(load16(p + 32 * s));
  };
  bf16x8 kf[KS], qf[KS];
  rows16(a.k, a.k_row, a.k_head, wave, kf);
  rows16(a.q, a.q_row, a.q_head, wave, qf);
  __syncthreads();

  // K_j K_w^T and K_j Q_w^T, tile j of the columns against the wave's own
  // rows: lane (g, n) gets row t = 16 w + n, columns 16 j + 4 g + i, which is
  // operand A's order (contraction index 8 g + 4 (j & 1) + i)
  const int t = 16 * wave + n;
  const double Gt = Gs[t];
  const float bt = DELTA ? bs[t] : 0.0f;
  f32x4 pt[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    pt[j] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    if (j > wave) continue;
    bf16x8 kj[KS];
    rows16(a.k, a.k_row, a.k_head, j, kj);
    f32x4 kk = {0.0f, 0.0f, 0.0f, 0.0f}, qk = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if constexpr (DELTA) kk = mfma(kj[s], kf[s], kk);
      qk = mfma(kj[s], qf[s], qk);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = 16 * j + 4 * g + i;
      const float e = m <= t && t < len ? expf((float)(Gt - Gs[m])) : 0.0f;
      qk[i] = m <= t && t < len ? qk[i] * e : 0.0f;
      kk[i] = m < t && t < len ? bt * (kk[i] * e) : 0.0f;
    }
    pt[j] = qk;
    if constexpr (DELTA) *reinterpret_cast<f32x4*>(&As[t * LD + 16 * j + 4 * g]) = kk;
  }
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    if (2 * ks > wave) continue;
    uint32_t lo[2][2], up[2][2];
    pieces<2>(pt[2 * ks], lo);
    pieces<2>(pt[2 * ks + 1], up);
    uint8_t* dst = ws + ChunkData<DELTA>::p + block_of(wave, ks) * 2 * kStep + lane * 16;
#pragma unroll
    for (int p = 0; p < 2; ++p)
      *reinterpret_cast<uint4*>(dst + p * kStep) = make_uint4(lo[p][0], lo[p][1], up[p][0], up[p][1]);
  }

  // K^T for the update, once for the value heads that share it: row m of the
  // wave's tile h is k's dim 32 ks + 8 (m / 4) + 4 h' + m % 4 (ks, h' the tile
  // number's upper part and lowest bit), the order in which the second
  // product of the state's own registers needs them
  if (hv % each == 0) {
    uint8_t* kt = static_cast<uint8_t*>(a.workspace) + a.kt_offset +
                  (c * a.k_heads + hk) * (int64_t)(8 * MT * kStep);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int tg = wave * MT + mt;
      const int d = 32 * (tg >> 1) + 8 * (n >> 2) + 4 * (tg & 1) + (n & 3);
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          uint32_t x[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int i = 32 * ks + 16 * ((j + e) >> 2) + 4 * g + ((j + e) & 3);
            x[e] = a.k[(row0 + (i < len ? i : len - 1)) * a.k_row + hk * a.k_head + d];
          }
          w[j >> 1] = x[0] | x[1] << 16;
        }
        *reinterpret_cast<uint4*>(kt + ((wave * MT + mt) * 2 + ks) * kStep + lane * 16) =
            make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  if constexpr (!DELTA) return;

  // T = (I + A)^-1: the four diagonal blocks by substitution, a column a
  // lane; then T_ij = -T_ii sum_k A_ik T_kj, one diagonal of blocks after
  // the other, on the fp32 matrix instruction.
  __syncthreads();
  {
    const int d0 = 16 * wave;
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float acc = i == n ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; ++j) acc = fmaf(-As[(d0 + i) * LD + d0 + j], x[j], acc);
      x[i] = acc;
    }
    if (g == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) Ts[(d0 + i) * LD + d0 + n] = x[i];
    }
  }
  __syncthreads();
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    if (wave + d < 4) {
      const int bi = wave + d, bj = wave;
      f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int k = bj; k < bi; ++k) {
        const f32x4 av = *reinterpret_cast<const f32x4*>(&As[(16 * bi + n) * LD + 16 * k + 4 * g]);
#pragma unroll
        for (int s = 0; s < 4; ++s)
          x = __builtin_amdgcn_mfma_f32_16x16x4f32(
              av[s], Ts[(16 * k + 4 * g + s) * LD + 16 * bj + n], x, 0, 0, 0);
      }
      const f32x4 dv = *reinterpret_cast<const f32x4*>(&Ts[(16 * bi + n) * LD + 16 * bi + 4 * g]);
      f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < 4; ++s) y = __builtin_amdgcn_mfma_f32_16x16x4f32(-dv[s], x[s], y, 0, 0, 0);
#pragma unroll
      for (int s = 0; s < 4; ++s) Ts[(16 * bi + 4 * g + s) * LD + 16 * bj + n] = y[s];
    }
    __syncthreads();
  }
  // times B, as operand A in three pieces
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    if (2 * ks > wave) continue;
    uint32_t w[2][3][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
      if (2 * ks + h <= wave) {
        const int col = 32 * ks + 16 * h + 4 * g;
        v = *reinterpret_cast<const f32x4*>(&Ts[t * LD + col]);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] *= bs[col + i];
      }
      pieces<3>(v, w[h]);
    }
    uint8_t* dst = ws + ChunkData<DELTA>::t + block_of(wave, ks) * 3 * kStep + lane * 16;
#pragma unroll
    for (int p = 0; p < 3; ++p)
      *reinterpret_cast<uint4*>(dst + p * kStep) =
          make_uint4(w[0][p][0], w[0][p][1], w[1][p][0], w[1][p][1]);
  }
}

template <int DK, bool DELTA>
__global__ __launch_bounds__(kLinThreads) void linear_chunk_kernel(const LinearArgs a) {
  constexpr int KS = DK / 32;
  constexpr int MT = DK / 64;
  constexpr int UP = DELTA ? 2 : 1;  // pieces of U in P U (without beta it is v, which is bf16)
  __shared__ uint4 Sf[3][KS][kWave];
  __shared__ uint4 Rf[DELTA ? 3 : 1][2][kWave];
  __shared__ uint4 Uf[UP + 3][2][kWave];

  // the column tiles of a head on one XCD, whose L2 holds the head's chunk
  const int tiles = a.dv / 16;
  const int64_t heads = (int64_t)a.requests * a.v_heads;
  const int64_t b = blockIdx.x;
  const int64_t per_xcd = (heads + 7) / 8 * tiles;
  const int64_t in_xcd = b >> 3;
  const int64_t head = (in_xcd / tiles) * 8 + (b & 7);
  if (in_xcd >= per_xcd || head >= heads) return;
  const int tile = (int)(in_xcd % tiles);
  const int r = (int)(head / a.v_heads), hv = (int)(head - (int64_t)r * a.v_heads);
  const int hk = hv / (a.v_heads / a.k_heads);
  const Seq sq = seq_of(a, r);
  const int64_t slot = slot_of(a, r);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int col = tile * 16 + n;

  // state: tile tg = wave MT + mt, lane (g, n): dims 32 (tg / 2) + 8 g +
  // 4 (tg % 2) + i of column n
  f32x4 S[MT];
  int64_t at[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int tg = wave * MT + mt;
    const int d = 32 * (tg >> 1) + 8 * g + 4 * (tg & 1);
    at[mt] = ((slot * a.v_heads + hv) * DK + d) * a.dv + col;
#pragma unroll
    for (int i = 0; i < 4; ++i) S[mt][i] = slot >= 0 ? a.state[at[mt] + (int64_t)i * a.dv] : 0.0f;
  }

  const int chunks = (sq.len + kChunk - 1) / kChunk;
  const int64_t c0 = chunk_base(a, r);
  const uint8_t* ws0 = static_cast<const uint8_t*>(a.workspace) +
                       (c0 * a.v_heads + hv) * (int64_t)ChunkData<DELTA>::bytes;
  const int64_t ws_step = (int64_t)a.v_heads * ChunkData<DELTA>::bytes;
  const uint8_t* kt0 = static_cast<const uint8_t*>(a.workspace) + a.kt_offset +
                       (c0 * a.k_heads + hk) * (int64_t)(8 * MT * kStep);
  const int64_t kt_step = (int64_t)a.k_heads * (8 * MT * kStep);
  const bool two = wave >= 2;  // blocks of the second 32 columns

  uint4 kf[KS], qf[KS], ktf[MT][2], tf[DELTA ? 3 : 1][2], pf[2][2];
  uint32_t vv[4];
  float eG[4], dec[4], eC;
  auto load_kq = [&](int c) {
    if (c >= chunks) return;
    const int i = c * kChunk + 16 * wave + n;
    const int64_t row = sq.begin + (i < sq.len ? i : sq.len - 1);
    const uint16_t* kp = a.k + row * a.k_row + hk * a.k_head + 8 * g;
    const uint16_t* qp = a.q + row * a.q_row + hk * a.q_head + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      if constexpr (DELTA) kf[s] = load16(kp + 32 * s);
      qf[s] = load16(qp + 32 * s);
    }
  };
  auto load_v = [&](int c) {
    if (c >= chunks) return;
    const float* scal = reinterpret_cast<const float*>(ws0 + c * ws_step + ChunkData<DELTA>::scal);
    const int i0 = 16 * wave + 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int j = c * kChunk + i0 + i;
      const int64_t row = sq.begin + (j < sq.len ? j : sq.len - 1);
      vv[i] = a.v[row * a.v_row + hv * a.v_head + col];
    }
    const f32x4 e = *reinterpret_cast<const f32x4*>(scal + i0);
    const f32x4 d = *reinterpret_cast<const f32x4*>(scal + kChunk + i0);
#pragma unroll
    for (int i = 0; i < 4; ++i) eG[i] = e[i], dec[i] = d[i];
    eC = scal[2 * kChunk];
  };
  auto load_t = [&](int c) {
    if (!DELTA || c >= chunks) return;
    const uint8_t* p = ws0 + c * ws_step + ChunkData<DELTA>::t + lane * 16;
#pragma unroll
    for (int i = 0; i < (DELTA ? 3 : 0); ++i) {
      tf[i][0] = load16(p + (block_of(wave, 0) * 3 + i) * kStep);
      if (two) tf[i][1] = load16(p + (block_of(wave, 1) * 3 + i) * kStep);
    }
  };
  auto load_p = [&](int c) {
    if (c >= chunks) return;
    const uint8_t* p = ws0 + c * ws_step + ChunkData<DELTA>::p + lane * 16;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      pf[i][0] = load16(p + (block_of(wave, 0) * 2 + i) * kStep);
      if (two) pf[i][1] = load16(p + (block_of(wave, 1) * 2 + i) * kStep);
    }
    const uint8_t* k = kt0 + c * kt_step + lane * 16;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) ktf[mt][ks] = load16(k + ((wave * MT + mt) * 2 + ks) * kStep);
  };
  load_kq(0);
  load_v(0);
  load_t(0);
  load_p(0);

  for (int c = 0; c < chunks; ++c) {
    // the state in three pieces, as operand B of the wave's dims
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int tg = wave * MT + mt;
      uint32_t w[3][2];
      pieces<3>(S[mt], w);
#pragma unroll
      for (int p = 0; p < 3; ++p)
        reinterpret_cast<uint2*>(&Sf[p][tg >> 1][lane])[tg & 1] = make_uint2(w[p][0], w[p][1]);
    }
    lds_barrier();
    f32x4 ksum[3], qsum[2];
#pragma unroll
    for (int p = 0; p < 3; ++p) ksum[p] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
    qsum[0] = qsum[1] = ksum[0];
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        if (!DELTA && p == 2) continue;
        const bf16x8 f = frag(Sf[p][s][lane]);
        if constexpr (DELTA) ksum[p] = mfma(frag(kf[s]), f, ksum[p]);
        if (p < 2) qsum[p] = mfma(frag(qf[s]), f, qsum[p]);
      }
    load_kq(c + 1);

    f32x4 u;
    if constexpr (DELTA) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        u[i] = bf16_to_f32(vv[i]) - eG[i] * (ksum[0][i] + (ksum[1][i] + ksum[2][i]));
      uint32_t w[3][2];
      pieces<3>(u, w);
#pragma unroll
      for (int p = 0; p < 3; ++p)
        reinterpret_cast<uint2*>(&Rf[p][wave >> 1][lane])[wave & 1] = make_uint2(w[p][0], w[p][1]);
      lds_barrier();
      f32x4 big = {0.0f, 0.0f, 0.0f, 0.0f}, small = big, least = big;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (ks && !two) continue;
        const bf16x8 r0 = frag(Rf[0][ks][lane]), r1 = frag(Rf[1][ks][lane]),
                     r2 = frag(Rf[2][ks][lane]);
        const bf16x8 t0 = frag(tf[0][ks]), t1 = frag(tf[1][ks]), t2 = frag(tf[2][ks]);
        big = mfma(t0, r0, big);
        small = mfma(t0, r1, small);
        least = mfma(t0, r2, least);
        small = mfma(t1, r0, small);
        least = mfma(t1, r1, least);
        least = mfma(t2, r0, least);
      }
      u = big + (small + least);
      load_t(c + 1);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = bf16_to_f32(vv[i]);
    }
    {
      uint32_t w[UP][2], x[3][2];
      pieces<UP>(u, w);
      f32x4 d;
#pragma unroll
      for (int i = 0; i < 4; ++i) d[i] = dec[i] * u[i];
      pieces<3>(d, x);
#pragma unroll
      for (int p = 0; p < UP; ++p)
        reinterpret_cast<uint2*>(&Uf[p][wave >> 1][lane])[wave & 1] = make_uint2(w[p][0], w[p][1]);
#pragma unroll
      for (int p = 0; p < 3; ++p)
        reinterpret_cast<uint2*>(&Uf[UP + p][wave >> 1][lane])[wave & 1] =
            make_uint2(x[p][0], x[p][1]);
    }
    lds_barrier();
    f32x4 o0 = {0.0f, 0.0f, 0.0f, 0.0f}, o1 = o0;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      if (ks && !two) continue;
      const bf16x8 u0 = frag(Uf[0][ks][lane]);
      o0 = mfma(frag(pf[0][ks]), u0, o0);
      o1 = mfma(frag(pf[1][ks]), u0, o1);
      if constexpr (DELTA) o1 = mfma(frag(pf[0][ks]), frag(Uf[1][ks][lane]), o1);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      f32x4 s0 = {0.0f, 0.0f, 0.0f, 0.0f}, s1 = s0, s2 = s0;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        const bf16x8 k = frag(ktf[mt][ks]);
        s0 = mfma(k, frag(Uf[UP][ks][lane]), s0);
        s1 = mfma(k, frag(Uf[UP + 1][ks][lane]), s1);
        s2 = mfma(k, frag(Uf[UP + 2][ks][lane]), s2);
      }
      S[mt] = eC * S[mt] + (s0 + (s1 + s2));
    }
    load_p(c + 1);
    const int i0 = c * kChunk + 16 * wave + 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float o = a.scale * (eG[i] * (qsum[0][i] + qsum[1][i]) + (o0[i] + o1[i]));
      if (i0 + i < sq.len)
        a.out[((sq.begin + i0 + i) * a.v_heads + hv) * a.dv + col] = (uint16_t)f32_to_bf16(o);
    }
    load_v(c + 1);
  }
  if (slot < 0) return;
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
#pragma unroll
    for (int i = 0; i < 4; ++i) a.state_out[at[mt] + (int64_t)i * a.dv] = S[mt][i];
}

template <int DK, bool DELTA>
hipError_t launch_linear_of(const LinearArgs& a, hipStream_t s) {
  const int clear = a.clear ? kClearParts : 0;
  const int64_t tiles = a.dv / 16;
  if (!a.workspace) {
    const int64_t waves = (int64_t)a.requests * a.v_heads * tiles;
    linear_step_kernel<DK, DELTA><<<(unsigned)((waves + 3) / 4 + clear), kLinThreads, 0, s>>>(a);
    return hipGetLastError();
  }
  linear_prepare_kernel<DK, DELTA>
      <<<(unsigned)(a.chunks * a.v_heads + clear), kLinThreads, 0, s>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t heads = (int64_t)a.requests * a.v_heads;
  linear_chunk_kernel<DK, DELTA>
      <<<(unsigned)((heads + 7) / 8 * 8 * tiles), kLinThreads, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace

bool linear_in_chunks(int64_t tokens, int requests) { return tokens > 16 * (int64_t)requests; }

LinearLayout linear_layout(int64_t tokens, int requests, int k_heads, int v_heads, int dk,
                           bool delta) {
  LinearLayout l;
  l.chunks = tokens / kChunk + requests;
  l.kt_offset = l.chunks * v_heads *
                (int64_t)(delta ? ChunkData<true>::bytes : ChunkData<false>::bytes);
  l.total = l.kt_offset + l.chunks * k_heads * (int64_t)(8 * (dk / 64) * kStep);
  return l;
}

hipError_t launch_linear(const LinearArgs& a, hipStream_t s) {
  if (a.dk == 64) return a.delta ? launch_linear_of<64, true>(a, s) : launch_linear_of<64, false>(a, s);
  return a.delta ? launch_linear_of<128, true>(a, s) : launch_linear_of<128, false>(a, s);
}

}  // namespace rmoe
