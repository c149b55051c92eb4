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
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

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

// 32-column waves from which the token form takes them (2048: 13.2 us against
// 12.8 with twice as many of 16, 4096: 28 against 31)
constexpr int64_t kWideStates = 4096;
constexpr int kClearParts = 16;  // workgroups that look for uncovered rows

// The sequences that go in chunks, more than a.by_token tokens: list[0] is their
// count, their numbers are from list[1] on, those with more chunks (by
// powers of two) first, so that the longest do not start last.  One workgroup.
__device__ void list_long(const LinearArgs& a) {
  __shared__ int counts[2][kLinThreads / kWave];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  auto length = [&](int r) { return r < a.requests ? seq_of(a, r).len : 0; };
  const bool few = a.requests <= kLinThreads;  // each thread's length stays with it
  const int first = few ? length(tid) : 0;
  int at = 0, turn = 0;
  for (int level = 31 - __clz((a.tokens + 63) / 64); level >= 0; --level) {
    for (int r0 = 0; r0 < a.requests; r0 += kLinThreads, turn ^= 1) {
      const int r = r0 + tid;
      const int len = few ? first : length(r);
      const bool mine = len > a.by_token && 31 - __clz((len + 63) / 64) == level;
      const uint64_t mask = __ballot(mine);
      if (lane == 0) counts[turn][wave] = __popcll(mask);
      __syncthreads();
      int before = 0, all = 0;
      for (int w = 0; w < kLinThreads / kWave; ++w) {
        before += w < wave ? counts[turn][w] : 0;
        all += counts[turn][w];
      }
      if (mine) a.list[1 + at + before + __popcll(mask & ((1ull << lane) - 1))] = r;
      at += all;
    }
  }
  if (tid == 0) a.list[0] = at;
}

// ------------------------------------------------------------ token by token
// Sum over the lanes equal modulo LC (4, 8 or 16): rotations inside 16 lanes,
// then the swaps across them, all without LDS.
template <int LC>
__device__ __forceinline__ float sum_over_rows(float v) {
  if constexpr (LC < 16)  // row_ror:8
    v += __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xF, 0xF, false));
  if constexpr (LC < 8)  // row_ror:4
    v += __int_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xF, 0xF, false));
  const uint32_t u = __float_as_uint(v);
  const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const uint32_t w = __float_as_uint(v);
  const auto b = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// A wave holds 4 LC columns of a state: lane (rg, c) the rows rg RW .. of
// columns 4 c .. 4 c + 3.  Both sums over the rows, S^T k and S^T q, are of
// the state before the token, so a token costs one round of exchanges:
// o = a S^T q + (q.k) u.  Bound by the state's read and write: 127 tokens x 32
// heads of 128 x 128 101 us, 5.3 TB/s.  LC 8 moves whole lines (there 106 us
// before the next token was loaded ahead, against 121 with LC 4 and 108 with
// 16), LC 4 has twice the waves for few states (one token x 32 heads: 4.4 us,
// 5.6 with LC 8).
template <int DK, bool DELTA, int LC>
__device__ __forceinline__ void by_token(const LinearArgs& a, int64_t group) {
  constexpr int RW = DK * LC / kWave;  // rows of a lane
  const int tiles = a.dv / (4 * LC);
  const int64_t id = group * 4 + (threadIdx.x >> 6);
  if (id >= (int64_t)a.requests * a.v_heads * tiles) return;
  const int lane = threadIdx.x & 63, c = lane % LC, rg = lane / LC;
  const int tile = (int)(id % tiles);
  const int hv = (int)(id / tiles % a.v_heads);
  const int r = (int)(id / tiles / a.v_heads);
  const int hk = hv / (a.v_heads / a.k_heads);
  const int col = (tile * LC + c) * 4;
  const Seq q = seq_of(a, r);
  if (a.list && q.len > a.by_token) return;
  const int64_t slot = slot_of(a, r);
  const int64_t at = ((slot * a.v_heads + hv) * DK + rg * RW) * a.dv + col;
  f32x4 s[RW];
#pragma unroll
  for (int i = 0; i < RW; ++i)
    s[i] = slot >= 0 ? *reinterpret_cast<const f32x4*>(a.state + at + (int64_t)i * a.dv)
                     : (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  // a token's inputs, asked for while the one before is worked on
  struct Token {
    uint2 k[RW / 4], q[RW / 4];
    uint16_t v[4];
    float g, beta;
  };
  auto load = [&](int t) {
    Token x;
    const int64_t row = q.begin + (t < q.len ? t : q.len - 1);
    const uint16_t* kp = a.k + row * a.k_row + hk * a.k_head + rg * RW;
    const uint16_t* qp = a.q + row * a.q_row + hk * a.q_head + rg * RW;
    const uint16_t* vp = a.v + row * a.v_row + hv * a.v_head + col;
#pragma unroll
    for (int i = 0; i < RW / 4; ++i) {
      x.k[i] = reinterpret_cast<const uint2*>(kp)[i];
      x.q[i] = reinterpret_cast<const uint2*>(qp)[i];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) x.v[j] = vp[j];
    x.g = log_decay(a, row, hv);
    x.beta = DELTA ? a.beta[row * a.beta_row + hv * a.beta_head] : 1.0f;
    return x;
  };
  Token next;
  if (q.len > 0) next = load(0);
  for (int t = 0; t < q.len; ++t) {
    const int64_t row = q.begin + t;
    const Token x = next;
    if (q.len > 1) next = load(t + 1);
    float kv[RW], qv[RW], u[4];
#pragma unroll
    for (int i = 0; i < RW / 4; ++i) {
      kv[4 * i] = bf16_lo(x.k[i].x), kv[4 * i + 1] = bf16_hi(x.k[i].x);
      kv[4 * i + 2] = bf16_lo(x.k[i].y), kv[4 * i + 3] = bf16_hi(x.k[i].y);
      qv[4 * i] = bf16_lo(x.q[i].x), qv[4 * i + 1] = bf16_hi(x.q[i].x);
      qv[4 * i + 2] = bf16_lo(x.q[i].y), qv[4 * i + 3] = bf16_hi(x.q[i].y);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) u[j] = bf16_to_f32(x.v[j]);
    const float decay = expf(x.g), beta = x.beta;

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
    for (int j = 0; j < 4; ++j) {
      if constexpr (DELTA) sk[j] = sum_over_rows<LC>(sk[j]);
      sq[j] = sum_over_rows<LC>(sq[j]);
    }
    qk = sum_over_rows<LC>(qk);
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

// Workgroups that take all sequences by token, 4 LC columns a wave.
__host__ __device__ __forceinline__ int64_t token_groups(const LinearArgs& a, int lc) {
  return ((int64_t)a.requests * a.v_heads * (a.dv / (4 * lc)) + 3) / 4;
}

template <int DK, bool DELTA, int LC>
__global__ __launch_bounds__(kLinThreads) void linear_step_kernel(const LinearArgs a) {
  const int64_t groups = token_groups(a, LC);
  if (blockIdx.x < groups)
    by_token<DK, DELTA, LC>(a, blockIdx.x);
  else
    clear_uncovered(a, (int)(blockIdx.x - groups), kClearParts);
}

// ------------------------------------------------------------------ in chunks
constexpr int kChunk = 64;
constexpr int kFewTokens = 8;
constexpr int kChunkThreads = 12 * kWave;
constexpr int kStep = 1024;  // bytes of one operand A of 16 x 32 values, in lane order

// Workspace of one (chunk, value head): the 16 x 16 tiles of T and P on and
// below the diagonal (tile (w, j) at number w (w + 1) / 2 + j), as operand A in
// pieces: for each lane its four values of a tile, T's first two pieces and
// P's two as 16 bytes, T's third as 8; then a line each for the four token
// waves (e^G and e^{G_C - G} of their tokens) and for the four state waves
// (e^{G_C}).  Of one (chunk, key head): q and k as operand A.  Every wave that
// reads these reads whole lines that no other wave of its workgroup does.
constexpr int kTiles = 10;
template <bool DELTA>
struct ChunkData {
  static constexpr int p = 0;
  static constexpr int t01 = kTiles * kStep;
  static constexpr int t2 = DELTA ? 2 * kTiles * kStep : t01;
  static constexpr int token = DELTA ? t2 + kTiles * kStep / 2 : t01;
  static constexpr int state = token + 4 * 128;
  static constexpr int bytes = state + 4 * 128;
};
template <int DK>
struct KeyData {
  static constexpr int part = DK / 32 * 4 * kStep;
  static constexpr int q = 0, k = part, bytes = 2 * part;
};
__device__ __forceinline__ int tile_of(int w, int j) { return w * (w + 1) / 2 + j; }

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

template <int CTRL, int ROWS>
__device__ __forceinline__ double from_lane(double v) {  // 0 where there is none
  return __hiloint2double(
      __builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, ROWS, 0xf, false),
      __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, ROWS, 0xf, false));
}

// Everything of a chunk that no state goes into, a workgroup per (chunk,
// value head), 16 tokens a wave.  Bound by the latency of its steps, so it
// keeps few registers and 30 KB of LDS: five workgroups a compute unit.  Each
// wave loads its own 16 rows of k and takes the others' from LDS (from memory
// each tile was a wait of its own); exponentials are of sums kept in base 2.
template <int DK, bool DELTA>
__device__ __forceinline__ void prepare(const LinearArgs& a, int64_t block) {
  constexpr int KS = DK / 32;
  constexpr int LD = 20;              // row of a 16 x 16 tile in LDS
  constexpr int TILE = 16 * LD;
  __shared__ double Gs[kChunk];
  __shared__ __align__(16) float bs[kChunk];
  __shared__ __align__(16) float As[DELTA ? kTiles * TILE : 4];
  // k as operand rows, then (with every wave past that) T
  constexpr int SHARED = KS * 4 * kWave * 4;
  __shared__ __align__(16) float Ts[SHARED > kTiles * TILE ? SHARED : kTiles * TILE];

  const int64_t c = block / a.v_heads;
  const int hv = (int)(block - c * a.v_heads);
  const int each = a.v_heads / a.k_heads;
  const int hk = hv / each;
  // the last r whose chunks start at or before c: 64 of them looked at at a
  // time, one a lane (9 sequences of 5 to 1500 tokens: prepared in 12.7 us,
  // 13.1 by bisection)
  int r = 0;
  for (int left = a.requests; left > 1;) {
    const int step = (left + kWave - 1) / kWave;
    const int at = (threadIdx.x & 63) * step;
    const uint64_t before = __ballot(at < left && chunk_base(a, r + at) <= c);
    const int skip = before ? (__popcll(before) - 1) * step : 0;
    r += skip;
    left = left - skip < step ? left - skip : step;
  }
  const Seq sq = seq_of(a, r);
  const int64_t first = (c - chunk_base(a, r)) * kChunk;
  if (first < 0 || first >= sq.len || (a.list && sq.len <= a.by_token)) return;
  const int64_t row0 = sq.begin + first;
  const int len = (int)(sq.len - first < kChunk ? sq.len - first : kChunk);

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  const int t = 16 * wave + n;  // the lane's token

  // 16 rows of k and of q as operands; rows past the end repeat the last one
  uint4 kf[KS], qf[KS];
  {
    const int64_t row = row0 + (t < len ? t : len - 1);
    const uint16_t* kp = a.k + row * a.k_row + hk * a.k_head + 8 * g;
    const uint16_t* qp = a.q + row * a.q_row + hk * a.q_head + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) kf[s] = load16(kp + 32 * s);
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = load16(qp + 32 * s);
  }
  // running sums of the log decays in base 2, one token a lane
  constexpr double kLog2e = 1.44269504088896340736;
  double G = lane < len ? (double)log_decay(a, row0 + lane, hv) * kLog2e : 0.0;
  float beta = 0.0f;
  if (DELTA && lane < len) beta = a.beta[(row0 + lane) * a.beta_row + hv * a.beta_head];
  G += from_lane<0x111, 0xf>(G);  // one lane to the left in a row of 16, then 2, 4, 8
  G += from_lane<0x112, 0xf>(G);
  G += from_lane<0x114, 0xf>(G);
  G += from_lane<0x118, 0xf>(G);
  G += from_lane<0x142, 0xa>(G);  // a row's last lane to the next row, of 32 to the next 32
  G += from_lane<0x143, 0xc>(G);
  const double Gc = __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(G), kWave - 1),
                                     __builtin_amdgcn_readlane(__double2loint(G), kWave - 1));
  uint8_t* ws = static_cast<uint8_t*>(a.workspace) +
                (c * a.v_heads + hv) * (int64_t)ChunkData<DELTA>::bytes;
  if (wave == 0) {
    Gs[lane] = G;
    if constexpr (DELTA) bs[lane] = beta;
    float* token = reinterpret_cast<float*>(ws + ChunkData<DELTA>::token) + 32 * g + n;
    token[0] = __builtin_amdgcn_exp2f((float)G);
    token[16] = lane < len ? __builtin_amdgcn_exp2f((float)(Gc - G)) : 0.0f;
    if (n == 0)
      *reinterpret_cast<float*>(ws + ChunkData<DELTA>::state + 128 * g) =
          __builtin_amdgcn_exp2f((float)Gc);
  }
  uint4* Ks = reinterpret_cast<uint4*>(Ts);
#pragma unroll
  for (int s = 0; s < KS; ++s) Ks[(s * 4 + wave) * kWave + lane] = kf[s];
  __syncthreads();

  // K_j K_w^T and K_j Q_w^T, tile j of the columns against the wave's own
  // rows: lane (g, n) gets row t = 16 w + n, columns 16 j + 4 g + i, which is
  // operand A's order (contraction index 8 g + 4 (j & 1) + i)
  const double Gt = Gs[t];
  const float bt = DELTA ? bs[t] : 0.0f;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j > wave) continue;
    f32x4 kk = {0.0f, 0.0f, 0.0f, 0.0f}, qk = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const bf16x8 kj = frag(Ks[(s * 4 + j) * kWave + lane]);
      if constexpr (DELTA) kk = mfma(kj, frag(kf[s]), kk);
      qk = mfma(kj, frag(qf[s]), qk);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int m = 16 * j + 4 * g + i;
      const bool in = m <= t && t < len;
      const float e = __builtin_amdgcn_exp2f((float)(Gt - Gs[m]));
      qk[i] = in ? qk[i] * e : 0.0f;
      kk[i] = in && m < t ? bt * (kk[i] * e) : 0.0f;
    }
    uint32_t w[2][2];
    pieces<2>(qk, w);
    *reinterpret_cast<uint4*>(ws + ChunkData<DELTA>::p + tile_of(wave, j) * kStep + lane * 16) =
        make_uint4(w[0][0], w[0][1], w[1][0], w[1][1]);
    if constexpr (DELTA) *reinterpret_cast<f32x4*>(&As[tile_of(wave, j) * TILE + n * LD + 4 * g]) = kk;
  }

  // q and k in operand order, once for the value heads that share them: rows
  // of all heads lie far apart, and a product needs half a line of each
  if (hv % each == 0) {
    uint8_t* key = static_cast<uint8_t*>(a.workspace) + a.key_offset +
                   (c * a.k_heads + hk) * (int64_t)KeyData<DK>::bytes + lane * 16;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      *reinterpret_cast<uint4*>(key + KeyData<DK>::q + (4 * s + wave) * kStep) = qf[s];
      *reinterpret_cast<uint4*>(key + KeyData<DK>::k + (4 * s + wave) * kStep) = kf[s];
    }
  }
  if constexpr (!DELTA) return;

  // T = (I + A)^-1: the four diagonal tiles by substitution, a column a lane;
  // then T_ij = -T_ii sum_k A_ik T_kj, one diagonal of tiles after the other,
  // on the fp32 matrix instruction.
  __syncthreads();
  {
    const float* d = &As[tile_of(wave, wave) * TILE];
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float acc = i == n ? 1.0f : 0.0f;
#pragma unroll
      for (int j = 0; j < i; ++j) acc = fmaf(-d[i * LD + j], x[j], acc);
      x[i] = acc;
    }
    if (g == 0) {
      float* o = &Ts[tile_of(wave, wave) * TILE];
#pragma unroll
      for (int i = 0; i < 16; ++i) o[i * LD + n] = x[i];
    }
  }
  __syncthreads();
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    if (wave + d < 4) {
      const int bi = wave + d, bj = wave;
      f32x4 x = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int e = 0; e < d; ++e) {
        const int k = bj + e;
        const f32x4 av = *reinterpret_cast<const f32x4*>(&As[tile_of(bi, k) * TILE + n * LD + 4 * g]);
        const float* tk = &Ts[tile_of(k, bj) * TILE + 4 * g * LD + n];
#pragma unroll
        for (int s = 0; s < 4; ++s)
          x = __builtin_amdgcn_mfma_f32_16x16x4f32(av[s], tk[s * LD], x, 0, 0, 0);
      }
      const f32x4 dv = *reinterpret_cast<const f32x4*>(&Ts[tile_of(bi, bi) * TILE + n * LD + 4 * g]);
      f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < 4; ++s) y = __builtin_amdgcn_mfma_f32_16x16x4f32(-dv[s], x[s], y, 0, 0, 0);
      float* o = &Ts[tile_of(bi, bj) * TILE + 4 * g * LD + n];
#pragma unroll
      for (int s = 0; s < 4; ++s) o[s * LD] = y[s];
    }
    __syncthreads();
  }
  // times B, as operand A in three pieces
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j > wave) continue;
    const int at = tile_of(wave, j);
    f32x4 v = *reinterpret_cast<const f32x4*>(&Ts[at * TILE + n * LD + 4 * g]);
    v *= *reinterpret_cast<const f32x4*>(&bs[16 * j + 4 * g]);
    uint32_t w[3][2];
    pieces<3>(v, w);
    *reinterpret_cast<uint4*>(ws + ChunkData<DELTA>::t01 + at * kStep + lane * 16) =
        make_uint4(w[0][0], w[0][1], w[1][0], w[1][1]);
    *reinterpret_cast<uint2*>(ws + ChunkData<DELTA>::t2 + at * (kStep / 2) + lane * 8) =
        make_uint2(w[2][0], w[2][1]);
  }
}

// The first launch of a call in chunks: the preparation of every chunk, and
// where lengths may differ the short sequences (whole, by token) and the list
// of the others beside it.
template <int DK, bool DELTA>
__global__ __launch_bounds__(kLinThreads, 5) void linear_prepare_kernel(const LinearArgs a) {
  int64_t block = blockIdx.x;
  if (a.list) {
    if (block == 0) return list_long(a);
    block -= 1;
    const int64_t groups = token_groups(a, 4);
    if (block < groups) return by_token<DK, DELTA, 4>(a, block);
    block -= groups;
  }
  const int64_t chunks = a.chunks * a.v_heads;
  if (block < chunks) return prepare<DK, DELTA>(a, block);
  clear_uncovered(a, (int)(block - chunks), kClearParts);
}

// One (sequence, head, 16 NT columns of the state) from chunk to chunk, twelve
// waves, three to a SIMD (one alone waits between its instructions):
//
//   - state waves 0 to 3 hold 32 dims of the state each and multiply them, as
//     they lie in their registers, by those dims of all 64 tokens: an
//     accumulator's lane holds rows 4 g + i of its column, four of the eight
//     contraction indices that the same lane needs in operand B;
//   - token waves 4 to 7 take 16 tokens each, add up the partial K S and make U;
//   - output waves 8 to 11 take 16 tokens each and make q S and, when U is
//     there, the outputs, while the others are in the next chunk.
//
// With the delta rule a chunk is a chain of three exchanges through LDS
// (partial K S, the residual, U) between the first two; what is not in the
// chain (outputs, q S, turning k, loads) is done by whoever is not in it.
// Without it U is v, and one exchange is left.
template <int DK, bool DELTA, int NT>
__device__ __forceinline__ void through_chunks(const LinearArgs& a, int r, int hv, int tile) {
  constexpr int KS = DK / 32;         // state waves
  constexpr int SP = DELTA ? 3 : 2;   // pieces of the state that a product takes
  constexpr int UP = DELTA ? 2 : 1;   // of U in P U (v alone is bf16 as it is)
  constexpr int BUF = DELTA ? 1 : 2;  // one exchange a chunk: two buffers in turn
  __shared__ f32x4 Kp[DELTA ? KS : 1][4 * NT][kWave];  // partial K S of each 16 tokens
  // q S: of the output waves, from two pieces of the state; without beta, where
  // they are the busiest, of the state waves, in parts
  __shared__ uint4 Sf[2][KS][NT][kWave];
  __shared__ f32x4 Qp[BUF][DELTA ? 1 : KS][4 * NT][kWave];
  __shared__ uint4 Rf[DELTA ? 3 : 1][2][NT][kWave];
  __shared__ uint4 Uf[BUF][UP + 3][2][NT][kWave];
  __shared__ uint4 Kt[KS][4][kWave];  // a state wave's dims of k, to be transposed

  const int hk = hv / (a.v_heads / a.k_heads);
  const Seq sq = seq_of(a, r);
  const int64_t slot = slot_of(a, r);

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int w4 = wave & 3;  // its dims 32 w4 .. or its tokens 16 w4 ..
  const int n = lane & 15, g = lane >> 4;
  const int col = tile * (16 * NT) + n;  // and every 16th on
  const int chunks = (sq.len + kChunk - 1) / kChunk;
  const int64_t c0 = chunk_base(a, r);
  const char* ws0 = static_cast<const char*>(a.workspace) +
                    (c0 * a.v_heads + hv) * (int64_t)ChunkData<DELTA>::bytes;
  const int64_t ws_step = (int64_t)a.v_heads * ChunkData<DELTA>::bytes;
  const uint32_t l16 = lane * 16;
  // State and token waves load their operands two chunks ahead, into two sets
  // used in turn, each kind while the chain is with the other; output waves,
  // which have time, one chunk ahead.  Past the end the last chunk's are loaded
  // again, which needs no branch.
  auto clamped = [&](int c) { return c < chunks ? c : chunks - 1; };

  if (wave < 4) {
    // -------------------------------------------------------- state waves
    if (w4 >= KS) {  // with 64 dims there are two
      for (int c = 0; c < chunks; ++c) {
        lds_barrier();
        if constexpr (DELTA) {
          lds_barrier();
          lds_barrier();
        }
      }
      return;
    }
    // lane (g, n) of tile h: dims 32 w4 + 8 g + 4 h + i of column 16 nt + n
    f32x4 S[NT][2];
    const int64_t at = ((slot * a.v_heads + hv) * DK + 32 * w4 + 8 * g) * a.dv + col;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          S[nt][h][i] = slot >= 0 ? a.state[at + (int64_t)(4 * h + i) * a.dv + 16 * nt] : 0.0f;

    const char* key0 = static_cast<const char*>(a.workspace) + a.key_offset +
                       (c0 * a.k_heads + hk) * (int64_t)KeyData<DK>::bytes + w4 * 4 * kStep;
    const int64_t key_step = (int64_t)a.k_heads * KeyData<DK>::bytes;
    struct Loads {
      uint4 k[4], q[DELTA ? 1 : 4];
      float eC;
    };
    // the wave's dims of 64 tokens of k and, without beta, of q
    auto load = [&](int c, Loads& x) {
      c = clamped(c);
      const char* k = key0 + c * key_step;
#pragma unroll
      for (int t = 0; t < 4; ++t) x.k[t] = load16(k + KeyData<DK>::k + t * kStep + l16);
      if constexpr (!DELTA) {
#pragma unroll
        for (int t = 0; t < 4; ++t) x.q[t] = load16(k + KeyData<DK>::q + t * kStep + l16);
      }
      x.eC = *reinterpret_cast<const float*>(ws0 + c * ws_step + ChunkData<DELTA>::state +
                                             128 * w4 + 4 * (uint32_t)(lane >> 6));
    };
    // K^T as operand A: the wave's own dims, turned in LDS.  The transposing
    // read gives lane m of 16 column m of the 4 rows of 16 values that the 16
    // lanes' addresses (4 values each) name: rows are tokens 4 g + i, columns
    // dims 8 (m / 4) + 4 h + m % 4, the order of the state's registers.
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4* lds_s16x4;
    const int turned = ((n & 3) * 16 + 4 * g + (n >> 2)) * 8;  // in 2-byte values
    auto transpose = [&](const Loads& x, bf16x8(&kt)[2][2]) {
#pragma unroll
      for (int t = 0; t < 4; ++t) Kt[w4][t][lane] = x.k[t];
      uint16_t* base = reinterpret_cast<uint16_t*>(&Kt[w4][0][0]) + turned;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          union {
            s16x4 half[2];
            bf16x8 v;
          } u;
#pragma unroll
          for (int e = 0; e < 2; ++e)
            u.half[e] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_s16x4)(base + (2 * ks + e) * (kStep / 2) + 4 * h));
          kt[h][ks] = u.v;
        }
    };
    auto step = [&](int c, Loads& now) {
      const int b = DELTA ? 0 : c & 1;
      bf16x8 sf[NT][SP];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint32_t lo[SP][2], up[SP][2];
        pieces<SP>(S[nt][0], lo);
        pieces<SP>(S[nt][1], up);
#pragma unroll
        for (int p = 0; p < SP; ++p) {
          const uint32_t w[4] = {lo[p][0], lo[p][1], up[p][0], up[p][1]};
          sf[nt][p] = frag(w);
        }
      }
      if constexpr (DELTA) {
        f32x4 x[4 * NT] = {};
#pragma unroll
        for (int p = SP - 1; p >= 0; --p)  // from the least up
#pragma unroll
          for (int t = 0; t < 4 * NT; ++t)
            x[t] = mfma(frag(now.k[t / NT]), sf[t % NT][p], x[t]);
#pragma unroll
        for (int t = 0; t < 4 * NT; ++t) Kp[w4][t][lane] = x[t];
        lds_barrier();
        __builtin_amdgcn_s_setprio(0);  // out of the chain until U is there
      }
      bf16x8 kt[2][2];
      if constexpr (DELTA) {
#pragma unroll
        for (int p = 0; p < 2; ++p)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            *reinterpret_cast<bf16x8*>(&Sf[p][w4][nt][lane]) = sf[nt][p];
        lds_barrier();
        transpose(now, kt);
      } else {
        transpose(now, kt);
        f32x4 x[4 * NT] = {};
#pragma unroll
        for (int p = 1; p >= 0; --p)
#pragma unroll
          for (int t = 0; t < 4 * NT; ++t)
            x[t] = mfma(frag(now.q[t / NT]), sf[t % NT][p], x[t]);
#pragma unroll
        for (int t = 0; t < 4 * NT; ++t) Qp[b][w4][t][lane] = x[t];
      }
      const float eC = now.eC;
      load(c + 2, now);
      lds_barrier();
      if constexpr (DELTA) __builtin_amdgcn_s_setprio(3);
      uint4 uf[NT][3][2];
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) uf[nt][p][ks] = Uf[b][UP + p][ks][nt][lane];
      issue_fence();
      f32x4 y[NT][2][2] = {};
#pragma unroll
      for (int p = 2; p >= 0; --p)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks)
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
              y[nt][h][ks] = mfma(kt[h][ks], frag(uf[nt][p][ks]), y[nt][h][ks]);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) S[nt][h] = eC * S[nt][h] + (y[nt][h][0] + y[nt][h][1]);
    };
    if (chunks > 0) {
      Loads even, odd;
      load(0, even);
      load(1, odd);
      int c = 0;
      for (; c + 1 < chunks; c += 2) {
        step(c, even);
        step(c + 1, odd);
      }
      if (c < chunks) step(c, even);
    }
    if (slot < 0) return;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          a.state_out[at + (int64_t)(4 * h + i) * a.dv + 16 * nt] = S[nt][h][i];
    return;
  }

  if (chunks == 0) return;
  const bool two = w4 >= 2;  // tiles of the second 32 columns
  const int tile0 = tile_of(w4, 0);
  const int i0 = 16 * w4 + 4 * g;
  auto load_scalars = [&](int c, int which) {
    return *reinterpret_cast<const f32x4*>(ws0 + c * ws_step + ChunkData<DELTA>::token +
                                           128 * w4 + 64 * which + 16 * (uint32_t)g);
  };

  if (wave >= 8) {
    // ------------------------------------------------------- output waves
    u32x4 p[4];
    uint4 qf[KS];
    f32x4 eG, qs[NT];
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = (u32x4){0, 0, 0, 0};  // above the diagonal: stay zero
    auto load = [&](int c) {
      c = clamped(c);
      const char* m = ws0 + c * ws_step + ChunkData<DELTA>::p + tile0 * kStep;
      eG = load_scalars(c, 0);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j <= w4) p[j] = *reinterpret_cast<const u32x4*>(m + j * kStep + l16);
    };
    auto load_q = [&](int c) {
      const char* m = static_cast<const char*>(a.workspace) + a.key_offset +
                      ((c0 + clamped(c)) * a.k_heads + hk) * (int64_t)KeyData<DK>::bytes +
                      KeyData<DK>::q + w4 * kStep;
#pragma unroll
      for (int s = 0; s < KS; ++s) qf[s] = load16(m + s * 4 * kStep + l16);
    };
    auto q_times_state = [&] {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint4 sf[2][KS];
#pragma unroll
        for (int s = 0; s < KS; ++s) sf[0][s] = Sf[0][s][nt][lane], sf[1][s] = Sf[1][s][nt][lane];
        f32x4 q0 = {0.0f, 0.0f, 0.0f, 0.0f}, q1 = q0;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
          q0 = mfma(frag(qf[s]), frag(sf[0][s]), q0);
          q1 = mfma(frag(qf[s]), frag(sf[1][s]), q1);
        }
        qs[nt] = q0 + q1;
      }
    };
    // scale (e^G q S + P U)
    uint16_t o16[NT][4];
    auto compute = [&](int b, int nt) {
      uint4 u[UP][2];
#pragma unroll
      for (int e = 0; e < UP; ++e) u[e][0] = Uf[b][e][0][nt][lane], u[e][1] = Uf[b][e][1][nt][lane];
      f32x4 part[DELTA ? 1 : KS];
      if constexpr (!DELTA) {
#pragma unroll
        for (int s = 0; s < KS; ++s) part[s] = Qp[b][s][w4 * NT + nt][lane];
      }
      issue_fence();
      f32x4 o0 = {0.0f, 0.0f, 0.0f, 0.0f}, o1 = o0, o2 = o0;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
        if (ks && !two) continue;
        const u32x4 l = p[2 * ks], r = p[2 * ks + 1];
        const bf16x8 p0 = frag(make_uint4(l.x, l.y, r.x, r.y));
        o0 = mfma(p0, frag(u[0][ks]), o0);
        o1 = mfma(frag(make_uint4(l.z, l.w, r.z, r.w)), frag(u[0][ks]), o1);
        if constexpr (DELTA) o2 = mfma(p0, frag(u[UP - 1][ks]), o2);
      }
      if constexpr (!DELTA) {
        qs[nt] = part[0] + part[1];
        if constexpr (KS == 4) qs[nt] += part[2] + part[3];
      }
      const f32x4 o = a.scale * (eG * qs[nt] + (o0 + (o1 + o2)));
#pragma unroll
      for (int i = 0; i < 4; ++i) o16[nt][i] = (uint16_t)f32_to_bf16(o[i]);
    };
    auto compute_all = [&](int b) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) compute(b, nt);
    };
    const int64_t o_row = (int64_t)a.v_heads * a.dv;
    auto store = [&](int c) {
      char* base = reinterpret_cast<char*>(
          a.out + (sq.begin + (int64_t)c * kChunk) * o_row + (int64_t)hv * a.dv);
      const int left = sq.len - c * kChunk;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (i0 + i < left) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
            *reinterpret_cast<uint16_t*>(base + ((uint32_t)(i0 + i) * ((uint32_t)o_row * 2u) +
                                                 2u * (uint32_t)(col + 16 * nt))) = o16[nt][i];
        }
    };
    // q S between a chunk's second and third exchange, P U between its third
    // and the next one's first, stores and loads behind that: no exchange
    // waits for an output wave.
    load(0);
    if constexpr (DELTA) load_q(0);
    for (int c = 0; c < chunks; ++c) {
      lds_barrier();
      if constexpr (DELTA) {
        if (c > 0) {
          store(c - 1);
          load(c);
        }
        lds_barrier();
        q_times_state();
        load_q(c + 1);
        lds_barrier();
        compute_all(0);
      } else {
        compute_all(c & 1);
        store(c);
        load(c + 1);
      }
    }
    if constexpr (DELTA) store(chunks - 1);
    return;
  }

  // ---------------------------------------------------------- token waves
  struct Loads {
    u32x4 t01[DELTA ? 4 : 1];
    u32x2 t2[DELTA ? 4 : 1];
    uint16_t v[NT][4];
    f32x4 eG, dec;
  };
  auto load = [&](int c, Loads& x) {
    c = clamped(c);
    const char* m = ws0 + c * ws_step;
    if constexpr (DELTA) x.eG = load_scalars(c, 0);
    x.dec = load_scalars(c, 1);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j > w4) continue;
      if constexpr (DELTA) {
        x.t01[j] = *reinterpret_cast<const u32x4*>(m + ChunkData<DELTA>::t01 + (tile0 + j) * kStep + l16);
        x.t2[j] = *reinterpret_cast<const u32x2*>(m + ChunkData<DELTA>::t2 +
                                                  (tile0 + j) * (kStep / 2) + l16 / 2);
      }
    }
    const int last = sq.len - c * kChunk - 1;
    const char* base = reinterpret_cast<const char*>(
        a.v + (sq.begin + (int64_t)c * kChunk) * a.v_row + hv * a.v_head);
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
        x.v[nt][e] = *reinterpret_cast<const uint16_t*>(
            base + ((uint32_t)min(i0 + e, last) * ((uint32_t)a.v_row * 2u) +
                    2u * (uint32_t)(col + 16 * nt)));
  };
  auto put_u = [&](int b, int nt, const f32x4 u, const f32x4 dec) {
    uint32_t w[UP][2], y[3][2];
    pieces<3>(dec * u, y);
#pragma unroll
    for (int p = 0; p < 3; ++p)
      reinterpret_cast<uint2*>(&Uf[b][UP + p][w4 >> 1][nt][lane])[w4 & 1] = make_uint2(y[p][0], y[p][1]);
    pieces<UP>(u, w);
#pragma unroll
    for (int p = 0; p < UP; ++p)
      reinterpret_cast<uint2*>(&Uf[b][p][w4 >> 1][nt][lane])[w4 & 1] = make_uint2(w[p][0], w[p][1]);
  };
  auto step = [&](int c, Loads& x) {
    const int b = DELTA ? 0 : c & 1;
    f32x4 u[NT];
    if constexpr (DELTA) {
      lds_barrier();
      __builtin_amdgcn_s_setprio(3);
      f32x4 k[NT][KS];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int s = 0; s < KS; ++s) k[nt][s] = Kp[s][w4 * NT + nt][lane];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        f32x4 ks = k[nt][0] + k[nt][1];
        if constexpr (KS == 4) ks += k[nt][2] + k[nt][3];
#pragma unroll
        for (int i = 0; i < 4; ++i) u[nt][i] = bf16_to_f32(x.v[nt][i]) - x.eG[i] * ks[i];
        uint32_t w[3][2];
        pieces<3>(u[nt], w);
#pragma unroll
        for (int p = 0; p < 3; ++p)
          reinterpret_cast<uint2*>(&Rf[p][w4 >> 1][nt][lane])[w4 & 1] = make_uint2(w[p][0], w[p][1]);
      }
      lds_barrier();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        uint4 rf[3][2];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int p = 0; p < 3; ++p) rf[p][s] = Rf[p][s][nt][lane];
        issue_fence();
        // six chains of one or two products; the sum goes from the least up
        f32x4 y[6] = {};
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          if (s && !two) continue;
          const u32x4 l = x.t01[2 * s], r = x.t01[2 * s + 1];
          const u32x2 l2 = x.t2[2 * s], r2 = x.t2[2 * s + 1];
          const bf16x8 t0 = frag(make_uint4(l.x, l.y, r.x, r.y));
          const bf16x8 t1 = frag(make_uint4(l.z, l.w, r.z, r.w));
          const bf16x8 t2 = frag(make_uint4(l2.x, l2.y, r2.x, r2.y));
          y[0] = mfma(t0, frag(rf[0][s]), y[0]);
          y[1] = mfma(t0, frag(rf[1][s]), y[1]);
          y[2] = mfma(t1, frag(rf[0][s]), y[2]);
          y[3] = mfma(t0, frag(rf[2][s]), y[3]);
          y[4] = mfma(t1, frag(rf[1][s]), y[4]);
          y[5] = mfma(t2, frag(rf[0][s]), y[5]);
        }
        u[nt] = y[0] + ((y[1] + y[2]) + (y[3] + (y[4] + y[5])));
      }
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 4; ++i) u[nt][i] = bf16_to_f32(x.v[nt][i]);
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) put_u(b, nt, u[nt], x.dec);
    lds_barrier();
    __builtin_amdgcn_s_setprio(0);
    load(c + 2, x);
  };
  Loads even, odd;
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // the tiles above the diagonal stay zero
    if constexpr (DELTA) {
      even.t01[j] = odd.t01[j] = (u32x4){0, 0, 0, 0};
      even.t2[j] = odd.t2[j] = (u32x2){0, 0};
    }
  }
  load(0, even);
  load(1, odd);
  int c = 0;
  for (; c + 1 < chunks; c += 2) {
    step(c, even);
    step(c + 1, odd);
  }
  if (c < chunks) step(c, even);
}

// The column tiles of a head on one XCD, whose L2 then holds the head's chunk,
// and with enough of them the heads that share q and k.
__host__ __device__ __forceinline__ int64_t chunk_items(const LinearArgs& a, int64_t sequences,
                                                        int nt) {
  const int64_t units = sequences * a.v_heads / a.span;
  return (units + 7) / 8 * 8 * a.span * (a.dv / (16 * nt));
}

template <int DK, bool DELTA, int NT>
__device__ __forceinline__ void chunk_item(const LinearArgs& a, int64_t id, int count) {
  const int tiles = a.dv / (16 * NT);
  const int64_t in_xcd = id >> 3;
  const int64_t at_xcd = in_xcd / tiles;
  const int64_t head = (at_xcd / a.span * 8 + (id & 7)) * a.span + at_xcd % a.span;
  if (head >= (int64_t)count * a.v_heads) return;
  const int which = (int)(head / a.v_heads);
  through_chunks<DK, DELTA, NT>(a, a.list ? a.list[1 + which] : 0,
                                (int)(head - (int64_t)which * a.v_heads), (int)(in_xcd % tiles));
}

// Workgroups of listed sequences' chunks: one a compute unit is all that the
// registers allow, and a workgroup without work would cost a turn.
constexpr int64_t kChunkGroups = 256;

// Whether an item takes 32 columns: its chain has waits that a second tile
// fills, and its operands are read once for both, so that two tiles take about
// 1.4 times one's time.  That pays where it saves more than a third of the
// rounds (32 heads of 128 x 128, with the delta rule and without: 4 sequences
// of 8192 tokens 1015 -> 781 and 721 -> 677 us, 16 of 512 303 -> 248 and
// 215 -> 189; 3 of 2048, three rounds against two, 183 -> 184 and 121 -> 135).
__host__ __device__ __forceinline__ bool two_tiles(const LinearArgs& a, int64_t sequences) {
  if (a.dv % 32) return false;
  const int64_t one = (chunk_items(a, sequences, 1) + kChunkGroups - 1) / kChunkGroups;
  const int64_t two = (chunk_items(a, sequences, 2) + kChunkGroups - 1) / kChunkGroups;
  return 3 * two < 2 * one;
}

// A workgroup takes one item of the only sequence, or of listed ones its item
// and those a grid further on, which are on the same XCD.  Only the list knows
// how many there are: where that could call for either width both kernels are
// launched, and one of them ends at once (2 us; with both in one kernel the
// registers spill, which costs 4 to 30%).
template <int DK, bool DELTA, int NT, bool LISTED>
__global__ __launch_bounds__(kChunkThreads) void linear_chunk_kernel(const LinearArgs a,
                                                                     bool either) {
  if constexpr (!LISTED) {
    chunk_item<DK, DELTA, NT>(a, blockIdx.x, 1);
  } else {
    const int count = a.list[0];
    if (either && two_tiles(a, count) != (NT == 2)) return;
    const int64_t items = chunk_items(a, count, NT);
    for (int64_t id = blockIdx.x; id < items; id += gridDim.x) {
      chunk_item<DK, DELTA, NT>(a, id, count);
      lds_barrier();  // the next one's first exchange writes where this one's last is read
    }
  }
}

template <int DK, bool DELTA, int NT>
hipError_t launch_chunks(const LinearArgs& a, int64_t sequences, bool either, hipStream_t s) {
  const int64_t items = chunk_items(a, sequences, NT);
  if (!a.list)
    linear_chunk_kernel<DK, DELTA, NT, false><<<(unsigned)items, kChunkThreads, 0, s>>>(a, false);
  else
    linear_chunk_kernel<DK, DELTA, NT, true>
        <<<(unsigned)(items < kChunkGroups ? items : kChunkGroups), kChunkThreads, 0, s>>>(a,
                                                                                          either);
  return hipGetLastError();
}

template <int DK, bool DELTA>
hipError_t launch_linear_of(const LinearArgs& a, hipStream_t s) {
  const int clear = a.clear ? kClearParts : 0;
  if (!a.workspace) {
    if (a.dv % 32 == 0 && (int64_t)a.requests * a.v_heads * (a.dv / 32) >= kWideStates)
      linear_step_kernel<DK, DELTA, 8>
          <<<(unsigned)(token_groups(a, 8) + clear), kLinThreads, 0, s>>>(a);
    else
      linear_step_kernel<DK, DELTA, 4>
          <<<(unsigned)(token_groups(a, 4) + clear), kLinThreads, 0, s>>>(a);
    return hipGetLastError();
  }
  const int64_t beside = a.list ? 1 + token_groups(a, 4) : 0;
  linear_prepare_kernel<DK, DELTA>
      <<<(unsigned)(beside + a.chunks * a.v_heads + clear), kLinThreads, 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t most = a.tokens / (a.by_token + 1);  // sequences that go in chunks
  const int64_t sequences = !a.list ? 1 : most < a.requests ? most : a.requests;
  const bool two = two_tiles(a, sequences);
  if (two) e = launch_chunks<DK, DELTA, 2>(a, sequences, true, s);
  if (e != hipSuccess || (two && !a.list)) return e;
  return launch_chunks<DK, DELTA, 1>(a, sequences, two, s);
}

}  // namespace

// Of several sequences, none empty, the longest has at most tokens - requests
// + 1 tokens.
bool linear_in_chunks(int64_t tokens, int requests) {
  return requests == 1 ? tokens > kFewTokens : tokens - requests > 32;
}

LinearLayout linear_layout(int64_t tokens, int requests, int k_heads, int v_heads, int dk,
                           bool delta) {
  LinearLayout l;
  l.chunks = tokens / kChunk + requests;
  l.key_offset = l.chunks * v_heads *
                 (int64_t)(delta ? ChunkData<true>::bytes : ChunkData<false>::bytes);
  l.list_offset = l.key_offset + l.chunks * k_heads *
                                     (int64_t)(dk == 64 ? KeyData<64>::bytes : KeyData<128>::bytes);
  l.total = l.list_offset + (requests > 1 ? ((int64_t)requests + 1) * 4 : 0);
  return l;
}

hipError_t launch_linear(const LinearArgs& in, hipStream_t s) {
  LinearArgs a = in;
  // Where lengths may differ, which sequences are taken by token.  Few states
  // leave most of the chip to a sequence's chunks, and a token costs its wave
  // 0.9 us (one sequence x 32 heads of 128 x 128: 8 tokens 10.8 us and 12.5 in
  // chunks, 16 tokens 18.8 and 12.6); many fill it either way (16 sequences:
  // 24 tokens 58 and 68, 32 tokens 73 and 67; 64: 64 tokens 356 and 301).
  a.by_token = (int64_t)a.requests * a.v_heads * (a.dv / 16) >= 4096 ? 24 : kFewTokens;
  // fewer than eight key heads would leave XCDs idle
  a.span = a.k_heads >= 8 ? a.v_heads / a.k_heads : 1;
  if (a.dk == 64) return a.delta ? launch_linear_of<64, true>(a, s) : launch_linear_of<64, false>(a, s);
  return a.delta ? launch_linear_of<128, true>(a, s) : launch_linear_of<128, false>(a, s);
}

}  // namespace rmoe
