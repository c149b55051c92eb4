// Attention of one new token of each request over its paged cache.
//
//   o_h = sum_j p_hj v_j / sum_j p_hj,  p_hj = exp(scale q_h . k_j - m_h)
//
// over the keys j of [length - window, length).  Bound by the read of K and
// V (2 bytes, or one, of each are used in at most `group` products), so the
// kernel is built around keeping loads in flight: K and V go from memory
// straight into the registers that feed the matrix instructions, with no
// LDS pass and no barrier before the end.
//
//   - 16 query heads of one key head (the group, padded) times 32 keys a
//     step: scores^T = K Q^T as 16x16x32 products, key rows as operand A.
//   - scores^T leaves lane (g, n) with keys 4 g + i of head n in each 16-key
//     half, which is just the operand layout of the second product with its
//     contraction index permuted (index 8 g + 4 half + i is key 16 half +
//     4 g + i), so the probabilities never move between lanes.
//   - out^T = V^T P^T: lane (g, n) loads for its 8 keys the dims n E ..
//     n E + E - 1 (E = 8 of 128: whole lines of V) and transposes them among
//     its own registers with byte permutes; tile e's row m is dim m E + e.
//   - running maximum and sum per head, in base 2 with the scale folded in.
//     The probabilities are rounded to bf16 for the second product (half a
//     step, 2^-9, of numbers that are averaged; the sum is of the unrounded
//     ones); everything else is fp32.
//
// Requests' keys are split over several workgroups and, in each, over its
// four waves; a second launch joins a request's parts in their order.
#include <type_traits>

#include "common.h"
#include "kernels.h"

namespace rmoe {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

constexpr int kAttWaves = 4;  // of a workgroup that shares a request's keys with others
constexpr int kAttTile = 32;  // keys of a step
constexpr float kLn2 = 0.69314718056f;
constexpr int kScanned = 256;  // requests up to which the parts are evened out over all

__device__ __forceinline__ bf16x8 frag(const uint32_t (&w)[4]) {
  union {
    uint32_t w[4];
    bf16x8 v;
  } u;
#pragma unroll
  for (int i = 0; i < 4; ++i) u.w[i] = w[i];
  return u.v;
}

__device__ __forceinline__ f32x4 mfma(const bf16x8 a, const bf16x8 b, const f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// Maximum / sum over the four lanes that hold one head (l ^ 16, l ^ 32).
__device__ __forceinline__ float head_max(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float head_sum(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  union {
    bf16x2 v;
    uint32_t u;
  } r;
  r.v = __builtin_convertvector((f32x2){lo, hi}, bf16x2);
  return r.u;
}

// Two e4m3 values (the low or high half of w) as packed bf16: exact.
template <bool HIGH>
__device__ __forceinline__ uint32_t e4m3_to_bf16(uint32_t w) {
  union {
    bf16x2 v;
    uint32_t u;
  } r;
  r.v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HIGH);
  return r.u;
}

// BYTES consecutive bytes (2, 4, 8, 16) as dwords.
template <int BYTES>
__device__ __forceinline__ void load_bytes(const uint8_t* p, uint32_t* w) {
  if constexpr (BYTES == 16) {
    const uint4 u = load16(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else if constexpr (BYTES == 8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x, w[1] = u.y;
  } else if constexpr (BYTES == 4) {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  } else {
    static_assert(BYTES == 2, "2, 4, 8 or 16 bytes");
    w[0] = *reinterpret_cast<const uint16_t*>(p);
  }
}

// A head's dims as runs of 128, 64 or 32: lane n of 16 holds P / 16
// consecutive ones of each run.
template <int D>
struct Runs {
  static constexpr int first = D >= 128 ? 128 : 64;
  static constexpr int second = D - first;
  static constexpr int row = first + 4;  // of LDS, where heads' rows then lie on other banks
};

// A request's keys [start, end) and the tiles of 32 they touch.
struct Keys {
  int start, end;
  int tile0, tiles;
};

__device__ __forceinline__ Keys keys_of(const AttentionArgs& a, int r) {
  Keys s;
  const int64_t most = (int64_t)a.width << a.shift;
  const int len = (int)(a.lengths[r] < most ? a.lengths[r] : most);
  s.end = len > 0 ? len : 0;
  s.start = a.window > 0 && s.end > a.window ? s.end - a.window : 0;
  s.tile0 = s.start / kAttTile;
  s.tiles = s.end > s.start ? (s.end - 1) / kAttTile + 1 - s.tile0 : 0;
  return s;
}

// Part `number` of `request`, whose parts are [first, first + as many as it
// has) of all requests' and take about `per` tiles each.
struct Part {
  int request, number, first, per;
};

__device__ __forceinline__ int ceil_div(int n, int d) { return (int)(((unsigned)n + d - 1) / d); }

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t from_lane(uint32_t v) {  // 0 where there is none
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}

// The sum of the lanes up to this one.
template <typename T>
__device__ __forceinline__ T running_sum(T v) {
  static_assert(sizeof(T) == 4, "one register");
  auto add = [&](uint32_t u) {
    T x;
    __builtin_memcpy(&x, &u, 4);
    v += x;
  };
  auto bits = [&] {
    uint32_t u;
    __builtin_memcpy(&u, &v, 4);
    return u;
  };
  add(from_lane<0x111, 0xf>(bits()));  // one lane to the left in a row of 16, then 2, 4, 8
  add(from_lane<0x112, 0xf>(bits()));
  add(from_lane<0x114, 0xf>(bits()));
  add(from_lane<0x118, 0xf>(bits()));
  add(from_lane<0x142, 0xa>(bits()));  // a row's last lane to the next row, of 32 to the next 32
  add(from_lane<0x143, 0xc>(bits()));
  return v;
}

// The greatest of all lanes.
__device__ __forceinline__ float wave_max(float v) {
  auto with = [&](auto ctrl, auto rows) {
    const int w = (int)__float_as_uint(v);  // its own where there is no other
    v = fmaxf(v, __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(
                     w, w, decltype(ctrl)::value, decltype(rows)::value, 0xf, false)));
  };
  constexpr std::integral_constant<int, 0xf> all;
  with(std::integral_constant<int, 0x111>(), all);
  with(std::integral_constant<int, 0x112>(), all);
  with(std::integral_constant<int, 0x114>(), all);
  with(std::integral_constant<int, 0x118>(), all);
  with(std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());
  with(std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());
  return __uint_as_float(
      (uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(v), kWave - 1));
}

// Part w of all.  Every wave works it out from the lengths (a load and two
// running sums across the wave for each 64 requests): the parts of all
// requests are of about one size, total / a.parts, and there is none without
// work but the one that a request without keys needs for its zeros.  (With a
// fixed number of parts for each request, as for more requests than a wave
// scans, 61 requests of 17 to 16000 keys took 84 us for 72, and 24 for 8 if
// none had a key: the time of workgroups that find nothing to do.)
__device__ __forceinline__ Part part_of(const AttentionArgs& a, int w) {
  if (!a.parts) return {w < a.requests ? w : -1, 0, w, 0x7FFFFFFF};
  if (a.requests == 1) {
    const int per = ceil_div(keys_of(a, 0).tiles, a.parts);
    return {0, w, 0, per > a.least ? per : a.least};
  }
  const int lane = threadIdx.x & 63;
  if (a.requests > kScanned) {  // each request by itself
    const int each = a.parts / a.requests;
    const int r = w / each;
    if (r >= a.requests) return {-1, 0, 0, 0};
    const int per = ceil_div(keys_of(a, r).tiles, each);
    return {r, w - r * each, r * each, per > a.least ? per : a.least};
  }
  constexpr int N = kScanned / kWave;
  int n[N];
  float total = 0.0f;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (kWave * j >= a.requests) break;
    const int i = lane + kWave * j;
    n[j] = i < a.requests ? keys_of(a, i).tiles : 0;
    total += (float)n[j];
  }
  total = running_sum(total);
  total = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(total), kWave - 1));
  const int even = (int)__builtin_ceilf(total / (float)a.parts);
  const int per = even > a.least ? even : a.least;
  int before = 0, r = -1, first = 0;
#pragma unroll
  for (int j = 0; j < N; ++j) {
    if (kWave * j >= a.requests) break;
    const int i = lane + kWave * j;
    int mine = ceil_div(n[j], per);
    mine = i >= a.requests ? 0 : mine > 0 ? mine : 1;
    const int upto = running_sum(mine);
    const int start = before + upto - mine;
    const uint64_t at = __ballot(start <= w && w < start + mine);
    if (at) {
      const int l = __builtin_ctzll(at);
      r = kWave * j + l;
      first = __builtin_amdgcn_readlane(start, l);
    }
    before += __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return {r, w - first, first, per};
}

template <int D, bool E4M3, int WAVES>
__global__ __launch_bounds__(WAVES * kWave, WAVES > 4 ? WAVES / 4 : D > 128 && !E4M3 ? 1 : 2)
void attention_kernel(const AttentionArgs a) {
  constexpr int EB = E4M3 ? 1 : 2;    // bytes of a cached value
  constexpr int KS = D / 32;          // steps of the first product
  constexpr int NT = D / 16;          // tiles of the second
  constexpr int P0 = Runs<D>::first, P1 = Runs<D>::second;
  constexpr int E0 = P0 / 16, E1 = P1 / 16;
  constexpr int V0 = (E0 * EB + 3) / 4, V1 = (E1 * EB + 3) / 4;  // dwords of a key's runs
  constexpr int KW = KS * 8 * EB / 4;                            // dwords of a key's share
  extern __shared__ __align__(16) float lds[];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, g = lane >> 4;
  // eight parts side by side, one for each XCD, which takes all heads of its
  // pages one after the other (heads on XCDs of their own: each XCD goes
  // through all pages, 8 requests of 100 to 60000 keys 83 us for 53); fewer
  // parts than that are spread with the heads
  const int all_heads = a.kv_heads * a.head_tiles;
  int w, h0;
  if (a.all_parts >= 8) {
    const int b = blockIdx.x >> 3;
    h0 = b % all_heads;
    w = b / all_heads * 8 + (blockIdx.x & 7);
  } else {
    h0 = blockIdx.x % all_heads;
    w = blockIdx.x / all_heads;
  }
  const Part part = part_of(a, w);
  const int r = __builtin_amdgcn_readfirstlane(part.request);
  if (r < 0) return;
  const int ht = h0 % a.head_tiles, hk = h0 / a.head_tiles;
  const Keys sh = keys_of(a, r);
  const int want = ceil_div(sh.tiles, part.per);
  const int per = want > 1 ? ceil_div(sh.tiles, want) : sh.tiles;
  const int parts = want > 1 ? ceil_div(sh.tiles, per) : 1;
  if (part.number >= parts) return;
  if (a.parts && h0 == 0 && part.number == 0 && tid == 0) a.list[r] = make_int2(part.first, parts);
  const int t_begin = part.number * per;
  const int t_end = t_begin + per < sh.tiles ? t_begin + per : sh.tiles;

  const int left = a.group - ht * 16;
  const int heads = left < 16 ? left : 16;  // of this workgroup
  const int head0 = hk * a.group + ht * 16;

  // queries, operand B: head n, the dims of each step as the keys have them
  bf16x8 qf[KS];
#pragma unroll
  for (int s = 0; s < KS; ++s) {
    uint32_t w[4] = {0, 0, 0, 0};
    int d = 32 * s + 8 * g;
    if (E4M3 && (s | 1) < KS) d = 64 * (s >> 1) + 16 * g + 8 * (s & 1);
    if (n < heads) {
      const uint16_t* p = a.q + (int64_t)r * a.q_row + (int64_t)(head0 + n) * a.q_head + d;
      const uint4 u = load16(p);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    }
    qf[s] = frag(w);
  }

  const uint8_t* kc = static_cast<const uint8_t*>(a.k_cache) + (int64_t)hk * a.head_stride * EB;
  const uint8_t* vc = static_cast<const uint8_t*>(a.v_cache) + (int64_t)hk * a.head_stride * EB;
  const int32_t* table = a.table + r * a.table_stride;
  const int in_page = (1 << a.shift) - 1;
  const int last = sh.end - 1;

  // page numbers of tile t: of key 16 half + n for K, of the four keys
  // 16 half + 4 g .. for V.  Keys past the end look the last key's page up.
  auto pages = [&](int t, int (&pk)[2], int (&pv)[2]) {
    const int key0 = (sh.tile0 + t) * kAttTile;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int jk = key0 + 16 * h + n, jv = key0 + 16 * h + 4 * g;
      pk[h] = table[(jk < last ? jk : last) >> a.shift];
      pv[h] = table[(jv < last ? jv : last) >> a.shift];
    }
  };
  // a page that is none of the cache's is read as page 0 and masked
  auto row_of = [&](int page, int key) {
    const int64_t p = (uint32_t)page < (uint32_t)a.pages ? page : 0;
    return (p * a.page_stride + (int64_t)(key & in_page) * a.row_stride) * EB;
  };
  uint32_t kw[2][KW];
  uint32_t v0[8][V0], v1[8][V1 ? V1 : 1];
  auto load_k = [&](int t, const int (&pk)[2]) {
    const int key0 = (sh.tile0 + t) * kAttTile;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* p = kc + row_of(pk[h], key0 + 16 * h + n);
      if constexpr (!E4M3) {
#pragma unroll
        for (int s = 0; s < KS; ++s) load_bytes<16>(p + (32 * s + 8 * g) * 2, &kw[h][4 * s]);
      } else {
#pragma unroll
        for (int s = 0; s + 1 < KS; s += 2) load_bytes<16>(p + 32 * s + 16 * g, &kw[h][2 * s]);
        if constexpr (KS & 1) load_bytes<8>(p + 32 * (KS - 1) + 8 * g, &kw[h][2 * (KS - 1)]);
      }
    }
  };
  auto load_v = [&](int t, const int (&pv)[2]) {
    const int key0 = (sh.tile0 + t) * kAttTile;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint8_t* p = vc + row_of(pv[j >> 2], key0 + 16 * (j >> 2) + 4 * g + (j & 3));
      load_bytes<E0 * EB>(p + n * E0 * EB, v0[j]);
      if constexpr (P1 > 0) load_bytes<E1 * EB>(p + (P0 + n * E1) * EB, v1[j]);
    }
  };

  f32x4 o[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) o[i] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
  float m = -INFINITY, l = 0.0f;

  int t = t_begin + wave;
  int pk[2], pv[2];
  if (t < t_end) {
    pages(t, pk, pv);
    load_k(t, pk);
    load_v(t, pv);
  }
  for (; t < t_end; t += WAVES) {
    const int next = t + WAVES;
    const int now_v[2] = {pv[0], pv[1]};
    if (next < t_end) pages(next, pk, pv);

    f32x4 sc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      sc[h] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint32_t w[4];
        if constexpr (!E4M3) {
#pragma unroll
          for (int i = 0; i < 4; ++i) w[i] = kw[h][4 * s + i];
        } else {
          w[0] = e4m3_to_bf16<false>(kw[h][2 * s]);
          w[1] = e4m3_to_bf16<true>(kw[h][2 * s]);
          w[2] = e4m3_to_bf16<false>(kw[h][2 * s + 1]);
          w[3] = e4m3_to_bf16<true>(kw[h][2 * s + 1]);
        }
        sc[h] = mfma(frag(w), qf[s], sc[h]);
      }
    }
    if (next < t_end) load_k(next, pk);

    // keys outside the request's or without a page: no weight, and their
    // values cleared, since 0 times a leftover infinity or NaN is NaN
    const int key0 = (sh.tile0 + t) * kAttTile;
    const bool bad_page = (uint32_t)now_v[0] >= (uint32_t)a.pages ||
                          (uint32_t)now_v[1] >= (uint32_t)a.pages;
    const bool edge = key0 < sh.start || key0 + kAttTile > sh.end || __any(bad_page);
    uint32_t dead = 0;
    if (edge) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int key = key0 + 16 * (j >> 2) + 4 * g + (j & 3);
        if (key < sh.start || key >= sh.end || (uint32_t)now_v[j >> 2] >= (uint32_t)a.pages)
          dead |= 1u << j;
      }
    }
    float x[8];
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = sc[j >> 2][j & 3] * a.scale_log2;
      if (edge && (dead >> j & 1)) x[j] = -INFINITY;
      top = fmaxf(top, x[j]);
    }
    top = fmaxf(m, head_max(top));
    if (__any(top > m)) {
      const float base = top == -INFINITY ? 0.0f : top;
      const float shrink = __builtin_amdgcn_exp2f(m - base);
      l *= shrink;
#pragma unroll
      for (int i = 0; i < NT; ++i) o[i] *= shrink;
      m = top;
    }
    const float base = m == -INFINITY ? 0.0f : m;
    uint32_t pw[4];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = __builtin_amdgcn_exp2f(x[j] - base);
      l += x[j];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) pw[j] = pack_bf16(x[2 * j], x[2 * j + 1]);
    const bf16x8 pf = frag(pw);

    // bf16 values of a run of key j, then the transposed fragments
    auto second = [&](const uint32_t* raw, int j, int dw) -> uint32_t {
      // dword dw (dims 2 dw, 2 dw + 1 of the lane's run) of key j as bf16
      uint32_t w;
      if constexpr (E4M3) {
        w = dw & 1 ? e4m3_to_bf16<true>(raw[dw >> 1]) : e4m3_to_bf16<false>(raw[dw >> 1]);
      } else {
        w = raw[dw];
      }
      return edge && (dead >> j & 1) ? 0u : w;
    };
#pragma unroll
    for (int dw = 0; dw < E0 / 2; ++dw) {
      uint32_t w[8], lo[4], hi[4];
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = second(v0[j], j, dw);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100);
        hi[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302);
      }
      o[2 * dw] = mfma(frag(lo), pf, o[2 * dw]);
      o[2 * dw + 1] = mfma(frag(hi), pf, o[2 * dw + 1]);
    }
    if constexpr (P1 > 0) {
#pragma unroll
      for (int dw = 0; dw < E1 / 2; ++dw) {
        uint32_t w[8], lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = second(v1[j], j, dw);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x05040100);
          hi[i] = __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], 0x07060302);
        }
        o[E0 + 2 * dw] = mfma(frag(lo), pf, o[E0 + 2 * dw]);
        o[E0 + 2 * dw + 1] = mfma(frag(hi), pf, o[E0 + 2 * dw + 1]);
      }
    }
    if (next < t_end) load_v(next, pv);
  }

  // The waves' parts together: first their maxima, so that each wave scales
  // what it has, then the sums of a run of dims and four waves at a time.
  // (Instruction fetch counts here: the code runs once.  With every sum's
  // factors at the sum, a value at a time, this took 7300 of a short part's
  // 16400 cycles.)
  l = head_sum(l);
  constexpr int THREADS = WAVES * kWave;
  constexpr int ROW = Runs<D>::row;
  constexpr int ITEMS = (16 * P0 / 4 + THREADS - 1) / THREADS;  // of a thread: four dims of a head
  float* ml = lds + 4 * heads * ROW;  // [wave][head] maximum, then sum, then both of all
  if (n < heads && g == 0) {
    ml[wave * 16 + n] = m;
    ml[(WAVES + wave) * 16 + n] = l;
  }
  __syncthreads();
  float* of_all = ml + 2 * WAVES * 16;
  if (n < heads) {
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = fmaxf(top, ml[w * 16 + n]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
      sum += __builtin_amdgcn_exp2f(ml[w * 16 + n] - base) * ml[(WAVES + w) * 16 + n];
    const float f = __builtin_amdgcn_exp2f(m - base);
#pragma unroll
    for (int i = 0; i < NT; ++i) o[i] *= f;
    if (wave == 0 && g == 0) of_all[n] = top, of_all[16 + n] = sum;
  }
  const int64_t row = (int64_t)r * a.kv_heads * a.group + head0;
  auto join = [&](auto run) {
    constexpr int P = decltype(run)::value ? P1 : P0, E = P / 16;
    constexpr int I0 = decltype(run)::value ? E0 : 0, D0 = decltype(run)::value ? P0 : 0;
    f32x4 acc[ITEMS];
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) acc[q] = (f32x4){0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w0 = 0; w0 < WAVES; w0 += 4) {
      if (w0 || D0) __syncthreads();
      if (n < heads && wave >= w0 && wave < w0 + 4) {
        float* mine = lds + ((wave - w0) * heads + n) * ROW + 4 * g * E;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if constexpr (E >= 4) {
#pragma unroll
            for (int i = 0; i < E; i += 4)
              *reinterpret_cast<f32x4*>(mine + k * E + i) =
                  (f32x4){o[I0 + i][k], o[I0 + i + 1][k], o[I0 + i + 2][k], o[I0 + i + 3][k]};
          } else {
            static_assert(E >= 4 || E == 2 || E == 0, "runs of 128, 64 or 32");
            *reinterpret_cast<f32x2*>(mine + k * E) = (f32x2){o[I0][k], o[I0 + 1][k]};
          }
        }
      }
      __syncthreads();
#pragma unroll
      for (int q = 0; q < ITEMS; ++q) {
        const int i = tid + q * THREADS, h = i / (P / 4), d = i % (P / 4) * 4;
        if (h >= heads) continue;
#pragma unroll
        for (int w = 0; w < 4; ++w)
          acc[q] += *reinterpret_cast<const f32x4*>(lds + (w * heads + h) * ROW + d);
      }
    }
#pragma unroll
    for (int q = 0; q < ITEMS; ++q) {
      const int i = tid + q * THREADS, h = i / (P / 4), d = D0 + i % (P / 4) * 4;
      if (h >= heads) continue;
      const float top = of_all[h], sum = of_all[16 + h];
      if (parts == 1) {
        const bool some = sum > 0.0f || sum != sum;
        uint32_t x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          x[k] = f32_to_bf16(some ? acc[q][k] / sum * a.v_scale : 0.0f);
        *reinterpret_cast<uint2*>(a.out + (row + h) * D + d) =
            make_uint2(x[0] | x[1] << 16, x[2] | x[3] << 16);
        if (a.lse && d == 0) a.lse[row + h] = top == -INFINITY ? top : (top + log2f(sum)) * kLn2;
      } else {
        const int64_t at = (int64_t)w * a.kv_heads * a.group + head0 + h;
        *reinterpret_cast<f32x4*>(a.part_o + at * D + d) = acc[q];
        if (d == 0) a.part_ml[at] = make_float2(top, sum);
      }
    }
  };
  join(std::integral_constant<int, 0>());
  if constexpr (P1 > 0) join(std::integral_constant<int, 1>());
}

// Joins the parts of one head, or of 32 dims of it: SLICE / 4 threads across
// the dims, the others across the parts.  Slices are for few heads, whose
// parts are many (16 heads of 256 dims, 128 parts: 4.9 us, whole heads 6.7);
// for many they are only more workgroups (1952 heads of 128 dims, 8 parts:
// 13.2 us, whole heads 5.5).
template <int D, int SLICE>
__global__ __launch_bounds__(256) void attention_join_kernel(const AttentionArgs a) {
  constexpr int C = SLICE / 4, Q = 256 / C, SLICES = D / SLICE;
  __shared__ float4 acc_s[Q][C];
  __shared__ float sum_s[Q];
  const int64_t row = blockIdx.x / SLICES;  // request and head
  const int slice = blockIdx.x % SLICES;
  const int heads = a.kv_heads * a.group;
  const int2 list = a.list[row / heads];
  const int parts = list.y;
  if (parts == 1) return;  // written in the first launch
  const int64_t first = (int64_t)list.x * heads + row % heads;
  const int tid = threadIdx.x, c = tid % C, q = tid / C;
  const float2* ml = a.part_ml + first;
  const float* o = a.part_o + first * D + slice * SLICE;
  auto load = [&](int i) {
    return reinterpret_cast<const float4*>(o + (int64_t)i * heads * D)[c];
  };
  // a thread's first part is on its way while the maximum is found
  const bool mine = q < Q && q < parts;
  float2 e = make_float2(-INFINITY, 0.0f);
  float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  if (mine) e = ml[(int64_t)q * heads], v = load(q);
  float top = -INFINITY;
  for (int i = tid & 63; i < parts; i += 64) top = fmaxf(top, ml[(int64_t)i * heads].x);
  top = wave_max(top);
  const float base = top == -INFINITY ? 0.0f : top;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  float sum = 0.0f;
  auto add = [&](const float2 e, const float4 v) {
    const float f = __builtin_amdgcn_exp2f(e.x - base);
    sum += f * e.y;
    acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
  };
  if (mine) add(e, v);
#pragma unroll 4
  for (int i = q + Q; i < (q < Q ? parts : 0); i += Q) add(ml[(int64_t)i * heads], load(i));
  if (q < Q) {
    acc_s[q][c] = acc;
    if (c == 0) sum_s[q] = sum;
  }
  __syncthreads();
  if (tid >= C) return;
  acc = acc_s[0][c];
  sum = sum_s[0];
#pragma unroll
  for (int i = 1; i < Q; ++i) {
    const float4 v = acc_s[i][c];
    acc.x += v.x, acc.y += v.y, acc.z += v.z, acc.w += v.w;
    sum += sum_s[i];
  }
  const bool some = sum > 0.0f || sum != sum;
  const float f = some ? a.v_scale / sum : 0.0f;
  uint2 w;
  w.x = f32_to_bf16(some ? acc.x * f : 0.0f) | f32_to_bf16(some ? acc.y * f : 0.0f) << 16;
  w.y = f32_to_bf16(some ? acc.z * f : 0.0f) | f32_to_bf16(some ? acc.w * f : 0.0f) << 16;
  reinterpret_cast<uint2*>(a.out + row * D + slice * SLICE)[c] = w;
  if (a.lse && tid == 0 && slice == 0)
    a.lse[row] = top == -INFINITY ? top : (top + log2f(sum)) * kLn2;
}

constexpr int kAloneWaves = 8;  // of a workgroup that has a request to itself

template <int D, bool E4M3>
hipError_t launch_attention_of(const AttentionArgs& a, hipStream_t s) {
  const int heads = a.group < 16 ? a.group : 16;
  const int64_t parts = a.all_parts >= 8 ? (a.all_parts + 7) / 8 * 8 : a.all_parts;
  const unsigned grid = (unsigned)(parts * a.kv_heads * a.head_tiles);
  auto lds = [&](int waves) {
    return (size_t)(4 * heads * Runs<D>::row + 2 * (waves + 1) * 16) * sizeof(float);
  };
  if (a.alone) {
    attention_kernel<D, E4M3, kAloneWaves>
        <<<grid, kAloneWaves * kWave, lds(kAloneWaves), s>>>(a);
    return hipGetLastError();
  }
  attention_kernel<D, E4M3, kAttWaves><<<grid, kAttWaves * kWave, lds(kAttWaves), s>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.parts) return e;
  const unsigned rows = (unsigned)(a.requests * a.kv_heads * a.group);
  if (rows <= 256)
    attention_join_kernel<D, 32><<<rows * (D / 32), 256, 0, s>>>(a);
  else
    attention_join_kernel<D, D><<<rows, 256, 0, s>>>(a);
  return hipGetLastError();
}

template <int D>
hipError_t launch_attention_dim(const AttentionArgs& a, hipStream_t s) {
  return a.bits == 8 ? launch_attention_of<D, true>(a, s) : launch_attention_of<D, false>(a, s);
}

}  // namespace

// Up to this many values of K a request that would be split is left whole to
// one workgroup of eight waves, without a second launch (one request, 2 key
// heads of 128 dims: 130 keys 6.4 us against 8.5, 500 keys 9.6 against 8.8 and
// a launch, 3 us, less on the host; 1000 keys 14.0 against 8.8: one compute
// unit reads 60 GB/s).
constexpr int64_t kAloneValues = 512 * 128;

AttentionPlan attention_plan(int requests, int kv_heads, int group, int dim, int64_t keys) {
  const int64_t heads = (int64_t)kv_heads * ((group + 15) / 16);
  const int64_t base = requests * heads;
  const int64_t tiles = (keys + kAttTile - 1) / kAttTile;
  const AttentionPlan whole = {0, requests, 0};
  if (base < 256 && tiles > kAttWaves && keys * dim <= kAloneValues) return {0, requests, 1};
  // many requests of few keys at most: the second launch would cost more than
  // uneven ones (64 requests x 8 heads x 2048 keys: 53 us whole, 63 in halves)
  if (tiles <= kAttWaves || (base >= 256 && keys <= 2048)) return whole;
  if (requests > kScanned) {
    const int64_t some = (keys + 2047) / 2048, each = 8192 / base < some ? 8192 / base : some;
    return each > 1 ? AttentionPlan{(int)(each * requests), (int)(each * requests), 0} : whole;
  }
  // Workgroups: of wide heads, whose registers leave room for one or two a
  // compute unit, whole rounds of one each with the rounding of every request's
  // parts counted in, the fewest in which a part is no more than the average
  // request (20 requests of 1000 to 30000 keys, 2 heads of 256: 76 us, 97 if
  // the rounding starts a second round; 4 of 1000 to 40000 28, 32 with two
  // rounds); of others two each for a single request (131071 keys, 8 heads of
  // 128, 8 bits: 57 us, 63 with six), and six where requests differ (61 of 17
  // to 16000 keys, 8 heads: 72 us, 83 with two, 75 with sixteen).  Where that
  // is less than a part a request, the parts are of the average request's size
  // (256 of 700 to 4100 keys, 16 heads of 64: 367 us, with larger ones 392).
  const int64_t units = 256 / heads;
  int64_t parts = requests == 1 ? (dim > 128 ? units : 512 / heads) : 1536 / heads;
  if (dim > 128 && requests > 1 && units > 0)
    parts = (2 * requests + units - 1) / units * units - requests;
  if (parts < requests) parts = requests;
  const int64_t most = (tiles + kAttWaves - 1) / kAttWaves * requests;
  if (parts > most) parts = most;
  if (parts < 2) return whole;
  return {(int)parts, (int)(requests == 1 ? parts : parts + requests), 0};
}

hipError_t launch_attention(const AttentionArgs& in, hipStream_t s) {
  AttentionArgs a = in;
  a.least = kAttWaves;  // a tile for each wave
  switch (a.dim) {
    case 64: return launch_attention_dim<64>(a, s);
    case 96: return launch_attention_dim<96>(a, s);
    case 128: return launch_attention_dim<128>(a, s);
    case 192: return launch_attention_dim<192>(a, s);
    default: return launch_attention_dim<256>(a, s);
  }
}

}  // namespace rmoe
