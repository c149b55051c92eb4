// A decode step's bookkeeping and the write into the paged cache: block
// tables and slot maps from request lengths, and rotary positions of one to
// four axes with the rotated key and the value written through by slot.
#include "common.h"
#include "kernels.h"

namespace rmoe {

// ------------------------------------------------- block tables, slot maps
// Running sums over the requests of their new tokens (cu) and of the pages
// these take from the free list (first), then one independent piece of work
// for each page taken and each row of the batch, found by bisection in the
// sums.  Every workgroup makes the sums for itself in LDS (at most 4096
// requests: 32 KB read from L2), which costs less than a second launch
// behind a workgroup that makes them for all.
constexpr int kTableThreads = 256;

__device__ __forceinline__ int ceil_shift(int64_t v, int shift) {
  return (int)((v + ((int64_t)1 << shift) - 1) >> shift);
}

struct Grown {  // one request's step
  int64_t c;    // cached tokens
  int64_t end;  // tokens after the step
  int have;     // pages it holds
  int take;     // pages it takes, as far as its row of the table goes
};

__device__ __forceinline__ Grown grown(const TableArgs& a, int r) {
  Grown g;
  g.c = max(a.cached[r], 0);
  g.end = g.c + max(a.added[r], 0);
  g.have = ceil_shift(g.c, a.shift);
  g.take = max(min(ceil_shift(g.end, a.shift), a.width) - g.have, 0);
  return g;
}

__device__ __forceinline__ int saturate(int64_t v) {
  return (int)(v < 0x7FFFFFFF ? v : 0x7FFFFFFF);
}

// The last r in [0, n) with sums[r] <= v (sums[0] == 0 <= v).
__device__ __forceinline__ int bisect(const int* sums, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= v)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kTableThreads) void tables_kernel(const TableArgs a) {
  __shared__ int cu[kMaxRequests + 1];
  __shared__ int first[kMaxRequests + 1];
  __shared__ int held[kMaxRequests];  // cached tokens
  __shared__ int64_t part[2][kTableThreads / kWave];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int R = a.requests;
  const int per = (R + kTableThreads - 1) / kTableThreads;
  const int r0 = min(tid * per, R), r1 = min(r0 + per, R);
  int64_t n = 0, p = 0;
  for (int r = r0; r < r1; ++r) {
    const Grown g = grown(a, r);
    n += g.end - g.c;
    p += g.take;
  }
  int64_t sn = n, sp = p;  // inclusive over the wave
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int64_t un = __shfl_up(sn, d, kWave), up = __shfl_up(sp, d, kWave);
    if (lane >= d) sn += un, sp += up;
  }
  if (lane == kWave - 1) part[0][wave] = sn, part[1][wave] = sp;
  __syncthreads();
  n = sn - n;
  p = sp - p;
  for (int w = 0; w < wave; ++w) n += part[0][w], p += part[1][w];
  for (int r = r0; r < r1; ++r) {
    const Grown g = grown(a, r);
    cu[r] = saturate(n);
    first[r] = saturate(p);
    held[r] = (int)g.c;
    n += g.end - g.c;
    p += g.take;
    if (r == R - 1) cu[R] = saturate(n), first[R] = saturate(p);
    if (blockIdx.x == 0) {
      a.cu[r] = cu[r];
      a.lengths[r] = saturate(g.end);
    }
  }
  __syncthreads();
  const int total = cu[R], taken = first[R];
  if (blockIdx.x == 0 && tid == 0) {
    a.cu[R] = total;
    a.counts[0] = total;
    a.counts[1] = min(taken, a.free_count);
    a.counts[2] = max(taken - a.free_count, 0);
  }
  const int64_t step = (int64_t)gridDim.x * kTableThreads;
  const int64_t at = (int64_t)blockIdx.x * kTableThreads + tid;
  for (int64_t i = at; i < taken; i += step) {
    const int r = bisect(first, R, (int)i);
    const int have = ceil_shift(held[r], a.shift);
    a.table[r * a.table_stride + have + ((int)i - first[r])] =
        i < a.free_count ? a.free_pages[i] : -1;
  }
  for (int64_t i = at; i < a.rows; i += step) {
    int64_t slot = -1;
    int position = 0, request = -1;
    if (i < total) {
      request = bisect(cu, R, (int)i);
      const int64_t pos = (int64_t)held[request] + (i - cu[request]);
      position = saturate(pos);
      const int64_t entry = pos >> a.shift;
      if (entry < a.width) {
        // pages of this step from the free list, since other threads are
        // writing their entries; the others were there before
        const int fresh = (int)entry - ceil_shift(held[request], a.shift);
        int page;
        if (fresh >= 0) {
          const int64_t f = (int64_t)first[request] + fresh;
          page = f < a.free_count ? a.free_pages[f] : -1;
        } else {
          page = a.table[request * a.table_stride + entry];
        }
        if (page >= 0)
          slot = ((int64_t)page << a.shift) + (pos & (((int64_t)1 << a.shift) - 1));
      }
    }
    a.slots[i] = slot;
    a.positions[i] = position;
    a.request_of[i] = request;
  }
}

hipError_t launch_tables(const TableArgs& a, hipStream_t s) {
  // a row a thread (509 requests, 125 thousand rows: 8.7 us at four rows) up
  // to four workgroups a compute unit
  const int64_t want = ((int64_t)a.rows + kTableThreads - 1) / kTableThreads;
  const int grid = (int)(want < 1 ? 1 : want > 1024 ? 1024 : want);
  tables_kernel<<<grid, kTableThreads, 0, s>>>(a);
  return hipGetLastError();
}

// --------------------------------------------------------- rotary positions
// Value pairs (a, b) of a head turn by angle(t, i) = pos[axis(i)][t] f_i:
// (a cos - b sin, a sin + b cos).  Bound by the stream of q, k and v.  A
// workgroup first works out the cosines and sines of its few tokens (shared
// by all heads) into LDS, then every thread turns 16-byte pieces.  The angle
// and its cosine and sine are made in 64 bits (in 32 position 200000 at
// frequency 1 would be off by up to 2^-7 of a radian), in revolutions, which
// need no reduction but a rounding.
constexpr int kRotThreads = 256;
constexpr int kRotMaxHalf = 128;

__device__ __forceinline__ int axis_of(const RotaryArgs& a, int i) {
  if (a.axes == 1) return 0;
  if (a.woven) {  // axis i mod axes, while it has a share left; else the first
    const int x = i % a.axes;
    return i / a.axes < a.sections[x] ? x : 0;
  }
  int x = 0;
  while (x + 1 < a.axes && i >= a.sections[x]) i -= a.sections[x], ++x;
  return x;
}

struct Eight {
  float v[8];
};

__device__ __forceinline__ Eight unpack8(const uint4 u) {
  Eight e;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) e.v[2 * i] = bf16_lo(w[i]), e.v[2 * i + 1] = bf16_hi(w[i]);
  return e;
}

// NaN stays NaN (f32_to_bf16 truncates one, which can leave an infinity).
__device__ __forceinline__ uint32_t bf16_bits(float v) {
  return v != v ? 0x7FC0u : f32_to_bf16(v);
}

__device__ __forceinline__ uint4 pack8(const Eight& e) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] = bf16_bits(e.v[2 * i]) | bf16_bits(e.v[2 * i + 1]) << 16;
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// e4m3 of v * inv, saturating at the type's largest value (an infinity
// would become NaN); one rounding, to nearest even, by the conversion.
__device__ __forceinline__ uint2 pack8_e4m3(const Eight& e, float inv) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float y = e.v[4 * h + i] * inv;
      x[i] = y > 448.0f ? 448.0f : y < -448.0f ? -448.0f : y;
    }
    int p = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    w[h] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], p, true);
  }
  return make_uint2(w[0], w[1]);
}

template <int TOKENS>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(const RotaryArgs a) {
  __shared__ float2 turn[TOKENS][kRotMaxHalf];
  const int tid = threadIdx.x;
  const int half = a.half, D = a.dim;
  const int64_t t0 = (int64_t)blockIdx.x * TOKENS;
  const int tokens = (int)(a.rows - t0 < TOKENS ? a.rows - t0 : TOKENS);
  for (int i = tid; i < tokens * half; i += kRotThreads) {
    const int t = i / half, f = i - t * half;
    const double pos = (double)a.positions[axis_of(a, f) * a.axis_stride + t0 + t];
    const double rev = pos * (double)a.inv_freq[f] * 0.15915494309189533577;
    double sn, cs;
    sincospi(2.0 * (rev - rint(rev)), &sn, &cs);
    turn[t][f] = make_float2((float)cs, (float)sn);
  }
  __syncthreads();
  // pieces of a head: pairs of 8 values half a turn apart (or 8 values of 4
  // adjacent pairs), then what does not turn, 8 values each
  const int turned = a.adjacent ? half / 4 : half / 8;
  const int pieces = turned + (D - 2 * half) / 8;
  const int heads = a.q_heads + a.kv_heads;
  const int all = heads * pieces;
  for (int i = tid; i < tokens * all; i += kRotThreads) {
    const int t = i / all, rest = i - t * all;
    const int h = rest / pieces, p = rest - h * pieces;
    const int64_t row = t0 + t;
    const bool is_q = h < a.q_heads;
    const int hk = h - a.q_heads;
    const uint16_t* src = is_q ? a.q + row * a.q_row + h * a.q_head
                               : a.k + row * a.k_row + hk * a.k_head;
    int64_t slot = 0;
    if (!is_q && a.slots) {
      slot = a.slots[row];
      if (slot < 0 || slot >= a.cache_slots) continue;
    }
    const bool pair = p < turned && !a.adjacent;
    const int d0 = p < turned ? p * 8 : 2 * half + (p - turned) * 8;
    const int d1 = d0 + half;
    Eight x = unpack8(load16(src + d0)), y;
    if (pair) {
      y = unpack8(load16(src + d1));
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 cs = turn[t][d0 + j];
        const float u = x.v[j], w = y.v[j];
        x.v[j] = u * cs.x - w * cs.y;
        y.v[j] = u * cs.y + w * cs.x;
      }
    } else if (p < turned) {
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        const float2 cs = turn[t][(d0 + j) >> 1];
        const float u = x.v[j], w = x.v[j + 1];
        x.v[j] = u * cs.x - w * cs.y;
        x.v[j + 1] = u * cs.y + w * cs.x;
      }
    }
    if (is_q || !a.slots) {
      uint16_t* dst = is_q ? a.q_out + (row * a.q_heads + h) * D
                           : a.k_out + (row * a.kv_heads + hk) * D;
      *reinterpret_cast<uint4*>(dst + d0) = pack8(x);
      if (pair) *reinterpret_cast<uint4*>(dst + d1) = pack8(y);
      continue;
    }
    const int64_t at = (slot >> a.shift) * a.page_stride + hk * a.head_stride +
                       (slot & ((1 << a.shift) - 1)) * a.row_stride;
    if (a.bits == 8) {
      uint8_t* dst = static_cast<uint8_t*>(a.k_cache) + at;
      *reinterpret_cast<uint2*>(dst + d0) = pack8_e4m3(x, a.k_inv);
      if (pair) *reinterpret_cast<uint2*>(dst + d1) = pack8_e4m3(y, a.k_inv);
    } else {
      uint16_t* dst = static_cast<uint16_t*>(a.k_cache) + at;
      *reinterpret_cast<uint4*>(dst + d0) = pack8(x);
      if (pair) *reinterpret_cast<uint4*>(dst + d1) = pack8(y);
    }
  }
  if (!a.slots) return;
  const int vp = D / 8;
  for (int i = tid; i < tokens * a.kv_heads * vp; i += kRotThreads) {
    const int t = i / (a.kv_heads * vp), rest = i - t * (a.kv_heads * vp);
    const int h = rest / vp, d0 = (rest - h * vp) * 8;
    const int64_t row = t0 + t, slot = a.slots[row];
    if (slot < 0 || slot >= a.cache_slots) continue;
    const uint4 u = load16(a.v + row * a.v_row + h * a.v_head + d0);
    const int64_t at = (slot >> a.shift) * a.page_stride + h * a.head_stride +
                       (slot & ((1 << a.shift) - 1)) * a.row_stride + d0;
    if (a.bits == 8)
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(a.v_cache) + at) =
          pack8_e4m3(unpack8(u), a.v_inv);
    else
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.v_cache) + at) = u;
  }
}

hipError_t launch_rotary(const RotaryArgs& a, hipStream_t s) {
  // one token a workgroup until the chip is full, then four, which share the
  // wait for the cosines
  if (a.rows <= 1024)
    rotary_kernel<1><<<(unsigned)a.rows, kRotThreads, 0, s>>>(a);
  else
    rotary_kernel<4><<<(unsigned)((a.rows + 3) / 4), kRotThreads, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace rmoe
