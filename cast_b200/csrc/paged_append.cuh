// Append of key / value rows to a paged cache, with the rotary position rotation on the way.
//
// Cache: per layer, K and V pages [num_pages, H_kv, page_size, D]; sequence b's row at slot s is row
// s % page_size of page table[b][s / page_size]. A new row (sequence b, j-th new row) goes to slot
// seq_len[b] + j. Its key is rotated by pos * inv_freq[i] (pos = the slot, or the caller's position):
//   (x_a, x_b) -> (x_a cos - x_b sin, x_b cos + x_a sin),   i < h,
// with (a, b) = (i, i + h) or (2i, 2i + 1); values from 2h on pass through. Queries beside the keys
// turn by the same angles into q_out. The angle is formed and reduced to [-pi/4, pi/4] in 64 bits (a
// 32-bit product is off by 0.004 rad at position 100,000), sine and cosine of the rest and the rotation
// are 32-bit, and each result is rounded once to the cache's type.
//
// Bound: memory traffic for prompts (2 bytes moved per byte of k, v and q), the latency of the chain
// length -> table entry -> store for a few rows. One CTA takes `tok` consecutive rows (what its threads
// load at once, fewer where that leaves SMs without eight CTAs) and all their heads, so an angle is
// computed once per row and shared by H_q + H_kv heads through shared memory. Thread (x, y): x = two
// 16-byte pieces of a head, y steps over (row, head); a piece of the first half travels with its partner
// of the second half, so both results come from one thread's registers. The first loads are issued before
// the row's sequence, page and angles are known.
#pragma once

#include "common.cuh"

namespace cast {
namespace papp {

constexpr int NT = 256;
constexpr int MAX_TOK = 8;      // rows per CTA
constexpr int MAX_D = 256;
constexpr int MAX_HEADS = 4096;
constexpr int MAXL = 64;        // layers per launch
constexpr int UNROLL = 3;       // (row, head) items a thread loads before it stores the first

struct Layers {
  const void* src[MAXL][2];   // new K, V rows
  void* dst[MAXL][2];         // K, V pages
};

struct Args {
  int H_kv, H_q, D, h;                 // h = rotated pairs per head
  int interleaved, tok;
  int X, np;                           // threads per head; those that hold the two pieces of a rotated pair
  uint32_t heads_inv;                  // ceil(2^32 / (H_q + 2 H_kv)): i / heads for i < 2^16
  float rope_scale;
  int num_pages, page_size, max_pages, B;
  int64_t table_stride;
  int64_t pk_p, pk_h, pk_r, pv_p, pv_h, pv_r;          // page strides (elements)
  int64_t sk_t, sk_h, sv_t, sv_h;                      // new-row strides
  int64_t sq_t, sq_h, so_t, so_h;                      // query strides (in, out)
  int64_t total;
  const int32_t *table, *seq_len, *cu_q, *keep, *accepted, *positions;
  int keep_stride;
  const float* inv_freq;
  const void* q;
  void* q_out;
};

// The last b in [0, B) with cu_q[b] <= t, or -1; by one whole warp (33 samples a round).
__device__ __forceinline__ int find_seq(const int32_t* cu_q, int B, int64_t t) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = B;
  while (n > 32) {
    const int step = (n + 31) / 32;
    const int i = lane * step;
    const int c = __popc(__ballot_sync(0xffffffffu, i < n && (int64_t)cu_q[lo + min(i, n - 1)] <= t));
    if (c == 0) return -1;
    lo += (c - 1) * step;
    n = min(step, n - (c - 1) * step);
  }
  const int c = __popc(__ballot_sync(0xffffffffu, lane < n && (int64_t)cu_q[lo + min(lane, n - 1)] <= t));
  return c == 0 ? -1 : lo + c - 1;
}

// cos and sin of pos * freq: quarter turns and the rest of one in 64 bits, the rest's functions in 32
// (sincospif: within half a quarter turn it needs no further reduction).
__device__ __forceinline__ void cos_sin(int pos, float freq, float& c, float& s) {
  constexpr double kTwoOverPi = 0.63661977236758134308;
  const double th = (double)pos * (double)freq;
  const double n = rint(th * kTwoOverPi);
  float sr, cr;
  sincospif(0.5f * (float)fma(th, kTwoOverPi, -n), &sr, &cr);
  const int k = (int)((long long)n & 3);
  c = (k & 1) ? sr : cr;
  s = (k & 1) ? cr : sr;
  if (k == 1 || k == 2) c = -c;
  if (k >= 2) s = -s;
}

__device__ __forceinline__ float2 pair_to_f(__nv_bfloat162 x) { return __bfloat1622float2(x); }
__device__ __forceinline__ float2 pair_to_f(__half2 x) { return __half22float2(x); }
__device__ __forceinline__ void pair_from_f(__nv_bfloat162& x, float a, float b) { x = __floats2bfloat162_rn(a, b); }
__device__ __forceinline__ void pair_from_f(__half2& x, float a, float b) { x = __floats2half2_rn(a, b); }

// VEC consecutive elements as one memory access
template <typename T, int VEC> struct alignas(VEC * sizeof(T)) Piece {
  T x[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Piece<T, VEC> load_piece(const T* p) {
  Piece<T, VEC> r;
  if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(r.x) = *reinterpret_cast<const uint4*>(p);
  else r.x[0] = *p;
  return r;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_piece(T* p, const Piece<T, VEC>& r) {
  if constexpr (VEC * sizeof(T) == 16) *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(r.x);
  else *p = r.x[0];
}

// The pairs (a[e], b[e]) turned by (c[e], s[e]), rounded once; 16-bit types convert two values at a time.
template <typename T, int VEC>
__device__ __forceinline__ void turn(Piece<T, VEC>& a, Piece<T, VEC>& b, const float* c, const float* s) {
  if constexpr (sizeof(T) == 2 && VEC == 8) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2* pa = reinterpret_cast<T2*>(a.x);
    T2* pb = reinterpret_cast<T2*>(b.x);
    const float4 c0 = *reinterpret_cast<const float4*>(c), c1 = *reinterpret_cast<const float4*>(c + 4);
    const float4 s0 = *reinterpret_cast<const float4*>(s), s1 = *reinterpret_cast<const float4*>(s + 4);
    const float2 cc[4] = {{c0.x, c0.y}, {c0.z, c0.w}, {c1.x, c1.y}, {c1.z, c1.w}};
    const float2 ss[4] = {{s0.x, s0.y}, {s0.z, s0.w}, {s1.x, s1.y}, {s1.z, s1.w}};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 u = pair_to_f(pa[e]), v = pair_to_f(pb[e]);
      pair_from_f(pa[e], u.x * cc[e].x - v.x * ss[e].x, u.y * cc[e].y - v.y * ss[e].y);
      pair_from_f(pb[e], v.x * cc[e].x + u.x * ss[e].x, v.y * cc[e].y + u.y * ss[e].y);
    }
  } else {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const float u = Elem<T>::to_f(a.x[e]), v = Elem<T>::to_f(b.x[e]);
      a.x[e] = Elem<T>::from_f(u * c[e] - v * s[e]);
      b.x[e] = Elem<T>::from_f(v * c[e] + u * s[e]);
    }
  }
}

// The pairs (a[2e], a[2e + 1]) turned by (c[e], s[e]).
template <typename T, int VEC>
__device__ __forceinline__ void turn_within(Piece<T, VEC>& a, const float* c, const float* s) {
  if constexpr (sizeof(T) == 2 && VEC == 8) {
    using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
    T2* pa = reinterpret_cast<T2*>(a.x);
    const float4 c4 = *reinterpret_cast<const float4*>(c), s4 = *reinterpret_cast<const float4*>(s);
    const float cc[4] = {c4.x, c4.y, c4.z, c4.w}, ss[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 u = pair_to_f(pa[e]);
      pair_from_f(pa[e], u.x * cc[e] - u.y * ss[e], u.y * cc[e] + u.x * ss[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e + 1 < VEC; e += 2) {
      const float u = Elem<T>::to_f(a.x[e]), v = Elem<T>::to_f(a.x[e + 1]);
      a.x[e] = Elem<T>::from_f(u * c[e / 2] - v * s[e / 2]);
      a.x[e + 1] = Elem<T>::from_f(v * c[e / 2] + u * s[e / 2]);
    }
  }
}

struct RowMeta {
  int64_t row;      // source row, -1: nothing to do
  int64_t dk, dv;   // element offset of the destination row (head 0) in the K / V pages
  int pos;
};

template <typename T, int VEC>
__global__ void __launch_bounds__(NT, 4) append_kernel(const Args a, const __grid_constant__ Layers ly) {
  __shared__ RowMeta meta[MAX_TOK];
  __shared__ __align__(16) float cs[MAX_TOK][MAX_D / 2], sn[MAX_TOK][MAX_D / 2];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int l = blockIdx.y;
  const T* sk = static_cast<const T*>(ly.src[l][0]);
  const T* sv = static_cast<const T*>(ly.src[l][1]);
  T* dk = static_cast<T*>(ly.dst[l][0]);
  T* dv = static_cast<T*>(ly.dst[l][1]);
  const T* q = static_cast<const T*>(a.q);
  T* qo = static_cast<T*>(a.q_out);
  const int X = a.X, Y = NT / X;           // threads beyond X * Y have no items
  const int x = tid % X, y = tid / X;
  // A thread's pieces, at off_a and off_b of a rotated head and voff_a and voff_b of a value head: two
  // halves of a pair (x < np), or two pieces of those that pass through or hold their pairs within
  // themselves (`inner`). Single elements (VEC = 1) that pass through come one to a thread.
  const bool paired = x < a.np, two = VEC > 1 || paired, inner = VEC > 1 && a.interleaved;
  const int voff_a = x * VEC, voff_b = (X + x) * VEC;
  int off_a = voff_a, off_b = voff_b;
  if (VEC == 1 && a.interleaved) {
    off_a = paired ? 2 * x : a.np + x;
    off_b = 2 * x + 1;
  } else if (!inner) {
    off_a = paired ? x * VEC : 2 * a.h + (x - a.np) * VEC;
    off_b = paired ? a.h + x * VEC : a.h + (X + x - a.np) * VEC;
  }
  const int heads = a.H_q + 2 * a.H_kv;      // H_q = 0 without queries
  // accept mode: one CTA per sequence walks its accepted rows; else one CTA per `tok` rows
  const bool accept = a.keep != nullptr;
  int rounds = 1, n_acc = 0;
  if (accept) {
    n_acc = a.accepted[blockIdx.x];
    if (n_acc < 0 || n_acc > a.keep_stride) {
      if (tid == 0 && l == 0) report(CAST_DEV_BAD_LAYOUT);
      return;
    }
    rounds = (n_acc + a.tok - 1) / a.tok;
  }
  const int items = a.tok * heads;
  const bool busy = y < Y;
  Piece<T, VEC> pa[UNROLL], pb[UNROLL];
  // source row of the CTA's k-th row; without lists it is known before the sequence it belongs to is
  auto row_of = [&](int k) -> int64_t {
    if (accept) return meta[k].row;
    const int64_t r = (int64_t)blockIdx.x * a.tok + k;
    return r < a.total ? r : -1;
  };
  auto load = [&](int i0) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int i = i0 + u * Y + y;
      if (!busy || i >= items) continue;
      const int k = (int)__umulhi((uint32_t)i, a.heads_inv), hd = i - k * heads;
      const int64_t row = row_of(k);
      if (row < 0) continue;
      const bool is_v = hd >= a.H_q + a.H_kv;
      const T* src;
      if (hd < a.H_q) src = q + row * a.sq_t + hd * a.sq_h;
      else if (!is_v) src = sk + row * a.sk_t + (hd - a.H_q) * a.sk_h;
      else src = sv + row * a.sv_t + (hd - a.H_q - a.H_kv) * a.sv_h;
      pa[u] = load_piece<T, VEC>(src + (is_v ? voff_a : off_a));
      if (two) pb[u] = load_piece<T, VEC>(src + (is_v ? voff_b : off_b));
    }
  };
  auto store = [&](int i0) {
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const int i = i0 + u * Y + y;
      if (!busy || i >= items) continue;
      const int k = (int)__umulhi((uint32_t)i, a.heads_inv), hd = i - k * heads;
      const RowMeta m = meta[k];
      if (m.row < 0) continue;
      const bool is_v = hd >= a.H_q + a.H_kv;
      T* dst;
      if (hd < a.H_q) dst = qo + m.row * a.so_t + hd * a.so_h;
      else if (!is_v) dst = dk + m.dk + (hd - a.H_q) * a.pk_h;
      else dst = dv + m.dv + (hd - a.H_q - a.H_kv) * a.pv_h;
      if (!is_v) {
        if (inner) {
          if (off_a < 2 * a.h) turn_within<T, VEC>(pa[u], cs[k] + off_a / 2, sn[k] + off_a / 2);
          if (off_b < 2 * a.h) turn_within<T, VEC>(pb[u], cs[k] + off_b / 2, sn[k] + off_b / 2);
        } else if (paired) {
          turn<T, VEC>(pa[u], pb[u], cs[k] + x * VEC, sn[k] + x * VEC);
        }
      }
      store_piece<T, VEC>(dst + (is_v ? voff_a : off_a), pa[u]);
      if (two) store_piece<T, VEC>(dst + (is_v ? voff_b : off_b), pb[u]);
    }
  };
  for (int rd = 0; rd < rounds; ++rd) {
    if (rd > 0) __syncthreads();             // the previous round's rows are done with meta, cs and sn
    if (!accept) load(0);
    for (int k = warp; k < a.tok; k += NT / 32) {
      int b, j;
      int64_t row;
      bool have;
      if (accept) {
        b = blockIdx.x;
        j = rd * a.tok + k;
        have = j < n_acc;
        row = -1;
        if (have) {
          const int pk = a.keep[(int64_t)b * a.keep_stride + j];
          const int64_t q0 = a.cu_q[b], q1 = a.cu_q[b + 1];
          row = q0 + pk;
          if (pk < 0 || q0 < 0 || row >= q1 || row >= a.total) {
            if (lane == 0) report(CAST_DEV_BAD_LAYOUT);
            have = false;
          }
        }
      } else {
        row = (int64_t)blockIdx.x * a.tok + k;
        have = row < a.total;
        if (a.cu_q == nullptr) {
          b = (int)row;
          j = 0;
          have = have && row < a.B;
        } else {
          b = have ? find_seq(a.cu_q, a.B, row) : -1;
          have = have && b >= 0;
          j = 0;
          if (have) {
            const int64_t q0 = a.cu_q[b];
            have = q0 >= 0 && row < a.cu_q[b + 1];   // rows behind the last sequence stay as they are
            j = (int)(row - q0);
          }
        }
      }
      if (lane == 0) {
        RowMeta m{-1, 0, 0, 0};
        if (have) {
          const int len = a.seq_len[b];
          const int64_t slot = (int64_t)len + j;
          const int64_t pi = slot / a.page_size;
          int page = -1;
          if (len >= 0 && pi < a.max_pages) page = a.table[(int64_t)b * a.table_stride + pi];
          if (page < 0 || page >= a.num_pages) {
            report(CAST_DEV_BAD_LAYOUT);
          } else {
            const int64_t r = slot - pi * a.page_size;
            m.row = row;
            m.dk = (int64_t)page * a.pk_p + r * a.pk_r;
            m.dv = (int64_t)page * a.pv_p + r * a.pv_r;
            m.pos = a.positions ? a.positions[row] : (int)min(slot, (int64_t)0x7fffffff);
          }
        }
        meta[k] = m;
      }
    }
    __syncthreads();
    if (accept) load(0);
    // the angles of this round's rows, while the first loads are under way
    for (int e = tid; e < a.tok * a.h; e += NT) {
      const int k = e / a.h, i = e - k * a.h;
      if (meta[k].row < 0) continue;
      float c, s;
      cos_sin(meta[k].pos, a.inv_freq[i], c, s);
      cs[k][i] = c * a.rope_scale;
      sn[k][i] = s * a.rope_scale;
    }
    __syncthreads();
    store(0);
    for (int i0 = Y * UNROLL; i0 < items; i0 += Y * UNROLL) {
      load(i0);
      store(i0);
    }
  }
}

}  // namespace papp
}  // namespace cast
