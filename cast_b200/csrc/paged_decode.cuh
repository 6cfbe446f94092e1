// Attention of one new token per sequence over a paged key-value cache.
//
//   s_n = q . k_n * scale;  s_n = cap tanh(s_n / cap);  s_n += slope (n - (len - 1));
//   out = sum_n softmax(s)_n v_n over the visible keys n in [max(0, len - window), len)
//
// Bound: one read of the visible keys and values from HBM (4 flops per byte and query head of a KV head).
//
// Split: every warp is a worker of its own. The visible keys of all (sequence, KV head, tile of query
// heads) units, in steps of KS keys, form one list of T steps; worker w of W takes steps [T w / W,
// T (w + 1) / W), whatever units they fall into, so ragged lengths load every warp alike and no host read
// of the lengths is needed. A worker streams its steps through a private ring of NST shared-memory stages
// with 16-byte asynchronous copies (no block barrier in the loop; the ring runs on across units), keeps a
// running maximum and sum, and at the end of a unit writes the output if the whole unit was its own, else
// an unnormalised partial. The join kernel (launched to overlap the tail) adds each unit's partials in
// worker order, so results do not depend on timing; it also writes the rows that see no key (0, -inf).
//
// 16-bit types: scores and outputs on mma.sync m16n8k16 with the KV head's query heads as the 16 rows
// (MT tiles of them). The loop is bound by memory, so the probabilities are carried as two 16-bit terms
// (p = hi + lo) and the only rounding of consequence is the output's. 32-bit: FMAs on the CUDA cores.
#pragma once

#include "common.cuh"
#include "tc_common.cuh"

namespace cast {
namespace pdec {

constexpr int NW = 4;            // warps (workers) per CTA
constexpr int NT = NW * 32;
constexpr int KS = 16;           // keys per step
constexpr int MIN_STEPS = 2;     // fewest steps worth a worker

// Ring stages per worker: 8 resident workers per SM hold at most 224 KB.
template <typename T, int D> __host__ __device__ constexpr int stage_bytes() { return 2 * KS * D * (int)sizeof(T); }
template <typename T, int D> __host__ __device__ constexpr int stages() {
  return sizeof(T) == 4 ? (D == 128 ? 3 : 6) : (D == 128 ? 3 : 6);
}
template <typename T, int D> __host__ __device__ constexpr int ctas_per_sm() { return sizeof(T) == 4 ? 1 : 2; }

struct Params {
  const void *q, *k, *v;
  void* out;
  float* lse;
  int64_t sq_b, sq_h, s_p, s_h, s_r, so_b, so_h;   // elements; keys and values share s_p, s_h, s_r
  const int32_t *table, *seq_len;
  int64_t table_stride;
  int B, H_q, H_kv, G, tiles, rows;                // tiles of `rows` query heads per KV head
  int num_pages, page_size, max_pages;
  int window;                                      // 0: none
  float scale, softcap;                            // softcap 0: none
  const float* slopes;                             // or NULL
  int W;                                           // workers
  float* ws_o;                                     // [2 W][rows][D]
  float* ws_ml;                                    // [2 W][rows][2]: running maximum (log2 units), sum
  int64_t* cum;                                    // [B + 1] first step of each sequence
};

// Visible keys [lo, len) of sequence b and the steps that cover them (step s = keys [s KS, (s + 1) KS)).
struct Span {
  int lo, len, s0, s1;
};
__device__ __forceinline__ Span span_of(const Params& p, int b) {
  Span z;
  int len = p.seq_len[b];
  // out of range (reported by plan_steps): nothing is visible
  if (len < 0 || len > 0x7fffffff - KS || (int64_t)len > (int64_t)p.max_pages * p.page_size) len = 0;
  z.len = len;
  z.lo = (p.window > 0 && len > p.window) ? len - p.window : 0;
  z.s0 = z.lo / KS;
  z.s1 = (int)(((int64_t)len + KS - 1) / KS);
  return z;
}

// Workers that share T steps, and worker w's first step.
__device__ __forceinline__ int active_workers(int64_t T, int W) {
  const int64_t n = (T + MIN_STEPS - 1) / MIN_STEPS;
  return n < W ? (int)n : W;
}
__device__ __forceinline__ int64_t first_step(int64_t T, int n, int w) { return T * w / n; }
__device__ __forceinline__ int worker_of(int64_t T, int n, int64_t step) { return (int)(((step + 1) * n + T - 1) / T) - 1; }

__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;      // 0: 16 zero bytes, nothing read
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t* r) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two probabilities as hi + lo pairs of 16-bit terms.
template <typename T> __device__ __forceinline__ void split2(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(p0, p1);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 r = __floats2bfloat162_rn(p0 - f.x, p1 - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
  } else {
    const __half2 h = __floats2half2_rn(p0, p1);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(p0 - f.x, p1 - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A score in log2 units: scaled, capped, biased by the distance to the newest key, masked.
__device__ __forceinline__ float score(const Params& p, float dot, int n, const Span& z, float slope) {
  if (n < z.lo || n >= z.len) return -INFINITY;
  float s = dot * p.scale;
  if (p.softcap > 0.f) s = p.softcap * tanhf(s / p.softcap);
  if (p.slopes != nullptr) s = fmaf(slope, (float)(n - (z.len - 1)), s);
  return s * kLog2e;
}

// Natural log-sum-exp from the running maximum (log2 units) and sum.
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

// Position of a worker in the step list.
struct Cursor {
  int b, u, s;      // sequence, unit of the sequence (KV head x tile), step
  Span z;
};
__device__ __forceinline__ void advance(const Params& p, Cursor& c) {
  if (++c.s < c.z.s1) return;
  if (++c.u == p.H_kv * p.tiles) {
    c.u = 0;
    do {
      if (++c.b >= p.B) return;
      c.z = span_of(p, c.b);
    } while (c.z.s1 <= c.z.s0);
  }
  c.s = c.z.s0;
}

// First step of every sequence: the block sums its threads' runs of sequences, scans the sums and finds
// the sequence that holds worker w's first step. CTA 0 writes the list for the join kernel.
struct Plan {
  int64_t T;
  int n;            // workers that take part
};
__device__ __forceinline__ Plan plan_steps(const Params& p, int w, Cursor& c, int64_t& begin, int64_t& end) {
  __shared__ int64_t sums[NT + 1];
  const int tid = threadIdx.x, lane = tid & 31;
  const int per = (p.B + NT - 1) / NT;
  const int64_t units = (int64_t)p.H_kv * p.tiles;
  const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    const Span z = span_of(p, b);
    mine += (z.s1 - z.s0) * units;
    if (blockIdx.x == 0 && z.len != p.seq_len[b]) report(CAST_DEV_BAD_LAYOUT);
  }
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  __shared__ int64_t wsum[NW];
  if (lane == 31) wsum[tid >> 5] = inc;
  __syncthreads();
  int64_t before = 0;
  for (int i = 0; i < (tid >> 5); ++i) before += wsum[i];
  sums[tid] = before + inc - mine;
  if (tid == NT - 1) sums[NT] = before + inc;
  __syncthreads();
  if (blockIdx.x == 0) {
    int64_t at = sums[tid];
    for (int b = b0; b < b1; ++b) {
      p.cum[b] = at;
      const Span z = span_of(p, b);
      at += (z.s1 - z.s0) * units;
    }
    if (tid == 0) p.cum[p.B] = sums[NT];
  }
  Plan pl;
  pl.T = sums[NT];
  pl.n = active_workers(pl.T, p.W);
  if (w >= pl.n) return pl;
  begin = first_step(pl.T, pl.n, w);
  end = first_step(pl.T, pl.n, w + 1);
  // the run of sequences that holds step `begin`: the last thread whose first step is <= begin
  int cnt = 0;
  for (int i = 0; i < NT / 32; ++i) cnt += __popc(__ballot_sync(0xffffffffu, sums[i * 32 + lane] <= begin));
  int b = (cnt - 1) * per;
  int64_t at = sums[cnt - 1];
  while (true) {
    c.z = span_of(p, b);
    const int64_t n = (c.z.s1 - c.z.s0) * units;
    if (begin < at + n) break;
    at += n;
    ++b;
  }
  c.b = b;
  const int steps = c.z.s1 - c.z.s0;
  c.u = (int)((begin - at) / steps);
  c.s = c.z.s0 + (int)((begin - at) % steps);
  return pl;
}

// Copies one step's keys and values into a stage: rows of D elements, 16-byte pieces permuted by the row
// (piece c of row r at c ^ (r & 7)) so that row-wise and piece-wise reads meet all banks.
// The caller passes this lane's key's page (lane & 15), fetched a step earlier.
template <typename T, int D>
__device__ __forceinline__ void issue_step(const Params& p, const Cursor& c, int page, uint32_t stage) {
  constexpr int CH = D * (int)sizeof(T) / 16;      // pieces per row
  const int lane = threadIdx.x & 31;
  const int n = c.s * KS + (lane & 15);
  int64_t off = -1;
  if (n >= c.z.lo && n < c.z.len) {
    if (page >= 0 && page < p.num_pages) off = (int64_t)page * p.s_p + (int64_t)(n % p.page_size) * p.s_r + (int64_t)(c.u / p.tiles) * p.s_h;
    else report(CAST_DEV_BAD_LAYOUT);
  }
  constexpr int IT = KS * CH / 32;
  const T* k = static_cast<const T*>(p.k);
  const T* v = static_cast<const T*>(p.v);
#pragma unroll
  for (int i = 0; i < IT; ++i) {
    const int e = i * 32 + lane;
    const int r = e / CH, ch = e % CH;
    const int64_t o = __shfl_sync(0xffffffffu, off, r);
    const bool ok = o >= 0;
    const int64_t src = (ok ? o : 0) + ch * (16 / (int)sizeof(T));
    const uint32_t dst = stage + r * (D * (int)sizeof(T)) + ((ch ^ (r & 7)) * 16);
    cp16(dst, k + src, ok);
    cp16(dst + KS * D * (int)sizeof(T), v + src, ok);
  }
}
__device__ __forceinline__ int page_of(const Params& p, const Cursor& c) {
  const int n = c.s * KS + (threadIdx.x & 15);
  if (c.b >= p.B || n < c.z.lo || n >= c.z.len) return -1;
  return p.table[(int64_t)c.b * p.table_stride + n / p.page_size];
}

// ---------------------------------------------------------------------------------------- 16-bit types
template <typename T, int D, int MT>
__global__ void __launch_bounds__(NT) decode_mma_kernel(const Params p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int NST = stages<T, D>(), SB = stage_bytes<T, D>();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int w = blockIdx.x * NW + warp;
  Cursor cc;
  int64_t at = 0, end = 0;
  const Plan pl = plan_steps(p, w, cc, at, end);
  if (w >= pl.n) return;
  const uint32_t ring = tc::smem_u32(smem) + warp * NST * SB;
  const int64_t begin = at;
  Cursor ci = cc;                      // where the copies are
  int64_t issued = at;
  int page = page_of(p, ci);
  auto issue = [&]() {
    if (issued < end) {
      issue_step<T, D>(p, ci, page, ring + (int)((issued - begin) % NST) * SB);
      ++issued;
      if (issued < end) {
        advance(p, ci);
        page = page_of(p, ci);
      }
    }
    cp_commit();
  };
  for (int i = 0; i < NST - 1; ++i) issue();

  uint32_t qf[MT][D / 16][4];
  float o[MT][D / 8][4], m[MT][2], l[MT][2], slope[MT][2];
  bool fresh = true;                   // the next step starts a piece of a unit
  bool whole = false;                  // that piece starts at the unit's first step
  int slot = 2 * w;
  int h = 0, h0 = 0, nrow = 0;
  for (; at < end; ++at) {
    if (fresh) {
      fresh = false;
      whole = cc.s == cc.z.s0;
      h = cc.u / p.tiles;
      h0 = h * p.G + (cc.u % p.tiles) * p.rows;
      nrow = min(p.rows, h * p.G + p.G - h0);
      const T* q = static_cast<const T*>(p.q) + (int64_t)cc.b * p.sq_b + (int64_t)h0 * p.sq_h;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = mt * 16 + g + (i & 1) * 8;
            qf[mt][k][i] = r < nrow ? *reinterpret_cast<const uint32_t*>(q + (int64_t)r * p.sq_h + k * 16 + t * 2 + (i >> 1) * 8) : 0u;
          }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          m[mt][i] = -INFINITY;
          l[mt][i] = 0.f;
          const int r = mt * 16 + g + i * 8;
          slope[mt][i] = (p.slopes != nullptr && r < nrow) ? p.slopes[h0 + r] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < D / 8; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[mt][j][i] = 0.f;
      }
    }
    cp_wait<NST - 2>();
    __syncwarp();
    const uint32_t sk = ring + (int)((at - begin) % NST) * SB, sv = sk + KS * D * (int)sizeof(T);
    issue();                        // into the stage that the previous step left

    float s[MT][2][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[mt][j][i] = 0.f;
    {
      const int r = (lane & 7) + (lane >> 4) * 8;   // matrices 0, 1: keys 0-7; 2, 3: keys 8-15
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        uint32_t b[4];
        const int ch = 2 * k + ((lane >> 3) & 1);
        ldsm4(sk + r * (D * 2) + ((ch ^ (r & 7)) * 16), b);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16816<T>(s[mt][0], qf[mt][k], b[0], b[1]);
          mma16816<T>(s[mt][1], qf[mt][k], b[2], b[3]);
        }
      }
    }
    const int n0 = cc.s * KS;
    uint32_t ph[MT][4], plo[MT][4];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[mt][j][i] = score(p, s[mt][j][i], n0 + j * 8 + t * 2 + (i & 1), cc.z, slope[mt][i >> 1]);
          mx[i >> 1] = fmaxf(mx[i >> 1], s[mt][j][i]);
        }
      float al[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        const float mn = fmaxf(m[mt][i], mx[i]);
        al[i] = mn == -INFINITY ? 1.f : ex2(m[mt][i] - mn);
        m[mt][i] = mn;
        l[mt][i] *= al[i];
      }
      if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          o[mt][j][0] *= al[0]; o[mt][j][1] *= al[0];
          o[mt][j][2] *= al[1]; o[mt][j][3] *= al[1];
        }
      }
      const float mu[2] = {m[mt][0] == -INFINITY ? 0.f : m[mt][0], m[mt][1] == -INFINITY ? 0.f : m[mt][1]};
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p0 = ex2(s[mt][j][2 * i] - mu[i]), p1 = ex2(s[mt][j][2 * i + 1] - mu[i]);
          l[mt][i] += p0 + p1;
          split2<T>(p0, p1, ph[mt][j * 2 + i], plo[mt][j * 2 + i]);
        }
    }
    {
      const int r = (lane & 7) + ((lane >> 3) & 1) * 8;   // matrices 0, 2: keys 0-7; 1, 3: keys 8-15
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t b[4];
        const int ch = 2 * j + (lane >> 4);
        ldsm4t(sv + r * (D * 2) + ((ch ^ (r & 7)) * 16), b);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          mma16816<T>(o[mt][2 * j], ph[mt], b[0], b[1]);
          mma16816<T>(o[mt][2 * j + 1], ph[mt], b[2], b[3]);
          mma16816<T>(o[mt][2 * j], plo[mt], b[0], b[1]);
          mma16816<T>(o[mt][2 * j + 1], plo[mt], b[2], b[3]);
        }
      }
    }
    const bool unit_end = cc.s + 1 == cc.z.s1;
    if (unit_end || at + 1 == end) {
      const bool direct = whole && unit_end;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float lt = l[mt][i] + __shfl_xor_sync(0xffffffffu, l[mt][i], 1);
          lt += __shfl_xor_sync(0xffffffffu, lt, 2);
          const int r = mt * 16 + g + i * 8;
          if (r >= nrow) continue;
          if (direct) {
            const float inv = lt == 0.f ? 0.f : 1.f / lt;
            T* out = static_cast<T*>(p.out) + (int64_t)cc.b * p.so_b + (int64_t)(h0 + r) * p.so_h + t * 2;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) {
              T y[2] = {Elem<T>::from_f(o[mt][j][2 * i] * inv), Elem<T>::from_f(o[mt][j][2 * i + 1] * inv)};
              *reinterpret_cast<uint32_t*>(out + j * 8) = *reinterpret_cast<const uint32_t*>(y);
            }
            if (p.lse != nullptr && t == 0)
              p.lse[(int64_t)cc.b * p.H_q + h0 + r] = lse_of(m[mt][i], lt);
          } else {
            float* wo = p.ws_o + ((int64_t)slot * p.rows + r) * D + t * 2;
#pragma unroll
            for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(wo + j * 8) = make_float2(o[mt][j][2 * i], o[mt][j][2 * i + 1]);
            if (t == 0) *reinterpret_cast<float2*>(p.ws_ml + ((int64_t)slot * p.rows + r) * 2) = make_float2(m[mt][i], lt);
          }
        }
      slot = 2 * w + 1;
      fresh = true;
    }
    if (at + 1 < end) advance(p, cc);
  }
  cp_wait<0>();
}

// ---------------------------------------------------------------------------------------- 32-bit type
// GT query heads of one KV head. Scores: lane = key (lane & 15) and half of the head dim (lane >> 4);
// outputs: lane = D / 32 dims, over the step's 16 keys.
template <int D, int GT>
__global__ void __launch_bounds__(NT) decode_f32_kernel(const Params p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int NST = stages<float, D>(), SB = stage_bytes<float, D>();
  constexpr int DV = D / 32;
  __shared__ __align__(16) float sq[NW][GT][D];
  __shared__ __align__(16) float sp[NW][GT][KS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int w = blockIdx.x * NW + warp;
  Cursor cc;
  int64_t at = 0, end = 0;
  const Plan pl = plan_steps(p, w, cc, at, end);
  if (w >= pl.n) return;
  uint8_t* ring_p = smem + (size_t)warp * NST * SB;
  const uint32_t ring = tc::smem_u32(ring_p);
  const int64_t begin = at;
  Cursor ci = cc;
  int64_t issued = at;
  int page = page_of(p, ci);
  auto issue = [&]() {
    if (issued < end) {
      issue_step<float, D>(p, ci, page, ring + (int)((issued - begin) % NST) * SB);
      ++issued;
      if (issued < end) {
        advance(p, ci);
        page = page_of(p, ci);
      }
    }
    cp_commit();
  };
  for (int i = 0; i < NST - 1; ++i) issue();

  float o[GT][DV], m[GT], l[GT], slope[GT];
  bool fresh = true, whole = false;
  int slot = 2 * w, h0 = 0, nrow = 0;
  const int key = lane & 15, half = lane >> 4;
  for (; at < end; ++at) {
    if (fresh) {
      fresh = false;
      whole = cc.s == cc.z.s0;
      const int h = cc.u / p.tiles;
      h0 = h * p.G + (cc.u % p.tiles) * p.rows;
      nrow = min(p.rows, h * p.G + p.G - h0);
      const float* q = static_cast<const float*>(p.q) + (int64_t)cc.b * p.sq_b + (int64_t)h0 * p.sq_h;
      __syncwarp();
#pragma unroll
      for (int a = 0; a < GT; ++a) {
        for (int d = lane; d < D; d += 32) sq[warp][a][d] = a < nrow ? q[(int64_t)a * p.sq_h + d] : 0.f;
        m[a] = -INFINITY;
        l[a] = 0.f;
        slope[a] = (p.slopes != nullptr && a < nrow) ? p.slopes[h0 + a] : 0.f;
#pragma unroll
        for (int i = 0; i < DV; ++i) o[a][i] = 0.f;
      }
    }
    cp_wait<NST - 2>();
    __syncwarp();
    const uint8_t* st = ring_p + (int)((at - begin) % NST) * SB;
    issue();

    float s[GT];
#pragma unroll
    for (int a = 0; a < GT; ++a) s[a] = 0.f;
#pragma unroll 4
    for (int c = 0; c < D / 8; ++c) {
      const int ch = half * (D / 8) + c;
      const float4 x = *reinterpret_cast<const float4*>(st + key * (D * 4) + ((ch ^ (key & 7)) * 16));
#pragma unroll
      for (int a = 0; a < GT; ++a) {
        const float4 y = *reinterpret_cast<const float4*>(&sq[warp][a][ch * 4]);
        s[a] = fmaf(x.x, y.x, s[a]);
        s[a] = fmaf(x.y, y.y, s[a]);
        s[a] = fmaf(x.z, y.z, s[a]);
        s[a] = fmaf(x.w, y.w, s[a]);
      }
    }
    const int n = cc.s * KS + key;
#pragma unroll
    for (int a = 0; a < GT; ++a) {
      s[a] += __shfl_xor_sync(0xffffffffu, s[a], 16);
      s[a] = score(p, s[a], n, cc.z, slope[a]);
      float mx = s[a];
#pragma unroll
      for (int i = 1; i < 16; i <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
      const float mn = fmaxf(m[a], mx);
      const float al = mn == -INFINITY ? 1.f : exp2f(m[a] - mn);
      const float pv = mn == -INFINITY ? 0.f : exp2f(s[a] - mn);
      m[a] = mn;
      l[a] = l[a] * al + pv;            // this lane's key; joined at the end of the unit
#pragma unroll
      for (int i = 0; i < DV; ++i) o[a][i] *= al;
      if (half == 0) sp[warp][a][key] = pv;
    }
    __syncwarp();
    const uint8_t* vt = st + KS * D * 4;
#pragma unroll
    for (int k4 = 0; k4 < KS; k4 += 4) {
      float4 pr[GT];
#pragma unroll
      for (int a = 0; a < GT; ++a) pr[a] = *reinterpret_cast<const float4*>(&sp[warp][a][k4]);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk) {
        const int r = k4 + kk;
        float x[DV];
        if constexpr (DV == 4) {
          const float4 v4 = *reinterpret_cast<const float4*>(vt + r * (D * 4) + ((lane ^ (r & 7)) * 16));
          x[0] = v4.x; x[1] = v4.y; x[2] = v4.z; x[3] = v4.w;
        } else {
          const float2 v2 = *reinterpret_cast<const float2*>(vt + r * (D * 4) + (((lane >> 1) ^ (r & 7)) * 16) + (lane & 1) * 8);
          x[0] = v2.x; x[1] = v2.y;
        }
#pragma unroll
        for (int a = 0; a < GT; ++a) {
          const float pa = kk == 0 ? pr[a].x : kk == 1 ? pr[a].y : kk == 2 ? pr[a].z : pr[a].w;
#pragma unroll
          for (int i = 0; i < DV; ++i) o[a][i] = fmaf(pa, x[i], o[a][i]);
        }
      }
    }
    const bool unit_end = cc.s + 1 == cc.z.s1;
    if (unit_end || at + 1 == end) {
      const bool direct = whole && unit_end;
#pragma unroll
      for (int a = 0; a < GT; ++a) {
        float lt = l[a];
#pragma unroll
        for (int i = 1; i < 16; i <<= 1) lt += __shfl_xor_sync(0xffffffffu, lt, i);
        if (a >= nrow) continue;
        float* dst;
        float f = 1.f;
        if (direct) {
          f = lt == 0.f ? 0.f : 1.f / lt;
          dst = static_cast<float*>(p.out) + (int64_t)cc.b * p.so_b + (int64_t)(h0 + a) * p.so_h;
          if (p.lse != nullptr && lane == 0)
            p.lse[(int64_t)cc.b * p.H_q + h0 + a] = lse_of(m[a], lt);
        } else {
          dst = p.ws_o + ((int64_t)slot * p.rows + a) * D;
          if (lane == 0) *reinterpret_cast<float2*>(p.ws_ml + ((int64_t)slot * p.rows + a) * 2) = make_float2(m[a], lt);
        }
#pragma unroll
        for (int i = 0; i < DV; ++i) dst[lane * DV + i] = o[a][i] * f;
      }
      slot = 2 * w + 1;
      fresh = true;
    }
    __syncwarp();
    if (at + 1 < end) advance(p, cc);
  }
  cp_wait<0>();
}

// ---------------------------------------------------------------------------------------- join
// One warp per (sequence, query head): adds the partials of the row's unit, in worker order. Units that
// one worker took whole are already written; rows without a visible key become 0 (lse -inf).
template <typename T, int D>
__global__ void __launch_bounds__(256) decode_join_kernel(const Params p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= (int64_t)p.B * p.H_q) return;
  const int b = (int)(row / p.H_q), hq = (int)(row % p.H_q);
  const int64_t T_all = p.cum[p.B];
  const int64_t c0 = p.cum[b], c1 = p.cum[b + 1];
  const int units = p.H_kv * p.tiles;
  T* out = static_cast<T*>(p.out) + (int64_t)b * p.so_b + (int64_t)hq * p.so_h;
  constexpr int DV = D / 32;
  if (c1 == c0) {
#pragma unroll
    for (int i = 0; i < DV; ++i) out[lane * DV + i] = Elem<T>::from_f(0.f);
    if (p.lse != nullptr && lane == 0) p.lse[row] = -INFINITY;
    return;
  }
  const int64_t steps = (c1 - c0) / units;
  const int u = (hq / p.G) * p.tiles + (hq % p.G) / p.rows, r = (hq % p.G) % p.rows;
  const int64_t us = c0 + u * steps;
  const int n = active_workers(T_all, p.W);
  const int w0 = worker_of(T_all, n, us), w1 = worker_of(T_all, n, us + steps - 1);
  if (w0 == w1) return;
  const int first = 2 * w0 + (first_step(T_all, n, w0) == us ? 0 : 1);
  auto slot_of = [&](int w) { return (int64_t)(w == w0 ? first : 2 * w) * p.rows + r; };
  float M = -INFINITY;
  for (int w = w0 + lane; w <= w1; w += 32) M = fmaxf(M, p.ws_ml[slot_of(w) * 2]);
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, i));
  const float mu = M == -INFINITY ? 0.f : M;
  float L = 0.f, acc[DV];
#pragma unroll
  for (int i = 0; i < DV; ++i) acc[i] = 0.f;
#pragma unroll 8
  for (int w = w0; w <= w1; ++w) {
    const int64_t sl = slot_of(w);
    const float2 ml = *reinterpret_cast<const float2*>(p.ws_ml + sl * 2);
    const float f = exp2f(ml.x - mu);
    L = fmaf(f, ml.y, L);
    const float* o = p.ws_o + sl * D + lane * DV;
#pragma unroll
    for (int i = 0; i < DV; ++i) acc[i] = fmaf(f, o[i], acc[i]);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int i = 0; i < DV; ++i) out[lane * DV + i] = Elem<T>::from_f(acc[i] * inv);
  if (p.lse != nullptr && lane == 0) p.lse[row] = lse_of(M, L);
}

}  // namespace pdec
}  // namespace cast
