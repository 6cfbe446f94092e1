// Attention of one new token per sequence over a paged key-value cache.
//
//   s_n = q . k_n * scale;  s_n = cap tanh(s_n / cap);  s_n += slope (n - (len - 1));
//   out = sum_n softmax(s)_n v_n over the visible keys n in [max(0, len - window), len)
//
// Bound: one read of the visible keys and values from HBM (4 flops per byte and query head of a KV head).
//
// Split: every warp is a worker of its own. The visible keys of all (sequence, KV head, tile of query
// heads) units, in steps of 4 KB of keys (16 keys of 128 16-bit values), form one list of T steps, cut into n even groups of steps whatever
// units they fall into, so ragged lengths load every warp alike and no host read of the lengths is needed.
// A long group is cut once more, into a head and NS short tails: the CTAs of the heads come first in the
// grid and fill the GPU, those of the tails start as slots get free. Some SMs read memory a tenth slower
// than the others (measured: 24 of 148, always the same), and the tails go to the fast ones.
// A worker streams its steps through a private ring of NST shared-memory stages with 16-byte asynchronous
// copies (no block barrier in the loop; the ring runs on across units), keeps a running maximum and sum,
// and at the end of a unit writes the output if the whole unit was its own, else an unnormalised partial.
// The join kernel (launched to overlap the tail) adds each unit's partials in the order of the list, so
// results do not depend on timing; it also writes the rows that see no key (0, -inf).
//
// 16-bit types: S^T = K Q^T and O^T = V^T P^T on mma.sync m16n8k16, so that keys and head dims fill the 16
// rows and the KV head's query heads are the 8 columns (NH tiles of them; with heads as rows a group of 4
// left 12 of 16 rows idle and held twice the registers). The probabilities are carried as two 16-bit
// terms (p = hi + lo, in half precision of 2^14 p): the loop is bound by memory, and the only rounding of
// consequence is the output's.
// 32-bit: FMAs on the CUDA cores.
#pragma once

#include "common.cuh"
#include "tc_common.cuh"

namespace cast {
namespace pdec {

constexpr int NW = 2;            // warps (workers) per CTA
constexpr int NT = NW * 32;
constexpr int NS = 2;            // short tails of a long group,
constexpr int TAIL = 12;         // each 1 / TAIL of it,
constexpr int MIN_TAIL = 8;      // and of at least this many steps (tails of 4 cost a sequence of 131072 keys a tenth)

// Keys per step, CTAs per SM, and ring stages per worker: 192 KB an SM. Two warps to a CTA start tails sooner
// than four (64 ragged sequences 239 against 244 us). 32-bit: the scores' FMAs want more warps than the
// copies want stages (64 sequences of 3000 keys, 32 / 8 heads: 250 us with 12 warps of two stages, 296 with 8
// of three; 16-bit 245 against 239 us).
template <typename T, int D> __host__ __device__ constexpr int step_keys() { return 4096 / (D * (int)sizeof(T)); }
template <typename T, int D> __host__ __device__ constexpr int stage_bytes() { return 2 * step_keys<T, D>() * D * (int)sizeof(T); }
template <typename T, int D> __host__ __device__ constexpr int stages() { return sizeof(T) == 4 ? 2 : 3; }
__host__ __device__ constexpr int ctas_per_sm(int elem_bytes) { return elem_bytes == 4 ? 6 : 4; }
constexpr int JOIN_NT = 256;

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
  float scale, softcap, cap_exp, cap_inv;          // softcap 0: none; 2 log2(e) / softcap, 1 / softcap
  int modified;                                    // softcap or slopes given
  int64_t v_minus_k;                               // byte distance of the value pages from the key pages
  int join_warps;                                  // warps of the join kernel per row
  const float* slopes;                             // or NULL
  int W, ns;                                       // groups of steps at most; tails per group (0 or NS)
  float* ws_o;                                     // [2 W (1 + ns)][rows][D]
  float* ws_ml;                                    // [2 W (1 + ns)][rows][2]: running maximum (log2 units), sum
};

// Visible keys [lo, len) of sequence b and the steps that cover them (step s = keys [s KS, (s + 1) KS)).
struct Span {
  int lo, len, s0, s1;
};
template <int KS> __device__ __forceinline__ Span span_of(const Params& p, int len) {
  Span z;
  // out of range (reported by plan_steps): nothing is visible. The copies look at table entries up to 63 ahead.
  if (len < 0 || len > 0x7fffffff - 8192 || (int64_t)len > (int64_t)p.max_pages * p.page_size) len = 0;
  z.len = len;
  z.lo = (p.window > 0 && len > p.window) ? len - p.window : 0;
  z.s0 = z.lo / KS;
  z.s1 = (int)(((int64_t)len + KS - 1) / KS);
  return z;
}

// a * b / c of non-negative numbers; 64-bit division takes some 100 instructions, so short lists go without
__device__ __forceinline__ int64_t mul_div(int64_t a, int b, int64_t c) {
  if (a * b <= 0xffffffffll && c <= 0xffffffffll) return (uint32_t)(a * b) / (uint32_t)c;
  return a * b / c;
}

// How T steps are cut: n groups, group g = steps [T g / n, T (g + 1) / n), of which the last ns * tail are
// ns tails. Piece j of group g (0: its head) is piece g (1 + ns) + j of the list.
struct Cut {
  int64_t T;
  int n, ns, tail;
  __device__ __forceinline__ Cut(int64_t steps, int W, int tails) : T(steps) {
    n = T < W ? (int)T : W;
    tail = tails > 0 && n > 0 ? (int)(mul_div(T, 1, n) / TAIL) : 0;
    ns = tail >= MIN_TAIL ? tails : 0;
  }
  __device__ __forceinline__ int64_t group(int g) const { return mul_div(T, g, n); }
  __device__ __forceinline__ int64_t first(int g, int j) const {
    return j == 0 ? group(g) : group(g + 1) - (int64_t)(ns - j + 1) * tail;
  }
  // the piece that holds a step, and that piece's first step
  __device__ __forceinline__ int piece_of(int64_t step, int64_t& begin) const {
    // the largest g with T g / n <= step, that is g < (step + 1) n / T
    int g = (int)mul_div(step + 1, n, T);
    if (g >= n || group(g) > step) --g;
    int j = 0;
    if (ns > 0) {
      const int64_t back = group(g + 1) - 1 - step;
      if (back < (int64_t)ns * tail) j = ns - (int)back / tail;
    }
    begin = first(g, j);
    return g * (1 + ns) + j;
  }
};

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::256B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp16_if(uint32_t dst, const void* src, bool valid) {
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

// 8 x 8 16-bit matrix spread over the warp (row lane / 4, columns 2 (lane % 4) and + 1), transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// The power of two that probabilities (1 at most) are multiplied by before they are split, and what takes it out
// of the sums of values again. Half precision ends at 2^-24: one split of p itself lost a sixth of p = 1.4e-7 and
// everything under 2^-25. Of 2^14 p the two terms are off by 2^-22 p or 2^-39, whichever is more, so 2^17 keys
// together by 2^-22 of the largest.
template <typename T> __host__ __device__ constexpr float p_scale() { return std::is_same<T, __half>::value ? 16384.f : 1.f; }

// Two probabilities, scaled, as hi + lo pairs of 16-bit terms.
template <typename T> __device__ __forceinline__ void split2(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(p0, p1);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 r = __floats2bfloat162_rn(p0 - f.x, p1 - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&r);
  } else {
    p0 *= p_scale<T>();
    p1 *= p_scale<T>();
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

__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A scaled score with its cap and its bias by the distance to the newest key, in log2 units. 32-bit: tanhf
// (which took a third of the 16-bit loop's instructions). 16-bit types: with x = |s| / cap, from a quarter up
// tanh x = 1 - 2 / (1 + e^2x), off by 2.5 x 2^-23, that is 2^-19 of the capped score at most; below, where that
// difference cancels (at a cap of 1e6 a score of 0.3 became 0.24, at 1e8 every score 0), s times the Taylor
// polynomial of tanh x / x to x^8, off by 2^-23: a large cap leaves the score as it is. 32 sequences with window
// and cap: 24.6 us without the polynomial, 25.0 with it.
template <bool EXACT>
__device__ __forceinline__ float modified_score(const Params& p, float s, int n, const Span& z, float slope) {
  if (p.softcap > 0.f) {
    if (EXACT) {
      s = p.softcap * tanhf(s / p.softcap);
    } else {
      const float a = fabsf(s), y = s * p.cap_inv * (s * p.cap_inv);
      const float far = copysignf(fmaf(-2.f * p.softcap, rcp(1.f + ex2(a * p.cap_exp)), p.softcap), s);
      const float near = fmaf(fmaf(fmaf(fmaf(62.f / 2835.f, y, -17.f / 315.f), y, 2.f / 15.f), y, -1.f / 3.f), y, 1.f) * s;
      s = y < 0.0625f ? near : far;
    }
  }
  if (p.slopes != nullptr) s = fmaf(slope, (float)(n - (z.len - 1)), s);
  return s * kLog2e;
}

// Natural log-sum-exp from the running maximum (log2 units) and sum.
__device__ __forceinline__ float lse_of(float m, float l) {
  return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}

// Position of a worker in the step list. Lane i holds the length of sequence `base` + i.
struct Cursor {
  int b, u, s;      // sequence, unit of the sequence (KV head x tile), step
  int base, lens;
  Span z;
};
template <int KS>
__device__ __forceinline__ void enter(const Params& p, Cursor& c) {
  if (c.b >= c.base + 32) {
    c.base = c.b;
    const int i = c.b + (threadIdx.x & 31);
    c.lens = i < p.B ? p.seq_len[i] : 0;
  }
  c.z = span_of<KS>(p, __shfl_sync(0xffffffffu, c.lens, c.b - c.base));
}
// To the next step; true when it starts another unit.
template <int KS>
__device__ __forceinline__ bool advance(const Params& p, Cursor& c) {
  if (++c.s < c.z.s1) return false;
  if (++c.u == p.H_kv * p.tiles) {
    c.u = 0;
    do {
      if (++c.b >= p.B) return true;
      enter<KS>(p, c);
    } while (c.z.s1 <= c.z.s0);
  }
  c.s = c.z.s0;
  return true;
}

// First step of every sequence, by a block of THREADS: thread t owns the run of `per` sequences from t * per
// and sums[t] is the run's first step; sums[THREADS] = T.
template <int KS, int THREADS>
__device__ __forceinline__ int scan_steps(const Params& p, int64_t* sums, int64_t* wsum, bool check) {
  const int tid = threadIdx.x, lane = tid & 31;
  const int per = (p.B + THREADS - 1) / THREADS;
  const int64_t units = (int64_t)p.H_kv * p.tiles;
  const int b0 = min(tid * per, p.B), b1 = min(b0 + per, p.B);
  int64_t mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int len = p.seq_len[b];
    const Span z = span_of<KS>(p, len);
    mine += (z.s1 - z.s0) * units;
    if (check && z.len != len) report(CAST_DEV_BAD_LAYOUT);
  }
  int64_t inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += x;
  }
  if (lane == 31) wsum[tid >> 5] = inc;
  __syncthreads();
  int64_t before = 0;
  for (int i = 0; i < (tid >> 5); ++i) before += wsum[i];
  sums[tid] = before + inc - mine;
  if (tid == THREADS - 1) sums[THREADS] = before + inc;
  __syncthreads();
  return per;
}

// What this warp does: its piece of the list and the cursor at the piece's first step.
struct Work {
  int piece;        // -1: nothing
  int steps;
  Cursor c;
};
template <int KS>
__device__ __forceinline__ Work plan_steps(const Params& p) {
  __shared__ int64_t sums[NT + 1], wsum[NW];
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t units = (int64_t)p.H_kv * p.tiles;
  const int per = scan_steps<KS, NT>(p, sums, wsum, blockIdx.x == 0);
  const Cut cut(sums[NT], p.W, p.ns);
  Work wk;
  Cursor& c = wk.c;
  wk.piece = -1;
  // the heads' CTAs come first; tail CTA x takes tail x % NS of NW neighbouring groups
  const int heads = p.W / NW;
  int g = blockIdx.x * NW + (tid >> 5), j = 0;
  if ((int)blockIdx.x >= heads) {
    const int x = blockIdx.x - heads;
    g = x / NS * NW + (tid >> 5);
    j = 1 + x % NS;
  }
  if (g >= cut.n || j > cut.ns) return wk;
  wk.piece = g * (1 + cut.ns) + j;
  const int64_t begin = cut.first(g, j);
  wk.steps = (int)((j == cut.ns ? cut.group(g + 1) : cut.first(g, j + 1)) - begin);
  // the run of sequences that holds step `begin`: the last thread whose first step is <= begin
  int cnt = 0;
  for (int i = 0; i < NT / 32; ++i) cnt += __popc(__ballot_sync(0xffffffffu, sums[i * 32 + lane] <= begin));
  c.b = (cnt - 1) * per;
  c.base = c.b - 32;
  int64_t at = sums[cnt - 1];
  while (true) {
    enter<KS>(p, c);
    const int64_t n = (c.z.s1 - c.z.s0) * units;
    if (begin < at + n) break;
    at += n;
    ++c.b;
  }
  const int steps = c.z.s1 - c.z.s0;
  c.u = (int)mul_div(begin - at, 1, steps);
  c.s = c.z.s0 + (int)(begin - at - (int64_t)c.u * steps);
  return wk;
}

// The copying side of a worker: its own cursor, ahead of the computing one. Lane i holds the sequence's
// table entry `base` + i, and entry `base` + 32 + i is under way.
// A stage holds KS rows of keys, then of values; 16-byte piece c of row r is kept at c ^ (r & 7), so that
// row-wise and piece-wise reads meet all banks.
template <typename T, int D>
struct Copier {
  static constexpr int KS = step_keys<T, D>();
  static constexpr int CH = D * (int)sizeof(T) / 16;      // pieces per row
  static constexpr int RPI = 32 / CH;                     // rows per warp-wide copy
  static constexpr int IT = KS * CH / 32;                 // copies per step (keys or values)
  static constexpr int ROW = D * (int)sizeof(T);
  Cursor c;
  int base, page, ahead;
  int pi, pr;             // page and row of the step's first key
  const char* head;       // keys of the unit's KV head

  __device__ __forceinline__ int entry(const Params& p, int i) const {
    return i <= (c.z.len - 1) / p.page_size ? p.table[(int64_t)c.b * p.table_stride + i] : -1;
  }
  __device__ __forceinline__ void start(const Params& p, const Cursor& at) {
    const int lane = threadIdx.x & 31, n0 = at.s * KS;
    c = at;
    head = static_cast<const char*>(p.k) + (int64_t)(c.u / p.tiles) * p.s_h * (int)sizeof(T);
    pi = n0 / p.page_size;
    pr = n0 - pi * p.page_size;
    base = pi;
    page = entry(p, base + lane);
    ahead = entry(p, base + 32 + lane);
  }
  __device__ __forceinline__ void next(const Params& p) {
    if (advance<KS>(p, c)) {
      start(p, c);
      return;
    }
    pr += KS;
    while (pr >= p.page_size) {
      pr -= p.page_size;
      ++pi;
    }
    if (pi >= base + 32) {      // by KS at most
      base += 32;
      page = ahead;
      ahead = entry(p, base + 32 + (threadIdx.x & 31));
    }
  }
  __device__ __forceinline__ void copy(const Params& p, uint32_t stage) const {
    const int lane = threadIdx.x & 31;
    const int ch = lane % CH, r0 = lane / CH;
    const int lo = c.z.lo - c.s * KS, hi = c.z.len - c.s * KS;     // visible rows of the step: [lo, hi)
    if (pr + KS <= p.page_size) {          // one page (always where page_size is a multiple of KS)
      const int pg = __shfl_sync(0xffffffffu, page, pi - base);
      const bool ok = pg >= 0 && pg < p.num_pages;
      if (!ok) report(CAST_DEV_BAD_LAYOUT);
      const int64_t step = p.s_r * (int)sizeof(T) * RPI;
      const char* src = head + ((int64_t)(ok ? pg : 0) * p.s_p + (int64_t)(pr + r0) * p.s_r) * (int)sizeof(T) + ch * 16;
      if (ok && lo <= 0 && hi >= KS) {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int r = i * RPI + r0;
          const uint32_t dst = stage + r * ROW + ((ch ^ (r & 7)) * 16);
          cp16(dst, src);
          cp16(dst + KS * ROW, src + p.v_minus_k);
          src += step;
        }
      } else {
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int r = i * RPI + r0;
          const uint32_t dst = stage + r * ROW + ((ch ^ (r & 7)) * 16);
          const bool in = ok && r >= lo && r < hi;
          cp16_if(dst, in ? src : head, in);
          cp16_if(dst + KS * ROW, (in ? src : head) + p.v_minus_k, in);
          src += step;
        }
      }
    } else {
      const int key = lane & (KS - 1), i = (pr + key) / p.page_size, row = pr + key - i * p.page_size;
      const int e = pi + i - base;         // up to 31 + KS
      const int e0 = __shfl_sync(0xffffffffu, page, e & 31), e1 = __shfl_sync(0xffffffffu, ahead, e & 31);
      const int pg = e < 32 ? e0 : e1;
      int64_t off = -1;
      if (key >= lo && key < hi) {
        if (pg >= 0 && pg < p.num_pages) off = ((int64_t)pg * p.s_p + (int64_t)row * p.s_r) * (int)sizeof(T);
        else report(CAST_DEV_BAD_LAYOUT);
      }
#pragma unroll
      for (int k = 0; k < IT; ++k) {
        const int r = k * RPI + r0;
        const int64_t o = __shfl_sync(0xffffffffu, off, r);
        const char* src = head + (o >= 0 ? o : 0) + ch * 16;
        const uint32_t dst = stage + r * ROW + ((ch ^ (r & 7)) * 16);
        cp16_if(dst, src, o >= 0);
        cp16_if(dst + KS * ROW, src + p.v_minus_k, o >= 0);
      }
    }
  }
};

// ---------------------------------------------------------------------------------------- 16-bit types
// NH tiles of 8 query heads of one KV head. Thread (g = lane / 4, t = lane % 4) holds the scores of keys
// g and g + 8 and the outputs of dims 16 j + g and + 8, for heads 2t and 2t + 1 of each tile.
template <typename T, int D, int NH>
__global__ void __launch_bounds__(NT) decode_mma_kernel(const Params p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int KS = step_keys<T, D>(), NST = stages<T, D>(), SB = stage_bytes<T, D>(), ROW = D * 2;
  constexpr int SUB = KS / 16;         // 16-key MMA rows per step
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const Work wk = plan_steps<KS>(p);
  if (wk.piece < 0) return;
  Cursor cc = wk.c;
  const uint32_t ring = tc::smem_u32(smem) + warp * NST * SB;
  int left = wk.steps;                 // steps to compute
  int to_copy = left;
  Copier<T, D> cp;
  cp.start(p, cc);
  uint32_t put = ring, take = ring;    // the stages of the next copy and of the next step
  auto issue = [&]() {
    if (to_copy > 0) {
      cp.copy(p, put);
      if (--to_copy > 0) cp.next(p);
      put = put + SB == ring + NST * SB ? ring : put + SB;
    }
    cp_commit();
  };
  for (int i = 0; i < NST - 1; ++i) issue();

  // ldmatrix row addresses within a stage: keys as the rows of A (matrices: keys 0-7 and 8-15 of piece 2k,
  // then of piece 2k + 1), values transposed (matrices: pieces 2j and 2j + 1 of keys 0-7, then of keys 8-15)
  const int kr = (lane & 7) + ((lane >> 3) & 1) * 8, kx = (lane >> 4) ^ (kr & 7);
  const int vr = (lane & 7) + (lane >> 4) * 8, vx = ((lane >> 3) & 1) ^ (vr & 7);
  const uint32_t koff = kr * ROW, voff = KS * ROW + vr * ROW;
  const float c = p.scale * kLog2e;

  uint32_t qf[NH][D / 16][2];
  float o[NH][D / 16][4], m[NH][2], l[NH][2], slope[NH][2];
  bool fresh = true;                   // the next step starts a piece of a unit
  bool whole = false;                  // that piece starts at the unit's first step
  int slot = 2 * wk.piece;
  int h0 = 0, nrow = 0;
  for (; left > 0; --left) {
    if (fresh) {
      fresh = false;
      whole = cc.s == cc.z.s0;
      const int h = cc.u / p.tiles;
      h0 = h * p.G + (cc.u - h * p.tiles) * p.rows;
      nrow = min(p.rows, h * p.G + p.G - h0);
      const T* q = static_cast<const T*>(p.q) + (int64_t)cc.b * p.sq_b + (int64_t)h0 * p.sq_h;
#pragma unroll
      for (int a = 0; a < NH; ++a) {
        const int r = a * 8 + g;
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
#pragma unroll
          for (int i = 0; i < 2; ++i)
            qf[a][k][i] = r < nrow ? *reinterpret_cast<const uint32_t*>(q + (int64_t)r * p.sq_h + k * 16 + t * 2 + i * 8) : 0u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          m[a][i] = -INFINITY;
          l[a][i] = 0.f;
          const int hr = a * 8 + t * 2 + i;
          slope[a][i] = (p.slopes != nullptr && hr < nrow) ? p.slopes[h0 + hr] : 0.f;
        }
#pragma unroll
        for (int j = 0; j < D / 16; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[a][j][i] = 0.f;
      }
    }
    cp_wait<NST - 2>();
    __syncwarp();
    const uint32_t st = take;
    take = take + SB == ring + NST * SB ? ring : take + SB;
    issue();                           // into the stage that the previous step left

    constexpr int NC = NH * SUB == 1 ? 2 : 1;      // one tile of heads and keys: two chains of dependent MMAs
    float s[SUB][NH][4], s2[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < SUB; ++e)
#pragma unroll
      for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[e][a][i] = 0.f;
#pragma unroll
    for (int k = 0; k < D / 16; ++k)
#pragma unroll
      for (int e = 0; e < SUB; ++e) {
        uint32_t ka[4];
        ldsm4(st + koff + e * 16 * ROW + ((kx ^ (2 * k)) * 16), ka);
#pragma unroll
        for (int a = 0; a < NH; ++a) mma16816<T>((k % NC) ? s2 : s[e][a], ka, qf[a][k][0], qf[a][k][1]);
      }
    if (NC == 2)
#pragma unroll
      for (int i = 0; i < 4; ++i) s[0][0][i] += s2[i];
    const int n0 = cc.s * KS + g;
    if (p.modified) {
#pragma unroll
      for (int e = 0; e < SUB; ++e)
#pragma unroll
        for (int a = 0; a < NH; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[e][a][i] = modified_score<false>(p, s[e][a][i] * p.scale, n0 + e * 16 + (i >> 1) * 8, cc.z, slope[a][i & 1]);
    } else {
#pragma unroll
      for (int e = 0; e < SUB; ++e)
#pragma unroll
        for (int a = 0; a < NH; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[e][a][i] *= c;
    }
    if (n0 - g < cc.z.lo || n0 - g + KS > cc.z.len) {
#pragma unroll
      for (int e = 0; e < SUB; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int n = n0 + e * 16 + i * 8;
          if (n < cc.z.lo || n >= cc.z.len)
#pragma unroll
            for (int a = 0; a < NH; ++a) s[e][a][2 * i] = s[e][a][2 * i + 1] = -INFINITY;
        }
    }
    uint32_t ph[SUB][NH][2], pl_[SUB][NH][2];
#pragma unroll
    for (int a = 0; a < NH; ++a) {
      float al[2], mu[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float mx = fmaxf(s[0][a][i], s[0][a][2 + i]);
#pragma unroll
        for (int e = 1; e < SUB; ++e) mx = fmaxf(mx, fmaxf(s[e][a][i], s[e][a][2 + i]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        const float mn = fmaxf(m[a][i], mx);
        mu[i] = mn == -INFINITY ? 0.f : mn;
        al[i] = ex2(m[a][i] - mu[i]);
        m[a][i] = mn;
      }
      if (__any_sync(0xffffffffu, al[0] != 1.f || al[1] != 1.f)) {
        l[a][0] *= al[0];
        l[a][1] *= al[1];
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          o[a][j][0] *= al[0]; o[a][j][1] *= al[1];
          o[a][j][2] *= al[0]; o[a][j][3] *= al[1];
        }
      }
#pragma unroll
      for (int e = 0; e < SUB; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float p0 = ex2(s[e][a][2 * i] - mu[0]), p1 = ex2(s[e][a][2 * i + 1] - mu[1]);
          l[a][0] += p0;
          l[a][1] += p1;
          split2<T>(p0, p1, ph[e][a][i], pl_[e][a][i]);
          ph[e][a][i] = transpose8(ph[e][a][i]);
          pl_[e][a][i] = transpose8(pl_[e][a][i]);
        }
    }
#pragma unroll
    for (int e = 0; e < SUB; ++e)
#pragma unroll
      for (int j = 0; j < D / 16; ++j) {
        uint32_t va[4];
        ldsm4t(st + voff + e * 16 * ROW + ((vx ^ (2 * j)) * 16), va);
#pragma unroll
        for (int a = 0; a < NH; ++a) {
          mma16816<T>(o[a][j], va, ph[e][a][0], ph[e][a][1]);
          mma16816<T>(o[a][j], va, pl_[e][a][0], pl_[e][a][1]);
        }
      }
    const bool unit_end = cc.s + 1 == cc.z.s1;
    if (unit_end || left == 1) {
      const bool direct = whole && unit_end;
#pragma unroll
      for (int a = 0; a < NH; ++a)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float lt = l[a][i] + __shfl_xor_sync(0xffffffffu, l[a][i], 4);
          lt += __shfl_xor_sync(0xffffffffu, lt, 8);
          lt += __shfl_xor_sync(0xffffffffu, lt, 16);
          const int r = a * 8 + t * 2 + i;
          if (r >= nrow) continue;
          if (direct) {
            const float inv = lt == 0.f ? 0.f : (1.f / p_scale<T>()) / lt;
            T* out = static_cast<T*>(p.out) + (int64_t)cc.b * p.so_b + (int64_t)(h0 + r) * p.so_h + g;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              out[j * 16] = Elem<T>::from_f(o[a][j][i] * inv);
              out[j * 16 + 8] = Elem<T>::from_f(o[a][j][2 + i] * inv);
            }
            if (p.lse != nullptr && g == 0) p.lse[(int64_t)cc.b * p.H_q + h0 + r] = lse_of(m[a][i], lt);
          } else {
            float* wo = p.ws_o + ((int64_t)slot * p.rows + r) * D + g;
#pragma unroll
            for (int j = 0; j < D / 16; ++j) {
              wo[j * 16] = o[a][j][i] * (1.f / p_scale<T>());
              wo[j * 16 + 8] = o[a][j][2 + i] * (1.f / p_scale<T>());
            }
            if (g == 0) *reinterpret_cast<float2*>(p.ws_ml + ((int64_t)slot * p.rows + r) * 2) = make_float2(m[a][i], lt);
          }
        }
      slot = 2 * wk.piece + 1;
      fresh = true;
    }
    if (left > 1) advance<KS>(p, cc);
  }
  cp_wait<0>();
}

// ---------------------------------------------------------------------------------------- 32-bit type
// GT query heads of one KV head. Scores: lane = key (lane % KS) and every (32 / KS)-th 16-byte piece of it;
// outputs: lane = D / 32 dims, over the step's keys.
template <int D, int GT>
__global__ void __launch_bounds__(NT) decode_f32_kernel(const Params p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int KS = step_keys<float, D>(), NST = stages<float, D>(), SB = stage_bytes<float, D>();
  constexpr int DV = D / 32, PARTS = 32 / KS;
  __shared__ __align__(16) float sq[NW][GT][D];
  __shared__ __align__(16) float sp[NW][GT][KS];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const Work wk = plan_steps<KS>(p);
  if (wk.piece < 0) return;
  Cursor cc = wk.c;
  uint8_t* ring_p = smem + (size_t)warp * NST * SB;
  const uint32_t ring = tc::smem_u32(ring_p);
  int left = wk.steps, to_copy = left;
  Copier<float, D> cp;
  cp.start(p, cc);
  uint32_t put = 0, take = 0;
  auto issue = [&]() {
    if (to_copy > 0) {
      cp.copy(p, ring + put);
      if (--to_copy > 0) cp.next(p);
      put = put + SB == NST * SB ? 0 : put + SB;
    }
    cp_commit();
  };
  for (int i = 0; i < NST - 1; ++i) issue();

  float o[GT][DV], m[GT], l[GT], slope[GT];
  bool fresh = true, whole = false;
  int slot = 2 * wk.piece, h0 = 0, nrow = 0;
  const int key = lane % KS, part = lane / KS;
  const float c = p.scale * kLog2e;
  for (; left > 0; --left) {
    if (fresh) {
      fresh = false;
      whole = cc.s == cc.z.s0;
      const int h = cc.u / p.tiles;
      h0 = h * p.G + (cc.u % p.tiles) * p.rows;
      nrow = min(p.rows, h * p.G + p.G - h0);
      const float* q = static_cast<const float*>(p.q) + (int64_t)cc.b * p.sq_b + (int64_t)h0 * p.sq_h;
      float x[GT][D / 32];                 // all loads before the first store
#pragma unroll
      for (int a = 0; a < GT; ++a) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) x[a][i] = a < nrow ? q[(int64_t)a * p.sq_h + i * 32 + lane] : 0.f;
        slope[a] = (p.slopes != nullptr && a < nrow) ? p.slopes[h0 + a] : 0.f;
        m[a] = -INFINITY;
        l[a] = 0.f;
#pragma unroll
        for (int i = 0; i < DV; ++i) o[a][i] = 0.f;
      }
      __syncwarp();
#pragma unroll
      for (int a = 0; a < GT; ++a)
#pragma unroll
        for (int i = 0; i < D / 32; ++i) sq[warp][a][i * 32 + lane] = x[a][i];
    }
    cp_wait<NST - 2>();
    __syncwarp();
    const uint8_t* st = ring_p + take;
    take = take + SB == NST * SB ? 0 : take + SB;
    issue();

    float s[GT];
#pragma unroll
    for (int a = 0; a < GT; ++a) s[a] = 0.f;
#pragma unroll 4
    for (int i = 0; i < D / 4 / PARTS; ++i) {
      const int ch = i * PARTS + part;
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
#pragma unroll
      for (int i = KS; i < 32; i <<= 1) s[a] += __shfl_xor_sync(0xffffffffu, s[a], i);
      s[a] = p.modified ? modified_score<true>(p, s[a] * p.scale, n, cc.z, slope[a]) : s[a] * c;
      if (n < cc.z.lo || n >= cc.z.len) s[a] = -INFINITY;
      float mx = s[a];
#pragma unroll
      for (int i = 1; i < KS; i <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, i));
      const float mn = fmaxf(m[a], mx);
      // the maximum ignores NaN, the probabilities must not: with nothing but hidden and NaN scores so far, 0 is
      // subtracted, and a NaN reaches the sum and the output
      const float mu = mn == -INFINITY ? 0.f : mn;
      const float al = exp2f(m[a] - mu);
      const float pv = exp2f(s[a] - mu);
      m[a] = mn;
      l[a] = l[a] * al + pv;            // this lane's key; joined at the end of the unit
#pragma unroll
      for (int i = 0; i < DV; ++i) o[a][i] *= al;
      if (part == 0) sp[warp][a][key] = pv;
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
    if (unit_end || left == 1) {
      const bool direct = whole && unit_end;
#pragma unroll
      for (int a = 0; a < GT; ++a) {
        float lt = l[a];
#pragma unroll
        for (int i = 1; i < KS; i <<= 1) lt += __shfl_xor_sync(0xffffffffu, lt, i);
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
      slot = 2 * wk.piece + 1;
      fresh = true;
    }
    __syncwarp();
    if (left > 1) advance<KS>(p, cc);
  }
  cp_wait<0>();
}

// ---------------------------------------------------------------------------------------- join
// Adds the partials of each (sequence, query head), in worker order: join_warps warps take every
// join_warps-th one of a row's partials, eight at a time (their sums and outputs are loaded together),
// and the first adds up the warps' results. Units that one piece held whole are already written; rows
// without a visible key become 0 (lse -inf).
template <typename T, int D>
__global__ void __launch_bounds__(JOIN_NT) decode_join_kernel(const Params p) {
  constexpr int DV = D / 32, NB = 8, KS = step_keys<T, D>();
  __shared__ float part[JOIN_NT / 32][D];
  __shared__ float2 part_ml[JOIN_NT / 32];
  __shared__ int64_t sums[JOIN_NT + 1], wsum[JOIN_NT / 32];
  // which partials: from the lengths alone, while the workers still run
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = scan_steps<KS, JOIN_NT>(p, sums, wsum, false);
  const int jw = p.join_warps, sub = warp % jw;
  const int64_t row = (int64_t)blockIdx.x * (JOIN_NT / 32 / jw) + warp / jw;
  const bool have = row < (int64_t)p.B * p.H_q;
  const int b = have ? (int)(row / p.H_q) : 0, hq = have ? (int)(row % p.H_q) : 0;
  const int units = p.H_kv * p.tiles;
  T* out = static_cast<T*>(p.out) + (int64_t)b * p.so_b + (int64_t)hq * p.so_h;
  int w0 = 0, w1 = 0, first = 0, r = 0;      // pieces of the row's unit
  const Span z = span_of<KS>(p, p.seq_len[b]);
  const int steps = z.s1 - z.s0;
  const bool split = have && steps > 0;
  if (split) {
    int64_t c0 = sums[b / per];
    for (int i = b / per * per; i < b; ++i) {
      const Span y = span_of<KS>(p, p.seq_len[i]);
      c0 += (int64_t)(y.s1 - y.s0) * units;
    }
    const int hr = hq % p.G, u = (hq / p.G) * p.tiles + hr / p.rows;
    r = hr % p.rows;
    const int64_t us = c0 + (int64_t)u * steps;
    const Cut cut(sums[JOIN_NT], p.W, p.ns);
    int64_t begin, last;
    w0 = cut.piece_of(us, begin);
    w1 = cut.piece_of(us + steps - 1, last);
    first = 2 * w0 + (begin == us ? 0 : 1);
  }
  asm volatile("griddepcontrol.wait;" ::: "memory");
  float M = -INFINITY, L = 0.f, acc[DV];
#pragma unroll
  for (int i = 0; i < DV; ++i) acc[i] = 0.f;
  if (split && w0 < w1) {
    for (int wb = w0 + sub; wb <= w1; wb += jw * NB) {
      float2 ml[NB];
      float x[NB][DV];
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const int w = wb + k * jw;
        ml[k] = make_float2(-INFINITY, 0.f);
        if (w <= w1) {
          const int64_t sl = (int64_t)(w == w0 ? first : 2 * w) * p.rows + r;
          ml[k] = *reinterpret_cast<const float2*>(p.ws_ml + sl * 2);
          if constexpr (DV == 4) *reinterpret_cast<float4*>(x[k]) = *reinterpret_cast<const float4*>(p.ws_o + sl * D + lane * 4);
          else *reinterpret_cast<float2*>(x[k]) = *reinterpret_cast<const float2*>(p.ws_o + sl * D + lane * 2);
        } else {
#pragma unroll
          for (int i = 0; i < DV; ++i) x[k][i] = 0.f;
        }
      }
      float mn = M;
#pragma unroll
      for (int k = 0; k < NB; ++k) mn = fmaxf(mn, ml[k].x);
      const float mu = mn == -INFINITY ? 0.f : mn, al = exp2f(M - mu);
      L *= al;
#pragma unroll
      for (int i = 0; i < DV; ++i) acc[i] *= al;
#pragma unroll
      for (int k = 0; k < NB; ++k) {
        const float f = exp2f(ml[k].x - mu);
        L = fmaf(f, ml[k].y, L);
#pragma unroll
        for (int i = 0; i < DV; ++i) acc[i] = fmaf(f, x[k][i], acc[i]);
      }
      M = mn;
    }
  }
  if (jw > 1) {
#pragma unroll
    for (int i = 0; i < DV; ++i) part[warp][lane * DV + i] = acc[i];
    if (lane == 0) part_ml[warp] = make_float2(M, L);
    __syncthreads();
    if (sub != 0) return;
    float mn = M;
    for (int k = 1; k < jw; ++k) mn = fmaxf(mn, part_ml[warp + k].x);
    const float mu = mn == -INFINITY ? 0.f : mn;
    float f = exp2f(M - mu);
    L *= f;
#pragma unroll
    for (int i = 0; i < DV; ++i) acc[i] *= f;
    for (int k = 1; k < jw; ++k) {
      f = exp2f(part_ml[warp + k].x - mu);
      L = fmaf(f, part_ml[warp + k].y, L);
#pragma unroll
      for (int i = 0; i < DV; ++i) acc[i] = fmaf(f, part[warp + k][lane * DV + i], acc[i]);
    }
    M = mn;
  }
  if (!have || (split && w0 == w1)) return;
  const float inv = L == 0.f ? 0.f : 1.f / L;
  T y[DV];
#pragma unroll
  for (int i = 0; i < DV; ++i) y[i] = Elem<T>::from_f(acc[i] * inv);
  if constexpr (DV * sizeof(T) == 16) *reinterpret_cast<uint4*>(out + lane * DV) = *reinterpret_cast<const uint4*>(y);
  else if constexpr (DV * sizeof(T) == 8) *reinterpret_cast<uint2*>(out + lane * DV) = *reinterpret_cast<const uint2*>(y);
  else *reinterpret_cast<uint32_t*>(out + lane * DV) = *reinterpret_cast<const uint32_t*>(y);
  if (p.lse != nullptr && lane == 0) p.lse[row] = lse_of(M, L);
}

}  // namespace pdec
}  // namespace cast
