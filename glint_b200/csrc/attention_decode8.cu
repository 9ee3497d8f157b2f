// Attention of single tokens over pages of 8-bit codes (cache8.cu), split evenly over the launch.
//
// Memory-bound work: 2 x head_dim bytes for every key of a (token, kv head) pair, shared by the query heads of its group.
// The pages of all pairs, in order, are one sequence; block b of two per SM takes units [b W, (b + 1) W) of it,
// whatever pairs they belong to (a unit is a page; every pair is preceded by `pair_cost` empty units that stand for
// what a pair costs a block beside its pages).  Every block finds W and where it begins by itself, from the
// positions: no launch goes before this one.  The warps take the block's pages in turn; each fills its own stages of a
// ring in shared memory (TMA boxes with the 128-byte swizzle, completion on an mbarrier) as soon as it has read them:
// one producer warp for all cannot issue pages of 4 KB fast enough.  A pair that lies inside one block is finished
// there; of a shared pair every block leaves a partial result in a workspace and the last one to arrive adds them up,
// in block order.
//
// Per 16 keys: scores^T = K q^T with mma.sync m16n8k32 over the codes themselves, in which N (8) holds the query heads of
// the group.  Queries become 16-bit integers (a power of two brings the largest element below 2^15: a bfloat16 query
// is then exact down to 2^-7 of it, and off by at most 2^-15 of it below), whose upper and lower bytes are two B operands;
// the products are exact integers, -127.5 sum(q) brings the codes' middle in, and the result becomes 32-bit float.
// out^T += V^T p^T with m16n8k16 in half precision: a byte permutation puts a code under an exponent of 2^10 and one
// subtraction gives c - 128, both exact; the half that a code stands above c - 128 enters at the end as 0.5 sum(p).
// A page's key scale multiplies its scores; its value scale goes into the probabilities (times 64, rounded to the 11
// bits of a half) as its ratio to a reference scale, which the accumulators follow when the ratio leaves [1/8, 8].
// Scores, soft cap, maxima, sums and accumulators are 32-bit.
//
// 64 requests of about 2,200 keys, 16 heads in 8 groups of 256: 581 MB of codes in 102 us = 5.7 TB/s, 0.87 of a copy's
// rate; one request of 2,000 keys 9.5 us, nearly all of it round trips (where a block begins, its pages' numbers, scales, the
// pages, the meeting of the parts), of which the first two pass under the kernel in front.  They do so only where the step's
// arrays come by copies: behind a kernel that may have written them, 103 and 11.1 us.
// Score = (q.k) * multiplier, then cap * tanh(score / cap); keys from max(0, pos - window + 1) to pos.
//
// No key is masked by zeroing values: codes are finite whatever bytes an unwritten row holds, and so is what
// the producer passes on as a scale (a page that is not finite gets NaN keys and finite values).
#include <cuda_fp16.h>

#include "common.cuh"
#include "tcgen05.cuh"

namespace glint {

// Measured, 64 requests of 2,200 keys in 8 groups of 256 / 16 of 4,200 keys in 16 groups of 128: 6 warps 101 / 54 us, 5 warps
// 101 / 60, 4 warps 100 / 64, 8 warps (whose registers spill) 123 / 54.
constexpr int D8_WARPS = 6;
constexpr int D8_THREADS = D8_WARPS * 32;
constexpr int D8_MAX_STAGES = 24;                 // a multiple of the warps (see the kernel)
constexpr int D8_CHUNK = 128;                     // pages looked up at a time
constexpr int D8_BLOCK_SMEM = 113 * 1024;         // of an SM's 228 KB: two blocks with 1 KB each of the system's
constexpr int D8_HEADS = 8;                       // query heads of a pair (the MMA's N); larger groups are several pairs
constexpr long long D8_BRIEF = 768 * 1024;        // bytes of a block's codes below which ...
constexpr long long D8_BRIEF_FLIGHT = 48 * 1024;  // ... so many of them are in flight
constexpr int D8_ROW = 128;                       // bytes of a swizzled row
constexpr int D8_MAX_TOKENS = 1024;               // of a launch
constexpr float D8_P_BASE = 64.f;                 // probabilities are multiplied by this before they become halves

struct Decode8Params {
  const __nv_bfloat16* q;       // [T][nh][hd]
  const int* positions;
  const int* token_seq;
  const int* block_table;
  const float* k_scale;         // [pages][kv heads]
  const float* v_scale;
  __nv_bfloat16* out;
  float* partials;              // [blocks][2][8][hd + 4]: a block's first pair (begun by another block) and its last
  int* arrive;                  // [pairs]: blocks that have left their part; back at 0 after the launch
  int* status;
  float multiplier, cap;
  int T, nh, nkv, hd, groups, page_size, splits, num_pages, max_pages, window, stages, whole_page, pair_cost, min_units;
  int early;                    // positions, requests and tables are no kernel's work: read before the wait
};

// Rows that a block reads: the first of them in the pools (-1: none), their scales.
struct Decode8Entry {
  int row;
  float ks, vs;
};

struct Decode8Shared {
  uint64_t full[D8_MAX_STAGES];
  Decode8Entry entry[2][D8_CHUNK];
  int walk[6];                  // where the last lookup ended
  int abort_flag;
  int last_one;
};

__device__ __forceinline__ void d8_mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// codes times the upper (signed) and lower (unsigned) bytes of 16-bit queries
__device__ __forceinline__ void d8_mma_hi(int* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void d8_mma_lo(int* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void d8_ldsm(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void d8_ldsm_trans(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ uint32_t d8_transpose(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t d8_pack(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// Bytes B0, B1 (0..3) of w as the halves c - 128: 0x6400 | c is 1024 + c.
template <int B0, int B1>
__device__ __forceinline__ uint32_t d8_halves(uint32_t w) {
  const uint32_t raised = __byte_perm(w, 0x64646464u, B0 | (4 << 4) | (B1 << 8) | (4 << 12));
  const __half2 v = __hsub2(*reinterpret_cast<const __half2*>(&raised), __half2half2(__ushort_as_half(0x6480)));   // 1152
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float d8_exp2(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float d8_rcp(float x) {
  float y;
  asm("rcp.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float d8_inverse(float power_of_two) { return __int_as_float((254 << 23) - __float_as_int(power_of_two)); }

struct Decode8Segment {
  int first, page_lo, pages;    // of a token: first key, first page, pages
};
// `last`: the last page that the block table has room for.  A position outside it is held to it here (units stay
// positive and bounded) and reported once, by d8_outside.
__device__ __forceinline__ Decode8Segment d8_segment(int pos, int window, int page_size, int last) {
  Decode8Segment s;
  pos = max(pos, 0);
  s.first = (window > 0 && pos - window + 1 > 0) ? pos - window + 1 : 0;
  s.page_lo = min(s.first / page_size, last);
  s.pages = min(pos / page_size, last) - s.page_lo + 1;
  return s;
}
__device__ __forceinline__ bool d8_outside(int pos, int page_size, int last) { return pos < 0 || pos / page_size > last; }

// What a warp has of a pair so far.
template <int HD>
struct Decode8State {
  float o[HD / 16][4];          // sums of (c - 128) p'' in units of `ref`
  float m[2], l[2], lp[2];      // heads 2 tq, 2 tq + 1: reference of the exponents (log2; within 4 of the maximum), sums of
                                // p and of p'' (this thread's keys only)
  float ref;                    // 1 / the value scale that o counts in (0: nothing yet)
};

// A pair's queries as this thread's part of the B operand: per 32 dims, the upper and lower bytes of dims
// 4 tq .. 4 tq + 3 and 16 + 4 tq .. of head g.
template <int HD>
struct Decode8Query {
  uint32_t hi[HD / 32][2], lo[HD / 32][2];
  int start[2];                 // heads 2 tq, 2 tq + 1: -128 sum(q)
  float half[2];                // sum(q) / 2
  float scale[2];               // of a score, without the page's scale
};

// One page of a stage; kaddr, vaddr: where this lane's rows of 16-byte chunks for ldmatrix begin.
template <int HD, bool FULL>
__device__ __forceinline__ void d8_page(Decode8State<HD>& st, const Decode8Query<HD>& qy, uint32_t kaddr, uint32_t vaddr,
                                        float ks, float vs, int page_key0, int pos, int first, int page_size, int hd,
                                        uint32_t sub_bytes, float cap2, int lane) {
  const int g = lane >> 2;
  // The page's value scale against the one that o counts in (the same in all lanes).  Upwards o follows all the way;
  // downwards by 2^64 at most, so that it cannot overflow: what a page 2^67 smaller still adds is nothing.
  if (st.ref == 0.f) st.ref = d8_inverse(vs);
  float ratio = vs * st.ref;
  for (int i = 0; ratio > 8.f || (i == 0 && ratio < 0.125f); ++i) {
    const int d = max(-64, min(64, 254 - ((__float_as_int(st.ref) >> 23) & 255) - ((__float_as_int(vs) >> 23) & 255)));
    const float f = __int_as_float((127 + d) << 23);
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) st.o[i][j] *= f;
    }
    st.lp[0] *= f;
    st.lp[1] *= f;
    st.ref *= f;
    ratio = vs * st.ref;
  }
  const float pscale = D8_P_BASE * ratio;
  const float f0 = qy.scale[0] * ks, f1 = qy.scale[1] * ks;
  for (int key0 = page_key0; key0 < page_key0 + page_size; key0 += 16, kaddr += 16 * D8_ROW, vaddr += 16 * D8_ROW) {
    if (key0 > pos || key0 + 15 < first) continue;             // the whole tile is masked
    int hi[4] = {0, 0, 0, 0}, lo[4] = {qy.start[0], qy.start[1], qy.start[0], qy.start[1]};
#pragma unroll
    for (int s = 0; s < HD / 32; ++s) {
      if (FULL || s * 32 < hd) {
        uint32_t a[4];
        d8_ldsm(a, (kaddr + (s >> 2) * sub_bytes) ^ ((s & 3) << 5));
        d8_mma_hi(hi, a, qy.hi[s][0], qy.hi[s][1]);
        d8_mma_lo(lo, a, qy.lo[s][0], qy.lo[s][1]);
      }
    }
    // [h]: key g, head 2 tq + h;  [2 + h]: key g + 8.  In log2 units; with a cap the scale holds 2 log2(e) / cap, and
    // tanh(y) = 1 - 2 / (1 + 2^(2 y log2 e)).
    float x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = ((float)(hi[i] * 256 + lo[i]) + qy.half[i & 1]) * ((i & 1) ? f1 : f0);
      if (cap2 > 0.f) x[i] = fmaf(-2.f * cap2, d8_rcp(1.f + d8_exp2(x[i])), cap2);
    }
    if (key0 < first || key0 + 15 > pos) {
      const bool va = key0 + g >= first && key0 + g <= pos, vb = key0 + g + 8 >= first && key0 + g + 8 <= pos;
      x[0] = va ? x[0] : -INFINITY;
      x[1] = va ? x[1] : -INFINITY;
      x[2] = vb ? x[2] : -INFINITY;
      x[3] = vb ? x[3] : -INFINITY;
    }
    // the exponents' reference follows the maximum only when that has grown by more than 4 (p is then at most 16)
    float t0 = fmaxf(x[0], x[2]), t1 = fmaxf(x[1], x[3]);
    if (__any_sync(0xffffffffu, t0 > st.m[0] + 4.f || t1 > st.m[1] + 4.f)) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, o));
        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, o));
      }
      const float n0 = fmaxf(st.m[0], t0), n1 = fmaxf(st.m[1], t1);
      const float c0 = st.m[0] == -INFINITY ? 0.f : d8_exp2(st.m[0] - n0), c1 = st.m[1] == -INFINITY ? 0.f : d8_exp2(st.m[1] - n1);
      st.m[0] = n0;
      st.m[1] = n1;
      st.l[0] *= c0; st.l[1] *= c1;
      st.lp[0] *= c0; st.lp[1] *= c1;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        st.o[i][0] *= c0;
        st.o[i][1] *= c1;
        st.o[i][2] *= c0;
        st.o[i][3] *= c1;
      }
    }
    const float base0 = st.m[0] == -INFINITY ? 0.f : st.m[0], base1 = st.m[1] == -INFINITY ? 0.f : st.m[1];
    const float p0 = d8_exp2(x[0] - base0), p1 = d8_exp2(x[1] - base1), p2 = d8_exp2(x[2] - base0), p3 = d8_exp2(x[3] - base1);
    st.l[0] += p0 + p2;
    st.l[1] += p1 + p3;
    st.lp[0] = fmaf(p0 + p2, pscale, st.lp[0]);
    st.lp[1] = fmaf(p1 + p3, pscale, st.lp[1]);
    // p''^T as the B operand: keys 2 tq, 2 tq + 1 (and + 8) of head g, by an 8x8 transpose in the warp
    const uint32_t b0 = d8_transpose(d8_pack(p0 * pscale, p1 * pscale)), b1 = d8_transpose(d8_pack(p2 * pscale, p3 * pscale));
    // values: the transposed load of 16-bit units gives dims (2 g, 2 g + 1) of keys 2 tq, 2 tq + 1; rows g and g + 8 of
    // the tile over a chunk of 16 dims are its dims 2 g and 2 g + 1
#pragma unroll
    for (int s = 0; s < HD / 32; ++s) {
      if (FULL || s * 32 < hd) {
        uint32_t a[4];
        d8_ldsm_trans(a, (vaddr + (s >> 2) * sub_bytes) ^ ((s & 3) << 5));
        d8_mma(st.o[2 * s], d8_halves<0, 2>(a[0]), d8_halves<1, 3>(a[0]), d8_halves<0, 2>(a[1]), d8_halves<1, 3>(a[1]), b0, b1);
        d8_mma(st.o[2 * s + 1], d8_halves<0, 2>(a[2]), d8_halves<1, 3>(a[2]), d8_halves<0, 2>(a[3]), d8_halves<1, 3>(a[3]), b0, b1);
      }
    }
  }
}

// Four output elements: sums over the sum of the probabilities.
__device__ __forceinline__ void d8_store(__nv_bfloat16* out, float4 acc, float L) {
  const float inv = L == 0.f ? 0.f : 1.f / L;
  const __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), hi = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
  *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}

// HD: register capacity (head_dim <= HD; head_dim and page_size are multiples of 16).
// FULL: head_dim is HD, no step is asked for (64 requests of 2,200 keys, heads of 256: 101 against 102 us; 16 of 4,200, heads
// of 128: 54 against 60).
template <int HD, bool FULL>
__global__ void __launch_bounds__(D8_THREADS, 2)
attention_decode8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                         const Decode8Params p) {
  extern __shared__ uint8_t d8_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(d8_raw) + 1023) & ~(uintptr_t)1023);
  const int hd = FULL ? HD : p.hd, G = p.nh / p.nkv;
  const int pairs = p.nkv * p.groups;                          // pairs of a token: (kv head, up to 8 query heads)
  const int nsub = (hd + 127) >> 7;
  const uint32_t sub_bytes = (uint32_t)p.page_size * D8_ROW;
  const uint32_t page_bytes = nsub * sub_bytes;
  const int stride_f = hd + 4;                                 // floats of a partial result: values, maximum, sum
  const int HP = G < D8_HEADS ? G : D8_HEADS;
  float* merge = reinterpret_cast<float*>(ring + (size_t)p.stages * 2 * page_bytes);      // [warps][HP][hd + 4]
  Decode8Shared* sh = reinterpret_cast<Decode8Shared*>(merge + (size_t)D8_WARPS * HP * stride_f);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &sh->abort_flag;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) tc::mbar_init(&sh->full[s], 1);
    sh->abort_flag = 0;
    tc::fence_barrier_init();
    tc::tma_prefetch_desc(&map_k);
    tc::tma_prefetch_desc(&map_v);
  }
  // ---- where this block begins: every warp scans the tokens' units for itself, some consecutive tokens per lane.  Where
  // positions, requests and block tables come by copies, all this passes under the kernel in front. ---------------------
  if (!p.early) pdl_wait();
  const int per = (p.T + 31) >> 5;
  const int r0 = min(lane * per, p.T), r1 = min(r0 + per, p.T);
  int mine = 0, row_first = 0;
  if (r0 < r1) row_first = p.token_seq[r0];
  const int last_page = p.max_pages * p.splits - 1;
  for (int r = r0; r < r1; ++r) {
    const int at = p.positions[r];
    if (d8_outside(at, p.page_size, last_page)) atomicExch(p.status, 3);
    mine += (p.pair_cost + d8_segment(at, p.window, p.page_size, last_page).pages) * pairs;
  }
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  const int total = __shfl_sync(0xffffffffu, incl, 31);
  const int W = max(p.min_units, (total + (int)gridDim.x - 1) / (int)gridDim.x);
  const long long begin = (long long)blockIdx.x * W;
  if (begin >= total) return;                                  // fewer units than blocks (the same for all threads)
  int t = 0, pos = 0, row = 0, inside = (int)begin - (incl - mine);
  const bool owner = inside >= 0 && inside < mine;             // one lane of the warp
  if (owner) {
    t = r0;
    row = row_first;
    for (;; ++t) {
      pos = p.positions[t];
      const int u = (p.pair_cost + d8_segment(pos, p.window, p.page_size, last_page).pages) * pairs;
      if (inside < u) break;
      inside -= u;
    }
    if (t > r0) row = p.token_seq[t];
  }
  const int who = __ffs(__ballot_sync(0xffffffffu, owner)) - 1;
  t = __shfl_sync(0xffffffffu, t, who);
  pos = __shfl_sync(0xffffffffu, pos, who);
  row = __shfl_sync(0xffffffffu, row, who);
  inside = __shfl_sync(0xffffffffu, inside, who);
  int remaining = min(W, total - (int)begin);                  // units
  Decode8Segment sg = d8_segment(pos, p.window, p.page_size, last_page);
  int pair = inside / (p.pair_cost + sg.pages);
  int voff = inside - pair * (p.pair_cost + sg.pages);

  // ---- the block's pages are looked up 128 at a time, one by a thread, into one of two halves of `entry`: chunk c + 1
  // when the block is in the middle of chunk c.  The walk over the pairs goes on where the last lookup ended. ------------
  auto look_up = [&](int half, int wt, int wpos, int wrow, int wpair, int woff, int wleft) -> int {
    int at = -1, first_row = -1;                               // place of this thread's page in the scales, -1: none
    const int i = threadIdx.x;
    for (int i0 = 0; i0 < D8_CHUNK && wleft > 0 && wt < p.T;) {           // the same walk in all threads, pair by pair
      const Decode8Segment ws = d8_segment(wpos, p.window, p.page_size, last_page);
      const int skipped = max(woff, p.pair_cost) - woff;       // empty units
      const int off = woff + skipped - p.pair_cost;            // first page of this pair here
      const int n = max(0, min(D8_CHUNK - i0, min(wleft - skipped, ws.pages - off)));
      if (i >= i0 && i < i0 + n) {
        const int unit = ws.page_lo + off + i - i0, place = unit / p.splits;
        int page = place < p.max_pages ? p.block_table[(size_t)wrow * p.max_pages + place] : -1;
        if (page < 0 || page >= p.num_pages) {                 // never read outside the pool; report it
          atomicExch(p.status, 3);
          page = 0;
        }
        at = page * p.nkv + wpair / p.groups;
        first_row = at * (p.page_size * p.splits) + (unit - place * p.splits) * p.page_size;
      }
      i0 += n;
      wleft -= skipped + n;
      woff += skipped + n;
      if (woff >= p.pair_cost + ws.pages) {
        woff = 0;
        if (++wpair == pairs) {
          wpair = 0;
          if (++wt < p.T && wleft > 0) {
            wpos = p.positions[wt];
            wrow = p.token_seq[wt];
          }
        }
      }
    }
    if (i < D8_CHUNK) sh->entry[half][i].row = first_row;
    if (i == 0) {
      sh->walk[0] = wt; sh->walk[1] = wpos; sh->walk[2] = wrow;
      sh->walk[3] = wpair; sh->walk[4] = woff; sh->walk[5] = wleft;
    }
    return at;
  };
  // Copies page i of the block into stage s: called by the warp whose page it is, which has read what was there before.
  auto fetch = [&](int i, int s) {
    const int first_row = sh->entry[(i / D8_CHUNK) & 1][i & (D8_CHUNK - 1)].row;
    if (first_row >= 0 && tc::elect_one()) {
      uint8_t* kdst = ring + (size_t)s * 2 * page_bytes;
      tc::mbar_expect_tx(&sh->full[s], 2 * page_bytes);
      if (p.whole_page) {
        tc::tma_load_3d(kdst, &map_k, &sh->full[s], 0, first_row, 0);
        tc::tma_load_3d(kdst + page_bytes, &map_v, &sh->full[s], 0, first_row, 0);
      } else {
        for (int sub = 0; sub < nsub; ++sub) {
          tc::tma_load_2d(kdst + sub * sub_bytes, &map_k, &sh->full[s], sub * 128, first_row);
          tc::tma_load_2d(kdst + page_bytes + sub * sub_bytes, &map_v, &sh->full[s], sub * 128, first_row);
        }
      }
    }
  };
  // The first pages' scales are requested before their copies: behind the burst of all blocks' first copies they would
  // arrive 5 us later.
  {
    const int at = look_up(0, t, pos, row, pair, voff, remaining);
    pdl_wait_release();
    const float ks = at >= 0 ? p.k_scale[at] : 0.f, vs = at >= 0 ? p.v_scale[at] : 1.f;
    __syncthreads();
    for (int s = warp; s < p.stages; s += D8_WARPS) fetch(s, s);          // a stage is always the same warp's
    if (at >= 0) {
      sh->entry[0][threadIdx.x].ks = ks;
      sh->entry[0][threadIdx.x].vs = vs;
    }
  }
  bool looked_up = false;                                      // by all threads: a barrier away

  const int g = lane >> 2, tq = lane & 3;
  const float LOG2E = 1.4426950408889634f;
  const float cap2 = p.cap > 0.f ? p.cap * LOG2E : 0.f;
  const float score_scale = p.cap > 0.f ? 2.f * LOG2E * p.multiplier / p.cap : p.multiplier * LOG2E;
  // for ldmatrix, lane 8 i + r gives row r + 8 (i mod 2) of 16 keys and chunk i / 2 of 32 dims; further chunks are an
  // exclusive or away (128-byte swizzle: chunk c of row r sits at c ^ (r mod 8))
  const uint32_t lane_addr = tc::smem_u32(ring) + (uint32_t)((lane & 7) + ((lane >> 3) & 1) * 8) * D8_ROW +
                             (uint32_t)(((lane >> 4) ^ (lane & 7)) << 4);
  int it = warp, stage = warp, phase = 0, it0 = 0;              // this warp's next page of the block; the pair's first
  int cursor = (int)begin;
  while (remaining > 0 && t < p.T) {
    const int units = min(remaining, p.pair_cost + sg.pages - voff);
    const int off = max(voff, p.pair_cost) - p.pair_cost;
    const int n = max(0, voff + units - p.pair_cost - off);
    const int pair_begin = cursor - voff + p.pair_cost;         // the pair's first page in the launch's sequence
    cursor += units;
    remaining -= units;
    voff = 0;
    if (n > 0) {
      const int kvh = pair / p.groups, h0 = (pair - kvh * p.groups) * D8_HEADS;   // of the group: first head
      const int H = min(G - h0, D8_HEADS);
      const bool begins = off == 0, ends = off + n == sg.pages;
      Decode8Query<HD> qy;
      {
        const __nv_bfloat16* qrow = p.q + ((size_t)t * p.nh + kvh * G + h0 + (g < H ? g : 0)) * hd;
        uint2 raw[HD / 32][2];
#pragma unroll
        for (int s = 0; s < HD / 32; ++s)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            raw[s][j] = make_uint2(0, 0);
            if ((FULL || s * 32 + j * 16 < hd) && g < H) raw[s][j] = *reinterpret_cast<const uint2*>(qrow + s * 32 + j * 16 + tq * 4);
          }
        unsigned top = 0;
#pragma unroll
        for (int s = 0; s < HD / 32; ++s)
#pragma unroll
          for (int j = 0; j < 2; ++j) top = __vmaxu2(top, __vmaxu2(raw[s][j].x & 0x7fff7fffu, raw[s][j].y & 0x7fff7fffu));
        top = max(top & 0xffffu, top >> 16);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^-e brings the largest element below 2^15; e is held where both powers are normal numbers
        const int e = max(-100, min(113, (int)(top >> 7) - 127 - 14));
        const float down = __int_as_float((127 - e) << 23);
#pragma unroll
        for (int s = 0; s < HD / 32; ++s)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            // x + 1.5 * 2^23 holds the rounded integer in its low bits
            const float magic = 12582912.f;
            const uint32_t v0 = __float_as_uint(fmaf(__uint_as_float(raw[s][j].x << 16), down, magic));
            const uint32_t v1 = __float_as_uint(fmaf(__uint_as_float(raw[s][j].x & 0xffff0000u), down, magic));
            const uint32_t v2 = __float_as_uint(fmaf(__uint_as_float(raw[s][j].y << 16), down, magic));
            const uint32_t v3 = __float_as_uint(fmaf(__uint_as_float(raw[s][j].y & 0xffff0000u), down, magic));
            const uint32_t w01 = __byte_perm(v0, v1, 0x5410), w23 = __byte_perm(v2, v3, 0x5410);
            qy.lo[s][j] = __byte_perm(w01, w23, 0x6420);
            qy.hi[s][j] = __byte_perm(w01, w23, 0x7531);
          }
        // sum(q) of every head, by a product with rows of ones: it arrives in the lanes that need it
        const uint32_t ones[4] = {0x01010101u, 0x01010101u, 0x01010101u, 0x01010101u};
        int sh_[4] = {0, 0, 0, 0}, sl_[4] = {0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < HD / 32; ++s) {
          d8_mma_hi(sh_, ones, qy.hi[s][0], qy.hi[s][1]);
          d8_mma_lo(sl_, ones, qy.lo[s][0], qy.lo[s][1]);
        }
        // a query that is not finite makes its scores NaN
        const float up = top < 0x7f80u ? __int_as_float((127 + e) << 23) : __int_as_float(0x7fc00000);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int sum = sh_[h] * 256 + sl_[h];
          qy.start[h] = -128 * sum;
          qy.half[h] = 0.5f * (float)sum;
          qy.scale[h] = score_scale * __shfl_sync(0xffffffffu, up, (2 * tq + h) * 4);
        }
      }
      Decode8State<HD> st;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) st.o[i][0] = st.o[i][1] = st.o[i][2] = st.o[i][3] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        st.m[h] = -INFINITY;
        st.l[h] = st.lp[h] = 0.f;
      }
      st.ref = 0.f;
      if (!looked_up) {
        __syncthreads();
        looked_up = true;
      }
      // Page `it` of the block belongs to warp it % warps and stage it % stages (a multiple of them: a stage is always
      // filled and read by the same warp, which therefore sees every phase of the stage's barrier).
      for (int done = it0; done < it0 + n;) {
        if ((done & (D8_CHUNK - 1)) == D8_CHUNK / 2) {         // all warps have left the chunk before
          __syncthreads();
          const int half = (done / D8_CHUNK + 1) & 1;
          const int* w = sh->walk;
          const int w0 = w[0], w1 = w[1], w2 = w[2], w3 = w[3], w4 = w[4], w5 = w[5];
          __syncthreads();                                     // all have read where to go on
          const int at = look_up(half, w0, w1, w2, w3, w4, w5);
          if (at >= 0) {
            sh->entry[half][threadIdx.x].ks = p.k_scale[at];
            sh->entry[half][threadIdx.x].vs = p.v_scale[at];
          }
          __syncthreads();
        }
        done = min(it0 + n, ((done + D8_CHUNK / 2) & ~(D8_CHUNK - 1)) + D8_CHUNK / 2);
        for (; it < done; it += D8_WARPS) {
          const Decode8Entry& en = sh->entry[(it / D8_CHUNK) & 1][it & (D8_CHUNK - 1)];
          float ks = en.ks, vs = en.vs;
          if (!(fabsf(vs) <= 3.4e38f)) {                        // not finite: the keys say so, the values stay finite
            ks = __int_as_float(0x7fc00000);
            vs = 1.f;
          }
          if (vs == 0.f) vs = 7.5231638e-37f;                   // 2^-120: a page that nothing was written to
          if (__all_sync(0xffffffffu, tc::mbar_wait(&sh->full[stage], phase, abort_flag))) {   // together: what follows is .aligned
            const uint32_t kaddr = lane_addr + (uint32_t)stage * 2 * page_bytes;
            d8_page<HD, FULL>(st, qy, kaddr, kaddr + page_bytes, ks, vs, (sg.page_lo + off + it - it0) * p.page_size, pos, sg.first,
                              p.page_size, hd, sub_bytes, cap2, lane);
            __syncwarp();
            fetch(it + p.stages, stage);
          }
          stage += D8_WARPS;
          if (stage >= p.stages) {
            stage -= p.stages;
            phase ^= 1;
          }
        }
      }
      it0 += n;
      // ---- this warp's totals; the warps are merged in shared memory, in warp order ------------------------------
      const float unit = st.ref == 0.f ? 0.f : d8_inverse(st.ref) * (1.f / D8_P_BASE);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          st.l[h] += __shfl_xor_sync(0xffffffffu, st.l[h], o);
          st.lp[h] += __shfl_xor_sync(0xffffffffu, st.lp[h], o);
        }
        const int head = 2 * tq + h;
        if (head < H) {
          float* dst = merge + ((size_t)warp * HP + head) * stride_f;
          const float half = 0.5f * st.lp[h];
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            const int d = i * 16 + 2 * g;
            if (FULL || d < hd) *reinterpret_cast<float2*>(dst + d) = make_float2((st.o[i][h] + half) * unit, (st.o[i][2 + h] + half) * unit);
          }
          if (g == 0) *reinterpret_cast<float2*>(dst + hd) = make_float2(st.m[h], st.l[h]);
        }
      }
      __syncthreads();
      const bool whole = begins && ends;
      float* partial = p.partials + ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * HP * stride_f;
      __nv_bfloat16* out = p.out + ((size_t)t * p.nh + kvh * G + h0) * hd;
      const int quads = hd >> 2;
      for (int e = threadIdx.x; e < H * quads; e += D8_THREADS) {
        const int j = e / quads, d = (e - j * quads) * 4;
        const float* part = merge + (size_t)j * stride_f;
        float2 ml[D8_WARPS];
        float M = -INFINITY;
#pragma unroll
        for (int wv = 0; wv < D8_WARPS; ++wv) {
          ml[wv] = *reinterpret_cast<const float2*>(part + (size_t)wv * HP * stride_f + hd);
          M = fmaxf(M, ml[wv].x);
        }
        float L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int wv = 0; wv < D8_WARPS; ++wv) {
          // a warp without pages has l = 0; one whose scores were all NaN has no maximum and l = NaN
          const float w = ml[wv].x == -INFINITY ? (ml[wv].y == 0.f ? 0.f : ml[wv].y) : d8_exp2(ml[wv].x - M);
          const float4 v = *reinterpret_cast<const float4*>(part + (size_t)wv * HP * stride_f + d);
          L += ml[wv].y * w;
          acc.x += v.x * w; acc.y += v.y * w; acc.z += v.z * w; acc.w += v.w * w;
        }
        if (whole) {
          d8_store(out + (size_t)j * hd + d, acc, L);
        } else {
          *reinterpret_cast<float4*>(partial + (size_t)j * stride_f + d) = acc;
          if (d == 0) *reinterpret_cast<float2*>(partial + (size_t)j * stride_f + hd) = make_float2(M, L);
        }
      }
      __syncthreads();                                          // the merge area is free, every part of the partial is written
      if (!whole) {
        // ---- the pair is shared: the block that leaves its part last adds the parts up, in block order.  With pages left
        // to do that is warp 0's work (the block whose last pair it is usually arrives later), else all warps'. -----------
        const int b_first = pair_begin / W, parts = (pair_begin + sg.pages - 1) / W - b_first + 1;
        const bool all = remaining <= 0;
        if (all || warp == 0) {
          int last = 0;
          if (threadIdx.x == 0) {
            // counted after this block's part is visible, and the others' parts are visible to the one that counts last
            int* counter = p.arrive + (size_t)t * pairs + pair;
            int seen;
            asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(seen) : "l"(counter) : "memory");
            last = seen == parts - 1;
            if (last) *counter = 0;                             // for the next launch
            if (all) sh->last_one = last;
          }
          if (all) __syncthreads();
          last = all ? sh->last_one : __shfl_sync(0xffffffffu, last, 0);
          __syncwarp();
          const int step = all ? D8_THREADS : 32;
          for (int e = threadIdx.x; last && e < H * quads; e += step) {
            const int j = e / quads, d = (e - j * quads) * 4;
            float M = -INFINITY, L = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i0 = 0; i0 < parts; i0 += 8) {             // up to eight parts in flight
              float2 ml[8];
              float4 v[8];
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const int bk = b_first + i0 + k;
                ml[k] = make_float2(-INFINITY, 0.f);
                v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (i0 + k < parts) {
                  const float* from = p.partials + (((size_t)bk * 2 + (bk == b_first ? 1 : 0)) * HP + j) * stride_f;
                  ml[k] = __ldcg(reinterpret_cast<const float2*>(from + hd));
                  v[k] = __ldcg(reinterpret_cast<const float4*>(from + d));
                }
              }
              float top = M;
#pragma unroll
              for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
              const float keep = M == -INFINITY ? (L == 0.f ? 0.f : L) : d8_exp2(M - top);
              L *= keep;
              acc.x *= keep; acc.y *= keep; acc.z *= keep; acc.w *= keep;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float wk = ml[k].x == -INFINITY ? (ml[k].y == 0.f ? 0.f : ml[k].y) : d8_exp2(ml[k].x - top);
                L += ml[k].y * wk;
                acc.x += v[k].x * wk; acc.y += v[k].y * wk; acc.z += v[k].z * wk; acc.w += v[k].w * wk;
              }
              M = top;
            }
            d8_store(out + (size_t)j * hd + d, acc, L);
          }
          __syncwarp();
        }
      }
    }
    if (++pair == pairs) {
      pair = 0;
      if (++t < p.T && remaining > 0) {
        pos = p.positions[t];
        sg = d8_segment(pos, p.window, p.page_size, last_page);
      }
    }
  }
  if (threadIdx.x == 0 && sh->abort_flag) atomicExch(p.status, 4);
}

// ---- host side -------------------------------------------------------------------------------------------------

typedef CUresult (*D8EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                               const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static D8EncodeFn d8_encode_fn() {
  static D8EncodeFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<D8EncodeFn>(ptr);
  }
  return fn;
}

// A pool of codes [pages][kv heads][page_size][head_dim] as rows of head_dim bytes, in boxes of a page's rows x 128
// columns with the 128-byte swizzle; columns past the head arrive as zeros.  When head_dim is a multiple of 128 the slices
// are a third dimension and one box brings a whole page.
static int d8_map(CUtensorMap* map, const void* pool, long long rows, int hd, int page_size, bool whole_page) {
  D8EncodeFn fn = d8_encode_fn();
  if (!fn) return GLINT_ERR_BAD_ARG;
  const cuuint32_t elem[3] = {1, 1, 1};
  if (whole_page) {
    const cuuint64_t dims[3] = {128, (cuuint64_t)rows, (cuuint64_t)(hd / 128)};
    const cuuint64_t strides[2] = {(cuuint64_t)hd, 128};
    const cuuint32_t box[3] = {128, (cuuint32_t)page_size, (cuuint32_t)(hd / 128)};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void*>(pool), dims, strides, box, elem,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? GLINT_OK : GLINT_ERR_BAD_ARG;
  }
  const cuuint64_t dims[2] = {(cuuint64_t)hd, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)hd};
  const cuuint32_t box[2] = {128, (cuuint32_t)page_size};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(pool), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? GLINT_OK : GLINT_ERR_BAD_ARG;
}

}  // namespace glint

using namespace glint;

// Head sizes in steps of 16 up to 256, pages in steps of 16.
GLINT_API int glint_attention_decode8_supported(int nh, int nkv, int hd, int page_size) {
  return nkv > 0 && nh > 0 && nh % nkv == 0 && hd % 16 == 0 && hd >= 16 && hd <= 256 && page_size % 16 == 0 && page_size >= 16 ? 1 : 0;
}

// Workspace of launches over `blocks` blocks: floats of partial results.
GLINT_API long long glint_attention_decode8_workspace(int blocks, int nh, int nkv, int hd) {
  const int G = nh / nkv;
  return (long long)blocks * 2 * (G < D8_HEADS ? G : D8_HEADS) * (hd + 4);
}

// q, out [T][nh][hd] bfloat16, pages of codes with their scales; T single tokens of which none attends more than
// `max_context` keys.  `partials`: glint_attention_decode8_workspace floats, 16-byte aligned; `arrive`: `arrive_ints`
// counters that are zero before the first launch (every launch leaves them zero).  Launches of more tokens than
// the counters or 1024 allow are cut.  `blocks`: at most that many blocks (two per SM).  `early`: positions, requests and
// block tables were on the device before the kernel in front began (copies, not a kernel's results).
GLINT_API int glint_attention_decode8(const void* q, const uint8_t* k_pool, const uint8_t* v_pool, const float* k_scale,
                                      const float* v_scale, const int* positions, const int* token_seq, const int* block_table,
                                      int max_pages, void* out, int T, int nh, int nkv, int hd, int page_size, int num_pages,
                                      float multiplier, float cap, int window, int max_context, int blocks, float* partials,
                                      int* arrive, int arrive_ints, int* status, int early, cudaStream_t stream) {
  if (T <= 0) return GLINT_OK;
  if (!partials || !arrive || blocks < 1 || max_pages < 1 || ((uintptr_t)partials & 15)) return GLINT_ERR_BAD_ARG;
  if (!glint_attention_decode8_supported(nh, nkv, hd, page_size)) return GLINT_ERR_UNSUPPORTED_SIZE;
  if (((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)q | (uintptr_t)out) & 15) return GLINT_ERR_UNSUPPORTED_SIZE;
  const long long rows = (long long)num_pages * nkv * page_size;
  if (rows > 0x7fffffffLL) return GLINT_ERR_UNSUPPORTED_SIZE;
  const int G = nh / nkv, groups = (G + D8_HEADS - 1) / D8_HEADS, pairs = nkv * groups;
  if (pairs > arrive_ints) return GLINT_ERR_UNSUPPORTED_SIZE;
  const int whole_page = hd % 128 == 0 ? 1 : 0;
  const long long fixed = (long long)D8_WARPS * (G < D8_HEADS ? G : D8_HEADS) * (hd + 4) * 4 + sizeof(Decode8Shared) + 1024;
  const long long row_bytes = (hd + 127) / 128 * D8_ROW;
  // A large page is read in parts of 64, 32 or 16 rows, the largest of which two stages per warp let two blocks share an SM
  int part = 64;
  while (part > 16 && (page_size % part || 2 * D8_WARPS * 2 * part * row_bytes + fixed > D8_BLOCK_SMEM)) part >>= 1;
  const int splits = page_size / part;
  page_size = part;
  CUtensorMap map_k, map_v;
  int rc = d8_map(&map_k, k_pool, rows, hd, page_size, whole_page);
  if (rc == GLINT_OK) rc = d8_map(&map_v, v_pool, rows, hd, page_size, whole_page);
  if (rc != GLINT_OK) return rc;
  const long long page_bytes = page_size * row_bytes;
  // What a pair costs a block beside its pages, and the least a block is given, in pages of this size.  Measured, one request
  // of 2,000 keys / 56 uneven ones of up to 4,600 (groups of 256) / 16 of 4,200 (groups of 128), a pair at 96 KB: 9.4 / 95.5 /
  // 54.0 us, at 24 KB 11.0 / 108.5 / 54.1, at 192 KB 9.4 / 94.4 / 58.4.  One request of 200 / 2,000 keys with its append, at
  // least 64 KB a block: 13.3 / 12.1 us, 48 KB 10.4 / 13.2, 96 KB 13.4 / 12.4.
  const long long unit = 2ll * page_size * hd;
  const int pair_cost = (int)((96 * 1024 + unit / 2) / unit) + 1;
  const int min_units = (int)((64 * 1024 + unit - 1) / unit) + 1;
  long long most_pages = ((long long)max_context + page_size - 1) / page_size;
  if (window > 0 && ((long long)window + page_size - 1) / page_size + 1 < most_pages)
    most_pages = ((long long)window + page_size - 1) / page_size + 1;
  // units are counted in 32 bits, whatever the positions turn out to be
  long long table_pages = (long long)max_pages * splits;
  if (table_pages > 0x7fffffffLL) return GLINT_ERR_UNSUPPORTED_SIZE;
  if (window > 0 && ((long long)window + page_size - 1) / page_size + 1 < table_pages)
    table_pages = ((long long)window + page_size - 1) / page_size + 1;
  const long long fits = 0x3fffffffLL / ((long long)pairs * (table_pages + pair_cost));
  if (fits < 1) return GLINT_ERR_UNSUPPORTED_SIZE;
  int step = arrive_ints / pairs < D8_MAX_TOKENS ? arrive_ints / pairs : D8_MAX_TOKENS;
  if (fits < step) step = (int)fits;
  if (step > T) step = T;
  // Shared memory for copies in flight: all of it for launches that stream long, 48 KB where a block has less than 768 KB to
  // read; the kernels on either side then find room beside it.  16 requests of 2,000 keys (16 heads in 8 groups of 256, 444 KB
  // a block) take 35.2 us with 48 KB and 36.8 with 96, 32 of them (886 KB) 57.8 and 56.3; a decode step of the 9B sizes
  // (21 layers) at one request 2.27 and 2.35 ms, at 32 requests 3.66 and 3.58.
  const bool brief = step * pairs * most_pages * unit < blocks * D8_BRIEF;
  long long flight = D8_BLOCK_SMEM - fixed;
  if (brief && flight > D8_BRIEF_FLIGHT) flight = D8_BRIEF_FLIGHT;
  int stages = (int)(flight / (2 * page_bytes * D8_WARPS)) * D8_WARPS;
  if (stages > D8_MAX_STAGES) stages = D8_MAX_STAGES;
  if (stages < D8_WARPS) stages = D8_WARPS;
  const long long smem = stages * 2 * page_bytes + fixed;
  for (int t0 = 0; t0 < T; t0 += step) {
    const int n = T - t0 < step ? T - t0 : step;
    Decode8Params p = {(const __nv_bfloat16*)q + (size_t)t0 * nh * hd, positions + t0, token_seq + t0, block_table, k_scale, v_scale,
                       (__nv_bfloat16*)out + (size_t)t0 * nh * hd, partials, arrive, status, multiplier, cap,
                       n, nh, nkv, hd, groups, page_size, splits, num_pages, max_pages, window, stages, whole_page, pair_cost, min_units,
                       early};
    const long long most = (long long)n * pairs * (most_pages + pair_cost);
    const long long useful = (most + min_units - 1) / min_units;
    const int grid = useful < blocks ? (int)useful : blocks;
#define LAUNCH(HD, FULL)                                                                                            \
  {                                                                                                                 \
    cudaError_t e = cudaFuncSetAttribute(attention_decode8_kernel<HD, FULL>, cudaFuncAttributeMaxDynamicSharedMemorySize, \
                                         (int)smem);                                                                \
    if (e != cudaSuccess) return (int)e;                                                                            \
    e = launch_kernel(attention_decode8_kernel<HD, FULL>, dim3(grid), dim3(D8_THREADS), (size_t)smem, stream, map_k, map_v, p); \
    if (e != cudaSuccess) return (int)e;                                                                            \
  }
    if (hd == 64) LAUNCH(64, true)
    else if (hd == 128) LAUNCH(128, true)
    else if (hd == 256) LAUNCH(256, true)
    else if (hd < 64) LAUNCH(64, false)
    else if (hd < 128) LAUNCH(128, false)
    else LAUNCH(256, false)
#undef LAUNCH
  }
  return (int)cudaGetLastError();
}
