// Attention of single tokens over pages of 8-bit codes (cache8.cu), split evenly over the launch.
//
// Memory-bound work: 2 x head_dim bytes for every key of a (token, kv head) pair, shared by the query heads of its group.
// The pages of all pairs, in order, are one sequence; block b of two per SM takes units [b W, (b + 1) W) of it,
// whatever pairs they belong to (a unit is a page; every pair is preceded by `pair_cost` empty units that stand for
// what a pair costs a block beside its pages).  Every block finds W and where it begins by itself, from the
// positions: no launch goes before this one.  A producer warp streams the pages into a ring of shared-memory stages
// (TMA boxes with the 128-byte swizzle, completion on an mbarrier) with each page's two scales beside them; the
// consumer warps take the pages in turn.  A pair that lies inside one block is finished there; of a shared pair every
// block leaves a partial result in a workspace and the last one to arrive adds them up, in block order.
//
// Per 16 keys: scores^T = K q^T and out^T += V^T p^T with mma.sync m16n8k16 tiles in half precision, in which N
// (8) holds the query heads of the group.  Codes become half-precision integers c - 128 by one byte permutation (the
// byte under an exponent of 2^10) and one subtraction, both exact; the half that a code's middle lies above c - 128
// enters through the accumulators: 0.5 sum(q) for the scores and 0.5 sum(p) for the values.  Queries are scaled by a
// power of two so that their largest element lies in [2^8, 2^9): bfloat16 queries are then exact down to 2^-24 of
// it.  A page's key scale multiplies its scores; its value scale goes into the probabilities (times 2^10, rounded to the
// 11 bits of a half) as its ratio to a reference scale, which the accumulators follow when the ratio leaves
// [2^-5, 2^5].  Scores, soft cap, maxima, sums and accumulators are 32-bit.
// Score = (q.k) * multiplier, then cap * tanh(score / cap); keys from max(0, pos - window + 1) to pos.
//
// No key is masked by zeroing values: codes are finite whatever bytes an unwritten row holds, and so is what
// the producer passes on as a scale (a page that is not finite gets NaN keys and finite values).
#include <cuda_fp16.h>

#include "common.cuh"
#include "tcgen05.cuh"

namespace glint {

constexpr int D8_WARPS = 4;                       // consumer warps; one more warp is the producer
constexpr int D8_THREADS = D8_WARPS * 32 + 32;
constexpr int D8_MAX_STAGES = 12;                 // a multiple of the consumer warps (see the kernel)
constexpr int D8_HEADS = 8;                       // query heads of a pair (the MMA's N); larger groups are several pairs
constexpr int D8_ROW = 128;                       // bytes of a swizzled row
constexpr int D8_MAX_TOKENS = 1024;               // of a launch
constexpr float D8_P_BASE = 1024.f;               // probabilities are multiplied by this before they become halves

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
  int T, nh, nkv, hd, groups, page_size, num_pages, max_pages, window, stages, whole_page, pair_cost, min_units;
};

struct Decode8Shared {
  uint64_t full[D8_MAX_STAGES];
  uint64_t empty[D8_MAX_STAGES];
  float2 scale[D8_MAX_STAGES];  // of the page in the stage: keys, values
  long long warp_sum[D8_THREADS / 32];
  long long total, W;
  int start_token, start_inside;
  int abort_flag;
  int last_one;
};

__device__ __forceinline__ void d8_consumer_sync() { asm volatile("bar.sync 1, %0;" ::"n"(D8_WARPS * 32) : "memory"); }

__device__ __forceinline__ void d8_mma(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
// Bytes b0, b1 of w (0..3) as the halves c - 128: 0x6400 | c is 1024 + c.
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
__device__ __forceinline__ uint4 d8_lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 d8_lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
// Byte offset of a 16-byte chunk of a row in a tile of 128-byte rows with the 128-byte swizzle.
__device__ __forceinline__ uint32_t d8_swz(int row, int chunk) { return (uint32_t)(row * D8_ROW + ((chunk ^ (row & 7)) << 4)); }

struct Decode8Segment {
  int first, page_lo, pages;    // of a token: first key, first page, pages
};
__device__ __forceinline__ Decode8Segment d8_segment(int pos, int window, int page_size) {
  Decode8Segment s;
  s.first = (window > 0 && pos - window + 1 > 0) ? pos - window + 1 : 0;
  s.page_lo = s.first / page_size;
  s.pages = pos / page_size - s.page_lo + 1;
  return s;
}

// What a warp has of a pair so far.
template <int HD>
struct Decode8State {
  float o[HD / 16][4];          // sums of (c - 128) p'' in units of `ref`
  float m[2], l[2], lp[2];      // heads 2 tq, 2 tq + 1: maximum (log2), sum of p, sum of p'' (this thread's keys only)
  float ref;                    // value scale that o counts in (0: nothing yet)
};

// One page of a stage.  Row g of a score tile is key kappa(g) = g / 2 + 4 (g mod 2) of the 16, row g + 8 is
// key kappa(g) + 8: the eight lanes that a 16-byte shared-memory load serves at a time then hit different banks, for
// keys (chunks tq of rows p and p + 4) and for values (chunks kappa(g) of rows tq) alike.
template <int HD>
__device__ __forceinline__ void d8_page(Decode8State<HD>& st, const uint32_t (&qb)[HD / 16][2], const float (&bias)[2],
                                        const float (&qscale)[2], uint32_t kbase, uint32_t vbase, float ks, float vs, int page_key0,
                                        int pos, int first, int page_size, int hd, uint32_t sub_bytes, float cap2, int lane) {
  constexpr int VW = HD == 64 ? 2 : 4;                         // words of a row of values that a lane holds
  const int g = lane >> 2, tq = lane & 3;
  const int kappa = (g >> 1) + 4 * (g & 1);
  // The page's value scale against the one that o counts in (the same in all lanes).  Upwards o follows all the way;
  // downwards by 2^64 at most, so that it cannot overflow: what a page 2^69 smaller still adds is nothing.
  if (st.ref == 0.f) st.ref = vs;
  float ratio = vs * (1.f / st.ref);
  for (int i = 0; ratio > 32.f || (i == 0 && ratio < 0.03125f); ++i) {
    const int d = max(-64, min(64, ((__float_as_int(st.ref) >> 23) & 255) - ((__float_as_int(vs) >> 23) & 255)));
    const float f = __int_as_float((127 + d) << 23);
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) st.o[i][j] *= f;
    }
    st.lp[0] *= f;
    st.lp[1] *= f;
    st.ref *= __int_as_float((127 - d) << 23);
    ratio = vs * (1.f / st.ref);
  }
  const float pscale = D8_P_BASE * ratio;
  for (int tile = 0; tile * 16 < page_size; ++tile) {
    const int key0 = page_key0 + tile * 16;
    if (key0 > pos || key0 + 15 < first) continue;             // the whole tile is masked
    float sc[4] = {bias[0], bias[1], bias[0], bias[1]};
    const uint32_t krow = kbase + (uint32_t)(tile * 16) * D8_ROW;
#pragma unroll
    for (int u = 0; u < HD / 64; ++u) {                        // 64 dims: a lane's 16 bytes of rows g and g + 8
      if (u * 64 < hd) {
        const uint32_t at = krow + (u >> 1) * sub_bytes + d8_swz(kappa, (u & 1) * 4 + tq);
        const uint4 a = d8_lds16(at), b = d8_lds16(at + 8 * D8_ROW);
        const uint32_t aw[4] = {a.x, a.y, a.z, a.w}, bw[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 4; ++j)
          d8_mma(sc, d8_halves<0, 1>(aw[j]), d8_halves<0, 1>(bw[j]), d8_halves<2, 3>(aw[j]), d8_halves<2, 3>(bw[j]),
                 qb[4 * u + j][0], qb[4 * u + j][1]);
      }
    }
    // sc[h]: key kappa, head 2 tq + h;  sc[2 + h]: key kappa + 8
    const bool inside = key0 >= first && key0 + 15 <= pos;
    const bool va = inside || (key0 + kappa >= first && key0 + kappa <= pos);
    const bool vb = inside || (key0 + kappa + 8 >= first && key0 + kappa + 8 <= pos);
    float corr[2], pp[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // log2 units; with a cap, qscale holds 2 log2(e) / cap and tanh(y) = 1 - 2 / (1 + 2^(2 y log2 e))
      const float f = qscale[h] * ks;
      float xa = sc[h] * f, xb = sc[2 + h] * f;
      if (cap2 > 0.f) {
        xa = cap2 - 2.f * cap2 * d8_rcp(1.f + d8_exp2(xa));
        xb = cap2 - 2.f * cap2 * d8_rcp(1.f + d8_exp2(xb));
      }
      xa = va ? xa : -INFINITY;
      xb = vb ? xb : -INFINITY;
      float mx = fmaxf(xa, xb);
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
      const float m_new = fmaxf(st.m[h], mx);
      const float base = m_new == -INFINITY ? 0.f : m_new;
      corr[h] = d8_exp2(st.m[h] - base);
      const float pa = d8_exp2(xa - base), pb = d8_exp2(xb - base);
      st.l[h] = st.l[h] * corr[h] + pa + pb;
      st.m[h] = m_new;
      pp[h] = pa * pscale;
      pp[2 + h] = pb * pscale;
      st.lp[h] = st.lp[h] * corr[h] + pp[h] + pp[2 + h];
    }
    if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) {
        st.o[i][0] *= corr[0];
        st.o[i][1] *= corr[1];
        st.o[i][2] *= corr[0];
        st.o[i][3] *= corr[1];
      }
    }
    // p^T as the B operand: keys (tq, tq + 4) and (tq + 8, tq + 12) of head g
    const uint32_t b0 = d8_transpose(d8_pack(pp[0], pp[1])), b1 = d8_transpose(d8_pack(pp[2], pp[3]));
    const uint32_t vrow = vbase + (uint32_t)(tile * 16) * D8_ROW;
#pragma unroll
    for (int s = 0; s < (HD + 127) / 128; ++s) {
      if (s * 128 < hd) {
        // this lane's 16 dims (8 of the 64 when heads are that small) of keys tq, tq + 4, tq + 8, tq + 12
        uint32_t w[4][VW];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = tq + 4 * k;
          const uint32_t at = vrow + s * sub_bytes;
          if (VW == 4) {
            const uint4 v = d8_lds16(at + d8_swz(row, kappa));
            w[k][0] = v.x; w[k][1] = v.y; w[k][VW == 4 ? 2 : 0] = v.z; w[k][VW == 4 ? 3 : 1] = v.w;
          } else {
            const uint2 v = d8_lds8(at + d8_swz(row, g >> 1) + (g & 1) * 8);
            w[k][0] = v.x; w[k][1] = v.y;
          }
        }
#pragma unroll
        for (int c = 0; c < VW; ++c) {                         // 4 dims: two tiles of (dim, dim + 1)
          const uint32_t lo0 = __byte_perm(w[0][c], w[1][c], 0x5140), hi0 = __byte_perm(w[0][c], w[1][c], 0x7362);
          const uint32_t lo1 = __byte_perm(w[2][c], w[3][c], 0x5140), hi1 = __byte_perm(w[2][c], w[3][c], 0x7362);
          d8_mma(st.o[s * 8 + 2 * c], d8_halves<0, 1>(lo0), d8_halves<2, 3>(lo0), d8_halves<0, 1>(lo1), d8_halves<2, 3>(lo1), b0, b1);
          d8_mma(st.o[s * 8 + 2 * c + 1], d8_halves<0, 1>(hi0), d8_halves<2, 3>(hi0), d8_halves<0, 1>(hi1), d8_halves<2, 3>(hi1), b0, b1);
        }
      }
    }
  }
}

// HD: register capacity (head_dim <= HD; head_dim and page_size are multiples of 16).
template <int HD>
__global__ void __launch_bounds__(D8_THREADS, 2)
attention_decode8_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                         const Decode8Params p) {
  extern __shared__ uint8_t d8_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(d8_raw) + 1023) & ~(uintptr_t)1023);
  const int hd = p.hd, G = p.nh / p.nkv;
  const int pairs = p.nkv * p.groups;                          // pairs of a token: (kv head, up to 8 query heads)
  const int nsub = (hd + 127) >> 7;
  const uint32_t sub_bytes = (uint32_t)p.page_size * D8_ROW;
  const uint32_t page_bytes = nsub * sub_bytes;
  const int stride_f = hd + 2, pstride = hd + 4;
  const int HP = G < D8_HEADS ? G : D8_HEADS;
  float* merge = reinterpret_cast<float*>(ring + (size_t)p.stages * 2 * page_bytes);      // [warps][HP][hd + 2]
  Decode8Shared* sh = reinterpret_cast<Decode8Shared*>(merge + (((size_t)D8_WARPS * HP * stride_f + 3) & ~(size_t)3));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      tc::mbar_init(&sh->full[s], 1);
      tc::mbar_init(&sh->empty[s], 1);
    }
    sh->abort_flag = 0;
    sh->last_one = 0;
    sh->start_token = -1;
    tc::fence_barrier_init();
    tc::tma_prefetch_desc(&map_k);
    tc::tma_prefetch_desc(&map_v);
  }
  pdl_wait_release();
  // ---- where this block begins: a scan over the tokens' units, some tokens per thread ---------------------------
  const int per = (p.T + D8_THREADS - 1) / D8_THREADS;
  const int r0 = min((int)threadIdx.x * per, p.T), r1 = min(r0 + per, p.T);
  long long mine = 0;
  for (int r = r0; r < r1; ++r) mine += (long long)(p.pair_cost + d8_segment(p.positions[r], p.window, p.page_size).pages) * pairs;
  long long incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) sh->warp_sum[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < D8_THREADS / 32; ++w) {
    if (w < warp) before += sh->warp_sum[w];
    total += sh->warp_sum[w];
  }
  const long long share = (total + gridDim.x - 1) / gridDim.x;
  const long long W = share > p.min_units ? share : p.min_units;
  const long long begin = (long long)blockIdx.x * W;
  if (begin >= total) return;                                  // fewer units than blocks (the same for all threads)
  if (begin >= before && begin < before + mine) {
    int r = r0;
    long long inside = begin - before;
    for (; r < r1; ++r) {
      const long long u = (long long)(p.pair_cost + d8_segment(p.positions[r], p.window, p.page_size).pages) * pairs;
      if (inside < u) break;
      inside -= u;
    }
    sh->start_token = r;
    sh->start_inside = (int)inside;
  }
  __syncthreads();
  int t = sh->start_token;
  int remaining = (int)min(W, total - begin);                  // units
  int pos = p.positions[t];
  Decode8Segment sg = d8_segment(pos, p.window, p.page_size);
  int pair = sh->start_inside / (p.pair_cost + sg.pages);
  int voff = sh->start_inside - pair * (p.pair_cost + sg.pages);
  int it0 = 0;
  volatile int* abort_flag = &sh->abort_flag;

  if (warp == D8_WARPS) {
    // ---- producer warp: 32 page lookups at a time with the pages' scales, one lane starts the copies --------------
    int row = p.token_seq[t];
    while (remaining > 0 && t < p.T) {
      const int units = min(remaining, p.pair_cost + sg.pages - voff);    // of this pair in this block
      const int off = max(voff, p.pair_cost) - p.pair_cost;               // first page
      const int n = max(0, voff + units - p.pair_cost - off);             // pages
      const int kvh = pair / p.groups;
      const int* table = p.block_table + (size_t)row * p.max_pages + sg.page_lo + off;
      for (int base = 0; base < n; base += 32) {
        int page = 0;
        float ks = 0.f, vs = 1.f;
        if (base + lane < n) {
          page = sg.page_lo + off + base + lane < p.max_pages ? table[base + lane] : -1;
          if (page < 0 || page >= p.num_pages) {               // never read outside the pool; report it
            atomicExch(p.status, 3);
            page = 0;
          }
          ks = p.k_scale[(size_t)page * p.nkv + kvh];
          vs = p.v_scale[(size_t)page * p.nkv + kvh];
          if (!(fabsf(vs) <= 3.4e38f)) {                       // not finite: the keys say so, the values stay finite
            ks = __int_as_float(0x7fc00000);
            vs = 1.f;
          }
          if (vs == 0.f) vs = 7.5231638e-37f;                  // 2^-120: a page that nothing was written to
        }
        for (int j = 0; j < 32 && base + j < n; ++j) {
          const int it = it0 + base + j;
          const int pg = __shfl_sync(0xffffffffu, page, j);
          const float pks = __shfl_sync(0xffffffffu, ks, j), pvs = __shfl_sync(0xffffffffu, vs, j);
          if (tc::elect_one()) {
            const int s = it % p.stages;
            bool ok = true;
            if (it >= p.stages) ok = tc::mbar_wait(&sh->empty[s], ((it / p.stages) - 1) & 1, abort_flag);
            if (ok) {
              uint8_t* kdst = ring + (size_t)s * 2 * page_bytes;
              const int at = (pg * p.nkv + kvh) * p.page_size;
              sh->scale[s] = make_float2(pks, pvs);            // before the arrival that completes with the copies
              tc::mbar_expect_tx(&sh->full[s], 2 * page_bytes);
              if (p.whole_page) {
                tc::tma_load_3d(kdst, &map_k, &sh->full[s], 0, at, 0);
                tc::tma_load_3d(kdst + page_bytes, &map_v, &sh->full[s], 0, at, 0);
              } else {
                for (int sub = 0; sub < nsub; ++sub) {
                  tc::tma_load_2d(kdst + sub * sub_bytes, &map_k, &sh->full[s], sub * 128, at);
                  tc::tma_load_2d(kdst + page_bytes + sub * sub_bytes, &map_v, &sh->full[s], sub * 128, at);
                }
              }
            }
          }
        }
      }
      remaining -= units;
      it0 += n;
      voff = 0;
      if (++pair == pairs) {
        pair = 0;
        if (++t < p.T && remaining > 0) {
          sg = d8_segment(p.positions[t], p.window, p.page_size);
          row = p.token_seq[t];
        }
      }
    }
    return;
  }

  // ---- consumer warps ------------------------------------------------------------------------------------------
  const int g = lane >> 2, tq = lane & 3;
  const float LOG2E = 1.4426950408889634f;
  const float cap2 = p.cap > 0.f ? p.cap * LOG2E : 0.f;
  const float score_scale = p.cap > 0.f ? 2.f * LOG2E * p.multiplier / p.cap : p.multiplier * LOG2E;
  const uint32_t ring_addr = tc::smem_u32(ring);
  long long cursor = begin;
  while (remaining > 0 && t < p.T) {
    const int units = min(remaining, p.pair_cost + sg.pages - voff);
    const int off = max(voff, p.pair_cost) - p.pair_cost;
    const int n = max(0, voff + units - p.pair_cost - off);
    const long long pair_begin = cursor - voff + p.pair_cost;   // the pair's first page in the launch's sequence
    cursor += units;
    remaining -= units;
    voff = 0;
    const int kvh = pair / p.groups, h0 = (pair - kvh * p.groups) * D8_HEADS;     // of the group: first head
    const int H = min(G - h0, D8_HEADS);
    if (n > 0) {
      const bool begins = off == 0, ends = off + n == sg.pages;
      // q^T as the B operand: this thread holds, per 64 dims, dims 16 tq .. 16 tq + 15 of head g, four to a tile
      uint32_t qb[HD / 16][2];
      float qscale[2], bias[2];
      {
        const __nv_bfloat16* qrow = p.q + ((size_t)t * p.nh + kvh * G + h0 + (g < H ? g : 0)) * hd;
        unsigned top = 0;
        uint32_t raw[HD / 16][2];
#pragma unroll
        for (int u = 0; u < HD / 64; ++u) {
          const bool in = u * 64 + tq * 16 < hd && g < H;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (in) v = *reinterpret_cast<const uint4*>(qrow + u * 64 + tq * 16 + half * 8);
            raw[4 * u + 2 * half][0] = v.x; raw[4 * u + 2 * half][1] = v.y;
            raw[4 * u + 2 * half + 1][0] = v.z; raw[4 * u + 2 * half + 1][1] = v.w;
          }
        }
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) top = max(top, max(raw[i][j] & 0x7fffu, (raw[i][j] >> 16) & 0x7fffu));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^-e brings the largest element to [2^8, 2^9); e is held where both powers are normal
        const int e = max(-100, min(118, (int)(top >> 7) - 127 - 8));
        const float down = __int_as_float((127 - e) << 23);
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float lo = __uint_as_float(raw[i][j] << 16) * down, hi = __uint_as_float(raw[i][j] & 0xffff0000u) * down;
            const __half2 hv = __floats2half2_rn(lo, hi);
            qb[i][j] = *reinterpret_cast<const uint32_t*>(&hv);
            sum += __low2float(hv) + __high2float(hv);
          }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        const float up = __int_as_float((127 + e) << 23);
#pragma unroll
        for (int h = 0; h < 2; ++h) {                           // from the lanes of head 2 tq + h
          bias[h] = 0.5f * __shfl_sync(0xffffffffu, sum, (2 * tq + h) * 4);
          qscale[h] = score_scale * __shfl_sync(0xffffffffu, up, (2 * tq + h) * 4);
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
      // Page `it` of the block belongs to warp it % warps and stage it % stages (a multiple of them: a stage is always
      // read by the same warp, which therefore sees every phase of the stage's barrier).
      for (int it = it0 + ((warp - it0) % D8_WARPS + D8_WARPS) % D8_WARPS; it < it0 + n; it += D8_WARPS) {
        const int s = it % p.stages;
        const bool ok = tc::mbar_wait(&sh->full[s], (it / p.stages) & 1, abort_flag);
        const uint32_t kbase = ring_addr + (uint32_t)s * 2 * page_bytes;
        if (ok) {
          const float2 scale = sh->scale[s];
          d8_page<HD>(st, qb, bias, qscale, kbase, kbase + page_bytes, scale.x, scale.y, (sg.page_lo + off + it - it0) * p.page_size,
                      pos, sg.first, p.page_size, hd, sub_bytes, cap2, lane);
        }
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sh->empty[s]);
      }
      // ---- this warp's totals; the warps are merged in shared memory, in warp order ------------------------------
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
          const float unit = st.ref * (1.f / D8_P_BASE), half = 0.5f * st.lp[h];
#pragma unroll
          for (int i = 0; i < HD / 16; ++i) {
            // tile i: dims (d, d + 1) of this lane's 16 (or 8) of the 128 (or 64)
            const int d = HD == 64 ? g * 8 + 2 * i : (i >> 3) * 128 + ((g >> 1) + 4 * (g & 1)) * 16 + 2 * (i & 7);
            if (d < hd) *reinterpret_cast<float2*>(dst + d) = make_float2((st.o[i][h] + half) * unit, (st.o[i][2 + h] + half) * unit);
          }
          if (g == 0) *reinterpret_cast<float2*>(dst + hd) = make_float2(st.m[h], st.l[h]);
        }
      }
      d8_consumer_sync();
      const bool whole = begins && ends;
      float* partial = p.partials + ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * HP * pstride;
      __nv_bfloat16* out = p.out + ((size_t)t * p.nh + kvh * G + h0) * hd;
      for (int j = 0; j < H; ++j) {
        float M = -INFINITY;
#pragma unroll
        for (int wv = 0; wv < D8_WARPS; ++wv) M = fmaxf(M, merge[((size_t)wv * HP + j) * stride_f + hd]);
        float L = 0.f, w[D8_WARPS];
#pragma unroll
        for (int wv = 0; wv < D8_WARPS; ++wv) {
          const float2 ml = *reinterpret_cast<const float2*>(merge + ((size_t)wv * HP + j) * stride_f + hd);
          // a warp without pages has l = 0; one whose scores were all NaN has the maximum -inf and l = NaN
          w[wv] = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : ml.y) : d8_exp2(ml.x - M);
          L += ml.y * w[wv];
        }
        for (int d = threadIdx.x; d < hd; d += D8_WARPS * 32) {
          float ov = 0.f;
#pragma unroll
          for (int wv = 0; wv < D8_WARPS; ++wv) ov += merge[((size_t)wv * HP + j) * stride_f + d] * w[wv];
          if (whole) out[(size_t)j * hd + d] = __float2bfloat16_rn(L == 0.f ? 0.f : ov / L);
          else partial[(size_t)j * pstride + d] = ov;
        }
        if (!whole && threadIdx.x == 0) *reinterpret_cast<float2*>(partial + (size_t)j * pstride + hd) = make_float2(M, L);
      }
      if (!whole) {
        // ---- the pair is shared: the block that leaves its part last adds the parts up, in block order --------------
        const int b_first = (int)(pair_begin / W), b_last = (int)((pair_begin + sg.pages - 1) / W);
        d8_consumer_sync();                                     // every thread's share of the partial result is written
        if (threadIdx.x == 0) {
          __threadfence();                                      // and visible before this block is counted
          int* counter = p.arrive + (size_t)t * pairs + pair;
          const int last = atomicAdd(counter, 1) == b_last - b_first;
          if (last) *counter = 0;                               // for the next launch
          __threadfence();
          sh->last_one = last;
        }
        d8_consumer_sync();
        if (sh->last_one) {
          const int parts = b_last - b_first + 1;
          const int quads = hd >> 2;
          for (int e = threadIdx.x; e < H * quads; e += D8_WARPS * 32) {
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
                  const float* from = p.partials + (((size_t)bk * 2 + (bk == b_first ? 1 : 0)) * HP + j) * pstride;
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
            const float inv = L == 0.f ? 0.f : 1.f / L;
            const __nv_bfloat162 lo = __floats2bfloat162_rn(acc.x * inv, acc.y * inv), hi = __floats2bfloat162_rn(acc.z * inv, acc.w * inv);
            *reinterpret_cast<uint2*>(out + (size_t)j * hd + d) =
                make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
          }
        }
      }
      d8_consumer_sync();                                       // the merge area and last_one are used again by the next pair
      it0 += n;
    }
    if (++pair == pairs) {
      pair = 0;
      if (++t < p.T && remaining > 0) {
        pos = p.positions[t];
        sg = d8_segment(pos, p.window, p.page_size);
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

static long long d8_fixed(int G, int hd) {
  const int HP = G < D8_HEADS ? G : D8_HEADS;
  return (((long long)D8_WARPS * HP * (hd + 2) + 3) & ~3ll) * 4 + (long long)sizeof(Decode8Shared) + 1024;
}

}  // namespace glint

using namespace glint;

// Head sizes in steps of 16 up to 256, pages in steps of 16 of which one per consumer warp fits a block's shared memory.
GLINT_API int glint_attention_decode8_supported(int nh, int nkv, int hd, int page_size) {
  if (!(nkv > 0 && nh > 0 && nh % nkv == 0 && hd % 16 == 0 && hd >= 16 && hd <= 256 && page_size % 16 == 0 && page_size >= 16 &&
        page_size <= 256))
    return 0;
  const long long page_bytes = (long long)((hd + 127) / 128) * page_size * D8_ROW;
  return D8_WARPS * 2 * page_bytes + d8_fixed(nh / nkv, hd) <= 227 * 1024 ? 1 : 0;
}

// Workspace of launches over `blocks` blocks: floats of partial results.
GLINT_API long long glint_attention_decode8_workspace(int blocks, int nh, int nkv, int hd) {
  const int G = nh / nkv;
  return (long long)blocks * 2 * (G < D8_HEADS ? G : D8_HEADS) * (hd + 4);
}

// q, out [T][nh][hd] bfloat16, pages of codes with their scales; T single tokens of which none attends more than
// `max_context` keys.  `partials`: glint_attention_decode8_workspace floats, 16-byte aligned; `arrive`: `arrive_ints`
// counters that are zero before the first launch (every launch leaves them zero).  Launches of more tokens than
// the counters or 1024 allow are cut.  `blocks`: at most that many blocks (two per SM).
GLINT_API int glint_attention_decode8(const void* q, const uint8_t* k_pool, const uint8_t* v_pool, const float* k_scale,
                                      const float* v_scale, const int* positions, const int* token_seq, const int* block_table,
                                      int max_pages, void* out, int T, int nh, int nkv, int hd, int page_size, int num_pages,
                                      float multiplier, float cap, int window, int max_context, int blocks, float* partials,
                                      int* arrive, int arrive_ints, int* status, cudaStream_t stream) {
  if (T <= 0) return GLINT_OK;
  if (!partials || !arrive || blocks < 1 || ((uintptr_t)partials & 15)) return GLINT_ERR_BAD_ARG;
  if (!glint_attention_decode8_supported(nh, nkv, hd, page_size)) return GLINT_ERR_UNSUPPORTED_SIZE;
  if (((uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)q | (uintptr_t)out) & 15) return GLINT_ERR_UNSUPPORTED_SIZE;
  const long long rows = (long long)num_pages * nkv * page_size;
  if (rows > 0x7fffffffLL) return GLINT_ERR_UNSUPPORTED_SIZE;
  const int G = nh / nkv, groups = (G + D8_HEADS - 1) / D8_HEADS, pairs = nkv * groups;
  if (pairs > arrive_ints) return GLINT_ERR_UNSUPPORTED_SIZE;
  const int whole_page = hd % 128 == 0 ? 1 : 0;
  CUtensorMap map_k, map_v;
  int rc = d8_map(&map_k, k_pool, rows, hd, page_size, whole_page);
  if (rc == GLINT_OK) rc = d8_map(&map_v, v_pool, rows, hd, page_size, whole_page);
  if (rc != GLINT_OK) return rc;
  const long long page_bytes = (long long)((hd + 127) / 128) * page_size * D8_ROW;
  const long long fixed = d8_fixed(G, hd);
  int stages = (int)((112 * 1024 - fixed) / (2 * page_bytes)) / D8_WARPS * D8_WARPS;     // two blocks share an SM
  if (stages > D8_MAX_STAGES) stages = D8_MAX_STAGES;
  if (stages < D8_WARPS) stages = D8_WARPS;
  const long long smem = stages * 2 * page_bytes + fixed;
  if (smem > 227 * 1024) return GLINT_ERR_UNSUPPORTED_SIZE;
  // what a pair costs a block beside its pages, and the least a block is given, in pages of this size
  const long long unit = 2ll * page_size * hd;
  const int pair_cost = (int)((48 * 1024 + unit / 2) / unit) + 1;
  const int min_units = (int)((32 * 1024 + unit - 1) / unit) + 1;
  long long most_pages = ((long long)max_context + page_size - 1) / page_size;
  if (window > 0 && ((long long)window + page_size - 1) / page_size + 1 < most_pages)
    most_pages = ((long long)window + page_size - 1) / page_size + 1;
  const int step = arrive_ints / pairs < D8_MAX_TOKENS ? arrive_ints / pairs : D8_MAX_TOKENS;
  for (int t0 = 0; t0 < T; t0 += step) {
    const int n = T - t0 < step ? T - t0 : step;
    Decode8Params p = {(const __nv_bfloat16*)q + (size_t)t0 * nh * hd, positions + t0, token_seq + t0, block_table, k_scale, v_scale,
                       (__nv_bfloat16*)out + (size_t)t0 * nh * hd, partials, arrive, status, multiplier, cap,
                       n, nh, nkv, hd, groups, page_size, num_pages, max_pages, window, stages, whole_page, pair_cost, min_units};
    const long long most = (long long)n * pairs * (most_pages + pair_cost);
    const long long useful = (most + min_units - 1) / min_units;
    const int grid = useful < blocks ? (int)useful : blocks;
#define LAUNCH(HD)                                                                                                       \
  {                                                                                                                      \
    cudaError_t e = cudaFuncSetAttribute(attention_decode8_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem); \
    if (e != cudaSuccess) return (int)e;                                                                                 \
    e = launch_kernel(attention_decode8_kernel<HD>, dim3(grid), dim3(D8_THREADS), (size_t)smem, stream, map_k, map_v, p); \
    if (e != cudaSuccess) return (int)e;                                                                                 \
  }
    if (hd <= 64) LAUNCH(64)
    else if (hd <= 128) LAUNCH(128)
    else LAUNCH(256)
#undef LAUNCH
  }
  return (int)cudaGetLastError();
}
