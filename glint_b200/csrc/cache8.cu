// The key/value cache held in 8 bits: rotation and append, and widening of pages.
//
// A page holds `page_size` tokens of one kv head: codes [page_size][head_dim] of 8 bits and one scale s = 2^e, for
// keys and for values each.  A code c stands for (c - 127.5) s and is made by floor(x / s) + 128; e is the
// largest over the page's tokens of floor(log2(max |x|)) - 6 (so that |x| < 128 s), at least -120.  When a later
// token raises the exponent by d, the codes of the rows before it move to ((c - 128) >> d) + 128.  Because
//     floor(floor(x / s) / 2^d) = floor(x / (s 2^d)),
// that is exactly the code that x would have got at the new scale: a page's content depends on its tokens and not
// on how they were cut into steps (rounding to nearest would round twice).  |value - x| <= s / 2, which is at
// most 1/128 of the page's largest magnitude; and every value is an odd integer of 8 bits times 2^(e-1), so
// that widening to bfloat16 is exact.
// A key or value that is not finite makes the page's scale NaN until the page is begun anew.
#include "common.cuh"

namespace glint {

constexpr int C8_LOWEST = -120;                   // smallest exponent of a scale
constexpr unsigned C8_NOT_FINITE = 0x7f800000u;   // |x| as bits: from here on infinities and NaN

// exponent of the scale for a largest magnitude given as the bits of |x|
__device__ __forceinline__ int c8_exponent(unsigned bits) { return max((int)(bits >> 23) - 133, C8_LOWEST); }
__device__ __forceinline__ float c8_pow2(int e) { return __int_as_float((e + 127) << 23); }    // -126 <= e <= 127
// Steps by which the 32-bit rotation can be off, in units u = 2^-24 of a pair's length (at most 128 sqrt(2) steps): the angle, two
// roundings and a constant of at most pi / 4, 1.9; sine and cosine 0.8 and 1.0, together 1.3; a product and a sum 2; an
// amplitude and its product 2: 7.2 u = 7.8e-5 (4.1 u is the most that a search found).  Keys nearer than that to a border
// between codes are rotated again in 64 bits (one in 6,000), so that codes are those of the definition to the last.
constexpr float C8_NEAR = 8e-5f;
__device__ __forceinline__ float c8_distance(float x, float inv) {
  const float h = x * inv, magic = 12582912.f;           // 1.5 * 2^23: the nearest whole number
  return fabsf(h - ((h + magic) - magic));
}
// A largest magnitude, given as bits, so near a power of two (16 steps of 32 bits; the rotation's 7.2 u of a pair's length
// are 10.2 of its larger part) that 64 bits have to say which exponent it has.
__device__ __forceinline__ bool c8_near_scale(unsigned bits) {
  return bits >= 13u << 23 && bits < C8_NOT_FINITE && ((bits + 16u) & 0x7fffffu) < 32u;
}
// floor(x / s) + 128.  The product is exact, but for the smallest numbers under the largest scales, where it may become
// -0: the floor of any negative number is at most -1.
__device__ __forceinline__ unsigned c8_code(float x, float inv) {
  const int q = __float2int_rd(x * inv);
  return (unsigned)((x < 0.f ? min(q, -1) : q) + 128) & 255u;
}

struct AppendParams {
  const float* qkv;              // [T][nh + 2 nkv][hd]
  const int* positions;
  const int* token_seq;
  const int* block_table;
  const double* turns;           // [rot / 2] turns per position
  void* q_out;                   // [T][nh][hd]
  void* k_pool;                  // null: q only
  void* v_pool;
  float* k_scale;                // null: pools of the activations' type
  float* v_scale;
  int* status;
  double amplitude;
  int T, nh, nkv, hd, rot, interleaved, page_size, num_pages, max_pages;
  int early;                     // positions, requests, tables and turns are no kernel's work: read before the wait
};

// (cos, sin) of 2 pi pos turns, times the amplitude.  The product is taken in 64 bits and reduced to an eighth of a turn
// either way before anything is rounded to 32: at position 100,000 the 32-bit product alone is off by 4e-3 radians.  Then
// the Taylor polynomials of sine and cosine to x^9 and x^10, |x| <= pi / 4: what they leave out is below 2e-9.
__device__ __forceinline__ float2 rope_angle(int pos, double turns, float amplitude) {
  const double quarters = 4.0 * turns * (double)pos;
  const double magic = 6755399441055744.0;                 // 1.5 * 2^52: the nearest whole number sits in the low bits
  const double shifted = quarters + magic;
  const int n = __double2loint(shifted);
  const float x = (float)(quarters - (shifted - magic)) * 1.57079632679f;
  const float y = x * x;
  float s = fmaf(y, 2.7557319e-6f, -1.9841270e-4f);        // 1/9!, 1/7!, 1/5!, 1/3!
  s = fmaf(s, y, 8.3333333e-3f);
  s = fmaf(s, y, -1.6666667e-1f);
  s = fmaf(s * y, x, x);
  float c = fmaf(y, -2.7557319e-7f, 2.4801587e-5f);        // 1/10!, 1/8!, 1/6!, 1/4!, 1/2!
  c = fmaf(c, y, -1.3888889e-3f);
  c = fmaf(c, y, 4.1666667e-2f);
  c = fmaf(c, y, -0.5f);
  c = fmaf(c, y, 1.f);
  const float cs = (n & 1) ? s : c, sn = (n & 1) ? c : s;
  return make_float2((((n + 1) & 2) ? -cs : cs) * amplitude, ((n & 2) ? -sn : sn) * amplitude);
}

// The pair (a, b) turned, in 64 bits: Taylor polynomials to x^17 and x^16, which leave out less than 1e-15.
__device__ __noinline__ double2 rope_exact(int pos, double turns, double amplitude, float a, float b) {
  const double quarters = 4.0 * turns * (double)pos;
  const double n = rint(quarters);
  const double x = (quarters - n) * 1.5707963267948966, y = x * x;
  double s = 0.0, c = 0.0, f = 1.0 / 355687428096000.0, g = 1.0 / 20922789888000.0;      // 1 / 17!, 1 / 16!
#pragma unroll
  for (int i = 17; i >= 3; i -= 2) {
    s = fma(s, y, ((i >> 1) & 1) ? -f : f);
    c = fma(c, y, ((i >> 1) & 1) ? -g : g);
    f *= (double)(i * (i - 1));
    g *= (double)((i - 1) * (i - 2));
  }
  s = fma(s * y, x, x);
  c = fma(c, y, 1.0);
  const int q = (int)((long long)n & 3);
  const double cs = ((q + 1) & 2 ? -1.0 : 1.0) * (q & 1 ? s : c) * amplitude, sn = (q & 2 ? -1.0 : 1.0) * (q & 1 ? c : s) * amplitude;
  return make_double2(a * cs - b * sn, a * sn + b * cs);
}
// (A value turned beyond what 32 bits hold is held to the largest code.)
__device__ __forceinline__ unsigned c8_code(double x, double inv) { return (unsigned)(max(-128, min(127, (int)floor(x * inv))) + 128); }

// ---- heads of up to 256: a lane holds NP pairs of a head ------------------------------------------------------------
//
// Memory-bound for portions (a float read and one to two bytes written per element), latency-bound for single tokens.
// One launch of two kinds of blocks of eight warps.  Cache blocks: a window of 16 tokens x one kv head x keys or values.  A
// block owns the runs (tokens of one request in one page) that begin in its window and takes them whole, so that the
// largest magnitude of a run, and with it the page's new scale, is found in one block whatever the windows cut: a warp
// per token, values kept in registers (two tokens a warp) between the maximum and the codes.  Query blocks: a warp
// rotates four heads of a token with one set of sines and cosines.
// Measured, 2,048 tokens of 8 heads in 4 groups of 256 with the widening behind it (34 MB of float read, 4 MB of codes and 8 MB
// of queries written; 11.3 + 4.2 us) / a mixed step of 997 tokens, 32 heads in 16 groups of 128: 16.6 / 22.9 us; two or eight
// heads a warp 17.4 / 24.6 and 23.1 / 23.9; one or four tokens held 18.0 / 24.2 and 17.4 / 23.6; room for three, five or
// six blocks an SM instead of four 18.5 / 22.8, 17.8 / 21.4 and 20.7 / 21.9, so that heads of 256 take four, smaller ones five.
// (All before keys next to a border were decided in 64 bits, which adds 0.8 / 1.0.)  One token takes 2.4 us behind a kernel
// that it can begin under.
constexpr int AP_WARPS = 8;
constexpr int AP_WINDOW = 16;                     // tokens
constexpr int AP_HELD = 2;                        // tokens of a warp whose values stay in registers
constexpr int AP_MOST_PAGE = AP_WARPS * 32 - AP_WINDOW;       // rows of a page: a thread per token of a block
constexpr int AP_HEADS = 4;                       // query heads of a unit

// Pair i of a head: its two dims.  The first rot / 2 are turned.
__device__ __forceinline__ int2 rope_pair(int i, int rot, int interleaved) {
  const int half = rot >> 1;
  return interleaved || i >= half ? make_int2(2 * i, 2 * i + 1) : make_int2(i, i + half);
}

// N values in as few accesses as they take; N x size is at most 16 or a multiple of it, and so is the address.
template <int N>
__device__ __forceinline__ void load_floats(const float* from, float* to) {
  if constexpr (N == 1) {
    to[0] = *from;
  } else if constexpr (N == 2) {
    const float2 v = *reinterpret_cast<const float2*>(from);
    to[0] = v.x; to[1] = v.y;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float4 v = *reinterpret_cast<const float4*>(from + i);
      to[i] = v.x; to[i + 1] = v.y; to[i + 2] = v.z; to[i + 3] = v.w;
    }
  }
}
template <int N>
__device__ __forceinline__ void store_values(float* to, const float* from) {
  if constexpr (N == 1) {
    *to = from[0];
  } else if constexpr (N == 2) {
    *reinterpret_cast<float2*>(to) = make_float2(from[0], from[1]);
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(to + i) = make_float4(from[i], from[i + 1], from[i + 2], from[i + 3]);
  }
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <int N>
__device__ __forceinline__ void store_values(__nv_bfloat16* to, const float* from) {
  if constexpr (N == 1) {
    *to = __float2bfloat16(from[0]);
  } else if constexpr (N == 2) {
    *reinterpret_cast<uint32_t*>(to) = pack_bf16(from[0], from[1]);
  } else if constexpr (N == 4) {
    *reinterpret_cast<uint2*>(to) = make_uint2(pack_bf16(from[0], from[1]), pack_bf16(from[2], from[3]));
  } else {
    *reinterpret_cast<uint4*>(to) = make_uint4(pack_bf16(from[0], from[1]), pack_bf16(from[2], from[3]), pack_bf16(from[4], from[5]),
                                              pack_bf16(from[6], from[7]));
  }
}
template <int N>
__device__ __forceinline__ void store_codes(uint8_t* to, const unsigned* c) {
  if constexpr (N == 1) {
    *to = (uint8_t)c[0];
  } else if constexpr (N == 2) {
    *reinterpret_cast<uint16_t*>(to) = (uint16_t)(c[0] | (c[1] << 8));
  } else {
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) w[i] = c[4 * i] | (c[4 * i + 1] << 8) | (c[4 * i + 2] << 16) | (c[4 * i + 3] << 24);
    if constexpr (N == 4) *reinterpret_cast<uint32_t*>(to) = w[0];
    else *reinterpret_cast<uint2*>(to) = make_uint2(w[0], w[1]);
  }
}
// Four codes at a scale 2^d larger, 1 <= d <= 7 (more gives what 7 gives): floor((c - 128) / 2^d) + 128 is
// (c >> d) + 128 - (128 >> d).
__device__ __forceinline__ uint32_t shift_codes(uint32_t w, int d) {
  return ((w >> d) & ((0xffu >> d) * 0x01010101u)) + (128u - (128u >> d)) * 0x01010101u;
}

// A lane's NP pairs of a head.  FULL: heads of 64 NP dims of which a multiple of 2 NP are turned, 16-byte aligned: NP
// consecutive pairs, all turned or none, moved together (2,048 tokens of 8 heads in 4 groups of 256: 13.8 -> 10.7 us against
// one by one).  Else pairs lane + 32 k.
template <int NP, bool FULL>
struct RopeLane {
  int lane, half, pairs, rot, interleaved;
  __device__ __forceinline__ int pair(int k) const { return FULL ? lane * NP + k : lane + 32 * k; }
  __device__ __forceinline__ bool in(int k) const { return FULL || lane + 32 * k < pairs; }
  __device__ __forceinline__ bool turned(int k) const { return (FULL ? lane * NP : lane + 32 * k) < half; }
  // FULL, not interleaved: where the pairs' first and second dims begin (those that are not turned pair up as they like)
  __device__ __forceinline__ int first() const { return lane * NP < half ? lane * NP : lane * 2 * NP; }
  __device__ __forceinline__ int second() const { return lane * NP < half ? half + lane * NP : lane * 2 * NP + NP; }
  __device__ __forceinline__ int2 dims(int k) const {
    if (!FULL) return at(k);
    return interleaved ? make_int2(2 * pair(k), 2 * pair(k) + 1) : make_int2(first() + k, second() + k);
  }
  __device__ __forceinline__ int2 at(int k) const { return rope_pair(lane + 32 * k, rot, interleaved); }
  __device__ __forceinline__ void load(const float* row, float (&a)[NP], float (&b)[NP]) const {
    if constexpr (FULL) {
      if (interleaved) {
        float v[2 * NP];
        load_floats<2 * NP>(row + lane * 2 * NP, v);
#pragma unroll
        for (int k = 0; k < NP; ++k) { a[k] = v[2 * k]; b[k] = v[2 * k + 1]; }
      } else {
        load_floats<NP>(row + first(), a);
        load_floats<NP>(row + second(), b);
      }
    } else {
#pragma unroll
      for (int k = 0; k < NP; ++k) {
        const int2 d = at(k);
        a[k] = in(k) ? row[d.x] : 0.f;
        b[k] = in(k) ? row[d.y] : 0.f;
      }
    }
  }
  template <typename S>
  __device__ __forceinline__ void store(S* row, const float (&a)[NP], const float (&b)[NP]) const {
    if constexpr (FULL) {
      if (interleaved) {
        float v[2 * NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) { v[2 * k] = a[k]; v[2 * k + 1] = b[k]; }
        store_values<2 * NP>(row + lane * 2 * NP, v);
      } else {
        store_values<NP>(row + first(), a);
        store_values<NP>(row + second(), b);
      }
    } else {
#pragma unroll
      for (int k = 0; k < NP; ++k)
        if (in(k)) {
          const int2 d = at(k);
          row[d.x] = from_float<S>(a[k]);
          row[d.y] = from_float<S>(b[k]);
        }
    }
  }
  __device__ __forceinline__ void store(uint8_t* row, const unsigned (&a)[NP], const unsigned (&b)[NP]) const {
    if constexpr (FULL) {
      if (interleaved) {
        unsigned v[2 * NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) { v[2 * k] = a[k]; v[2 * k + 1] = b[k]; }
        store_codes<2 * NP>(row + lane * 2 * NP, v);
      } else {
        store_codes<NP>(row + first(), a);
        store_codes<NP>(row + second(), b);
      }
    } else {
#pragma unroll
      for (int k = 0; k < NP; ++k)
        if (in(k)) {
          const int2 d = at(k);
          row[d.x] = (uint8_t)a[k];
          row[d.y] = (uint8_t)b[k];
        }
    }
  }
};

template <typename S, int NP, bool FULL>
__global__ void __launch_bounds__(AP_WARPS * 32, NP == 4 ? 4 : 5) rope_append_kernel(const AppendParams p, int cache_blocks) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int width = (p.nh + 2 * p.nkv) * p.hd, pairs = p.hd >> 1;
  const RopeLane<NP, FULL> mine = {lane, p.rot >> 1, pairs, p.rot, p.interleaved};
  if (!p.early) pdl_wait();
  double turns[NP];
#pragma unroll
  for (int k = 0; k < NP; ++k) turns[k] = mine.turned(k) ? p.turns[mine.pair(k)] : 0.0;

  if ((int)blockIdx.x >= cache_blocks) {
    // ---- queries ---------------------------------------------------------------------------------------------------
    const int groups = (p.nh + AP_HEADS - 1) / AP_HEADS;
    const long long unit = (long long)(blockIdx.x - cache_blocks) * AP_WARPS + warp;
    const int t = (int)(unit / groups), h0 = (int)(unit - (long long)t * groups) * AP_HEADS;
    if (t >= p.T) return;
    const int pos = p.positions[t];
    float2 turned_by[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) turned_by[k] = mine.turned(k) ? rope_angle(pos, turns[k], (float)p.amplitude) : make_float2(1.f, 0.f);
    pdl_wait_release();
    const float* src = p.qkv + (size_t)t * width + (size_t)h0 * p.hd;
    S* dst = (S*)p.q_out + ((size_t)t * p.nh + h0) * p.hd;
    float a[AP_HEADS][NP], b[AP_HEADS][NP];
#pragma unroll
    for (int h = 0; h < AP_HEADS; ++h)
      if (h0 + h < p.nh) mine.load(src + h * p.hd, a[h], b[h]);
#pragma unroll
    for (int h = 0; h < AP_HEADS; ++h)
      if (h0 + h < p.nh) {
        float x[NP], y[NP];
#pragma unroll
        for (int k = 0; k < NP; ++k) {
          const float2 cs = turned_by[k];
          x[k] = mine.turned(k) ? a[h][k] * cs.x - b[h][k] * cs.y : a[h][k];
          y[k] = mine.turned(k) ? a[h][k] * cs.y + b[h][k] * cs.x : b[h][k];
        }
        mine.store(dst + h * p.hd, x, y);
      }
    return;
  }

  // ---- keys and values.  Where positions, requests and block tables come by copies (`early`), all that follows from them
  // passes under the kernel in front. --------------------------------------------------------------------------------------
  // Of the window's tokens and those behind it that may belong to its runs: what a thread finds out for all.
  __shared__ unsigned starts[AP_WARPS], bad[AP_WARPS];    // does a run begin there; does it break the order
  __shared__ int poss[AP_WARPS * 32], offs[AP_WARPS * 32];
  __shared__ int runs[AP_WARPS * 32];                     // the run's first token
  __shared__ int pages[AP_WARPS * 32];                    // of a run, at its first token: page (-1: none), ...
  __shared__ unsigned olds[AP_WARPS * 32];                // ... bits of the scale it had (0 when the run begins the page), ...
  __shared__ unsigned tops[AP_WARPS * 32];                // ... bits of its largest magnitude
  const int kv = blockIdx.x % (2 * p.nkv), is_v = kv & 1, h = kv >> 1;
  const int t0 = (int)(blockIdx.x / (2 * p.nkv)) * AP_WINDOW;
  const int reach = min(AP_WINDOW + p.page_size, p.T - t0);
  const int me = threadIdx.x;
  int seq = 0, pos = 0, place = 0;
  {
    bool start = true, wrong = false;                     // what lies behind the reach ends every run
    if (me < reach) {
      seq = p.token_seq[t0 + me];
      pos = p.positions[t0 + me];
      place = pos / p.page_size;
      poss[me] = pos;
      offs[me] = pos - place * p.page_size;
      if (t0 + me > 0) {
        const int before = p.token_seq[t0 + me - 1], pos_before = p.positions[t0 + me - 1];
        wrong = before > seq || (before == seq && pos_before + 1 != pos);
        start = wrong || before != seq || offs[me] == 0;
      }
      if (wrong && me < AP_WINDOW) atomicExch(p.status, 5);
    }
    const unsigned s = __ballot_sync(0xffffffffu, start), w = __ballot_sync(0xffffffffu, wrong);
    if (lane == 0) {
      starts[warp] = s;
      bad[warp] = w;
    }
  }
  __syncthreads();
  // the block's tokens: from the first run that begins in the window to the end of the last one that does
  const unsigned in_window = starts[0] & 0xffffu;
  const int first = __ffs(in_window) - 1;
  if (first < 0 || first >= reach) return;
  int last = reach;
  if (starts[0] >> AP_WINDOW) {
    last = min(reach, AP_WINDOW + __ffs(starts[0] >> AP_WINDOW) - 1);
  } else {
    for (int w = 1; w < AP_WARPS; ++w)
      if (starts[w]) {
        last = min(reach, w * 32 + __ffs(starts[w]) - 1);
        break;
      }
  }
  const float* src = p.qkv + (size_t)t0 * width + (size_t)(p.nh + (is_v ? p.nkv : 0) + h) * p.hd;
  auto load = [&](int i, float (&a)[NP], float (&b)[NP]) { mine.load(src + (size_t)i * width, a, b); };
  const bool coded = p.k_scale != nullptr;
  float* scale = is_v ? p.v_scale : p.k_scale;
  int owned = -2;                                         // page of the run that this thread's token begins
  if (me >= first && me < last) {
    int w = me >> 5;
    unsigned m = starts[w] & (0xffffffffu >> (31 - (me & 31)));
    while (!m) m = starts[--w];                           // `first` begins a run
    const int s = w * 32 + 31 - __clz(m);
    runs[me] = s;
    if (s == me) {
      int page = -1;
      if (!((bad[me >> 5] >> (me & 31)) & 1u)) {
        if (pos >= 0 && place < p.max_pages) page = p.block_table[(size_t)seq * p.max_pages + place];
        if (page < 0 || page >= p.num_pages) {
          atomicExch(p.status, 2);
          page = -1;
        }
      }
      pages[me] = page;
      tops[me] = 0u;
      owned = page;
    }
  }
  pdl_wait_release();
  float a[AP_HELD][NP], b[AP_HELD][NP];
#pragma unroll
  for (int c = 0; c < AP_HELD; ++c)
    if (first + warp + c * AP_WARPS < last) load(first + warp + c * AP_WARPS, a[c], b[c]);
  if (owned > -2) olds[me] = coded && owned >= 0 && offs[me] ? __float_as_uint(scale[(size_t)owned * p.nkv + h]) & 0x7fffffffu : 0u;
  __syncthreads();
  auto rotate = [&](int i, float (&x)[NP], float (&y)[NP]) {
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      if (!is_v && mine.turned(k)) {
        const float2 cs = rope_angle(poss[i], turns[k], (float)p.amplitude);
        const float u = x[k], v = y[k];
        x[k] = u * cs.x - v * cs.y;
        y[k] = u * cs.y + v * cs.x;
      }
    }
  };
  // The largest magnitude of token i's values in this lane, as bits.  Next to a power of two, where it decides the scale,
  // that of the pairs turned in 64 bits, cut to 32 (which keeps its exponent).
  auto magnitude = [&](int i, const float (&x)[NP], const float (&y)[NP]) {
    unsigned m = 0;
#pragma unroll
    for (int k = 0; k < NP; ++k) m = max(m, max(__float_as_uint(x[k]) & 0x7fffffffu, __float_as_uint(y[k]) & 0x7fffffffu));
    if (!is_v && coded && c8_near_scale(m)) {
      const float* row = src + (size_t)i * width;
      m = 0;
      for (int k = 0; k < NP; ++k) {
        if (!mine.in(k)) continue;
        const int2 d = mine.dims(k);
        double2 u = make_double2(row[d.x], row[d.y]);
        if (mine.turned(k)) u = rope_exact(poss[i], p.turns[mine.pair(k)], p.amplitude, row[d.x], row[d.y]);
        m = max(m, __float_as_uint(__double2float_rz(fmax(fabs(u.x), fabs(u.y)))));
      }
    }
    return m;
  };
#pragma unroll
  for (int c = 0; c < AP_HELD; ++c) {
    const int i = first + warp + c * AP_WARPS;
    if (i >= last) continue;
    rotate(i, a[c], b[c]);
    const unsigned m = __reduce_max_sync(0xffffffffu, magnitude(i, a[c], b[c]));
    if (lane == 0) atomicMax(&tops[runs[i]], m);
  }
  for (int i = first + warp + AP_HELD * AP_WARPS; i < last; i += AP_WARPS) {    // a run cut by the window, pages of many rows
    float x[NP], y[NP];
    load(i, x, y);
    rotate(i, x, y);
    const unsigned m = __reduce_max_sync(0xffffffffu, magnitude(i, x, y));
    if (lane == 0) atomicMax(&tops[runs[i]], m);
  }
  __syncthreads();
  // returns the pairs whose codes have to be looked at again
  auto store = [&](int i, const float (&x)[NP], const float (&y)[NP]) -> unsigned {
    const int s = runs[i], page = pages[s];
    if (page < 0) return 0u;
    const size_t row = ((size_t)page * p.nkv + h) * p.page_size;
    if (!coded) {
      mine.store((S*)(is_v ? p.v_pool : p.k_pool) + (row + offs[i]) * p.hd, x, y);
      return 0u;
    }
    const unsigned m = tops[s], before = olds[s];
    const int off0 = offs[s];
    const bool finite = m < C8_NOT_FINITE && before < C8_NOT_FINITE;
    const int e_old = (int)(before >> 23) - 127;
    const int e = off0 > 0 ? max(c8_exponent(m), e_old) : c8_exponent(m);
    uint8_t* dst = (uint8_t*)(is_v ? p.v_pool : p.k_pool) + row * p.hd;
    if (i == s) {
      if (lane == 0) scale[(size_t)page * p.nkv + h] = finite ? c8_pow2(e) : __int_as_float(0x7fc00000);
      if (finite && off0 > 0 && e > e_old) {              // the rows before move to the new scale
        const int d = min(e - e_old, 7);
        if constexpr (FULL) {
          uint4* q = reinterpret_cast<uint4*>(dst);
          for (int j = lane; j < off0 * (4 * NP); j += 32) {
            const uint4 v = q[j];
            q[j] = make_uint4(shift_codes(v.x, d), shift_codes(v.y, d), shift_codes(v.z, d), shift_codes(v.w, d));
          }
        } else {
          uint16_t* q = reinterpret_cast<uint16_t*>(dst);
          for (int j = lane; j < off0 * pairs; j += 32) q[j] = (uint16_t)shift_codes(q[j], d);
        }
      }
    }
    dst += (size_t)offs[i] * p.hd;
    const float inv = c8_pow2(-e);
    unsigned cx[NP], cy[NP];
#pragma unroll
    for (int k = 0; k < NP; ++k) {
      cx[k] = finite ? c8_code(x[k], inv) : 128u;
      cy[k] = finite ? c8_code(y[k], inv) : 128u;
    }
    unsigned near = 0;
    if (!is_v && finite) {
#pragma unroll
      for (int k = 0; k < NP; ++k)
        if (fminf(c8_distance(x[k], inv), c8_distance(y[k], inv)) < C8_NEAR) near |= 1u << k;
    }
    mine.store(dst, cx, cy);
    return near;
  };
  auto again = [&](int i, unsigned near) {
    const int r = runs[i];
    const float* row = src + (size_t)i * width;
    uint8_t* dst = (uint8_t*)p.k_pool + (((size_t)pages[r] * p.nkv + h) * p.page_size + offs[i]) * p.hd;
    const int e = max(c8_exponent(tops[r]), offs[r] > 0 ? (int)(olds[r] >> 23) - 127 : C8_LOWEST);
    const double inv = (double)c8_pow2(-e);
    for (; near; near &= near - 1) {
      const int k = __ffs(near) - 1;
      if (!mine.turned(k)) continue;
      const int2 d = mine.dims(k);
      const float a = row[d.x], b = row[d.y];
      if (a == 0.f && b == 0.f) continue;
      const double2 u = rope_exact(poss[i], p.turns[mine.pair(k)], p.amplitude, a, b);
      dst[d.x] = (uint8_t)c8_code(u.x, inv);
      dst[d.y] = (uint8_t)c8_code(u.y, inv);
    }
  };
  unsigned near[AP_HELD] = {};
#pragma unroll
  for (int c = 0; c < AP_HELD; ++c)
    if (first + warp + c * AP_WARPS < last) near[c] = store(first + warp + c * AP_WARPS, a[c], b[c]);
#pragma unroll
  for (int c = 0; c < AP_HELD; ++c)
    if (near[c]) again(first + warp + c * AP_WARPS, near[c]);
  for (int i = first + warp + AP_HELD * AP_WARPS; i < last; i += AP_WARPS) {
    float x[NP], y[NP];
    load(i, x, y);
    rotate(i, x, y);
    const unsigned some = store(i, x, y);
    if (some) again(i, some);
  }
}

// ---- any head size -------------------------------------------------------------------------------------------------
// Element d of a head of token t (row of hd floats), rotated (in 64 bits: these sizes are not those that count).
__device__ __forceinline__ double rope_element(const AppendParams& p, const float* row, int pos, int d) {
  if (d >= p.rot) return row[d];
  const int half = p.rot >> 1;
  const int j = p.interleaved ? d >> 1 : (d < half ? d : d - half);
  const int ia = p.interleaved ? 2 * j : j, ib = p.interleaved ? 2 * j + 1 : j + half;
  const double2 r = rope_exact(pos, p.turns[j], p.amplitude, row[ia], row[ib]);
  return d == ia ? r.x : r.y;
}

// Grid (tokens, 1 + 2 kv heads): y = 0 rotates the token's queries; y = 1 + 2 h + w writes keys (w = 0) or values
// of kv head h, for the whole run of tokens of the request that lie in one page, in the block of the run's first token.
template <typename S>
__global__ void __launch_bounds__(128) rope_append_simple_kernel(const AppendParams p) {
  __shared__ unsigned top[4];
  pdl_wait_release();
  const int t0 = blockIdx.x;
  const int width = (p.nh + 2 * p.nkv) * p.hd;
  const int pos0 = p.positions[t0];
  if (blockIdx.y == 0) {
    const float* row = p.qkv + (size_t)t0 * width;
    S* q = (S*)p.q_out + (size_t)t0 * p.nh * p.hd;
    for (int i = threadIdx.x; i < p.nh * p.hd; i += blockDim.x) {
      const int head = i / p.hd;
      q[i] = from_float<S>((float)rope_element(p, row + head * p.hd, pos0, i - head * p.hd));
    }
    return;
  }
  const int is_v = (blockIdx.y - 1) & 1, h = (blockIdx.y - 1) >> 1;
  const int seq = p.token_seq[t0];
  const int place = pos0 / p.page_size, off0 = pos0 - place * p.page_size;
  if (t0 > 0) {
    const int before = p.token_seq[t0 - 1], pos_before = p.positions[t0 - 1];
    if (before > seq || (before == seq && pos_before + 1 != pos0)) {
      if (threadIdx.x == 0) atomicExch(p.status, 5);
      return;
    }
    if (before == seq && pos_before / p.page_size == place) return;       // not the first of its run
  }
  const int page = pos0 < 0 || place >= p.max_pages ? -1 : p.block_table[(size_t)seq * p.max_pages + place];
  if (page < 0 || page >= p.num_pages) {
    if (threadIdx.x == 0) atomicExch(p.status, 2);
    return;
  }
  int n = 1;
  while (off0 + n < p.page_size && t0 + n < p.T && p.token_seq[t0 + n] == seq && p.positions[t0 + n] == pos0 + n) ++n;
  const float* src = p.qkv + (size_t)t0 * width + (size_t)(p.nh + (is_v ? p.nkv : 0) + h) * p.hd;
  const size_t at = ((size_t)page * p.nkv + h) * p.page_size;              // row of the pool
  auto element = [&](int i) -> double {
    const int r = i / p.hd, d = i - r * p.hd;
    return is_v ? (double)src[(size_t)r * width + d] : rope_element(p, src + (size_t)r * width, pos0 + r, d);
  };
  if (!p.k_scale) {
    S* dst = (S*)(is_v ? p.v_pool : p.k_pool) + (at + off0) * p.hd;
    for (int i = threadIdx.x; i < n * p.hd; i += blockDim.x) dst[i] = from_float<S>((float)element(i));
    return;
  }
  uint8_t* dst = (uint8_t*)(is_v ? p.v_pool : p.k_pool) + at * p.hd;
  float* scale = (is_v ? p.v_scale : p.k_scale) + (size_t)page * p.nkv + h;
  unsigned mine = 0;
  for (int i = threadIdx.x; i < n * p.hd; i += blockDim.x) mine = max(mine, __float_as_uint(__double2float_rz(element(i))) & 0x7fffffffu);
  mine = __reduce_max_sync(0xffffffffu, mine);
  if ((threadIdx.x & 31) == 0) top[threadIdx.x >> 5] = mine;
  const unsigned old = off0 > 0 ? __float_as_uint(*scale) & 0x7fffffffu : 0u;
  __syncthreads();
  mine = max(max(top[0], top[1]), max(top[2], top[3]));
  const bool finite = mine < C8_NOT_FINITE && old < C8_NOT_FINITE;
  const int e_old = (int)(old >> 23) - 127;
  const int e = off0 > 0 ? max(c8_exponent(mine), e_old) : c8_exponent(mine);
  if (threadIdx.x == 0) *scale = finite ? c8_pow2(e) : __int_as_float(0x7fc00000);
  if (finite && off0 > 0 && e > e_old) {
    const int d = min(e - e_old, 7);
    for (int i = threadIdx.x; i < off0 * p.hd; i += blockDim.x) dst[i] = (uint8_t)shift_codes(dst[i], d);
  }
  const float inv = c8_pow2(-e);
  for (int i = threadIdx.x; i < n * p.hd; i += blockDim.x)
    dst[off0 * p.hd + i] = finite ? (uint8_t)c8_code(element(i), (double)inv) : (uint8_t)128;
}

struct UnpackParams {
  const uint8_t* k;
  const uint8_t* v;
  const float* k_scale;
  const float* v_scale;
  const int* seq_start;
  const int* cu_seqlens;
  const int* block_table;
  void* k_out;
  void* v_out;
  int* status;
  int max_pages, window, nkv, page_elems, page_size, num_pages, early;
};

// A page that a request can reach: its place in the pools, -1 if there is none.
__device__ __forceinline__ int unpack_page(const UnpackParams& p, int r, int ordinal) {
  const int start = p.seq_start[r], n = p.cu_seqlens[r + 1] - p.cu_seqlens[r];
  if (n <= 0) return -1;
  const int lo = p.window > 0 && start - p.window + 1 > 0 ? (start - p.window + 1) / p.page_size : 0;
  const int place = lo + ordinal, last = (start + n - 1) / p.page_size;
  if (place > last) return -1;
  if (ordinal == (int)gridDim.x - 1 && place < last && threadIdx.x == 0) atomicExch(p.status, 6);    // the rest stays as it was
  const int page = place >= p.max_pages ? -1 : p.block_table[(size_t)r * p.max_pages + place];
  if (page < 0 || page >= p.num_pages) {
    if (threadIdx.x == 0) atomicExch(p.status, 3);
    return -1;
  }
  return page;
}

// The scales of a page as the readers take them.  One that is not finite becomes NaN keys and finite values: a query
// that sees the page gets NaN, and a tile that holds it behind a mask (probability 0) gets no 0 x NaN from its values.
__device__ __forceinline__ float2 unpack_scales(const UnpackParams& p, size_t at) {
  float ks = p.k_scale[at], vs = p.v_scale[at];
  if (!(fabsf(vs) <= 3.4e38f)) {
    ks = __int_as_float(0x7fc00000);
    vs = 0.f;
  }
  if (!(fabsf(ks) <= 3.4e38f)) ks = __int_as_float(0x7fc00000);
  return make_float2(ks, vs);
}

// Four codes as values, exactly: a byte permutation puts a code c under the exponent of 2^15 as 32768 + c.
__device__ __forceinline__ float widen(uint32_t raised, float s) { return (__uint_as_float(raised) - 32895.5f) * s; }
__device__ __forceinline__ float4 widen4(uint32_t w, float s) {
  const uint32_t under = 0x47000000u;
  return make_float4(widen(__byte_perm(w, under, 0x7404), s), widen(__byte_perm(w, under, 0x7414), s),
                     widen(__byte_perm(w, under, 0x7424), s), widen(__byte_perm(w, under, 0x7434), s));
}
__device__ __forceinline__ void store16(__nv_bfloat16* to, const float4 (&v)[4]) {
  uint4* t = reinterpret_cast<uint4*>(to);
  t[0] = make_uint4(pack_bf16(v[0].x, v[0].y), pack_bf16(v[0].z, v[0].w), pack_bf16(v[1].x, v[1].y), pack_bf16(v[1].z, v[1].w));
  t[1] = make_uint4(pack_bf16(v[2].x, v[2].y), pack_bf16(v[2].z, v[2].w), pack_bf16(v[3].x, v[3].y), pack_bf16(v[3].z, v[3].w));
}
__device__ __forceinline__ void store16(float* to, const float4 (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) reinterpret_cast<float4*>(to)[i] = v[i];
}

// Memory-bound: a byte read and two written per element (8,150 keys of 8 heads of 256, 100 MB: 16.9 us = 5.9 TB/s, the part of
// it that stays in L2 included; 4,096 keys 10.5 us, of which 3 are the launch's start and end).  Grid (pages of the longest range,
// requests, parts of 8192 elements of a page's keys, then of its values): a page's heads lie one behind the other, a thread
// takes 16 codes at a time of one of them (a page of a head is a multiple of 16 elements).
constexpr int UP_THREADS = 256;                   // 128: a mixed step 8.1 instead of 6.4 us; 512: 2,282 tokens 13.7 instead of 13.0
constexpr int UP_EACH = 2;                        // sixteens of a thread; 1: 16.5 instead of 13.0, 4: 15.0

template <typename S>
__global__ void __launch_bounds__(UP_THREADS) cache8_unpack_kernel(const UnpackParams p, int parts) {
  if (!p.early) pdl_wait();
  const int page = unpack_page(p, blockIdx.y, blockIdx.x);
  pdl_wait_release();
  if (page < 0) return;
  const int is_v = (int)blockIdx.z >= parts;
  const int first = ((int)blockIdx.z - (is_v ? parts : 0)) * (UP_THREADS * UP_EACH) + (int)threadIdx.x;
  const int sixteens = p.nkv * (p.page_elems >> 4), per_head = p.page_elems >> 4;
  const size_t base = (size_t)page * sixteens;
  const uint4* from = reinterpret_cast<const uint4*>(is_v ? p.v : p.k) + base;
  S* to = (S*)(is_v ? p.v_out : p.k_out) + base * 16;
  uint4 c[UP_EACH];
#pragma unroll
  for (int j = 0; j < UP_EACH; ++j)
    if (first + j * UP_THREADS < sixteens) c[j] = from[first + j * UP_THREADS];
#pragma unroll
  for (int j = 0; j < UP_EACH; ++j) {
    const int i = first + j * UP_THREADS;
    if (i >= sixteens) break;
    const float2 both = unpack_scales(p, (size_t)page * p.nkv + i / per_head);
    const float s = is_v ? both.y : both.x;
    const float4 v[4] = {widen4(c[j].x, s), widen4(c[j].y, s), widen4(c[j].z, s), widen4(c[j].w, s)};
    store16(to + (size_t)i * 16, v);
  }
}

// Any size, element by element.  Grid (pages of the longest request, kv heads, requests): the pages that the request's new
// tokens can reach, each to its own place in the wide pools.
template <typename S>
__global__ void __launch_bounds__(256) cache8_unpack_simple_kernel(const UnpackParams p) {
  pdl_wait_release();
  const int page = unpack_page(p, blockIdx.z, blockIdx.x);
  if (page < 0) return;
  const size_t at = (size_t)page * p.nkv + blockIdx.y;
  const float2 scale = unpack_scales(p, at);
  const size_t base = at * p.page_elems;
  for (int i = threadIdx.x; i < p.page_elems; i += blockDim.x) {
    ((S*)p.k_out)[base + i] = from_float<S>(((float)p.k[base + i] - 127.5f) * scale.x);
    ((S*)p.v_out)[base + i] = from_float<S>(((float)p.v[base + i] - 127.5f) * scale.y);
  }
}

}  // namespace glint

using namespace glint;

#define C8_DISPATCH(dtype, ...)                              \
  if ((dtype) == GLINT_DTYPE_F32) { using S = float; __VA_ARGS__; } \
  else if ((dtype) == GLINT_DTYPE_BF16) { using S = __nv_bfloat16; __VA_ARGS__; } \
  else return GLINT_ERR_BAD_ARG;

// qkv [T][nh + 2 nkv][hd] float32: the first `rot` dims of every query and key head are turned in pairs, (j, j + rot/2)
// or, interleaved, (2 j, 2 j + 1), by positions[t] * turns[j] of a full turn, scaled by `amplitude`; queries go to
// q_out, keys and values to the pages: coded when there are scales, else in `dtype`.  k_pool null: queries only.
// The tokens of a request stand together in ascending positions (status 5 otherwise).  `early`: positions, requests, block
// tables and turns were on the device before the kernel in front began (copies, not a kernel's results).
GLINT_API int glint_rope_append(const float* qkv, const int* positions, const int* token_seq, const int* block_table,
                                int max_pages, const double* turns, int rot, int interleaved, double amplitude, void* q_out,
                                int dtype, void* k_pool, void* v_pool, float* k_scale, float* v_scale, int T, int nh,
                                int nkv, int hd, int page_size, int num_pages, int* status, int early, cudaStream_t stream) {
  if (T <= 0) return GLINT_OK;
  if (hd <= 0 || hd % 2 || rot % 2 || rot < 0 || rot > hd || nh <= 0 || nkv <= 0 || page_size <= 0) return GLINT_ERR_BAD_ARG;
  if (!k_pool != !v_pool || !k_scale != !v_scale || (k_scale && !k_pool)) return GLINT_ERR_BAD_ARG;
  if (k_scale && (((uintptr_t)k_pool | (uintptr_t)v_pool) & 1)) return GLINT_ERR_BAD_ARG;      // codes are moved in pairs
  if (nkv > 32767) return GLINT_ERR_UNSUPPORTED_SIZE;
  AppendParams p = {qkv, positions, token_seq, block_table, turns, q_out, k_pool, v_pool, k_scale, v_scale, status, amplitude,
                    T, nh, nkv, hd, rot, interleaved ? 1 : 0, page_size, num_pages, max_pages, early};
  cudaError_t e = cudaSuccess;
  if (hd <= 256 && page_size <= AP_MOST_PAGE) {
    const long long cache_blocks = k_pool ? (long long)((T + AP_WINDOW - 1) / AP_WINDOW) * 2 * nkv : 0;
    const long long units = (long long)T * ((nh + AP_HEADS - 1) / AP_HEADS);
    const long long blocks = cache_blocks + (units + AP_WARPS - 1) / AP_WARPS;
    if (blocks > 0x7fffffffLL) return GLINT_ERR_UNSUPPORTED_SIZE;
    const dim3 grid((unsigned)blocks), block(AP_WARPS * 32);
    const int cb = (int)cache_blocks;
#define APPEND(NP, FULL) C8_DISPATCH(dtype, e = launch_kernel(rope_append_kernel<S, NP, FULL>, grid, block, 0, stream, p, cb))
    const bool full = hd % 64 == 0 && rot % (hd / 32) == 0 && !(((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15);
    if (hd == 64 && full) { APPEND(1, true) }
    else if (hd == 128 && full) { APPEND(2, true) }
    else if (hd == 256 && full) { APPEND(4, true) }
    else if (hd <= 64) { APPEND(1, false) }
    else if (hd <= 128) { APPEND(2, false) }
    else { APPEND(4, false) }
#undef APPEND
  } else {
    const dim3 grid(T, k_pool ? 1 + 2 * nkv : 1);
    C8_DISPATCH(dtype, e = launch_kernel(rope_append_simple_kernel<S>, grid, dim3(128), 0, stream, p))
  }
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

// Codes of the pages that the new tokens of each request can reach (from the page of the first key that the first of
// them sees, to the page of the last of them) as values of `dtype`, at the same places of the wide pools.
// `most_pages`: at least the pages of any request's range (status 6 where it is less).  `early` as for glint_rope_append.
GLINT_API int glint_cache8_unpack(const uint8_t* k, const uint8_t* v, const float* k_scale, const float* v_scale,
                                  const int* seq_start, const int* cu_seqlens, const int* block_table, int max_pages,
                                  void* k_out, void* v_out, int dtype, int n_seqs, int most_pages, int window, int nkv,
                                  int hd, int page_size, int num_pages, int* status, int early, cudaStream_t stream) {
  if (n_seqs <= 0 || most_pages <= 0) return GLINT_OK;
  if (nkv <= 0 || hd <= 0 || page_size <= 0 || (long long)page_size * hd > 0x7fffffffLL) return GLINT_ERR_BAD_ARG;
  if (nkv > 65535 || n_seqs > 65535) return GLINT_ERR_UNSUPPORTED_SIZE;
  UnpackParams p = {k, v, k_scale, v_scale, seq_start, cu_seqlens, block_table, k_out, v_out, status, max_pages, window, nkv,
                    page_size * hd, page_size, num_pages, early};
  cudaError_t e = cudaSuccess;
  const long long parts = ((long long)nkv * page_size * hd / 16 + UP_THREADS * UP_EACH - 1) / (UP_THREADS * UP_EACH);
  const bool aligned = !(((uintptr_t)k | (uintptr_t)v | (uintptr_t)k_out | (uintptr_t)v_out) & 15);
  if ((long long)page_size * hd % 16 == 0 && aligned && 2 * parts <= 65535) {
    const dim3 grid(most_pages, n_seqs, (unsigned)(2 * parts));
    C8_DISPATCH(dtype, e = launch_kernel(cache8_unpack_kernel<S>, grid, dim3(UP_THREADS), 0, stream, p, (int)parts))
  } else {
    const dim3 grid(most_pages, nkv, n_seqs);
    C8_DISPATCH(dtype, e = launch_kernel(cache8_unpack_simple_kernel<S>, grid, dim3(256), 0, stream, p))
  }
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}
