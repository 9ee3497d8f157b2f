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
  float amplitude;
  int T, nh, nkv, hd, rot, interleaved, page_size, num_pages, max_pages;
};

// (cos, sin) of 2 pi pos turns, times the amplitude.  The product is taken in 64 bits and reduced to half a turn either
// way before anything is rounded to 32: at position 100,000 the 32-bit product alone is off by 4e-3 radians.
__device__ __forceinline__ float2 rope_angle(int pos, double turns, float amplitude) {
  const double t = (double)pos * turns;
  float s, c;
  sincospif((float)(2.0 * (t - rint(t))), &s, &c);
  return make_float2(c * amplitude, s * amplitude);
}

// Element d of a head of token t (row of hd floats), rotated.
__device__ __forceinline__ float rope_element(const AppendParams& p, const float* row, int pos, int d) {
  if (d >= p.rot) return row[d];
  const int half = p.rot >> 1;
  const int j = p.interleaved ? d >> 1 : (d < half ? d : d - half);
  const int ia = p.interleaved ? 2 * j : j, ib = p.interleaved ? 2 * j + 1 : j + half;
  const float2 cs = rope_angle(pos, p.turns[j], p.amplitude);
  const float a = row[ia], b = row[ib];
  return d == ia ? a * cs.x - b * cs.y : a * cs.y + b * cs.x;
}

// Grid (tokens, 1 + 2 kv heads): y = 0 rotates the token's queries; y = 1 + 2 h + w writes keys (w = 0) or values
// of kv head h, for the whole run of tokens of the request that lie in one page, in the block of the run's first token.
template <typename S>
__global__ void __launch_bounds__(128) rope_append_simple_kernel(const AppendParams p) {
  __shared__ unsigned top[4];
  const int t0 = blockIdx.x;
  const int width = (p.nh + 2 * p.nkv) * p.hd;
  const int pos0 = p.positions[t0];
  if (blockIdx.y == 0) {
    const float* row = p.qkv + (size_t)t0 * width;
    S* q = (S*)p.q_out + (size_t)t0 * p.nh * p.hd;
    for (int i = threadIdx.x; i < p.nh * p.hd; i += blockDim.x) {
      const int head = i / p.hd;
      q[i] = from_float<S>(rope_element(p, row + head * p.hd, pos0, i - head * p.hd));
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
  auto element = [&](int i) -> float {
    const int r = i / p.hd, d = i - r * p.hd;
    return is_v ? src[(size_t)r * width + d] : rope_element(p, src + (size_t)r * width, pos0 + r, d);
  };
  if (!p.k_scale) {
    S* dst = (S*)(is_v ? p.v_pool : p.k_pool) + (at + off0) * p.hd;
    for (int i = threadIdx.x; i < n * p.hd; i += blockDim.x) dst[i] = from_float<S>(element(i));
    return;
  }
  uint8_t* dst = (uint8_t*)(is_v ? p.v_pool : p.k_pool) + at * p.hd;
  float* scale = (is_v ? p.v_scale : p.k_scale) + (size_t)page * p.nkv + h;
  unsigned mine = 0;
  for (int i = threadIdx.x; i < n * p.hd; i += blockDim.x) mine = max(mine, __float_as_uint(element(i)) & 0x7fffffffu);
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
    const int d = min(e - e_old, 31);
    for (int i = threadIdx.x; i < off0 * p.hd; i += blockDim.x) dst[i] = (uint8_t)((((int)dst[i] - 128) >> d) + 128);
  }
  const float inv = c8_pow2(-e);
  for (int i = threadIdx.x; i < n * p.hd; i += blockDim.x)
    dst[off0 * p.hd + i] = finite ? (uint8_t)c8_code(element(i), inv) : (uint8_t)128;
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
  int max_pages, window, nkv, page_elems, page_size, num_pages;
};

// Grid (pages of the longest request, kv heads, requests): the pages that the request's new tokens can reach, each to
// its own place in the wide pools.  A page whose scale is not finite gives NaN keys and finite values: a query that
// sees it gets NaN, and a tile that holds it behind a mask (probability 0) gets no 0 x NaN from its values.
template <typename S>
__global__ void __launch_bounds__(256) cache8_unpack_simple_kernel(const UnpackParams p) {
  const int r = blockIdx.z, h = blockIdx.y;
  const int start = p.seq_start[r], n = p.cu_seqlens[r + 1] - p.cu_seqlens[r];
  if (n <= 0) return;
  const int lo = p.window > 0 && start - p.window + 1 > 0 ? (start - p.window + 1) / p.page_size : 0;
  const int place = lo + (int)blockIdx.x;
  if (place > (start + n - 1) / p.page_size) return;
  const int page = place >= p.max_pages ? -1 : p.block_table[(size_t)r * p.max_pages + place];
  if (page < 0 || page >= p.num_pages) {
    if (threadIdx.x == 0) atomicExch(p.status, 3);
    return;
  }
  const size_t at = (size_t)page * p.nkv + h;
  float ks = p.k_scale[at], vs = p.v_scale[at];
  if (!(fabsf(vs) <= 3.4e38f)) {
    ks = __int_as_float(0x7fc00000);
    vs = 0.f;
  }
  if (!(fabsf(ks) <= 3.4e38f)) ks = __int_as_float(0x7fc00000);
  const size_t base = at * p.page_elems;
  for (int i = threadIdx.x; i < p.page_elems; i += blockDim.x) {
    ((S*)p.k_out)[base + i] = from_float<S>(((float)p.k[base + i] - 127.5f) * ks);
    ((S*)p.v_out)[base + i] = from_float<S>(((float)p.v[base + i] - 127.5f) * vs);
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
// The tokens of a request stand together in ascending positions (status 5 otherwise).
GLINT_API int glint_rope_append(const float* qkv, const int* positions, const int* token_seq, const int* block_table,
                                int max_pages, const double* turns, int rot, int interleaved, float amplitude, void* q_out,
                                int dtype, void* k_pool, void* v_pool, float* k_scale, float* v_scale, int T, int nh,
                                int nkv, int hd, int page_size, int num_pages, int* status, cudaStream_t stream) {
  if (T <= 0) return GLINT_OK;
  if (hd <= 0 || hd % 2 || rot % 2 || rot < 0 || rot > hd || nh <= 0 || nkv <= 0 || page_size <= 0) return GLINT_ERR_BAD_ARG;
  if (!k_pool != !v_pool || !k_scale != !v_scale || (k_scale && !k_pool)) return GLINT_ERR_BAD_ARG;
  if (nkv > 32767) return GLINT_ERR_UNSUPPORTED_SIZE;
  AppendParams p = {qkv, positions, token_seq, block_table, turns, q_out, k_pool, v_pool, k_scale, v_scale, status, amplitude,
                    T, nh, nkv, hd, rot, interleaved ? 1 : 0, page_size, num_pages, max_pages};
  const dim3 grid(T, k_pool ? 1 + 2 * nkv : 1);
  C8_DISPATCH(dtype, rope_append_simple_kernel<S><<<grid, 128, 0, stream>>>(p));
  return (int)cudaGetLastError();
}

// Codes of the pages that the new tokens of each request can reach (from the page of the first key that the first of
// them sees, to the page of the last of them) as values of `dtype`, at the same places of the wide pools.
// `most_pages`: at least the pages of any request's range.
GLINT_API int glint_cache8_unpack(const uint8_t* k, const uint8_t* v, const float* k_scale, const float* v_scale,
                                  const int* seq_start, const int* cu_seqlens, const int* block_table, int max_pages,
                                  void* k_out, void* v_out, int dtype, int n_seqs, int most_pages, int window, int nkv,
                                  int hd, int page_size, int num_pages, int* status, cudaStream_t stream) {
  if (n_seqs <= 0 || most_pages <= 0) return GLINT_OK;
  if (nkv <= 0 || hd <= 0 || page_size <= 0 || (long long)page_size * hd > 0x7fffffffLL) return GLINT_ERR_BAD_ARG;
  if (nkv > 65535 || n_seqs > 65535) return GLINT_ERR_UNSUPPORTED_SIZE;
  UnpackParams p = {k, v, k_scale, v_scale, seq_start, cu_seqlens, block_table, k_out, v_out, status, max_pages, window, nkv,
                    page_size * hd, page_size, num_pages};
  const dim3 grid(most_pages, nkv, n_seqs);
  C8_DISPATCH(dtype, cache8_unpack_simple_kernel<S><<<grid, 256, 0, stream>>>(p));
  return (int)cudaGetLastError();
}
