// Attention of prompt portions over wide pages on the 5th-generation tensor cores, for the coded cache: its pages are
// widened in front (cache8.cu), this kernel reads them.
//
// A block owns 128 query rows, rows being (token, query head of the group) pairs, and walks their keys in tiles of 64.
// What bounds such a walk here is not the products (a tile of head size 256 takes the tensor pipe 0.55 us) but the soft cap
// and the exponential of 8,192 scores, two operations of the special-function unit each: 0.55 us of its time if it
// never pauses.  So nothing waits that need not:
//   warps 0, 3 TMA: the query tile once and key tiles; value tiles: page by page into rings as deep as shared memory allows
//              (head size 256: three tiles of keys, two of values)
//   warp 1     tcgen05.mma: S = Q K^T into one of two score buffers of tensor memory, as soon as that has been read.  With
//              64 keys a tile, products from shared memory alone read Q again for every tile (head size 256: 64 KB beside 64
//              of K and V read and 64 written, 1,536 cycles of shared memory, about the tile's time), so the first 128 dims
//              of Q lie in tensor memory where there is room (4,096 tokens 136.6 -> 133.6 us)
//   warp 2     tcgen05.mma: O += P V, P (bfloat16 pairs) from one of two buffers of tensor memory
//   warps 4-7  softmax of the even tiles, warps 8-11 of the odd ones, one thread per row: no maximum or sum is exchanged
//              within a tile, and one group computes while the other loads, stores and waits
// With a soft cap of up to 55 the exponentials need no running maximum at all: scores lie within +-cap (80 log2 units), and
// probabilities relative to 2^10, between 2^-90 and 2^70, keep the precision they always have in float32 sums and as bfloat16.
// So do their products with values of up to 2^36 (a row of 2^20 keys that all reach +cap) and down to 2^-36 (one whose
// keys all stay at -cap); sums of larger ones that overflow are reported (status 7).  Otherwise the groups hand each row's
// reference from tile to tile (it follows the maximum when that has grown by more than 8 log2 units, and O is rescaled then).
// Where SMs would stay empty (fewer blocks than SMs, or a few blocks behind the last full round of them) the keys of a tile of
// rows are split over several blocks, whose partial results a second kernel adds up in order.
// Blocks are found from the portions' lengths, so that short portions beside long ones cost no empty blocks.
// 4,096 tokens, 16 heads in 8 groups of 256: 137 GFLOP in 124 us (and 10 for the wide pages) = 1.11 PFLOP/s, 0.68 of what a
// large product reaches (call after call 145 us: the power cap); tensor pipe and special-function unit are busy 55 % of the
// time.  Neither binds alone: what is left is the hand-over between the warps of a tile.
// Score = (q.k) * multiplier, then cap * tanh(score / cap) with tanh.approx: 2^-11 of a capped score, so up to 0.02 in the
// exponent of a score of 40, beside the 2^-8 of a probability's rounding.  The single-token kernel has its cap to 32 bits;
// exponential and reciprocal in place of tanh.approx would be a third special-function operation a score where two of them
// bind.  Keys of a token at position p from max(0, p - window + 1) to p.  Sums, references and accumulators are 32-bit;
// probabilities are rounded to bfloat16 for the second product, and their sum is that of the rounded ones.
#include "common.cuh"
#include "tcgen05.cuh"

namespace glint {

constexpr int AT_M = 128;             // query rows of a block
constexpr int AT_N = 64;              // keys of a tile
constexpr int AT_THREADS = 384;
constexpr int AT_Q_SUB = AT_M * 128;  // bytes of a 64-column slice of the query tile
constexpr int AT_KV_SUB = AT_N * 128;
constexpr int AT_STAGES = 4;          // most tiles of keys, or of values, in shared memory
constexpr int AT_LEAST = 4;           // key tiles of a split
constexpr float AT_GROW = 8.f;        // log2 units
constexpr float AT_FIXED_CAP = 55.f;  // largest soft cap whose exponentials need no maximum
constexpr float AT_FIXED_REF = 10.f;  // log2 units: their reference

struct PortionParams {
  const int* cu_seqlens;
  const int* seq_start;
  const int* block_table;
  __nv_bfloat16* out;
  float* part_o;                // [splits][split tiles][128][hd]
  float2* part_ml;              // [splits][split tiles][128] (reference in log2 units, sum)
  int4* part_info;              // [split tiles]: parts (below 2: nothing to add up), rows, first token, kv head
  int* status;
  float multiplier, cap;
  int max_pages, nh, nkv, hd, page_size, num_pages, window, n_seqs, whole, k_stages, v_stages;
  int split_from, splits;       // tiles (query tile, kv head) from there on have their keys split over that many blocks
  int split_tiles;              // and are that many
  int early;                    // offsets and starts are no kernel's work: read before the wait
};

struct PortionShared {
  uint64_t q_full, o_full, q_ready;
  uint64_t s_full[2], s_free[2], p_ready[2], pv_done[2], turn[2];
  uint64_t k_full[AT_STAGES], k_empty[AT_STAGES], v_full[AT_STAGES], v_empty[AT_STAGES];
  uint32_t tmem_base;
  int abort_flag;
  int part_tile;                // where this block's partial results go, in tiles of rows (-1: it has all keys)
  float row_ref[AT_M];
  float row_sum[2][AT_M];
  float row_own[2][AT_M];
};

// A wait of a whole warp: its lanes go on together (what follows is .aligned), or not at all.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, tc::mbar_wait(bar, parity, abort_flag));
}

// The query tile of a block, counted from the last: late tiles have the most keys and start first.
struct PortionTile {
  int seq, tile, begin, len, start;      // request, tile of its portion, first token, tokens, position of the first
};
// False: there are fewer.  A warp looks at 32 requests at a time; up to 32 cost one trip to memory.
__device__ __forceinline__ bool portion_tile(const PortionParams& p, int tok_per_tile, int index, PortionTile& found) {
  const int lane = threadIdx.x & 31;
  int total = 0, lo = 0, hi = 0, start = 0;
  auto look = [&](int b) -> int {        // tiles of request b + lane
    lo = hi = start = 0;
    if (b + lane < p.n_seqs) {
      lo = p.cu_seqlens[b + lane];
      hi = p.cu_seqlens[b + lane + 1];
      start = p.seq_start[b + lane];
    }
    return max(0, (hi - lo + tok_per_tile - 1) / tok_per_tile);
  };
  int n = 0;
  for (int b = 0; b < p.n_seqs; b += 32) {
    n = look(b);
    total += __reduce_add_sync(0xffffffffu, n);
  }
  int at = total - 1 - index;
  if (at < 0) return false;
  for (int b = 0; b < p.n_seqs; b += 32) {
    if (p.n_seqs > 32) n = look(b);
    int incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, at < incl);
    if (hit) {
      const int who = __ffs(hit) - 1;
      found.seq = b + who;
      found.tile = at - __shfl_sync(0xffffffffu, incl - n, who);
      found.begin = __shfl_sync(0xffffffffu, lo, who);
      found.len = __shfl_sync(0xffffffffu, hi, who) - found.begin;
      found.start = __shfl_sync(0xffffffffu, start, who);
      return true;
    }
    at -= __shfl_sync(0xffffffffu, incl, 31);
  }
  return false;
}

// The keys of a query tile, and what a split of them takes: tiles of 64, an even share of at least AT_LEAST.
struct PortionKeys {
  int pos0, pos_last, kv_first, begin, tiles, per, parts;
};
__device__ __forceinline__ PortionKeys portion_keys(const PortionParams& p, const PortionTile& w, int tok_per_tile, bool split) {
  PortionKeys k;
  const int tok0 = w.tile * tok_per_tile;
  k.pos0 = w.start + tok0;
  // a position that the block table has no room for (the widening in front has reported it) is held to its last page
  k.pos_last = (int)min((long long)k.pos0 + min(tok_per_tile, w.len - tok0) - 1, (long long)p.max_pages * p.page_size - 1);
  k.kv_first = p.window > 0 ? max(0, k.pos0 - p.window + 1) : 0;
  k.begin = k.kv_first & ~(AT_N - 1);
  k.tiles = (k.pos_last - k.begin + AT_N) / AT_N;
  k.per = split ? max(AT_LEAST, (k.tiles + p.splits - 1) / p.splits) : k.tiles;
  k.parts = split ? (k.tiles + k.per - 1) / k.per : 1;
  return k;
}

// FIXED: the soft cap spares the running maximum (with the widening, at cap 50 / without a cap / at cap 56: 4,096 tokens, 16 heads
// in 8 groups of 256, 136 / 170 / 188 us; 2,282 ragged ones, 32 heads in 16 groups of 128, 92 / 134 / 166, where the columns that
// do not fit the registers are computed twice).
// PAIR: two blocks on an SM (head sizes up to 128): each has half of the tensor memory, so that P is written over the scores
// it came from and the scores two tiles on wait for the product that reads it; one block's beginning and end pass under the
// other's tiles (the ragged portions 90 us, 105 with one block).
template <bool FIXED, bool PAIR>
__global__ void __launch_bounds__(AT_THREADS, PAIR ? 2 : 1)
attention_portion_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                         const __grid_constant__ CUtensorMap map_v, const PortionParams p) {
  extern __shared__ __align__(1024) uint8_t at_raw[];    // begins at a multiple of 1024: there is no room for less (checked)
  uint8_t* smem = at_raw;
  const int hd = p.hd, hd16 = hd >> 4, nsub = (hd + 63) >> 6;
  const int G = p.nh / p.nkv;
  const int tok_per_tile = AT_M / G;
  constexpr int TMEM_COLS = PAIR ? 256 : 512;
  uint8_t* sq = smem;
  uint8_t* sk = sq + (size_t)nsub * AT_Q_SUB;            // [stages][nsub][64 keys x 128 B]
  uint8_t* sv = sk + (size_t)p.k_stages * nsub * AT_KV_SUB;
  PortionShared* sh = reinterpret_cast<PortionShared*>(sv + (size_t)p.v_stages * nsub * AT_KV_SUB);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  {
    // a barrier per thread; arrivals of a group's rows where threads arrive, of one thread or copy elsewhere
    uint64_t* const single[] = {&sh->q_full, &sh->o_full, sh->s_full, sh->pv_done, sh->k_full, sh->k_empty, sh->v_full, sh->v_empty};
    const int many[] = {1, 1, 2, 2, AT_STAGES, AT_STAGES, AT_STAGES, AT_STAGES};
    uint64_t* const rows[] = {sh->s_free, sh->p_ready, sh->turn, &sh->q_ready};
    const int rows_many[] = {2, 2, 2, 1};
    int i = threadIdx.x;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (i >= 0 && i < many[k]) tc::mbar_init(single[k] + i, 1);
      i -= many[k];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (i >= 0 && i < rows_many[k]) tc::mbar_init(rows[k] + i, AT_M);
      i -= rows_many[k];
    }
    if (i == 0) sh->abort_flag = 0;
    if (threadIdx.x < 32) tc::fence_barrier_init();
    if (threadIdx.x == 64) tc::tma_prefetch_desc(&map_q);
    if (threadIdx.x == 65) tc::tma_prefetch_desc(&map_k);
    if (threadIdx.x == 66) tc::tma_prefetch_desc(&map_v);
  }
  __syncthreads();
  // blocks count (query tile from the last, kv head); from split_from on every such tile has `splits` blocks
  const bool may_split = (int)blockIdx.x >= p.split_from;
  const int behind = may_split ? (int)blockIdx.x - p.split_from : 0;
  const int split = may_split ? behind / p.split_tiles : 0, split_tile = behind - split * p.split_tiles;
  const int index = may_split ? p.split_from + split_tile : (int)blockIdx.x;
  const int kvh = index % p.nkv;
  if (!p.early) pdl_wait();
  PortionTile work;
  const bool found = portion_tile(p, tok_per_tile, index / p.nkv, work);
  pdl_wait();
  if (tc::smem_u32(at_raw) & 1023) {                     // the operands' swizzle wants it
    if (threadIdx.x == 0) atomicExch(p.status, 4);
    return;
  }
  if (!found) {
    if (may_split && threadIdx.x == 0) p.part_info[split_tile] = make_int4(0, 0, 0, 0);
    return;
  }
  const int seq = work.seq, tile = work.tile, t_begin = work.begin, q_len = work.len;
  const int tok0 = tile * tok_per_tile;
  const int n_tok = min(tok_per_tile, q_len - tok0);
  const int n_rows = n_tok * G;
  const PortionKeys keys = portion_keys(p, work, tok_per_tile, may_split);
  const int pos0 = keys.pos0, pos_last = keys.pos_last, kv_first = keys.kv_first;
  const int kv_begin = keys.begin + split * keys.per * AT_N;                      // this split's first tile
  const int n_tiles = min(keys.per, keys.tiles - split * keys.per);
  if (n_tiles <= 0) {                                    // fewer parts than blocks, or no key (the same for all threads)
    if (may_split && split == 0 && threadIdx.x == 0) p.part_info[split_tile] = make_int4(0, 0, 0, 0);
    return;
  }
  if (threadIdx.x == 4 * 32) {
    sh->part_tile = keys.parts > 1 ? split * p.split_tiles + split_tile : -1;
    if (may_split && split == 0) p.part_info[split_tile] = make_int4(keys.parts, n_rows, t_begin + tok0, kvh);
  }
  if (warp != 0 && warp != 3) {                          // the producers begin at once
    // Tensor memory is taken before the successor is released: one that takes its own before it waits for this kernel could
    // else leave a block here without.  (With the allocation in front of everything the ragged portions took 1 us more.)
    if (warp == 1) tc::tmem_alloc(&sh->tmem_base, TMEM_COLS);
    tc::fence_before_thread_sync();
    asm volatile("bar.sync 3, %0;" ::"n"(AT_THREADS - 64) : "memory");
    tc::fence_after_thread_sync();
    pdl_launch_dependents();
  }
  const uint32_t tmem_s = warp != 0 && warp != 3 ? sh->tmem_base : 0u;      // two score buffers of 64 columns
  // two of P as bfloat16 pairs, 32 columns each; O, up to 256 columns (PAIR: 128)
  const uint32_t tmem_p = PAIR ? tmem_s : tmem_s + 2 * AT_N, p_step = PAIR ? AT_N : AT_N / 2;
  const uint32_t tmem_o = tmem_s + (PAIR ? 2 * AT_N : 3 * AT_N);
  const uint32_t tmem_q = tmem_s + 448;                  // not PAIR: the first 128 dims of the queries
  volatile int* abort_flag = &sh->abort_flag;

  if (warp == 0 || warp == 3) {
    // ---- producers, of keys and of values: each at the pace of its own ring.  The whole warp walks the tiles; lane pi looks
    // up page pi of the next tile, one elected thread issues. ----------------------------------------------------------
    const bool values = warp == 3;
    if (!values && tc::elect_one()) {
      tc::mbar_expect_tx(&sh->q_full, (uint32_t)nsub * tok_per_tile * G * 128);
      for (int sub = 0; sub < nsub; ++sub)
        tc::tma_load_4d(sq + (size_t)sub * AT_Q_SUB, &map_q, &sh->q_full, sub * 64, 0, kvh, t_begin + tok0);
    }
    __syncwarp();
    const int ppt = AT_N / p.page_size;                  // pages per tile: 4, 2 or 1
    const int* table = p.block_table + (size_t)seq * p.max_pages;
    const int page_lo = kv_first / p.page_size, page_hi = min(pos_last / p.page_size, p.max_pages - 1);
    const int first_page = kv_begin / p.page_size;
    const CUtensorMap* map = values ? &map_v : &map_k;
    uint64_t* full = values ? sh->v_full : sh->k_full;
    uint64_t* empty = values ? sh->v_empty : sh->k_empty;
    uint8_t* ring = values ? sv : sk;
    const int stages = values ? p.v_stages : p.k_stages;
    // pages outside [page_lo, page_hi] are masked; they are filled from page 0, whose values are finite as all wide ones are
    auto fetch = [&](int j) -> int {
      const int page_idx = first_page + j * ppt + lane;
      return lane < ppt ? table[min(max(page_idx, page_lo), page_hi)] : 0;
    };
    int next = fetch(0), stage = 0, lap = 0;
    bool ok = true;
    for (int j = 0; j < n_tiles && ok; ++j) {
      int mine = next;
      const int page_idx = first_page + j * ppt + lane;
      if (lane >= ppt || page_idx < page_lo || page_idx > page_hi) {
        mine = 0;
      } else if (mine < 0 || mine >= p.num_pages) {
        atomicExch(p.status, 3);
        mine = 0;
      }
      if (j + 1 < n_tiles) next = fetch(j + 1);
      int pages[4];
#pragma unroll
      for (int pi = 0; pi < 4; ++pi) pages[pi] = __shfl_sync(0xffffffffu, mine, pi);
      if (lap > 0) ok = warp_wait(&empty[stage], (lap - 1) & 1, abort_flag);
      if (!ok) break;
      if (tc::elect_one()) {
        tc::mbar_expect_tx(&full[stage], (uint32_t)nsub * AT_KV_SUB);
        uint8_t* to = ring + (size_t)stage * nsub * AT_KV_SUB;
        if (p.whole && values) {                         // values: a box per page, [slice][row of the page][64 columns]
#pragma unroll
          for (int pi = 0; pi < 4; ++pi)
            if (pi < ppt)
              tc::tma_load_3d(to + (size_t)pi * nsub * p.page_size * 128, map, &full[stage], 0, (pages[pi] * p.nkv + kvh) * p.page_size, 0);
        } else if (p.whole) {                            // keys: a box per 8 rows, [slice][8 rows][64 columns]
#pragma unroll
          for (int a = 0; a < AT_N / 8; ++a) {
            const int key = a * 8;
            const int pg = p.page_size == 16 ? pages[a >> 1] : p.page_size == 32 ? pages[a >> 2] : pages[0];
            tc::tma_load_3d(to + (size_t)a * nsub * 1024, map, &full[stage], 0, (pg * p.nkv + kvh) * p.page_size + (key & (p.page_size - 1)), 0);
          }
        } else {
#pragma unroll
          for (int pi = 0; pi < 4; ++pi) {
            if (pi < ppt) {
              const int row = (pages[pi] * p.nkv + kvh) * p.page_size;
              uint8_t* dst = to + (size_t)pi * p.page_size * 128;
              for (int sub = 0; sub < nsub; ++sub) tc::tma_load_2d(dst + (size_t)sub * AT_KV_SUB, map, &full[stage], sub * 64, row);
            }
          }
        }
      }
      __syncwarp();
      if (++stage == stages) {
        stage = 0;
        ++lap;
      }
    }
  } else if (warp == 1) {
    // ---- S = Q K^T, a tile ahead of the softmax as soon as a score buffer has been read -----------------------------------
    if (tc::elect_one()) {
      const uint32_t idesc = tc::idesc_bf16_f32(AT_M, AT_N);
      const uint64_t qd = tc::smem_desc_k_sw128(tc::smem_u32(sq));
      const uint32_t k_slice = p.whole ? 1024u : (uint32_t)AT_KV_SUB;          // bytes between slices of keys
      const uint32_t k_sbo = p.whole ? (uint32_t)nsub * 1024u : 1024u;         // bytes between groups of 8 keys
      const uint64_t kd0 = tc::smem_desc_k_sw128_sbo(tc::smem_u32(sk), k_sbo);
      const uint32_t k_tile = ((uint32_t)nsub * AT_KV_SUB) >> 4;
      bool ok = tc::mbar_wait(&sh->q_full, 0, abort_flag);
      if (!PAIR && ok) ok = tc::mbar_wait(&sh->q_ready, 0, abort_flag);
      for (int j = 0, stage = 0, phase = 0; j < n_tiles && ok; ++j) {
        const int b = j & 1;
        ok = tc::mbar_wait(&sh->k_full[stage], phase, abort_flag);
        if (ok && j >= 2) ok = tc::mbar_wait(PAIR ? &sh->pv_done[b] : &sh->s_free[b], ((j >> 1) - 1) & 1, abort_flag);
        if (!ok) break;
        tc::fence_after_thread_sync();
        const uint32_t d = tmem_s + b * AT_N;
        const uint64_t kd = kd0 + stage * k_tile;
#pragma unroll
        for (int ks = 0; ks < 16; ++ks) {
          if (ks < hd16) {
            const uint32_t oq = ((ks >> 2) * AT_Q_SUB + (ks & 3) * 32) >> 4;
            const uint32_t ok_ = ((ks >> 2) * k_slice + (ks & 3) * 32) >> 4;
            if (!PAIR && ks < 8) tc::mma_bf16_ts(d, tmem_q + 8 * ks, kd + ok_, idesc, ks > 0 ? 1u : 0u);
            else tc::mma_bf16_ss(d, qd + oq, kd + ok_, idesc, ks > 0 ? 1u : 0u);
          }
        }
        tc::mma_commit(&sh->s_full[b]);
        tc::mma_commit(&sh->k_empty[stage]);
        if (++stage == p.k_stages) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    // ---- O += P V --------------------------------------------------------------------------------------------------------
    if (tc::elect_one()) {
      const uint32_t idesc = tc::idesc_bf16_f32_b_mn(AT_M, hd);
      const uint32_t v_lbo = p.whole ? (uint32_t)p.page_size * 128u : (uint32_t)AT_KV_SUB;
      const uint32_t v_page = (uint32_t)nsub * p.page_size * 128u;             // whole boxes: bytes of a page
      const uint64_t vd0 = tc::smem_desc_mn_sw128(tc::smem_u32(sv), v_lbo, 1024);
      const uint32_t v_tile = ((uint32_t)nsub * AT_KV_SUB) >> 4;
      uint32_t v_step[AT_N / 16];                                              // start of keys 16 kk, in 16 bytes
#pragma unroll
      for (int kk = 0; kk < AT_N / 16; ++kk)
        v_step[kk] = p.whole ? (((kk * 16) / p.page_size) * v_page + ((kk * 16) % p.page_size) * 128u) >> 4
                             : (uint32_t)(kk * 2048) >> 4;
      bool ok = true;
      for (int j = 0, stage = 0, phase = 0; j < n_tiles && ok; ++j) {
        const int b = j & 1;
        ok = tc::mbar_wait(&sh->v_full[stage], phase, abort_flag);
        if (ok) ok = tc::mbar_wait(&sh->p_ready[b], (j >> 1) & 1, abort_flag);
        if (!ok) break;
        tc::fence_after_thread_sync();
#pragma unroll
        for (int kk = 0; kk < AT_N / 16; ++kk)
          tc::mma_bf16_ts(tmem_o, tmem_p + b * p_step + 8 * kk, vd0 + stage * v_tile + v_step[kk], idesc, (j > 0 || kk > 0) ? 1u : 0u);
        tc::mma_commit(&sh->v_empty[stage]);
        tc::mma_commit(&sh->pv_done[b]);
        if (++stage == p.v_stages) {
          stage = 0;
          phase ^= 1;
        }
      }
      tc::mma_commit(&sh->o_full);
    }
    __syncwarp();
  } else if (warp >= 4) {
    // ---- softmax: group 0 takes the even tiles, group 1 the odd ones; a thread has a row -------------------------------
    const int quarter = warp & 3, group = (warp - 4) >> 2;
    const int r = quarter * 32 + lane;
    const bool rv = r < n_rows;
    const int qpos = pos0 + (rv ? r / G : 0);
    const int lo = p.window > 0 ? qpos - p.window + 1 : 0;
    const uint32_t lane_base = ((uint32_t)(quarter * 32) << 16);
    const uint32_t my_s = tmem_s + group * AT_N + lane_base, my_p = tmem_p + group * p_step + lane_base;
    const float LOG2E = 1.4426950408889634f;
    const float in_scale = p.cap > 0.f ? p.multiplier / p.cap : p.multiplier;
    const float out_scale = p.cap > 0.f ? p.cap * LOG2E : LOG2E;   // scores are kept in log2 units
    float ref = -INFINITY, l = 0.f;
    bool ok = true;                                      // the same in all lanes of a warp
    if (!PAIR && group == 0) {                           // the queries' first 128 dims, as pairs, into tensor memory
      ok = warp_wait(&sh->q_full, 0, abort_flag);
      if (ok) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int chunk = (c & 1) * 4 + i;
            const uint4 x = *reinterpret_cast<const uint4*>(sq + (size_t)(c >> 1) * AT_Q_SUB + r * 128 + ((chunk ^ (r & 7)) << 4));
            v[4 * i] = x.x; v[4 * i + 1] = x.y; v[4 * i + 2] = x.z; v[4 * i + 3] = x.w;
          }
          tc::tmem_st_16(tmem_q + lane_base + 16 * c, v);
        }
        tc::tmem_st_wait();
        tc::fence_before_thread_sync();
        tc::mbar_arrive(&sh->q_ready);
      }
    }
    constexpr int CH = PAIR ? 32 : AT_N;                 // columns in registers at a time
    for (int j = group; j < n_tiles && ok; j += 2) {
      ok = warp_wait(&sh->s_full[group], (j >> 1) & 1, abort_flag);
      if (!ok) break;
      tc::fence_after_thread_sync();
      const int key0 = kv_begin + j * AT_N;
      // Most tiles lie wholly inside every row's range.  Lanes without a row compute what nobody reads: asked for the mask in
      // every tile, they made 250 tokens behind 7,900 take 67.3 us instead of 59.7.
      const bool inside = __all_sync(0xffffffffu, !rv || (key0 >= lo && key0 + AT_N - 1 <= qpos));
      uint32_t raw[CH];
      // scores of columns c0 .. c0 + CH - 1 in log2 units, masked; FIXED: less the fixed reference
      auto scores = [&](int c0) {
#pragma unroll
        for (int c = 0; c < CH; c += 16) tc::tmem_ld_16(my_s + c0 + c, raw + c);
        tc::tmem_ld_wait();
        if (!PAIR) {
          tc::fence_before_thread_sync();
          tc::mbar_arrive(&sh->s_free[group]);
        }
        if (FIXED || p.cap > 0.f) {
#pragma unroll
          for (int c = 0; c < CH; ++c) {
            const float v = tc::tanh_approx(__uint_as_float(raw[c]) * in_scale);
            raw[c] = __float_as_uint(FIXED ? fmaf(v, out_scale, -AT_FIXED_REF) : v * out_scale);
          }
        } else {
#pragma unroll
          for (int c = 0; c < CH; ++c) raw[c] = __float_as_uint(__uint_as_float(raw[c]) * (in_scale * out_scale));
        }
        if (!inside) {
#pragma unroll
          for (int c = 0; c < CH; ++c)
            if (!(rv && key0 + c0 + c <= qpos && key0 + c0 + c >= lo)) raw[c] = 0xff800000u;      // -inf
        }
      };
      if (!FIXED) {
        float top = -INFINITY;
#pragma unroll
        for (int c0 = 0; c0 < AT_N; c0 += CH) {
          scores(c0);
#pragma unroll
          for (int c = 0; c < CH; ++c) top = fmaxf(top, __uint_as_float(raw[c]));
        }
        // the row's reference comes from the tile before, goes to the tile behind
        if (j > 0) ok = warp_wait(&sh->turn[group], ((j + group) / 2 - 1) & 1, abort_flag);
        if (!ok) break;
        const float before = j > 0 ? sh->row_ref[r] : -INFINITY;
        const bool grow = top > before + AT_GROW || (before == -INFINITY && top > -INFINITY);
        const float now = grow ? top : before;
        if (grow || j == 0) sh->row_ref[r] = now;
        tc::mbar_arrive(&sh->turn[group ^ 1]);
        if (now != ref) {                                // what this group has summed so far follows
          l *= ref == -INFINITY ? 0.f : tc::exp2_approx(ref - now);
          ref = now;
        }
        if (j > 0 && __any_sync(0xffffffffu, grow)) {    // O follows when the product of the tile before is in
          ok = warp_wait(&sh->pv_done[(j - 1) & 1], ((j - 1) >> 1) & 1, abort_flag);
          if (!ok) break;
          tc::fence_after_thread_sync();
          const float corr = grow ? (before == -INFINITY ? 0.f : tc::exp2_approx(before - now)) : 1.f;
          for (int c0 = 0; c0 < hd; c0 += 16) {
            uint32_t o[16];
            tc::tmem_ld_16(tmem_o + lane_base + c0, o);
            tc::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
            tc::tmem_st_16(tmem_o + lane_base + c0, o);
          }
          tc::tmem_st_wait();
        }
      }
      const float base = FIXED || ref == -INFINITY ? 0.f : ref;
      float l4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c0 = 0; c0 < AT_N; c0 += CH) {
        if (FIXED || PAIR) scores(c0);                   // else they are in registers still
#pragma unroll
        for (int c = 0; c < CH; c += 2) {
          const float p0 = tc::exp2_approx(FIXED ? __uint_as_float(raw[c]) : __uint_as_float(raw[c]) - base);
          const float p1 = tc::exp2_approx(FIXED ? __uint_as_float(raw[c + 1]) : __uint_as_float(raw[c + 1]) - base);
          const __nv_bfloat162 h = __floats2bfloat162_rn(p0, p1);
          const uint32_t both = *reinterpret_cast<const uint32_t*>(&h);
          l4[c & 3] += __uint_as_float(both << 16);      // the sum of what the product will see
          l4[(c + 1) & 3] += __uint_as_float(both & 0xffff0000u);
          raw[c >> 1] = both;
        }
        if (!PAIR && j >= 2) {                           // P of two tiles ago was read
          ok = warp_wait(&sh->pv_done[group], ((j >> 1) - 1) & 1, abort_flag);
          if (!ok) break;
          tc::fence_after_thread_sync();
        }
#pragma unroll
        for (int c = 0; c < CH / 2; c += 16) tc::tmem_st_16(my_p + c0 / 2 + c, raw + c);
      }
      if (!ok) break;
      l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
      tc::tmem_st_wait();
      tc::fence_before_thread_sync();
      tc::mbar_arrive(&sh->p_ready[group]);
    }
    // ---- epilogue: O over the row's sum, a half of the columns each --------------------------------------------------
    sh->row_sum[group][r] = l;
    sh->row_own[group][r] = ref;
    asm volatile("bar.sync 2, 256;" ::: "memory");
    const bool partial = sh->part_tile >= 0;
    const size_t part_row = (size_t)max(sh->part_tile, 0) * AT_M;
    if (ok) ok = warp_wait(&sh->o_full, 0, abort_flag);
    if (ok) {
      tc::fence_after_thread_sync();
      float total = sh->row_sum[0][r] + sh->row_sum[1][r], last = 0.f;
      if (!FIXED) {
        last = sh->row_ref[r];
        total = 0.f;
#pragma unroll
        for (int b = 0; b < 2; ++b)
          if (sh->row_own[b][r] != -INFINITY) total += sh->row_sum[b][r] * tc::exp2_approx(sh->row_own[b][r] - last);
          else total += sh->row_sum[b][r];               // 0, or NaN where every score was
      }
      const int o_lo = group ? ((hd16 + 1) >> 1) * 16 : 0, o_hi = group ? hd : ((hd16 + 1) >> 1) * 16;
      const float inv = total == 0.f ? 0.f : 1.0f / total;
      if (partial && rv && group == 0) p.part_ml[part_row + r] = make_float2(last, total);
      // Rows go out by way of shared memory, which all copies and products have left: a thread has a row of O, but a
      // warp should write rows as a whole (a thread writing its own row's 32 bytes at a time took 5 us).  16-byte chunk c of
      // row r sits at c ^ (r mod 8), as far as the chunks of a row are a multiple of a power of two.
      const int chunk_shift = partial ? 2 : 3;          // elements of a chunk: 4 floats, 8 bfloat16
      const int chunks = hd >> chunk_shift, swizzle = r & 7 & ((chunks & -chunks) - 1);
      uint4* row_at = reinterpret_cast<uint4*>(smem) + (size_t)r * chunks;
      uint32_t largest = 0, pairs = 0;                   // magnitudes of 32 bits, of two times 16
      for (int c0 = o_lo; c0 < o_hi; c0 += 32) {
        uint32_t o[32];
        tc::tmem_ld_16(tmem_o + lane_base + c0, o);
        if (c0 + 16 < o_hi) tc::tmem_ld_16(tmem_o + lane_base + c0 + 16, o + 16);
        tc::tmem_ld_wait();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (c0 + 16 * half >= o_hi) break;
          const uint32_t* v = o + 16 * half;
          const int c = (c0 + 16 * half) >> chunk_shift;
          if (partial) {
#pragma unroll
            for (int i = 0; i < 4; ++i) row_at[(c + i) ^ swizzle] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
#pragma unroll
            for (int i = 0; i < 16; ++i) largest = max(largest, v[i] & 0x7fffffffu);
          } else {
            uint32_t h[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const __nv_bfloat162 x = __floats2bfloat162_rn(__uint_as_float(v[2 * i]) * inv, __uint_as_float(v[2 * i + 1]) * inv);
              h[i] = *reinterpret_cast<const uint32_t*>(&x);
              pairs = __vmaxu2(pairs, h[i] & 0x7fff7fffu);
            }
            row_at[c ^ swizzle] = make_uint4(h[0], h[1], h[2], h[3]);
            row_at[(c + 1) ^ swizzle] = make_uint4(h[4], h[5], h[6], h[7]);
          }
        }
      }
      // values are finite, and a score that is not makes the row's sum NaN: what else is not finite has overflowed
      if (rv && total < INFINITY && max(largest, max(pairs, pairs << 16)) >= 0x7f800000u) atomicExch(p.status, 7);
    }
    asm volatile("bar.sync 2, 256;" ::: "memory");
    if (ok) {
      // 8, 16 or 32 lanes to a row; a warp's rows are 8 x (rows at once) apart, their (token, head) counted without division
      const int chunks = hd >> (partial ? 2 : 3);
      const int lanes = chunks <= 8 ? 8 : chunks <= 16 ? 16 : 32, at_once = 32 / lanes, step = 8 * at_once;
      const int step_tok = step / G, step_head = step - step_tok * G, wrap = (chunks & -chunks) - 1;
      uint4* to = partial ? reinterpret_cast<uint4*>(p.part_o + part_row * hd) : reinterpret_cast<uint4*>(p.out);
      int row = (warp - 4) * at_once + lane / lanes;
      int tok = row / G, head = row - tok * G;
      const int c0 = lane & (lanes - 1);
      constexpr int AHEAD = 4;                           // rows on their way through registers
      auto advance = [&](int& t, int& h) {
        t += step_tok;
        h += step_head;
        if (h >= G) {
          h -= G;
          ++t;
        }
      };
      for (; row < n_rows; row += AHEAD * step) {
        for (int c = c0; c < chunks; c += lanes) {
          uint4 v[AHEAD];
#pragma unroll
          for (int k = 0; k < AHEAD; ++k) {
            const int r_ = row + k * step;
            if (r_ < n_rows) v[k] = reinterpret_cast<const uint4*>(smem)[(size_t)r_ * chunks + (c ^ (r_ & 7 & wrap))];
          }
          int t_ = tok, h_ = head;
#pragma unroll
          for (int k = 0; k < AHEAD; ++k) {
            const size_t to_row = partial ? (size_t)(row + k * step) : (size_t)(t_begin + tok0 + t_) * p.nh + kvh * G + h_;
            if (row + k * step < n_rows) to[to_row * chunks + c] = v[k];
            advance(t_, h_);
          }
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) advance(tok, head);
      }
    }
  }
  tc::fence_before_thread_sync();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after_thread_sync();
    tc::tmem_dealloc(sh->tmem_base, TMEM_COLS);
  }
  if (threadIdx.x == 0 && sh->abort_flag) atomicExch(p.status, 4);
}

// Adds up the parts of every row of the split tiles, in order: a warp per row, 16 blocks per tile.  Short and bound by its
// round trips (7 us for 32 tiles of 4 parts, 16.8 MB): few registers, so that its blocks wait beside the last ones of
// the kernel in front (with four parts in flight, 70 registers, they did not fit and the two took 1 us more).
__global__ void __launch_bounds__(256) attention_portion_merge_kernel(const PortionParams p) {
  pdl_wait_release();
  const int split_tile = blockIdx.x >> 4, r = (blockIdx.x & 15) * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int4 info = p.part_info[split_tile];
  const int parts = info.x, G = p.nh / p.nkv;
  if (parts < 2 || r >= info.y) return;
  const size_t from = (size_t)split_tile * AT_M + r, stride = (size_t)p.split_tiles * AT_M;
  const size_t row = (size_t)(info.z + r / G) * p.nh + info.w * G + r % G;
  float M = -INFINITY;
  for (int s = 0; s < parts; ++s) M = fmaxf(M, p.part_ml[s * stride + from].x);
  float L = 0.f;
  float4 acc[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};
  for (int s = 0; s < parts; ++s) {
    const float2 ml = p.part_ml[s * stride + from];
    // a split whose keys are all masked for this row has no reference and L = 0; one whose scores were NaN has L = NaN
    const float w = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : ml.y) : tc::exp2_approx(ml.x - M);
    L += ml.y * w;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int d = lane * 4 + k * 128;
      if (d < p.hd) {
        const float4 v = *reinterpret_cast<const float4*>(p.part_o + (s * stride + from) * p.hd + d);
        acc[k].x += v.x * w; acc[k].y += v.y * w; acc[k].z += v.z * w; acc[k].w += v.w * w;
      }
    }
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int d = lane * 4 + k * 128;
    if (d < p.hd) {
      if (L < INFINITY && !(fmaxf(fmaxf(fabsf(acc[k].x), fabsf(acc[k].y)), fmaxf(fabsf(acc[k].z), fabsf(acc[k].w))) < INFINITY))
        atomicExch(p.status, 7);                          // (parts that are finite each)
      const __nv_bfloat162 a = __floats2bfloat162_rn(acc[k].x * inv, acc[k].y * inv), b = __floats2bfloat162_rn(acc[k].z * inv, acc[k].w * inv);
      *reinterpret_cast<uint2*>(p.out + row * p.hd + d) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
  }
}

// ---- host side -------------------------------------------------------------------------------------------------

typedef CUresult (*AtEncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                               const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                               CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static AtEncodeFn at_encode_fn() {
  static AtEncodeFn fn = nullptr;
  if (!fn) {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult qres;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &qres) == cudaSuccess &&
        qres == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<AtEncodeFn>(ptr);
  }
  return fn;
}

static int at_map(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                  const cuuint32_t* box) {
  AtEncodeFn fn = at_encode_fn();
  if (!fn) return GLINT_ERR_BAD_ARG;
  const cuuint32_t elem[4] = {1, 1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? GLINT_OK : GLINT_ERR_BAD_ARG;
}

}  // namespace glint

using namespace glint;

// head_dim a multiple of 16 up to 256; at most 128 query heads per kv head; pages of 16, 32 or 64.
GLINT_API int glint_attention_portion_supported(int nh, int nkv, int hd, int page_size) {
  return (nkv > 0 && nh % nkv == 0 && nh / nkv <= AT_M && hd % 16 == 0 && hd >= 16 && hd <= 256 &&
          (page_size == 16 || page_size == 32 || page_size == 64)) ? 1 : 0;
}

// q, out: [T, nh * hd] bf16; pools [pages][nkv][page_size][hd] bf16, finite everywhere; cu_seqlens (absolute token offsets),
// seq_start and block_table of the n_seqs portions, which have `tokens` tokens in all and of which none is longer than max_q_len or attends more than
// max_context keys.  `scratch`: floats for partial results, 16-byte aligned (none, or too few: the keys are not split).
// `early`: cu_seqlens and seq_start were on the device before the kernel in front began (copies, not a kernel's results).
GLINT_API int glint_attention_portion(const void* q, const void* k_pool, const void* v_pool, const int* cu_seqlens,
                                      const int* seq_start, const int* block_table, int max_pages, void* out, int T,
                                      int tokens, int n_seqs, int max_q_len, int max_context, int nh, int nkv, int hd, int page_size,
                                      int num_pages, float multiplier, float cap, int window, int sms, float* scratch,
                                      long long scratch_floats, int* status, int early, cudaStream_t stream) {
  if (n_seqs <= 0 || max_q_len <= 0 || tokens <= 0 || T < tokens) return GLINT_OK;
  if (!glint_attention_portion_supported(nh, nkv, hd, page_size)) return GLINT_ERR_UNSUPPORTED_SIZE;
  if (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)out) & 15) return GLINT_ERR_UNSUPPORTED_SIZE;
  if ((long long)num_pages * nkv * page_size > 0x7fffffffLL) return GLINT_ERR_UNSUPPORTED_SIZE;
  const int G = nh / nkv;
  const int tok_per_tile = AT_M / G;
  CUtensorMap map_q, map_k, map_v;
  {
    const cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)G, (cuuint64_t)nkv, (cuuint64_t)T};
    const cuuint64_t strides[3] = {(cuuint64_t)hd * 2, (cuuint64_t)G * hd * 2, (cuuint64_t)nh * hd * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)G, 1, (cuuint32_t)tok_per_tile};
    const int rc = at_map(&map_q, q, 4, dims, strides, box);
    if (rc != GLINT_OK) return rc;
  }
  // With head_dim a multiple of 64 the 64-column slices are a third dimension of the pools, and one box brings all
  // slices of its rows (the copy unit spends about 65 cycles on a box whatever its size).
  const int whole = hd % 64 == 0 ? 1 : 0;
  const cuuint64_t rows = (cuuint64_t)num_pages * nkv * page_size;
  int rc;
  if (whole) {
    const cuuint64_t dims[3] = {64, rows, (cuuint64_t)(hd / 64)};
    const cuuint64_t strides[2] = {(cuuint64_t)hd * 2, 128};
    const cuuint32_t box_k[3] = {64, 8, (cuuint32_t)(hd / 64)};
    const cuuint32_t box_v[3] = {64, (cuuint32_t)page_size, (cuuint32_t)(hd / 64)};
    rc = at_map(&map_k, k_pool, 3, dims, strides, box_k);
    if (rc == GLINT_OK) rc = at_map(&map_v, v_pool, 3, dims, strides, box_v);
  } else {
    const cuuint64_t dims[2] = {(cuuint64_t)hd, rows};
    const cuuint64_t strides[1] = {(cuuint64_t)hd * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)page_size};
    rc = at_map(&map_k, k_pool, 2, dims, strides, box);
    if (rc == GLINT_OK) rc = at_map(&map_v, v_pool, 2, dims, strides, box);
  }
  if (rc != GLINT_OK) return rc;
  PortionParams p = {};
  p.cu_seqlens = cu_seqlens; p.seq_start = seq_start; p.block_table = block_table; p.max_pages = max_pages;
  p.out = (__nv_bfloat16*)out; p.nh = nh; p.nkv = nkv; p.hd = hd; p.page_size = page_size; p.num_pages = num_pages;
  p.multiplier = multiplier; p.cap = cap; p.window = window; p.whole = whole; p.status = status; p.n_seqs = n_seqs; p.early = early;
  const int nsub = (hd + 63) / 64;
  // As many tiles ahead as fit, up to four: two of each do nearly as well (ragged portions, heads of 128: 91 against 90 us;
  // heads of 256, which have room for three of keys and two of values: 4,096 tokens 134.5 against 133.9, 250 behind 7,900 61.6
  // against 59.8)
  auto bytes = [&](int k, int v) { return nsub * AT_Q_SUB + (k + v) * nsub * AT_KV_SUB + (int)sizeof(PortionShared); };
  const bool pair = hd <= 128;                           // two blocks on an SM
  p.k_stages = p.v_stages = AT_STAGES;
  while (bytes(p.k_stages, p.v_stages) > (pair ? 113 * 1024 : 227 * 1024)) {
    if (p.v_stages >= p.k_stages) --p.v_stages;
    else --p.k_stages;
  }
  const int smem = bytes(p.k_stages, p.v_stages);
  // n tokens make at most (n - 1) / tok_per_tile + 1 tiles of a portion
  const long long blocks = ((tokens > n_seqs ? ((long long)tokens - n_seqs) / tok_per_tile : 0) + n_seqs) * nkv;
  if (blocks > 0x3fffffffLL) return GLINT_ERR_UNSUPPORTED_SIZE;
  // Keys are split where SMs would stay empty: those of all tiles when these are fewer than the SMs, else of the tiles
  // behind the last full round.  A key tile takes about 1 us of an SM, 1.75 us when two blocks share it; partial results and
  // their sum cost about as much as 9 key tiles (12 behind full rounds, whose blocks do not all end together; 16 with two
  // blocks to an SM).  Measured (us, unsplit / one split block to an SM / two): heads of 128, 96 tiles (one part only fits)
  // over 7,000 keys 116 / - / 84, over 1,024 keys 24 / - / 30; 64 tiles over 7,000 - / 71 / 66, 16 tiles - / 29 / 33; 304 tiles
  // over 7,000 keys 278 / 208 and over 1,024 53 / 46; heads of 256, 152 tiles over 3,000 keys 95 / 74, over 500 32 / 36.
  const long long before = ((long long)max_context - max_q_len) / (n_seqs > 1 ? 2 : 1);     // cached tokens, of several portions half the most
  const bool tail = blocks > sms;
  const long long keys = tail ? (window > 0 && window < before ? window : before) + tok_per_tile
                              : window > 0 && (long long)window + tok_per_tile + AT_N < max_context ? (long long)window + tok_per_tile + AT_N : max_context;
  const int tiles = (int)((keys + AT_N - 1) / AT_N);
  p.split_from = tail ? (int)(blocks / sms * sms) : 0;
  p.split_tiles = (int)blocks - p.split_from;
  p.splits = 1;
  if (p.split_tiles) {
    const int most = tiles / AT_LEAST, one = min(sms / p.split_tiles, most), two = min(2 * sms / p.split_tiles, most);
    float least = (float)tiles;
    if (one > 1 && (float)tiles / one + (tail ? 12.f : 9.f) < least) {
      p.splits = one;
      least = (float)tiles / one + 9.f;
    }
    if (pair && !tail && two > one && 1.75f * tiles / two + 16.f < least) p.splits = two;
  }
  const long long part = (long long)p.split_tiles * (AT_M * (hd + 2) + 4);      // floats of a split, and of what is said of its tiles
  if (p.splits > 1 && (!scratch || ((uintptr_t)scratch & 15) || part * p.splits > scratch_floats))
    p.splits = scratch && !((uintptr_t)scratch & 15) ? (int)(scratch_floats / part) : 1;
  if (p.splits < 2) {
    p.splits = 1;
    p.split_tiles = 0;
    p.split_from = (int)blocks;
  } else {
    p.part_info = reinterpret_cast<int4*>(scratch);
    p.part_o = scratch + (long long)p.split_tiles * 4;
    p.part_ml = reinterpret_cast<float2*>(p.part_o + (long long)p.splits * p.split_tiles * AT_M * hd);
  }
  const dim3 grid((unsigned)(p.split_from + p.split_tiles * p.splits));
  const bool fixed = cap > 0.f && cap <= AT_FIXED_CAP;
  cudaError_t e = cudaSuccess;
#define LAUNCH(FIXED, PAIR)                                                                                             \
  {                                                                                                                     \
    e = cudaFuncSetAttribute(attention_portion_kernel<FIXED, PAIR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem); \
    if (e == cudaSuccess)                                                                                               \
      e = launch_kernel(attention_portion_kernel<FIXED, PAIR>, grid, dim3(AT_THREADS), (size_t)smem, stream, map_q, map_k, map_v, p); \
  }
  if (pair) {
    if (fixed) LAUNCH(true, true) else LAUNCH(false, true)
  } else {
    if (fixed) LAUNCH(true, false) else LAUNCH(false, false)
  }
#undef LAUNCH
  if (e == cudaSuccess && p.split_tiles)
    e = launch_kernel(attention_portion_merge_kernel, dim3((unsigned)(p.split_tiles * (AT_M / 8))), dim3(256), 0, stream, p);
  return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}
