// Attention of one new token per sequence over the paged cache, in the prover's integers
// (grape_kv_attend): every row's scores, exp arguments and values, softmax and output, exactly.
//
// The softmax is rounded with the whole row's sum before it meets the values, so nothing can be rescaled
// later: three passes, joined by an integer maximum and integer sums, whose order changes no bit.
#include <algorithm>
#include <exception>

#include <cooperative_groups.h>

#include "kv.cuh"

namespace grape {

struct AttendArgs {
  KvView c;
  const int32_t *len, *selected;
  uint32_t n_select;
  const int32_t* q;
  uint64_t q_stride;
  uint32_t heads, group, score_shift, soft_shift;
  const int32_t* exp;
  int32_t exp_low;
  uint32_t exp_len;
  uint64_t max_keys;
  int32_t *out, *score, *score_rem, *exp_in, *exp_out, *softmax, *out_rem;
  int64_t* sum;
  int32_t* piece_max;      // [row + block of the grid][heads of a tile]: the largest score of a row's piece
  uint32_t* before;        // [batch + 1]: key sets of the sequences before
  int64_t* acc;            // [batch][heads][head_dim]
  uint32_t* done;          // warps that have added to acc, per (row, part of a row's values, unit of a block)
  unsigned char* valid;    // [batch][kv_heads][padded columns]: 1 where a column holds a position
  int64_t* row_at;         // [batch][kv_heads][padded columns]: offset of a column's key and value (of some row where there is none)
  unsigned char* digits;   // [batch][heads][3][padded columns]: the softmax in bytes
  int64_t* weight;         // [batch][heads]: sum of the softmax
  uint64_t padded, acc_count, done_count;
  uint32_t tiles, split, stages;                       // scores: head tiles of a key head, warps of a row, stages of a queue
  uint32_t score_grid, score_heads, score_keys;
  uint32_t v_tiles, v_parts, v_split, v_heads;         // values: head tiles, parts of a row, segments of a part, heads of a tile
};

// Columns of a row that can hold a position: its length, or the slots of the selected pages.
__device__ __forceinline__ uint32_t columns(const AttendArgs& a, uint32_t n) {
  if (!a.selected) return n;
  return n == 0 ? 0 : (uint32_t)min((uint64_t)a.n_select * a.c.page_size, a.max_keys);
}
__device__ __forceinline__ uint32_t length(const AttendArgs& a, uint32_t b, bool report) {
  return kv_length(a.c, a.len, b, a.selected ? ~0ull : a.max_keys, report);
}

// Page and slot of column i of a sequence of n tokens, or page -1 where the column holds no position.
__device__ __forceinline__ int32_t column_page(const AttendArgs& a, uint32_t b, uint32_t g, uint32_t n, uint32_t i, uint32_t& slot,
                                               bool report) {
  const KvView& c = a.c;
  uint32_t at = c.by_page.div(i);
  slot = i - at * c.page_size;
  if (a.selected) {
    const int32_t s = __ldg(a.selected + ((uint64_t)b * c.kv_heads + g) * a.n_select + at);
    if (s < 0) return -1;
    at = (uint32_t)s;
    if (at >= c.width) {
      if (report) kv_flag(c, STATUS_KV_PLACE);
      return -1;
    }
  }
  if ((uint64_t)at * c.page_size + slot >= n) return -1;
  const int32_t page = kv_page(c, b, at);
  if (page < 0 && report) kv_flag(c, STATUS_KV_PLACE);
  return page;
}

// Entry of the exp table for an argument in [exp_low, 0]: up to 2^31, so the difference is an unsigned one.
__device__ __forceinline__ uint32_t exp_index(const AttendArgs& a, int32_t x) { return (uint32_t)x - (uint32_t)a.exp_low; }

// ---- how scores and values are split --------------------------------------------------------------
// The rows (sequence, key head, head tile, ...) are laid end to end, each cut into sets of 16 or 32 keys, and
// every block of the grid takes one span of sets, the same number for all: however ragged the lengths, the
// blocks end together.  A row counts for AT_EXTRA sets more than it has, behind its own, which is about what
// beginning and ending it costs: without them the blocks that meet many short rows end last (32 caches of 301
// to 4096 tokens: scores 80 us against 65 us for 32 equal ones).  A block walks the pieces of the rows that its
// span covers.  Pieces of row r in block i are numbered r + i: unique, and the pieces of a row lie together.
constexpr uint32_t AT_BATCH = 256;  // sequences of a launch
constexpr uint32_t AT_EXTRA = 8;
constexpr uint32_t AT_SMEM = 110 * 1024;     // dynamic shared memory of a block that shares its SM with another
constexpr uint32_t AT_SMEM_ALONE = 222 * 1024;

// s_before[b] = what the rows of the sequences before b count for; returns that of all.
__device__ __forceinline__ uint32_t plan_sets(const AttendArgs& a, uint32_t* s_before, uint32_t keys, uint32_t rows, bool report) {
  for (uint32_t b = threadIdx.x; b < a.c.batch; b += blockDim.x) {
    const uint32_t sets = (columns(a, length(a, b, report)) + keys - 1) / keys;
    s_before[b + 1] = sets ? (sets + AT_EXTRA) * rows : 0;
  }
  if (threadIdx.x == 0) s_before[0] = 0;
  __syncthreads();
  if (threadIdx.x < 32) {
    uint32_t carry = 0;
    for (uint32_t base = 0; base < a.c.batch; base += 32) {
      const uint32_t b = base + threadIdx.x;
      uint32_t v = b < a.c.batch ? s_before[b + 1] : 0;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(~0u, v, o);
        if ((int)threadIdx.x >= o) v += u;
      }
      if (b < a.c.batch) s_before[b + 1] = carry + v;
      carry += __shfl_sync(~0u, v, 31);
    }
  }
  __syncthreads();
  return s_before[a.c.batch];
}

struct Piece {
  uint32_t b, row, sets;      // sequence, row within it, key sets of the whole row
  uint32_t first_set, count;  // the piece; count may be 0
  uint32_t begin, next;       // where the row begins, and where the block's span goes on
};
__device__ __forceinline__ Piece piece_at(const AttendArgs& a, const uint32_t* s_before, uint32_t rows, uint32_t at, uint32_t end) {
  uint32_t lo = 0, hi = a.c.batch;  // the last b with s_before[b] <= at
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (s_before[mid] <= at) lo = mid; else hi = mid;
  }
  Piece p;
  p.b = lo;
  const uint32_t units = (s_before[lo + 1] - s_before[lo]) / rows;
  p.sets = units - AT_EXTRA;
  p.row = (at - s_before[lo]) / units;
  p.begin = s_before[lo] + p.row * units;
  p.first_set = at - p.begin;
  p.next = min(p.begin + units, end);
  p.count = p.first_set < p.sets ? min(p.sets - p.first_set, end - at) : 0;
  return p;
}

// ---- one pass after another -----------------------------------------------------------------------------
// The three passes are launched so that the blocks of the next begin as SMs come free of the last: what they do
// before after_previous() touches nothing that the pass before writes.  A pass lets the next one begin once
// its own wait is over, so that whoever runs has all passes before the last one complete behind it.
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_begin() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// ---- copies ------------------------------------------------------------------------------------------
// A lane's own queue in shared memory: asynchronous copies that this lane alone reads back, so that no barrier
// is needed, only the wait for its own copies, and what is under way costs no registers.  What the warps of an
// SM have under way (about 150 KB) is what carries the kernels: one step at a time in registers (64 KB) gave
// 3 TB/s.  Whole rows by bulk copies of one warp for all gave 3.4 TB/s, the same copies by a warp's lanes 3.1 to
// 4.3: the issuing warps could not keep up.
__device__ __forceinline__ void mma_u8s8(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_u8u8(int32_t (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.u8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- scores --------------------------------------------------------------------------------------
// q . k exactly, on the 8-bit matrix instruction.  k is read as it lies: 4 (or 2) unsigned bytes once its sign
// bit is flipped (k' = k + bias, bias = 2^31 or 2^15), and q in five balanced digits base 256 (four in
// [-128, 127] and a fifth of 0 or 1).  Byte p of k' meets digit r of q at weight 256^(p + r), so ONE operand
// column per weight c, holding digit c - p at byte p, gives
//   q . k = sum_c 256^c (k' bytes . column c) - bias sum_d q_d,      c = 0 .. 7
// and the eight weights are the eight columns of an m16n8k32: 16 keys, 32 bytes of each, one head.  A sum
// of a column is at most 4096 elements x 4 bytes x 255 x 128 < 2^31.
// What bounds it: bytes of the keys.  The instruction takes 2 cycles of an SM (measured, 570 T products/s) for
// 512 bytes of keys and a head, which arrive every 22 cycles.
// Columns 0..7 of the bytes of a word: byte p of column c is digit c - p of the element (two elements a word when
// they have 16 bits).  u = q + 0x80808080: its four low bytes are the digits + 128, its fifth the fifth digit.
template <int EB>
__device__ __forceinline__ void column_words(const uint64_t (&u)[4 / EB], uint32_t (&w)[8]) {
  uint32_t d[4 / EB], top[4 / EB];
#pragma unroll
  for (int e = 0; e < 4 / EB; e++) {
    d[e] = (uint32_t)u[e] ^ 0x80808080u;
    top[e] = (uint32_t)(u[e] >> 32);  // bytes 5..7 of the pair (d, top) are zero
  }
  if (EB == 4) {
    w[0] = __byte_perm(d[0], top[0], 0x5550);
    w[1] = __byte_perm(d[0], top[0], 0x5501);
    w[2] = __byte_perm(d[0], top[0], 0x5012);
    w[3] = __byte_perm(d[0], top[0], 0x0123);
    w[4] = __byte_perm(d[0], top[0], 0x1234);
    w[5] = __byte_perm(d[0], top[0], 0x2345);
    w[6] = __byte_perm(d[0], top[0], 0x3455);
    w[7] = __byte_perm(d[0], top[0], 0x4555);
  } else {
    constexpr uint32_t pick[8] = {0x5550, 0x5501, 0x5512, 0x5523, 0x5534, 0x5545, 0x5555, 0x5555};
#pragma unroll
    for (int c = 0; c < 8; c++)
      w[c] = __byte_perm(__byte_perm(d[0], top[0], pick[c]), __byte_perm(d[4 / EB - 1], top[4 / EB - 1], pick[c]), 0x5410);
  }
}

// A block builds the columns of HT heads' queries, hn of them real, in s_w ([blk][HT][32 lanes]: 4 words, those of a
// lane's 16 bytes), and bias * sum_d q_d of each.  s_bias is zero before.
template <int EB, int HT>
__device__ __forceinline__ void build_columns(uint4* s_w, unsigned long long* s_bias, const int32_t* q, uint32_t hn, uint32_t D, uint32_t blks) {
  constexpr uint32_t PER = 4 / EB;  // elements of a word
  const uint32_t share = blockDim.x / HT, h = threadIdx.x / share;
  q += (uint64_t)h * D;
  int64_t sum = 0;
  for (uint32_t i = threadIdx.x % share; i < blks * 16; i += share) {
    uint64_t u[PER];
#pragma unroll
    for (uint32_t e = 0; e < PER; e++) {
      const uint32_t d = i * PER + e;
      const int32_t v = h < hn && d < D ? __ldg(q + d) : 0;
      sum += v;
      u[e] = (uint64_t)((int64_t)v + 0x80808080ll);
    }
    // word i of the row: block i / 16, lane group (i / 4) % 4, word i % 4
    uint32_t* to = reinterpret_cast<uint32_t*>(s_w + ((uint64_t)(i / 16) * HT + h) * 32 + (i / 4) % 4) + i % 4;
    uint32_t w[8];
    column_words<EB>(u, w);
#pragma unroll
    for (int k = 0; k < 8; k++) to[k * 16] = w[k];
  }
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if (threadIdx.x % 32 == 0) atomicAdd(&s_bias[h], (unsigned long long)sum << (EB == 4 ? 31 : 15));
}

// The eight column sums of a (head, key) at their weights.
__device__ __forceinline__ uint64_t weigh(const int32_t (&v)[8]) {
  const int64_t v01 = (int64_t)v[0] + (int64_t)v[1] * 256, v23 = (int64_t)v[2] + (int64_t)v[3] * 256;
  const int64_t v45 = (int64_t)v[4] + (int64_t)v[5] * 256, v67 = (int64_t)v[6] + (int64_t)v[7] * 256;
  return (uint64_t)v01 + ((uint64_t)v23 << 16) + ((uint64_t)v45 << 32) + ((uint64_t)v67 << 48);
}

// A step: 64 bytes of 32 keys (MT = 2), or of 16 where a row is shared by the warps of a block.
constexpr uint32_t SC_SLAB = 1024;  // bytes of a warp's slab of sums
__host__ __device__ constexpr int sc_stages(int mt) { return mt == 2 ? 5 : 4; }
__host__ __device__ constexpr uint32_t sc_warp(int mt) { return sc_stages(mt) * mt * 1024 + SC_SLAB; }

// MT: sixteens of keys of a set.  HT: heads of a tile.  A block builds the columns of a piece's tile; its warps (a
// team of `split` where rows are long, each a part of the row) take the sets in turn.
template <int EB, int HT, int MT>
__global__ void __launch_bounds__(MT == 2 ? 256 : 512) k_kv_scores(AttendArgs a) {
  constexpr int SLABS = HT * MT >= 2 ? HT * MT / 2 : 1;  // (head, key) pairs in 32s
  constexpr uint32_t KEYS = 16 * MT;
  constexpr int STAGES = sc_stages(MT);
  extern __shared__ uint4 s_dyn[];  // columns, [blk][HT][32 lanes]: 4 words, those of a lane's 16 bytes; the warps' queues and slabs
  __shared__ unsigned long long s_bias[HT];
  __shared__ int32_t s_max[HT];
  __shared__ uint32_t s_before[AT_BATCH + 1];
  const KvView& c = a.c;
  const uint32_t D = c.head_dim, row_bytes = D * EB, blks = (row_bytes + 63) / 64;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gl = lane >> 2, t = lane & 3;
  const uint32_t rows = c.kv_heads * a.tiles, split = MT == 2 ? 1 : a.split, teams = (blockDim.x >> 5) / split;
  const uint32_t wd = warp % split, team = warp / split, blk0 = blks * wd / split, blk1 = blks * (wd + 1) / split;
  const uint32_t total = plan_sets(a, s_before, KEYS, rows, blockIdx.x == 0);
  const uint32_t span = (total + gridDim.x - 1) / gridDim.x;
  const uint32_t begin = min(total, blockIdx.x * span), end = min(total, begin + span);

  // `fetch` walks the warp's steps STAGES - 1 ahead of their use, through the sets of a piece and on to the next.  A
  // column that holds no position reads some other row of the cache and is dropped at the end; `fifo` has a bit
  // for this lane's key of every set under way.
  char* const mine = reinterpret_cast<char*>(s_dyn + (uint64_t)blks * HT * 32) + (uint64_t)warp * sc_warp(MT);
  uint4* const queue = reinterpret_cast<uint4*>(mine) + lane;
  Piece ahead = {};
  uint32_t ahead_at = begin, ahead_k = team, ahead_blk = blk0, ahead_stage = 0, fifo = 0, under_way = 0;
  const char* key[2 * MT];
  auto settle = [&]() {  // on to the piece that holds the warp's next set
    while (ahead_at < end && ahead_k >= ahead.count) {
      ahead_at = ahead.next;
      ahead_k = team;
      if (ahead_at < end) ahead = piece_at(a, s_before, rows, ahead_at, end);
    }
  };
  if (begin < end) ahead = piece_at(a, s_before, rows, begin, end);
  settle();
  auto fetch = [&]() {
    if (ahead_at < end) {
      if (ahead_blk == blk0) {
        const uint32_t g = ahead.row / a.tiles, tile = ahead.row % a.tiles, n = length(a, ahead.b, false), cols = columns(a, n);
        const uint32_t i = (ahead.first_set + ahead_k) * KEYS + (lane & (KEYS - 1));
        uint32_t slot = 0;
        int32_t page = i < cols ? column_page(a, ahead.b, g, n, i, slot, tile == 0 && wd == 0) : -1;
        fifo |= (page >= 0 ? 1u : 0u) << under_way++;
        const bool first = tile == 0 && wd == 0 && lane < KEYS;
        const uint64_t note = ((uint64_t)ahead.b * c.kv_heads + g) * a.padded + i;
        if (first) a.valid[note] = page >= 0;
        if (page < 0) page = slot = 0;
        const int64_t offset = page * c.page_stride + g * c.head_stride + slot * c.slot_stride;
        if (first) a.row_at[note] = offset;
        // the values' pass takes 32 keys at a time: what lies behind an odd last sixteen is some row too
        const uint32_t set = ahead.first_set + ahead_k;
        if (KEYS == 16 && tile == 0 && wd == 0 && lane >= 16 && set % 2 == 0 && (set + 1) * 16 >= cols)
          a.row_at[((uint64_t)ahead.b * c.kv_heads + g) * a.padded + set * 16 + lane] = g * c.head_stride;
        const uint64_t row = reinterpret_cast<uint64_t>(c.k + offset);
#pragma unroll
        for (int m = 0; m < 2 * MT; m++) key[m] = reinterpret_cast<const char*>(__shfl_sync(~0u, row, m * 8 + gl)) + t * 16;
      }
      if (ahead_blk * 64 + t * 16 < row_bytes) {
#pragma unroll
        for (int m = 0; m < 2 * MT; m++) copy_async<16>(queue + (ahead_stage * 2 * MT + m) * 32, key[m] + ahead_blk * 64);
      }
      ahead_stage = ahead_stage + 1 == STAGES ? 0 : ahead_stage + 1;
      if (++ahead_blk == blk1) {
        ahead_blk = blk0;
        ahead_k += teams;
        settle();
      }
    }
    copy_commit();
  };
#pragma unroll 1
  for (int i = 0; i < STAGES - 1; i++) fetch();

  {
    // what the later passes add to, the plan, and the rows that have no column
    const uint64_t at = (uint64_t)blockIdx.x * blockDim.x + tid, step = (uint64_t)gridDim.x * blockDim.x;
    for (uint64_t i = at; i < a.acc_count; i += step) a.acc[i] = 0;
    for (uint64_t i = at; i < a.done_count; i += step) a.done[i] = 0;
    for (uint64_t i = at; i < (uint64_t)c.batch * a.heads; i += step) a.weight[i] = 0;
    for (uint64_t i = at; i <= c.batch; i += step) a.before[i] = s_before[i];
    for (uint32_t b = 0; b < c.batch; b++) {
      if (s_before[b] != s_before[b + 1]) continue;
      for (uint64_t i = at; i < (uint64_t)a.heads * D; i += step) {
        a.out[(uint64_t)b * a.heads * D + i] = 0;
        if (a.out_rem) a.out_rem[(uint64_t)b * a.heads * D + i] = 0;
        if (i < a.heads) a.sum[(uint64_t)b * a.heads + i] = 0;
      }
    }
  }

  uint32_t stage = 0;
  bool range = false;
  for (uint32_t at = begin; at < end;) {
    const Piece p = piece_at(a, s_before, rows, at, end);
    at = p.next;
    if (p.count == 0) continue;
    const uint32_t g = p.row / a.tiles, tile = p.row % a.tiles;
    const uint32_t h0 = g * a.group + tile * HT, hn = min((uint32_t)HT, a.group - tile * HT);
    const uint64_t row0 = (uint64_t)p.b * a.heads + h0;
    // the operand columns, and the sum of each head's query
    if (tid < HT) { s_bias[tid] = 0; s_max[tid] = INT32_MIN; }
    __syncthreads();
    build_columns<EB, HT>(s_dyn, s_bias, a.q + (uint64_t)p.b * a.q_stride + (uint64_t)h0 * D, hn, D, blks);
    __syncthreads();

    int32_t best[SLABS];
#pragma unroll
    for (int j = 0; j < SLABS; j++) best[j] = INT32_MIN;
    // teams of several warps meet in every set: all of a block's teams take the same number of turns
    for (uint32_t k = team; k < (split == 1 ? p.count : (p.count + teams - 1) / teams * teams); k += teams) {
      const bool real = split == 1 || k < p.count;
      int32_t acc[HT][MT][4];
#pragma unroll
      for (int h = 0; h < HT; h++)
#pragma unroll
        for (int m = 0; m < MT; m++) acc[h][m][0] = acc[h][m][1] = acc[h][m][2] = acc[h][m][3] = 0;
      if (real) {
#pragma unroll 1
        for (uint32_t blk = blk0; blk < blk1; blk++) {
          constexpr uint32_t FLIP = EB == 4 ? 0x80000000u : 0x80008000u;
          copy_wait<STAGES - 2>();
          uint4 y[2 * MT];
#pragma unroll
          for (int m = 0; m < 2 * MT; m++) {
            y[m] = queue[(stage * 2 * MT + m) * 32];
            y[m].x ^= FLIP;
            y[m].y ^= FLIP;
            y[m].z ^= FLIP;
            y[m].w ^= FLIP;
          }
          stage = stage + 1 == STAGES ? 0 : stage + 1;
          fetch();  // into the place that was read a step ago
          const uint4* w = s_dyn + (uint64_t)blk * HT * 32 + lane;
#pragma unroll
          for (int h = 0; h < HT; h++) {
            if (HT > 2 && h >= hn) break;
            const uint4 z = w[h * 32];
#pragma unroll
            for (int m = 0; m < MT; m++) {
              mma_u8s8(acc[h][m], y[2 * m].x, y[2 * m + 1].x, y[2 * m].y, y[2 * m + 1].y, z.x, z.y);
              mma_u8s8(acc[h][m], y[2 * m].z, y[2 * m + 1].z, y[2 * m].w, y[2 * m + 1].w, z.z, z.w);
            }
          }
        }
      }
      bool there = false;
      if (real) {
        there = fifo & 1;
        fifo >>= 1;
        under_way--;
      }
      const uint32_t i = (p.first_set + k) * KEYS + (lane & (KEYS - 1));
      // Lane (g, t) holds columns 2t and 2t + 1 of keys g and g + 8.  Through a slab of shared memory the eight sums
      // of a (head, key) come to one lane, the lane of the key; warps that share a row add theirs up on the way
      // (a column's sum over the whole row stays below 2^31).
#pragma unroll
      for (int j = 0; j < SLABS; j++) {
        int2* slab = reinterpret_cast<int2*>(mine + sc_warp(MT) - SC_SLAB);
#pragma unroll
        for (int z = 0; z < (HT * MT >= 2 ? 4 : 2); z++) {
          const int h = MT == 2 ? j : 2 * j + z / 2, m = MT == 2 ? z / 2 : 0, e = z % 2;
          slab[(z * 8 + gl) * 4 + t] = make_int2(acc[h][m][2 * e], acc[h][m][2 * e + 1]);
        }
        if (split == 1) __syncwarp(); else __syncthreads();
        if (split == 1 || j % split == wd) {
          int32_t v[8] = {};
          for (uint32_t w = 0; w < split; w++) {
            const int4* from = reinterpret_cast<const int4*>(mine + ((int32_t)(team * split + w) - (int32_t)warp) * (int32_t)sc_warp(MT) + sc_warp(MT) - SC_SLAB) + lane * 2;
            const int4 p0 = from[0], p1 = from[1];
            v[0] += p0.x; v[1] += p0.y; v[2] += p0.z; v[3] += p0.w;
            v[4] += p1.x; v[5] += p1.y; v[6] += p1.z; v[7] += p1.w;
          }
          const uint32_t h = MT == 2 ? j : 2 * j + lane / 16;
          if (h < hn && there && (HT * MT >= 2 || lane < 16)) {
            const uint64_t sum = weigh(v) - s_bias[h];
            const int64_t quotient = rdiv((int64_t)sum, a.score_shift);
            const int32_t score = saturate(quotient, INT32_MIN, INT32_MAX, range);
            const uint64_t to = (row0 + h) * a.max_keys + i;
            a.score[to] = score;
            if (a.score_rem) a.score_rem[to] = (int32_t)(uint32_t)(sum - ((uint64_t)quotient << a.score_shift));
            best[j] = max(best[j], score);
          }
        }
        if (split == 1) __syncwarp(); else __syncthreads();
      }
    }
    // the piece's largest score per head
#pragma unroll
    for (int j = 0; j < SLABS; j++) {
      for (int o = MT == 2 ? 16 : 8; o; o >>= 1) best[j] = max(best[j], __shfl_xor_sync(~0u, best[j], o));
      const uint32_t h = MT == 2 ? j : 2 * j + lane / 16;
      if (lane % KEYS == 0 && h < HT) atomicMax(&s_max[h], best[j]);
    }
    __syncthreads();
    if (tid < HT) a.piece_max[((uint64_t)p.b * rows + p.row + blockIdx.x) * HT + tid] = s_max[tid];
  }
  let_next_begin();
  copy_wait<0>();
  if (range) kv_flag(c, STATUS_KV_RANGE);
}

// ---- softmax -------------------------------------------------------------------------------------------
// exp_in, exp_out, the row's sum and the softmax of one row, by a cluster of up to 8 blocks that share their sums
// through distributed shared memory: no pass over the scores for the sum alone.  The table (4 MB for the layer
// prover's) lives in L2; a thread has four columns under way, since what it waits for is a chain of loads.
constexpr uint32_t EX_COLS = 4, EX_MAX_THREADS = 1024;

// Two blocks of 1024 threads an SM leave 32 registers, of which 20 to 28 bytes spill.
// A warp takes 128 columns at a time, a lane four that lie together where the rows of the witness begin on 16 bytes
// (ALIGNED: one access each), else every 32nd.
template <bool ALIGNED>
__global__ void __launch_bounds__(EX_MAX_THREADS, 2) k_kv_softmax(AttendArgs a, uint32_t blocks) {
  __shared__ int64_t s_part[32];
  __shared__ int64_t s_sum;
  __shared__ uint64_t s_inverse;
  namespace cg = cooperative_groups;
  constexpr uint32_t STEP = ALIGNED ? 1 : 32;  // between a lane's columns
  const KvView& c = a.c;
  const uint32_t rank = blockIdx.x % blocks, row = blockIdx.x / blocks, h = row % a.heads, b = row / a.heads, g = h / a.group;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, turn = blocks * blockDim.x * EX_COLS;
  const uint32_t cols = columns(a, length(a, b, false));
  after_previous();
  let_next_begin();
  if (cols == 0) return;
  const uint32_t first = (rank * warps + warp) * 128 + lane * (ALIGNED ? 4 : 1), up = (cols + 31) & ~31u;
  const uint64_t at = (uint64_t)row * a.max_keys;
  const unsigned char* valid = a.valid + ((uint64_t)b * c.kv_heads + g) * a.padded;
  auto which = [&](uint32_t i) {  // of the lane's four columns hold a position
    uint32_t in = 0;
    if (ALIGNED && i < up) {
      const uchar4 v = *reinterpret_cast<const uchar4*>(valid + i);
      in = v.x | v.y << 1 | v.z << 2 | v.w << 3;
      if (i + 4 > cols) in &= i < cols ? (1u << (cols - i)) - 1 : 0;
    }
#pragma unroll
    for (uint32_t j = 0; j < 4; j++)
      if (!ALIGNED && i + j * STEP < cols && valid[i + j * STEP]) in |= 1u << j;
    return in;
  };
  auto load = [&](const int32_t* from, uint32_t i, int32_t (&v)[4]) {
    if (ALIGNED && i + 4 <= cols) {
      const int4 x = *reinterpret_cast<const int4*>(from + at + i);
      v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) v[j] = i + j * STEP < cols ? from[at + i + j * STEP] : 0;
    }
  };
  auto store = [&](int32_t* to, uint32_t i, uint32_t in, const int32_t (&v)[4]) {
    if (!to) return;
    if (ALIGNED && in == 15) {
      *reinterpret_cast<int4*>(to + at + i) = make_int4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (uint32_t j = 0; j < 4; j++)
        if (in >> j & 1) to[at + i + j * STEP] = v[j];
    }
  };

  // the row's largest score: its pieces are those of the blocks whose spans it meets
  const uint32_t rows = c.kv_heads * a.tiles, tile = h % a.group / a.score_heads, r = g * a.tiles + tile;
  const uint32_t before = a.before[b], units = (a.before[b + 1] - before) / rows, begin = before + r * units;
  const uint32_t span = (a.before[c.batch] + a.score_grid - 1) / a.score_grid, first_block = begin / span, last_block = (begin + units - AT_EXTRA - 1) / span;
  int32_t best = INT32_MIN;
  for (uint32_t i = first_block + lane; i <= last_block; i += 32)
    best = max(best, a.piece_max[((uint64_t)b * rows + r + i) * a.score_heads + h % a.group % a.score_heads]);
  best = __reduce_max_sync(~0u, best);

  int64_t sum = 0;
  bool outside = false;
  for (uint32_t i = first; i < cols; i += turn) {
    const uint32_t in = which(i);
    int32_t s[4], e[4];
    load(a.score, i, s);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const int64_t d = in >> j & 1 ? (int64_t)s[j] - best : 0;
      outside |= d < a.exp_low;
      s[j] = (int32_t)max(d, (int64_t)a.exp_low);
      e[j] = __ldg(a.exp + exp_index(a, s[j]));
    }
    store(a.exp_in, i, in, s);
#pragma unroll
    for (int j = 0; j < 4; j++) {
      if (!(in >> j & 1)) e[j] = 0;
      if (e[j] < 0) { e[j] = 0; outside = true; }
      sum += e[j];
    }
    store(a.exp_out, i, in, e);
  }
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if (lane == 0) s_part[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    sum = lane < warps ? s_part[lane] : 0;
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
    if (lane == 0) s_sum = sum;
  }
  // floor(top / sum) by the reciprocal floor((2^64 - 1) / sum): short by one at most.  The digits are written up to a
  // multiple of 32 columns, zeros where a column holds no position.
  if (blocks > 1) {
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    if (threadIdx.x == 0) {
      sum = 0;
      for (uint32_t i = 0; i < blocks; i++) sum += *cluster.map_shared_rank(&s_sum, i);
    }
    cluster.sync();  // nobody's sum is overwritten or goes while another reads it
  }
  if (threadIdx.x == 0) {
    s_sum = sum;
    s_inverse = sum ? ~0ull / (uint64_t)sum : 0;
    if (rank == 0) {
      a.sum[row] = sum;
      outside |= sum == 0;
    }
  }
  if (outside) kv_flag(c, STATUS_KV_EXP);
  __syncthreads();
  const uint64_t total = (uint64_t)s_sum, inverse = s_inverse;
  unsigned char* const digits = a.digits + (uint64_t)row * 3 * a.padded;
  int64_t weights = 0;
  for (uint32_t i = first; i < up; i += turn) {
    const uint32_t in = which(i);
    int32_t o[4];
    load(a.exp_out, i, o);  // this thread's own
    uint32_t weight = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const uint64_t top = ((uint64_t)(uint32_t)o[j] << a.soft_shift) + total / 2, q = __umul64hi(top, inverse);
      o[j] = in >> j & 1 && total ? (int32_t)((uint32_t)q + (top - q * total >= total ? 1u : 0u)) : 0;
      weight += (uint32_t)o[j];
    }
    weights += weight;
    store(a.softmax, i, in, o);
#pragma unroll
    for (int d = 0; d < 3; d++) {
      unsigned char* to = digits + d * a.padded + i;
      if (ALIGNED) {
        *reinterpret_cast<uint32_t*>(to) = __byte_perm(__byte_perm(o[0], o[1], d | (4 + d) << 4), __byte_perm(o[2], o[3], d | (4 + d) << 4), 0x5410);
      } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
          if (i + j * STEP < up) to[j * STEP] = (unsigned char)(o[j] >> 8 * d);
      }
    }
  }
  for (int o = 16; o; o >>= 1) weights += __shfl_xor_sync(~0u, weights, o);
  if (lane == 0 && weights) atomicAdd(reinterpret_cast<unsigned long long*>(a.weight + row), (unsigned long long)weights);
}

// ---- values ----------------------------------------------------------------------------------------
// sum_j o_j v_j exactly, on the same instruction.  o is at most 2^20: three unsigned digits base 256, which are
// operand columns; the rows are the bytes of v (v' = v + bias unsigned), so that
//   sum_j o_j v_j = sum_p,r 256^(p + r) (byte plane p of v' . digit r of o) - bias sum_j o_j.
// Sums of a block's keys stay below 2^31 (see VA_SETS).
// A warp takes 128 bytes of 32 rows for 4 heads (or for the 1 or 2 that there are): lane (g, t) has 16 bytes of the
// rows 8 t .. 8 t + 7, and turning 4 keys x 4 bytes in registers (8 byte permutes) gives the A registers, keys
// along the instruction's inner dimension; the 8 bytes of a column's digits are a lane's B registers as they
// lie.  The three digits of a head are columns of one lane (one pair of lanes with fewer than 4 heads), so a
// warp adds its heads' sums to the output without meeting another warp.
// What bounds it: bytes of the values; 32 keys x 128 bytes cost a warp about 160 instructions of the 700 that an
// SM quarter issues while they arrive.
constexpr uint32_t VA_SETS = 512;  // sets of 32 keys whose products a register takes: 16384 x 255 x 255 < 2^31
constexpr int VA_THREADS = 256, VA_WARPS = VA_THREADS / 32, VA_STAGES = 3;
constexpr uint32_t VA_STEP = 4096 + 512;   // bytes of a step: 32 rows x 128 bytes, and digits

// bytes [key][plane] of 4 words -> words [plane] of 4 keys
__device__ __forceinline__ void turn4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&o)[4]) {
  const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362);
  const uint32_t cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
  o[0] = __byte_perm(ab0, cd0, 0x5410);
  o[1] = __byte_perm(ab0, cd0, 0x7632);
  o[2] = __byte_perm(ab1, cd1, 0x5410);
  o[3] = __byte_perm(ab1, cd1, 0x7632);
}

// What a warp of the values' pass holds in its 8 x NT products, channel by channel: f(e, sum) for the 16 / EB channels of
// the lane's 16 bytes, of head t (NH = 4) or t / 2, every second lane then.  Columns 2t and 2t + 1 of each eight: with
// four heads digits 0 and 1 of head t lie there and digit 2 in the second eight; with one or two, digit 2 lies in
// the next lane.
template <int EB, int NH, int NT, class F>
__device__ __forceinline__ void each_channel(const int32_t (&acc)[8][NT][4], F&& f) {
  auto join = [&](uint64_t c0, uint64_t c1, uint64_t c2) {
    if (NH != 4) c2 = __shfl_xor_sync(~0u, c0, 1);
    return c0 + (c1 << 8) + (c2 << 16);
  };
#pragma unroll
  for (int w = 0; w < 4; w++) {
    uint64_t plane[3][2];  // digit columns: bytes 0 and 1, bytes 2 and 3 of the word
#pragma unroll
    for (int z = 0; z < 3; z++) {
      const int k = z == 2 ? NT - 1 : 0, half = z == 1 ? 1 : 0;
#pragma unroll
      for (int m = 0; m < 2; m++)
        plane[z][m] = (uint64_t)(int64_t)acc[2 * w + m][k][half] + ((uint64_t)(int64_t)acc[2 * w + m][k][2 + half] << 8);
    }
    if (EB == 4) {
      f(w, join(plane[0][0] + (plane[0][1] << 16), plane[1][0] + (plane[1][1] << 16), plane[2][0] + (plane[2][1] << 16)));
    } else {
#pragma unroll
      for (int m = 0; m < 2; m++) f(2 * w + m, join(plane[0][m], plane[1][m], plane[2][m]));
    }
  }
}

// 32 keys x 128 bytes of their values, a lane's 16 bytes of rows 8 t .. 8 t + 7 at from + 512 j, against the digits d.
// 8 bytes of the rows at a time: all 16 together would not leave registers for two blocks an SM.
template <int EB, int NT>
__device__ __forceinline__ void multiply_step(int32_t (&acc)[8][NT][4], const char* from, const uint2 (&d)[NT]) {
#pragma unroll
  for (int half = 0; half < 2; half++) {
    uint2 v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = *reinterpret_cast<const uint2*>(from + j * 512 + half * 8);
#pragma unroll
    for (int z = 0; z < 2; z++) {
      const int w = 2 * half + z;
      uint32_t lo[4], hi[4];
      auto word = [&](int j) { return z == 0 ? v[j].x : v[j].y; };
      turn4(word(0), word(1), word(2), word(3), lo);
      turn4(word(4), word(5), word(6), word(7), hi);
      lo[3] ^= 0x80808080u;
      hi[3] ^= 0x80808080u;
      if (EB == 2) { lo[1] ^= 0x80808080u; hi[1] ^= 0x80808080u; }
#pragma unroll
      for (int k = 0; k < NT; k++) {
        mma_u8u8(acc[2 * w][k], lo[0], lo[1], hi[0], hi[1], d[k].x, d[k].y);
        mma_u8u8(acc[2 * w + 1][k], lo[2], lo[3], hi[2], hi[3], d[k].x, d[k].y);
      }
    }
  }
}

// NH: heads of a warp, 1, 2 or 4.  A block takes a.v_heads = NH or 8.  Two blocks an SM leave 128 registers: with four heads
// 86 bytes a thread spill with 32-bit values and 158 with 16.
template <int EB, int NH>
__global__ void __launch_bounds__(VA_THREADS, 2) k_kv_values(AttendArgs a) {
  constexpr int NT = NH == 4 ? 2 : 1;      // columns of a warp in eights
  constexpr uint32_t ELEMS = 128 / EB;     // channels of a warp
  extern __shared__ uint4 s_dyn[];         // the lanes' queues
  __shared__ uint32_t s_before[AT_BATCH + 1];
  const KvView& c = a.c;
  const uint32_t D = c.head_dim, row_bytes = D * EB, segments = (row_bytes + 127) / 128;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gl = lane >> 2, t = lane & 3;
  const uint32_t rows = c.kv_heads * a.v_parts * a.v_tiles, members = a.v_split * (a.v_heads / NH), teams = VA_WARPS / members;
  const uint32_t team = warp / members, member = warp % members, seg = member % a.v_split, hg = member / a.v_split;
  const uint32_t total = plan_sets(a, s_before, 32, rows, false);
  const uint32_t span = (total + gridDim.x - 1) / gridDim.x;
  const uint32_t begin = min(total, blockIdx.x * span), end = min(total, begin + span);

  // what a row of the plan is to this warp: its heads and its segment; hn 0: nothing
  auto place_of = [&](uint32_t row, uint32_t& g, uint32_t& h0, uint32_t& segment) {
    const uint32_t tile = row % a.v_tiles, part = row / a.v_tiles % a.v_parts, in_tile = min(a.v_heads, a.group - tile * a.v_heads);
    g = row / a.v_tiles / a.v_parts;
    h0 = g * a.group + tile * a.v_heads + hg * NH;
    segment = part * a.v_split + seg;
    return in_tile > hg * NH && segment < segments ? min((uint32_t)NH, in_tile - hg * NH) : 0u;
  };
  // the column that this lane brings for: head and digit; with four heads, digit 2 of the even ones in the second eight
  const uint32_t col_head = NH == 4 ? gl / 2 : gl / 4, col_digit = NH == 4 ? gl % 2 : gl % 4;

  // `fetch` walks the warp's sets VA_STAGES - 1 ahead of their use, and where their rows lie one more.  A lane's place in
  // a step: the 128 bytes of a row side by side (they arrive together), their order turned with t so that the lanes
  // that read together meet different banks; behind the rows the digits, 8 bytes a lane and eight of columns.
  char* const queue = reinterpret_cast<char*>(s_dyn) + warp * VA_STAGES * VA_STEP;
  const uint32_t my_rows = (t * 8 + (gl ^ (2 * t))) * 16, my_digits = 4096 + lane * 8;
  const bool in_page = c.page_size % 8 == 0;  // then the rows 8 t .. 8 t + 7 lie one slot apart
  uint32_t ahead_at = begin, ahead_left = 0, ahead_stage = 0;
  bool ahead_has = false, ahead_in = false;
  const char* ahead_base = nullptr;
  const int64_t* ahead_rows = nullptr;
  const unsigned char* ahead_digits = nullptr;
  int64_t next_row = 0;
  auto settle = [&]() {  // on to the piece that holds the warp's next set, if its sets of this one are over
    while (ahead_left == 0 && ahead_at < end) {
      const Piece p = piece_at(a, s_before, rows, ahead_at, end);
      uint32_t g, h0, segment;
      const uint32_t hn = place_of(p.row, g, h0, segment);
      ahead_at = p.next;
      if (!hn || p.count <= team) continue;
      ahead_left = (p.count - team + teams - 1) / teams;
      ahead_in = segment * 128 + gl * 16 < row_bytes;
      ahead_base = c.v + segment * 128 + gl * 16;
      ahead_has = col_head < hn && col_digit < 3;
      const uint64_t key0 = (uint64_t)(p.first_set + team) * 32;
      ahead_rows = a.row_at + ((uint64_t)p.b * c.kv_heads + g) * a.padded + key0 + (in_page ? 8 * t : lane);
      ahead_digits = a.digits + (((uint64_t)p.b * a.heads + h0 + (ahead_has ? col_head : 0)) * 3 + (ahead_has ? col_digit : 0)) * a.padded + key0 + 8 * t;
      next_row = *ahead_rows;
    }
  };
  settle();
  auto fetch_digits = [&](char* to, const unsigned char* from, bool has) {
    if (has) {
      copy_async<8>(to + my_digits, from);
      if (NT == 2 && col_digit == 0) copy_async<8>(to + my_digits + 256, from + 2 * a.padded);
    }
  };
  auto fetch = [&](bool with_digits) {
    if (ahead_left) {
      char* const to = queue + ahead_stage * VA_STEP;
      const char* from = ahead_base + next_row;
      if (in_page) {
        if (ahead_in) {
#pragma unroll
          for (int j = 0; j < 8; j++) {
            copy_async<16>(to + my_rows + j * 512, from);
            from += c.slot_stride;
          }
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; j++) {
          const int64_t row = __shfl_sync(~0u, next_row, 8 * t + j);
          if (ahead_in) copy_async<16>(to + my_rows + j * 512, ahead_base + row);
        }
      }
      if (with_digits) fetch_digits(to, ahead_digits, ahead_has);
      ahead_stage = ahead_stage + 1 == VA_STAGES ? 0 : ahead_stage + 1;
      ahead_rows += teams * 32;
      ahead_digits += teams * 32;
      if (--ahead_left) next_row = *ahead_rows;
      else settle();
    }
  };
  // the rows of the first steps before the softmax is complete, their digits behind it
  const unsigned char* first_digits[VA_STAGES - 1];
  bool first_has[VA_STAGES - 1];
#pragma unroll
  for (int i = 0; i < VA_STAGES - 1; i++) {
    first_digits[i] = ahead_digits;
    first_has[i] = ahead_left && ahead_has;
    fetch(false);
  }
  after_previous();
#pragma unroll
  for (int i = 0; i < VA_STAGES - 1; i++) {
    fetch_digits(queue + i * VA_STEP, first_digits[i], first_has[i]);
    copy_commit();
  }

  uint32_t stage = 0;
  bool range = false;
  for (uint32_t at = begin; at < end;) {
    const uint32_t here = at;
    uint32_t count;
    {
      const Piece p = piece_at(a, s_before, rows, at, end);
      uint32_t g, h0, segment;
      count = p.count;
      at = p.next;
      if (!place_of(p.row, g, h0, segment) || count <= team) continue;
    }
    int32_t acc[8][NT][4];
#pragma unroll
    for (int k = 0; k < NT; k++)
#pragma unroll
      for (int m = 0; m < 8; m++) acc[m][k][0] = acc[m][k][1] = acc[m][k][2] = acc[m][k][3] = 0;
#pragma unroll 1
    for (uint32_t k = team; k < count; k += teams) {
      copy_wait<VA_STAGES - 2>();
      const char* const step = queue + stage * VA_STEP;
      stage = stage + 1 == VA_STAGES ? 0 : stage + 1;
      fetch(true);  // into the place that was read a step ago
      copy_commit();
      uint2 d[NT];
#pragma unroll
      for (int z = 0; z < NT; z++) d[z] = *reinterpret_cast<const uint2*>(step + my_digits + z * 256);
      multiply_step<EB, NT>(acc, step + my_rows, d);
    }
    const Piece p = piece_at(a, s_before, rows, here, end);
    uint32_t g, h0, segment;
    const uint32_t hn = place_of(p.row, g, h0, segment);
    // how many sums come together in the row's output: of each of its pieces, the teams that have a set of it
    const uint32_t start = min(p.sets, span - p.begin % span), others = p.sets - start;
    const uint32_t adders = min(teams, start) + others / span * min(teams, span) + min(teams, others % span);
    const uint32_t head = NH == 4 ? t : t / 2, channel = segment * ELEMS + gl * (16 / EB);
    const bool mine = head < hn && (NH == 4 || t % 2 == 0);
    const uint64_t row = (uint64_t)p.b * a.heads + h0 + (mine ? head : 0), to = row * D + channel;
    const uint64_t below = (uint64_t)a.weight[row] << (EB == 4 ? 31 : 15);  // bias times the sum of the softmax
    auto finish = [&](uint64_t biased, uint64_t where) {
      const int64_t sum = (int64_t)(biased - below), y = rdiv(sum, a.soft_shift);
      a.out[where] = saturate(y, INT32_MIN, INT32_MAX, range);
      if (a.out_rem) a.out_rem[where] = (int32_t)(uint32_t)((uint64_t)sum - ((uint64_t)y << a.soft_shift));
    };
    each_channel<EB, NH, NT>(acc, [&](uint32_t e, uint64_t value) {
      if (mine && channel + e < D) {
        if (adders == 1) finish(value, to + e);
        else atomicAdd(reinterpret_cast<unsigned long long*>(a.acc + to + e), (unsigned long long)value);
      }
    });
    if (adders > 1) {
      // the last of the warps that add to these channels brings the sums to the output
      __threadfence();
      __syncwarp();
      uint32_t nth = 0;
      if (lane == 0) nth = atomicAdd(a.done + ((uint64_t)p.b * rows + p.row) * VA_WARPS + member, 1u);
      nth = __shfl_sync(~0u, nth, 0);
      if (nth == adders - 1) {
        __threadfence();
        for (uint32_t e = 0; e < 16 / EB; e++)
          if (mine && channel + e < D) finish((uint64_t)__ldcg(reinterpret_cast<const long long*>(a.acc) + to + e), to + e);
      }
    }
  }
  copy_wait<0>();
  if (range) kv_flag(c, STATUS_KV_RANGE);
}

// ---- short rows ------------------------------------------------------------------------------------------
// All three passes over the columns of one head tile by one block: where a key head's rows are short, three launches
// and their beginnings cost more than the bytes.  Scores, softmax and digits stay in shared memory between the
// passes; the arithmetic is that of the passes above.
// Measured against the three passes (us): 32 caches of 64 / 256 / 512 keys, 32 heads on 8 of 128: 15 / 29 / 44 against
// 31 / 47 / 62 (their bytes alone 3 / 11 / 22); 4 caches of 512: 25 against 27; one cache of 256, 4 heads of 64: 14 against 23.  With few rows and
// long ones a block alone is too slow: 2 caches of 1024 keys of 16 bits, 16 heads on 4: 31 against 25.
constexpr uint32_t SM_BYTES = 256 * 1024;     // keys of a row at most
constexpr uint32_t SM_BYTES_FEW = 128 * 1024; // where there are fewer than SM_MANY blocks
constexpr uint32_t SM_MANY = 32;
constexpr int SM_THREADS = 256, SM_WARPS = SM_THREADS / 32, SM_STAGES = 4, SM_VALUE_STAGES = 2;
constexpr uint32_t SM_QUEUE = 8192;  // bytes of a warp's queue: four steps of keys or two of values

struct SmallLayout {  // of the dynamic shared memory, in bytes
  uint32_t queue, slabs, row_at, score, digits, valid, all;
};
__host__ __device__ inline SmallLayout small_layout(uint32_t blks, uint32_t ht, uint32_t padded) {
  SmallLayout l;
  l.queue = blks * ht * 512;
  l.slabs = l.queue + SM_WARPS * SM_QUEUE;
  l.row_at = l.slabs + SM_WARPS * SC_SLAB;
  l.score = l.row_at + padded * 8;
  l.digits = l.score + ht * padded * 4;
  l.valid = l.digits + (ht == 4 ? 16 : 8) * (padded + 32);
  l.all = l.valid + padded;
  return l;
}

template <int EB, int HT>
__global__ void __launch_bounds__(SM_THREADS) k_kv_small(AttendArgs a) {
  constexpr int SLABS = HT, NT = HT == 4 ? 2 : 1;
  extern __shared__ uint4 s_dyn[];
  __shared__ unsigned long long s_bias[HT], s_sum[HT], s_inverse[HT], s_weight[HT];
  __shared__ int32_t s_max[HT];
  const KvView& c = a.c;
  const uint32_t D = c.head_dim, row_bytes = D * EB, blks = (row_bytes + 63) / 64, padded = (uint32_t)a.padded;
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gl = lane >> 2, t = lane & 3;
  const uint32_t tile = blockIdx.x % a.tiles, g = blockIdx.x / a.tiles % c.kv_heads, b = blockIdx.x / a.tiles / c.kv_heads;
  const uint32_t n = length(a, b, tid == 0 && tile == 0 && g == 0), cols = columns(a, n);
  const uint32_t h0 = g * a.group + tile * HT, hn = min((uint32_t)HT, a.group - tile * HT);
  const uint64_t row0 = (uint64_t)b * a.heads + h0;
  if (cols == 0) {
    for (uint32_t i = tid; i < hn * D; i += SM_THREADS) {
      a.out[row0 * D + i] = 0;
      if (a.out_rem) a.out_rem[row0 * D + i] = 0;
    }
    if (a.sum && tid < hn) a.sum[row0 + tid] = 0;
    return;
  }
  const SmallLayout at = small_layout(blks, HT, padded);
  char* const base = reinterpret_cast<char*>(s_dyn);
  char* const mine = base + at.queue + warp * SM_QUEUE;
  char* const slab0 = base + at.slabs + warp * SC_SLAB;
  int64_t* const s_row = reinterpret_cast<int64_t*>(base + at.row_at);
  int32_t* const s_score = reinterpret_cast<int32_t*>(base + at.score);
  unsigned char* const s_digits = reinterpret_cast<unsigned char*>(base + at.digits);
  unsigned char* const s_valid = reinterpret_cast<unsigned char*>(base + at.valid);
  const uint32_t sets = (cols + 31) / 32, digits_row = padded + 32;

  // where the columns lie (some row where there is none), and the operand columns
  if (tid < HT) {
    s_bias[tid] = s_sum[tid] = s_weight[tid] = 0;
    s_max[tid] = INT32_MIN;
  }
  for (uint32_t i = tid; i < sets * 32; i += SM_THREADS) {
    uint32_t slot = 0;
    int32_t page = i < cols ? column_page(a, b, g, n, i, slot, tile == 0) : -1;
    s_valid[i] = page >= 0;
    if (page < 0) page = slot = 0;
    s_row[i] = page * c.page_stride + g * c.head_stride + slot * c.slot_stride;
  }
  __syncthreads();

  // scores: a warp every eighth set, `fetch` SM_STAGES - 1 steps of 64 bytes ahead
  {
    uint4* const queue = reinterpret_cast<uint4*>(mine) + lane;
    uint32_t ahead_set = warp, ahead_blk = 0, ahead_stage = 0, stage = 0;
    auto fetch = [&]() {
      if (ahead_set < sets) {
        if (ahead_blk * 64 + t * 16 < row_bytes) {
#pragma unroll
          for (int m = 0; m < 4; m++) copy_async<16>(queue + (ahead_stage * 4 + m) * 32, c.k + s_row[ahead_set * 32 + m * 8 + gl] + ahead_blk * 64 + t * 16);
        }
        ahead_stage = ahead_stage + 1 == SM_STAGES ? 0 : ahead_stage + 1;
        if (++ahead_blk == blks) {
          ahead_blk = 0;
          ahead_set += SM_WARPS;
        }
      }
      copy_commit();
    };
#pragma unroll 1
    for (int i = 0; i < SM_STAGES - 1; i++) fetch();
    build_columns<EB, HT>(s_dyn, s_bias, a.q + (uint64_t)b * a.q_stride + (uint64_t)h0 * D, hn, D, blks);
    __syncthreads();
    int32_t best[SLABS];
#pragma unroll
    for (int j = 0; j < SLABS; j++) best[j] = INT32_MIN;
    bool range = false;
    for (uint32_t set = warp; set < sets; set += SM_WARPS) {
      int32_t acc[HT][2][4];
#pragma unroll
      for (int h = 0; h < HT; h++)
#pragma unroll
        for (int m = 0; m < 2; m++) acc[h][m][0] = acc[h][m][1] = acc[h][m][2] = acc[h][m][3] = 0;
#pragma unroll 1
      for (uint32_t blk = 0; blk < blks; blk++) {
        constexpr uint32_t FLIP = EB == 4 ? 0x80000000u : 0x80008000u;
        copy_wait<SM_STAGES - 2>();
        uint4 y[4];
#pragma unroll
        for (int m = 0; m < 4; m++) {
          y[m] = queue[(stage * 4 + m) * 32];
          y[m].x ^= FLIP;
          y[m].y ^= FLIP;
          y[m].z ^= FLIP;
          y[m].w ^= FLIP;
        }
        stage = stage + 1 == SM_STAGES ? 0 : stage + 1;
        fetch();  // into the place that was read a step ago
        const uint4* w = s_dyn + (uint64_t)blk * HT * 32 + lane;
#pragma unroll
        for (int h = 0; h < HT; h++) {
          const uint4 z = w[h * 32];
#pragma unroll
          for (int m = 0; m < 2; m++) {
            mma_u8s8(acc[h][m], y[2 * m].x, y[2 * m + 1].x, y[2 * m].y, y[2 * m + 1].y, z.x, z.y);
            mma_u8s8(acc[h][m], y[2 * m].z, y[2 * m + 1].z, y[2 * m].w, y[2 * m + 1].w, z.z, z.w);
          }
        }
      }
      const uint32_t i = set * 32 + lane;
#pragma unroll
      for (int j = 0; j < SLABS; j++) {
        int2* slab = reinterpret_cast<int2*>(slab0);
#pragma unroll
        for (int z = 0; z < 4; z++) slab[(z * 8 + gl) * 4 + t] = make_int2(acc[j][z / 2][2 * (z % 2)], acc[j][z / 2][2 * (z % 2) + 1]);
        __syncwarp();
        const int4 p0 = reinterpret_cast<const int4*>(slab0)[lane * 2], p1 = reinterpret_cast<const int4*>(slab0)[lane * 2 + 1];
        const int32_t v[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
        if (j < hn && s_valid[i]) {
          const uint64_t sum = weigh(v) - s_bias[j];
          const int64_t quotient = rdiv((int64_t)sum, a.score_shift);
          const int32_t score = saturate(quotient, INT32_MIN, INT32_MAX, range);
          const uint64_t to = (row0 + j) * a.max_keys + i;
          s_score[j * padded + i] = score;
          if (a.score) a.score[to] = score;
          if (a.score_rem) a.score_rem[to] = (int32_t)(uint32_t)(sum - ((uint64_t)quotient << a.score_shift));
          best[j] = max(best[j], score);
        }
        __syncwarp();
      }
    }
    copy_wait<0>();
    if (range) kv_flag(c, STATUS_KV_RANGE);
#pragma unroll
    for (int j = 0; j < SLABS; j++) {
      best[j] = __reduce_max_sync(~0u, best[j]);
      if (lane == 0) atomicMax(&s_max[j], best[j]);
    }
  }
  __syncthreads();

  // the first values, while the softmax is made
  const uint32_t segments = (row_bytes + 127) / 128, teams = SM_WARPS / a.v_split, team = warp / a.v_split, segment = warp % a.v_split;
  const uint32_t my_rows = (t * 8 + (gl ^ (2 * t))) * 16, byte = segment * 128 + gl * 16;
  uint32_t ahead = team, ahead_stage = 0;
  auto fetch = [&]() {
    if (ahead < sets) {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (byte < row_bytes) copy_async<16>(mine + ahead_stage * 4096 + my_rows + j * 512, c.v + s_row[ahead * 32 + 8 * t + j] + byte);
      ahead_stage = ahead_stage + 1 == SM_VALUE_STAGES ? 0 : ahead_stage + 1;
      ahead += teams;
    }
    copy_commit();
  };
#pragma unroll 1
  for (int i = 0; i < SM_VALUE_STAGES; i++) fetch();

  // softmax: a warp a head (two or eight warps where there are fewer heads)
  {
    constexpr uint32_t SHARE = SM_WARPS / HT;
    const uint32_t h = warp / SHARE, first = warp % SHARE * 32 + lane;
    const uint64_t to = (row0 + h) * a.max_keys;
    bool outside = false;
    if (h < hn) {
      const int32_t top = s_max[h];
      int64_t sum = 0;
      for (uint32_t i = first; i < cols; i += SHARE * 32) {
        if (!s_valid[i]) continue;
        const int64_t d = (int64_t)s_score[h * padded + i] - top;
        outside |= d < a.exp_low;
        const int32_t x = (int32_t)max(d, (int64_t)a.exp_low);
        int32_t e = __ldg(a.exp + exp_index(a, x));
        if (e < 0) { e = 0; outside = true; }
        sum += e;
        s_score[h * padded + i] = e;
        if (a.exp_in) a.exp_in[to + i] = x;
        if (a.exp_out) a.exp_out[to + i] = e;
      }
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
      if (lane == 0) atomicAdd(&s_sum[h], (unsigned long long)sum);
    }
    __syncthreads();
    if (tid < HT) {
      s_inverse[tid] = s_sum[tid] ? ~0ull / s_sum[tid] : 0;
      if (tid < hn) {
        if (a.sum) a.sum[row0 + tid] = (int64_t)s_sum[tid];
        outside |= s_sum[tid] == 0;
      }
    }
    if (outside) kv_flag(c, STATUS_KV_EXP);
    __syncthreads();
    const uint64_t total = s_sum[h], inverse = s_inverse[h];
    uint64_t weights = 0;
    for (uint32_t i = first; i < sets * 32; i += SHARE * 32) {
      uint32_t o = 0;
      if (h < hn && s_valid[i] && total) {
        const uint64_t up = ((uint64_t)(uint32_t)s_score[h * padded + i] << a.soft_shift) + total / 2, q = __umul64hi(up, inverse);
        o = (uint32_t)q + (up - q * total >= total ? 1u : 0u);
        weights += o;
      }
      if (a.softmax && h < hn && s_valid[i]) a.softmax[to + i] = (int32_t)o;
      // a column of the instruction a digit, as the values' pass has them
      unsigned char* digits = s_digits + (HT == 4 ? 2 * h : 4 * h) * digits_row + i;
      digits[0] = (unsigned char)o;
      digits[digits_row] = (unsigned char)(o >> 8);
      digits[(HT == 4 ? 8 : 2) * digits_row] = (unsigned char)(o >> 16);
    }
    for (int o = 16; o; o >>= 1) weights += __shfl_xor_sync(~0u, weights, o);
    if (lane == 0) atomicAdd(&s_weight[h], (unsigned long long)weights);
  }
  // the columns' places are the sums of the output from here on
  unsigned long long* const s_out = reinterpret_cast<unsigned long long*>(s_dyn);
  for (uint32_t i = tid; i < HT * D; i += SM_THREADS) s_out[i] = 0;
  __syncthreads();

  int32_t acc[8][NT][4];
#pragma unroll
  for (int k = 0; k < NT; k++)
#pragma unroll
    for (int m = 0; m < 8; m++) acc[m][k][0] = acc[m][k][1] = acc[m][k][2] = acc[m][k][3] = 0;
  uint32_t stage = 0;
#pragma unroll 1
  for (uint32_t set = team; set < sets; set += teams) {
    copy_wait<SM_VALUE_STAGES - 1>();
    uint2 d[NT];
#pragma unroll
    for (int z = 0; z < NT; z++) d[z] = *reinterpret_cast<const uint2*>(s_digits + (z * 8 + gl) * digits_row + set * 32 + 8 * t);
    const char* from = mine + stage * 4096 + my_rows;
    stage = stage + 1 == SM_VALUE_STAGES ? 0 : stage + 1;
    multiply_step<EB, NT>(acc, from, d);
    fetch();  // into the place that has just been read
  }
  copy_wait<0>();
  {
    const uint32_t head = HT == 4 ? t : t / 2, channel = segment * (128 / EB) + gl * (16 / EB);
    const bool own = head < hn && (HT == 4 || t % 2 == 0) && segment < segments;
    each_channel<EB, HT, NT>(acc, [&](uint32_t e, uint64_t value) {
      if (own && channel + e < D) atomicAdd(&s_out[head * D + channel + e], (unsigned long long)value);
    });
  }
  __syncthreads();
  bool range = false;
  for (uint32_t i = tid; i < hn * D; i += SM_THREADS) {
    const int64_t sum = (int64_t)(s_out[i] - (s_weight[i / D] << (EB == 4 ? 31 : 15))), y = rdiv(sum, a.soft_shift);
    a.out[row0 * D + i] = saturate(y, INT32_MIN, INT32_MAX, range);
    if (a.out_rem) a.out_rem[row0 * D + i] = (int32_t)(uint32_t)((uint64_t)sum - ((uint64_t)y << a.soft_shift));
  }
  if (range) kv_flag(c, STATUS_KV_RANGE);
}

// `overlap`: the blocks may begin before the launch before has ended (see after_previous).
template <class K, class... Args>
static int launch(grape_ctx* ctx, K kernel, uint64_t grid, uint32_t threads, size_t smem, uint32_t cluster, bool overlap, const Args&... args) {
  if (smem)  // the limit of 48 KB is for this and the kernel's own arrays together
    if (int rc = kv_allow_shared(ctx, kernel, AT_SMEM_ALONE)) return rc;
  cudaLaunchAttribute attributes[2] = {};
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((uint32_t)grid);
  config.blockDim = dim3(threads);
  config.dynamicSmemBytes = smem;
  config.stream = ctx->stream;
  config.attrs = attributes;
  if (overlap) {
    attributes[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[config.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attributes[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attributes[config.numAttrs].val.clusterDim.x = cluster;
    attributes[config.numAttrs].val.clusterDim.y = 1;
    attributes[config.numAttrs++].val.clusterDim.z = 1;
  }
  GRAPE_CUDA_TRY(ctx, cudaLaunchKernelEx(&config, kernel, args...));
  ctx->launches += 1;
  return GRAPE_OK;
}

template <int EB>
static int launch_scores(grape_ctx* ctx, const AttendArgs& a, uint32_t threads, size_t smem) {
  const uint32_t h = a.score_heads;
  auto kernel = a.score_keys == 32 ? (h == 1 ? k_kv_scores<EB, 1, 2> : h == 2 ? k_kv_scores<EB, 2, 2> : k_kv_scores<EB, 4, 2>)
                                   : (h == 1 ? k_kv_scores<EB, 1, 1> : h == 2 ? k_kv_scores<EB, 2, 1> : k_kv_scores<EB, 4, 1>);
  return launch(ctx, kernel, a.score_grid, threads, smem, 1, false, a);
}

static int launch_softmax(grape_ctx* ctx, const AttendArgs& a, uint64_t rows, uint64_t cols) {
  // As many threads as the GPU holds at a time (phases of several blocks on an SM cover one another), at most one
  // for every four columns.  Threads of a block first, up to 1024, then blocks of a cluster, up to 8.
  const uint64_t room = (uint64_t)ctx->sm_count * 2048;
  uint32_t blocks = 1, threads = 256;
  while (threads < EX_MAX_THREADS && (uint64_t)threads * EX_COLS < cols && rows * threads * 2 <= room) threads *= 2;
  while (blocks < 8 && (uint64_t)blocks * threads * EX_COLS < cols && rows * blocks * threads * 2 <= room) blocks *= 2;
  return launch(ctx, a.max_keys % 4 ? k_kv_softmax<false> : k_kv_softmax<true>, rows * blocks, threads, 0, blocks, true, a, blocks);
}

template <int EB>
static int launch_values(grape_ctx* ctx, const AttendArgs& a, uint64_t grid) {
  const uint32_t h = a.v_heads;
  return launch(ctx, h == 1 ? k_kv_values<EB, 1> : h == 2 ? k_kv_values<EB, 2> : k_kv_values<EB, 4>, grid, VA_THREADS, VA_WARPS * VA_STAGES * VA_STEP, 1, true, a);
}

template <int EB>
static int launch_small(grape_ctx* ctx, const AttendArgs& a, uint32_t ht, uint64_t grid, size_t smem) {
  return launch(ctx, ht == 1 ? k_kv_small<EB, 1> : ht == 2 ? k_kv_small<EB, 2> : k_kv_small<EB, 4>, grid, SM_THREADS, smem, 1, false, a);
}

static int attend_launch(grape_ctx* ctx, const grape_kv_cache* cache, AttendArgs a) {
  const uint64_t rows = (uint64_t)a.c.batch * a.heads, D = cache->head_dim, kv_rows = (uint64_t)a.c.batch * cache->kv_heads;
  const uint64_t all = a.selected ? (uint64_t)a.n_select * cache->page_size : (uint64_t)a.c.width * cache->page_size;
  const uint64_t cols = std::min(all, a.max_keys);
  // without arrays of the caller's, whose rows are max_keys apart, the workspace's rows are as long as a row can be
  if (!a.score && !a.score_rem && !a.exp_in && !a.exp_out && !a.softmax) a.max_keys = std::min((all + 3) & ~uint64_t(3), a.max_keys);
  const uint32_t row_bytes = (uint32_t)(D * cache->bits / 8), blks = (row_bytes + 63) / 64, sms = (uint32_t)ctx->sm_count;

  // Short rows: one block for all passes of a head tile, while what it keeps fits an SM.
  {
    const uint32_t ht = a.group >= 3 ? 4 : a.group;
    a.padded = (cols + 31) & ~uint64_t(31);
    a.tiles = (a.group + ht - 1) / ht;
    a.v_split = 1;
    while (a.v_split < 8 && a.v_split < (row_bytes + 127) / 128) a.v_split *= 2;
    if (row_bytes <= 1024 && a.padded * row_bytes <= (kv_rows * a.tiles < SM_MANY ? SM_BYTES_FEW : SM_BYTES) && kv_rows * a.tiles <= 0x7fffffffu) {
      const SmallLayout l = small_layout(blks, ht, (uint32_t)a.padded);
      if (l.all <= AT_SMEM_ALONE && ht * D * 8 <= l.queue)
        return cache->bits == 32 ? launch_small<4>(ctx, a, ht, kv_rows * a.tiles, l.all) : launch_small<2>(ctx, a, ht, kv_rows * a.tiles, l.all);
    }
  }

  // Scores.  Rows up to 1 KB: two blocks of 8 warps an SM, a warp a set of 32 keys.  Longer ones: one block of 16
  // warps, 16 keys at a time, a row shared by as many warps as have 8 blocks of it (a few rows of a long head are
  // few sets).  Heads of a tile: as many as there are up to 4, while their columns fit.
  const int mt = row_bytes <= 1024 ? 2 : 1;
  const uint32_t threads = mt == 2 ? 256 : 512, warps = threads / 32;
  a.score_keys = 16 * mt;
  a.split = 1;
  while (mt == 1 && a.split < warps && blks / (2 * a.split) >= 8) a.split *= 2;
  const size_t room = (mt == 2 ? AT_SMEM : AT_SMEM_ALONE) - warps * sc_warp(mt);
  uint32_t ht = 1;
  while (ht < 4 && ht < a.group && (size_t)2 * ht * blks * 512 <= room) ht *= 2;
  a.score_heads = ht;
  a.tiles = (a.group + ht - 1) / ht;
  const size_t smem = (size_t)blks * ht * 512 + warps * sc_warp(mt);
  const uint64_t units = kv_rows * a.tiles * ((cols + a.score_keys - 1) / a.score_keys + AT_EXTRA);
  a.score_grid = (uint32_t)std::min<uint64_t>((mt == 2 ? 2 : 1) * sms, units);

  // Values: 4 heads a warp, 8 a block where a key head has more than 4 and the segments of a row leave warps for
  // it; up to 8 segments of 128 bytes a block, the rest of a row in other parts; teams share the keys.
  const uint32_t segments = (row_bytes + 127) / 128;
  a.v_split = 1;
  while (a.v_split < VA_WARPS && a.v_split < segments) a.v_split *= 2;
  a.v_heads = a.group == 1 ? 1 : a.group == 2 ? 2 : a.group <= 4 || a.v_split == VA_WARPS ? 4 : 8;
  a.v_tiles = (a.group + a.v_heads - 1) / a.v_heads;
  a.v_parts = (segments + a.v_split - 1) / a.v_split;
  const uint64_t v_rows = kv_rows * a.v_parts * a.v_tiles, v_units = v_rows * ((cols + 31) / 32 + AT_EXTRA);
  // a block's span of sets bounds the sums of a register
  const uint64_t v_grid = std::max<uint64_t>(std::min<uint64_t>(2 * sms, v_units), (v_units + VA_SETS - 1) / VA_SETS);

  const uint64_t most = 0x7fffffffu;
  if (units > most || rows > most || v_units > most || rows * D > (uint64_t(1) << 38))
    return kv_refuse(ctx, GRAPE_ERR_LIMIT, "too many rows and columns for one call");
  a.acc_count = rows * D;
  a.done_count = v_rows * VA_WARPS;
  a.padded = (cols + 31) & ~uint64_t(31);
  auto up = [](uint64_t n) { return (n + 255) & ~uint64_t(255); };
  const uint64_t b_max = up((kv_rows * a.tiles + a.score_grid) * ht * 4), b_before = up((a.c.batch + 1) * 4), b_acc = up(a.acc_count * 8);
  const uint64_t b_done = up(a.done_count * 4), b_valid = up(kv_rows * a.padded), b_digits = up(rows * 3 * a.padded), b_rows = up(kv_rows * a.padded * 8), b_weight = up(rows * 8), b_sum = a.sum ? 0 : up(rows * 8);
  const uint64_t b_keys = up(rows * a.max_keys * 4);
  void* w = nullptr;
  if (int rc = kv_workspace(ctx, b_max + b_before + b_acc + b_done + b_valid + b_digits + b_rows + b_weight + b_sum + (a.score ? 0 : b_keys) + (a.exp_out ? 0 : b_keys), &w))
    return rc;
  char* p = reinterpret_cast<char*>(w);
  auto take = [&](uint64_t bytes) {
    char* at = p;
    p += bytes;
    return reinterpret_cast<void*>(at);
  };
  a.piece_max = (int32_t*)take(b_max);
  a.before = (uint32_t*)take(b_before);
  a.acc = (int64_t*)take(b_acc);
  a.done = (uint32_t*)take(b_done);
  a.valid = (unsigned char*)take(b_valid);
  a.digits = (unsigned char*)take(b_digits);
  a.row_at = (int64_t*)take(b_rows);
  a.weight = (int64_t*)take(b_weight);
  if (!a.sum) a.sum = (int64_t*)take(b_sum);
  if (!a.score) a.score = (int32_t*)take(b_keys);
  if (!a.exp_out) a.exp_out = (int32_t*)take(b_keys);
  if (int rc = cache->bits == 32 ? launch_scores<4>(ctx, a, threads, smem) : launch_scores<2>(ctx, a, threads, smem)) return rc;
  if (int rc = launch_softmax(ctx, a, rows, cols)) return rc;
  if (int rc = cache->bits == 32 ? launch_values<4>(ctx, a, v_grid) : launch_values<2>(ctx, a, v_grid)) return rc;
  GRAPE_CUDA_TRY(ctx, cudaGetLastError());
  return GRAPE_OK;
}

}  // namespace grape

using namespace grape;

extern "C" int grape_kv_attend(grape_ctx* ctx, const grape_kv_cache* cache, const int32_t* d_table, uint32_t table_width,
                               uint32_t batch, const int32_t* d_len, const int32_t* d_selected, uint32_t n_select,
                               const int32_t* d_q, uint64_t q_stride, uint32_t heads, uint32_t score_shift,
                               const int32_t* d_exp, int32_t exp_low, uint32_t exp_len, uint32_t soft_shift,
                               uint64_t max_keys, int32_t* d_out, const grape_kv_witness* witness) try {
  if (int rc = kv_check_cache(ctx, cache, d_table, table_width, batch, true, true, false)) return rc;
  if (heads < 1 || heads > 65535 || heads % cache->kv_heads)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "heads must be a multiple of kv_heads up to 65535, not %u", heads);
  if (score_shift > 31) return kv_refuse(ctx, GRAPE_ERR_INVALID, "score_shift must be at most 31, not %u", score_shift);
  if (soft_shift < 1 || soft_shift > 20) return kv_refuse(ctx, GRAPE_ERR_INVALID, "soft_shift must be 1 to 20, not %u", soft_shift);
  if (max_keys < 1 || max_keys > 0x7fffffffu) return kv_refuse(ctx, GRAPE_ERR_INVALID, "max_keys must be 1 to 2^31 - 1");
  if (!d_exp || misaligned(d_exp, 4) || exp_low > 0 || (int64_t)exp_low + exp_len < 1)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "the exp table must be given and hold the argument 0");
  if (d_selected ? n_select < 1 || n_select > (1u << 20) : n_select != 0)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "n_select must be 1 to 2^20 with selected pages and 0 without, not %u", n_select);
  if ((uint64_t)n_select * cache->page_size > 0x7fffffffu) return kv_refuse(ctx, GRAPE_ERR_LIMIT, "n_select * page_size must stay below 2^31");
  const grape_kv_witness none = {};
  const grape_kv_witness& w = witness ? *witness : none;
  if (batch) {
    if (int rc = kv_check_rows(ctx, "queries", d_q, q_stride, (uint64_t)heads * cache->head_dim)) return rc;
    if (!d_len || misaligned(d_len, 4)) return kv_refuse(ctx, GRAPE_ERR_INVALID, "lengths must be given, on 4 bytes");
    if (!d_out) return kv_refuse(ctx, GRAPE_ERR_INVALID, "no output");
  }
  if (misaligned(d_selected, 4) || misaligned(d_out, 16) || misaligned(w.d_out_rem, 16) || misaligned(w.d_score, 16) || misaligned(w.d_score_rem, 16) ||
      misaligned(w.d_exp_in, 16) || misaligned(w.d_exp_out, 16) || misaligned(w.d_softmax, 16) || misaligned(w.d_sum, 8))
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "outputs must be on 16 bytes");
  if ((uint64_t)batch * heads > 0x7fffffffu) return kv_refuse(ctx, GRAPE_ERR_LIMIT, "too many sequences and heads for one call");
  if (!ctx) return kv_refuse(ctx, GRAPE_ERR_INVALID, "null context");
  make_device_current(ctx);
  if (!batch) return GRAPE_OK;
  AttendArgs a{};
  a.c = kv_view(ctx, cache, d_table, table_width, batch);
  a.len = d_len;
  a.selected = d_selected;
  a.n_select = n_select;
  a.q = d_q;
  a.q_stride = q_stride;
  a.heads = heads;
  a.group = heads / cache->kv_heads;
  a.score_shift = score_shift;
  a.soft_shift = soft_shift;
  a.exp = d_exp;
  a.exp_low = exp_low;
  a.exp_len = exp_len;
  a.max_keys = max_keys;
  a.out = d_out;
  a.score = w.d_score;
  a.score_rem = w.d_score_rem;
  a.exp_in = w.d_exp_in;
  a.exp_out = w.d_exp_out;
  a.softmax = w.d_softmax;
  a.sum = w.d_sum;
  a.out_rem = w.d_out_rem;
  // launches of AT_BATCH sequences, one after another on the same workspace
  for (uint32_t b = 0; b < batch; b += AT_BATCH) {
    AttendArgs s = a;
    s.c.batch = std::min(AT_BATCH, batch - b);
    s.c.table += (uint64_t)b * table_width;
    s.len += b;
    s.q += (uint64_t)b * q_stride;
    if (s.selected) s.selected += (uint64_t)b * cache->kv_heads * n_select;
    const uint64_t keys = (uint64_t)b * heads * max_keys, channels = (uint64_t)b * heads * cache->head_dim;
    for (int32_t** p : {&s.score, &s.score_rem, &s.exp_in, &s.exp_out, &s.softmax})
      if (*p) *p += keys;
    s.out += channels;
    if (s.out_rem) s.out_rem += channels;
    if (s.sum) s.sum += (uint64_t)b * heads;
    if (int rc = attend_launch(ctx, cache, s)) return rc;
  }
  if (max_keys < (uint64_t)n_select * cache->page_size)
    return kv_refuse(ctx, GRAPE_CUT, "max_keys %llu cuts the %llu columns of the selected pages", (unsigned long long)max_keys,
                     (unsigned long long)n_select * cache->page_size);
  return GRAPE_OK;
} catch (const std::exception& e) {
  return kv_refuse(nullptr, GRAPE_ERR_NOMEM, "%s", e.what());
}
