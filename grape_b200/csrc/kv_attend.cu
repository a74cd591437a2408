// Attention of one new token per sequence over the paged cache, in the prover's integers
// (grape_kv_attend): every row's scores, exp arguments and values, softmax and output, exactly.
//
// The softmax is rounded with the whole row's sum before it meets the values, so nothing can be rescaled
// later: three passes, joined by an integer maximum and integer sums, whose order changes no bit.
#include <algorithm>
#include <exception>

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
  int32_t* chunk_max;  // [batch][heads][chunks]
  int64_t* acc;        // [batch][heads][head_dim]
  uint32_t* done;      // blocks of a key head's tile and part that have added to acc
  uint32_t tiles, split, chunks, chunk_keys;  // scores: head tiles of a key head, warps of a row, blocks of a row
  uint32_t exp_chunks;
  uint32_t v_tiles, v_parts, v_split, v_chunks, v_chunk_keys;  // values: head tiles, parts of a row, warps of a part, ...
  uint32_t done_per_row;
  unsigned char* valid;   // [batch][kv_heads][columns]: 1 where a column holds a position
  uint64_t valid_stride;
};

// Columns of a row that can hold a position: its length, or the slots of the selected pages.
__device__ __forceinline__ uint32_t columns(const AttendArgs& a, uint32_t b, bool report) {
  const uint32_t n = kv_length(a.c, a.len, b, a.selected ? ~0ull : a.max_keys, report);
  if (!a.selected) return n;
  if (n == 0) return 0;
  const uint64_t all = (uint64_t)a.n_select * a.c.page_size;
  return (uint32_t)min(all, a.max_keys);
}

// Page and slot of column i, or page -1 where the column holds no position.
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

// A lane's own queue in shared memory: 16-byte copies from global memory that this lane alone reads back, so
// that no barrier is needed, only the wait for its own copies, and what is under way costs no registers.
__device__ __forceinline__ void copy_async(uint4* to, const char* from, bool there) {
  // nothing is read where `there` is false: the 16 bytes become zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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
// A warp takes 16 keys (rows g and g + 8 of a lane), 64 bytes of them per step: a lane's 16 bytes are the A
// registers of two instructions, no shuffles, no staging.  The columns (8 words per 4 bytes of a key) are
// built once per block in shared memory.
// What bounds it: bytes of the keys.  The instruction takes 2 cycles of an SM (measured, 570 T products/s) for
// 512 bytes of keys and a head, which arrive every 22 cycles.
constexpr int SC_MAX_THREADS = 512;
constexpr int SC_SMEM = 128 * 1024;      // bytes of a block's columns at most
constexpr int SC_SMEM_ALL = 224 * 1024;  // and of all that it keeps in shared memory

template <int EB>
__device__ __forceinline__ uint32_t column_word(const uint64_t (&u)[4 / EB], int c) {
  // u: q + 0x80808080 per element, whose bytes are the digits + 128 and whose fifth byte is the fifth digit
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4 / EB; e++) {
#pragma unroll
    for (int p = 0; p < EB; p++) {
      const int r = c - p;
      if (r >= 0 && r <= 4) {
        uint32_t digit = (uint32_t)(u[e] >> (8 * r)) & 0xffu;
        if (r < 4) digit ^= 0x80u;
        w |= digit << (8 * (e * EB + p));
      }
    }
  }
  return w;
}

__host__ __device__ constexpr int sc_sixteens(int ht) { return ht >= 4 ? 2 : 1; }  // sixteens of keys that share a read of the columns
__host__ __device__ constexpr int sc_stages(int ht) { return ht >= 4 ? 4 : 5; }    // steps in a lane's queue

template <int EB, int HT>
__global__ void __launch_bounds__(SC_MAX_THREADS) k_kv_scores(AttendArgs a) {
  constexpr int MT = sc_sixteens(HT), STAGES = sc_stages(HT);
  constexpr int NV = 2 * MT * HT;               // values of a lane group: (head, eight of keys)
  constexpr int OWN = NV >= 4 ? NV / 4 : 1;     // those that a lane finishes
  constexpr int HEADS = HT >= 4 ? HT / 4 : 1;   // and the heads they belong to
  extern __shared__ uint4 s_w[];  // [blk][HT][32 lanes]: 4 words, the columns of a lane's 16 bytes; the lanes' queues; partial sums
  __shared__ unsigned long long s_bias[HT];
  __shared__ int32_t s_max[HT];
  __shared__ unsigned char s_valid[SC_MAX_THREADS / 32][16 * MT];
  const KvView& c = a.c;
  const uint32_t D = c.head_dim, row_bytes = D * EB, blks = (row_bytes + 63) / 64;
  uint32_t x = blockIdx.x;
  const uint32_t tile = x % a.tiles;
  x /= a.tiles;
  const uint32_t chunk = x % a.chunks, row = x / a.chunks, g = row % c.kv_heads, b = row / c.kv_heads;
  const uint32_t h0 = g * a.group + tile * HT, hn = min((uint32_t)HT, a.group - tile * HT);
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = blockDim.x >> 5;
  const uint32_t n = kv_length(c, a.len, b, a.selected ? ~0ull : a.max_keys, false);
  const uint32_t cols = columns(a, b, chunk == 0 && tid == 0);
  const uint64_t row0 = (uint64_t)b * a.heads + h0;  // first of the block's rows
  if (chunk == 0) {
    // what the later passes add to
    for (uint32_t i = tid; i < hn * D; i += blockDim.x) a.acc[row0 * D + i] = 0;
    for (uint32_t i = tid; i < hn; i += blockDim.x) a.sum[row0 + i] = 0;
    for (uint32_t i = tid; tile == 0 && i < a.done_per_row; i += blockDim.x) a.done[(uint64_t)row * a.done_per_row + i] = 0;
    if (cols == 0) {
      for (uint32_t i = tid; i < hn * D; i += blockDim.x) {
        a.out[row0 * D + i] = 0;
        if (a.out_rem) a.out_rem[row0 * D + i] = 0;
      }
    }
  }
  const uint32_t first = chunk * a.chunk_keys, last = min(cols, first + a.chunk_keys);
  if (first >= last) return;

  const uint32_t gl = lane >> 2, t = lane & 3;
  const uint32_t wd = warp % a.split, wk = warp / a.split, keys_at_once = warps / a.split * 16 * MT;
  const uint32_t blk0 = blks * wd / a.split, blk1 = blks * (wd + 1) / a.split;

  // A step is 64 bytes of the warp's 16 MT keys.  `fetch` walks the steps STAGES - 1 ahead of their use; which of
  // a lane's keys exist goes through `fifo`, four bits for each set of keys under way.
  uint4* const queue = s_w + (uint64_t)blks * HT * 32 + (uint64_t)warp * STAGES * MT * 64 + lane;
  const char* key[2 * MT];
  uint32_t ahead_base = first, ahead_blk = blk0, ahead_slot = 0, fifo = 0, under_way = 0;
  auto fetch = [&]() {
    if (ahead_base < last) {
      if (ahead_blk == blk0) {
        uint32_t mask = 0;
#pragma unroll
        for (int m = 0; m < 2 * MT; m++) {
          const uint32_t i = ahead_base + wk * 16 * MT + m * 8 + gl;
          uint32_t slot;
          const int32_t page = i < last ? column_page(a, b, g, n, i, slot, t == 0 && wd == 0) : -1;
          key[m] = page >= 0 ? c.k + page * c.page_stride + g * c.head_stride + slot * c.slot_stride + t * 16 : nullptr;
          if (page >= 0) mask |= 1u << m;
        }
        fifo |= mask << (4 * under_way++);
      }
      const bool in = ahead_blk * 64 + t * 16 < row_bytes;
#pragma unroll
      for (int m = 0; m < 2 * MT; m++) {
        const bool there = in && key[m];
        copy_async(queue + (ahead_slot * 2 * MT + m) * 32, there ? key[m] + ahead_blk * 64 : c.k, there);
      }
      ahead_slot = ahead_slot + 1 == STAGES ? 0 : ahead_slot + 1;
      if (++ahead_blk == blk1) {
        ahead_blk = blk0;
        ahead_base += keys_at_once;
      }
    }
    copy_commit();
  };
#pragma unroll 1
  for (int i = 0; i < STAGES - 1; i++) fetch();

  // the operand columns, and the sum of each head's query
  if (tid < HT) { s_bias[tid] = 0; s_max[tid] = INT32_MIN; }
  __syncthreads();
  {
    constexpr uint32_t PER = 4 / EB;  // elements of a word
    const uint32_t share = blockDim.x / HT, h = tid / share;
    const int32_t* q = a.q + (uint64_t)b * a.q_stride + (uint64_t)(h0 + h) * D;
    int64_t total = 0;
    for (uint32_t i = tid % share; i < blks * 16; i += share) {
      uint64_t u[PER];
#pragma unroll
      for (uint32_t e = 0; e < PER; e++) {
        const uint32_t d = i * PER + e;
        const int32_t v = h < hn && d < D ? __ldg(q + d) : 0;
        total += v;
        u[e] = (uint64_t)((int64_t)v + 0x80808080ll);
      }
      // word i of the row: block i / 16, lane group (i / 4) % 4, word i % 4
      uint32_t* to = reinterpret_cast<uint32_t*>(s_w + ((uint64_t)(i / 16) * HT + h) * 32 + (i / 4) % 4) + i % 4;
#pragma unroll
      for (int k = 0; k < 8; k++) to[k * 16] = column_word<EB>(u, k);
    }
    for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(~0u, total, o);
    if (lane == 0) atomicAdd(&s_bias[h], (unsigned long long)total);
  }
  __syncthreads();

  const uint64_t bias = EB == 4 ? uint64_t(1) << 31 : uint64_t(1) << 15;
  constexpr uint32_t FLIP = EB == 4 ? 0x80000000u : 0x80008000u;
  int32_t best[HEADS];
#pragma unroll
  for (int j = 0; j < HEADS; j++) best[j] = INT32_MIN;
  bool range = false;
  auto finish = [&](uint64_t acc, uint32_t h, uint32_t i) {
    acc -= bias * (uint64_t)s_bias[h];
    const int64_t s = rdiv((int64_t)acc, a.score_shift);
    const int32_t v = saturate(s, INT32_MIN, INT32_MAX, range);
    const uint64_t at = (row0 + h) * a.max_keys + i;
    a.score[at] = v;
    if (a.score_rem) a.score_rem[at] = (int32_t)(uint32_t)(acc - ((uint64_t)s << a.score_shift));
    return v;
  };

  uint32_t slot = 0;
  for (uint32_t base = first; base < last; base += keys_at_once) {
    int32_t acc[HT][MT][4];
#pragma unroll
    for (int h = 0; h < HT; h++)
#pragma unroll
      for (int m = 0; m < MT; m++) acc[h][m][0] = acc[h][m][1] = acc[h][m][2] = acc[h][m][3] = 0;
#pragma unroll 1
    for (uint32_t blk = blk0; blk < blk1; blk++) {
      copy_wait<STAGES - 2>();
      uint4 y[2 * MT];
#pragma unroll
      for (int m = 0; m < 2 * MT; m++) {
        y[m] = queue[(slot * 2 * MT + m) * 32];
        y[m].x ^= FLIP;
        y[m].y ^= FLIP;
        y[m].z ^= FLIP;
        y[m].w ^= FLIP;
      }
      slot = slot + 1 == STAGES ? 0 : slot + 1;
      fetch();  // into the place that was read a step ago
      const uint4* w = s_w + (uint64_t)blk * HT * 32 + lane;
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
    const uint32_t mask = fifo & 15;
    fifo >>= 4;
    under_way--;
    // Lane (g, t) holds columns 2t and 2t + 1 of keys g and g + 8.  The sum over t leaves lane t with the values
    // t OWN .. of (head * MT + sixteen) * 2 + eight: each lane finishes its own.
    uint64_t v[NV];
#pragma unroll
    for (int h = 0; h < HT; h++)
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int e = 0; e < 2; e++)
          v[(h * MT + m) * 2 + e] = ((uint64_t)(int64_t)acc[h][m][2 * e] + ((uint64_t)(int64_t)acc[h][m][2 * e + 1] << 8)) << (16 * t);
    if (NV >= 4) {
#pragma unroll
      for (int j = 0; j < NV / 2; j++) {
        const uint64_t keep = t & 2 ? v[j + NV / 2] : v[j], give = t & 2 ? v[j] : v[j + NV / 2];
        v[j] = keep + __shfl_xor_sync(~0u, give, 2);
      }
    } else {
      v[0] += __shfl_xor_sync(~0u, v[0], 2);
      v[1] += __shfl_xor_sync(~0u, v[1], 2);
    }
#pragma unroll
    for (int j = 0; j < OWN; j++) {
      const uint64_t keep = t & 1 ? v[j + OWN] : v[j], give = t & 1 ? v[j] : v[j + OWN];
      v[j] = keep + __shfl_xor_sync(~0u, give, 1);
    }
    const uint32_t own0 = NV >= 4 ? t * OWN : t & 1, key0 = base + wk * 16 * MT + gl;
    if (tile == 0 && wd == 0 && t < 2 * MT && key0 + t * 8 < last) a.valid[(uint64_t)row * a.valid_stride + key0 + t * 8] = (mask >> t) & 1;
    if (a.split == 1) {
#pragma unroll
      for (int j = 0; j < OWN; j++) {
        const uint32_t own = own0 + j, h = own / (2 * MT), e = own % (2 * MT);
        if (h < hn && (NV >= 4 || t < 2) && ((mask >> e) & 1)) best[j * HEADS / OWN] = max(best[j * HEADS / OWN], finish(v[j], h, key0 + e * 8));
      }
    } else {
      // warps that share the keys add up in shared memory, [warp][value][g]
      int64_t* s_part = reinterpret_cast<int64_t*>(s_w + (uint64_t)blks * HT * 32 + (uint64_t)warps * STAGES * MT * 64);
      __syncthreads();
#pragma unroll
      for (int j = 0; j < OWN; j++)
        if (NV >= 4 || t < 2) s_part[((uint64_t)warp * NV + own0 + j) * 8 + gl] = (int64_t)v[j];
      if (wd == 0 && t < 2 * MT) s_valid[wk][t * 8 + gl] = (mask >> t) & 1;
      __syncthreads();
      for (uint32_t i = wd * 32 + lane; i < NV * 8; i += a.split * 32) {
        const uint32_t own = i / 8, h = own / (2 * MT), at = own % (2 * MT) * 8 + i % 8;
        if (h >= hn || !s_valid[wk][at]) continue;
        uint64_t sum = 0;
        for (uint32_t w = 0; w < a.split; w++) sum += (uint64_t)s_part[((uint64_t)(wk * a.split + w) * NV + own) * 8 + i % 8];
        atomicMax(&s_max[h], finish(sum, h, base + wk * 16 * MT + at));
      }
    }
  }
  if (range) kv_flag(c, STATUS_KV_RANGE);
  if (a.split == 1) {
#pragma unroll
    for (int j = 0; j < HEADS; j++) {
      for (int o = 16; o >= 4; o >>= 1) best[j] = max(best[j], __shfl_xor_sync(~0u, best[j], o));
      const uint32_t h = HT >= 4 ? t * HEADS + j : HT == 2 ? t >> 1 : 0;
      if (gl == 0) atomicMax(&s_max[h], best[j]);
    }
  }
  __syncthreads();
  if (tid < hn) a.chunk_max[(row0 + tid) * a.chunks + chunk] = s_max[tid];
}

// ---- exp -----------------------------------------------------------------------------------------
// exp_in, exp_out and the row's sum.  The table (4 MB for the layer prover's) lives in L2; a thread has four
// columns under way, since what it waits for is a chain of three loads.
constexpr int EX_THREADS = 256, EX_COLS = 4;
constexpr uint32_t EX_KEYS = EX_THREADS * EX_COLS;  // columns of a block

__global__ void __launch_bounds__(EX_THREADS) k_kv_exp(AttendArgs a) {
  __shared__ int32_t s_max[EX_THREADS / 32];
  __shared__ int64_t s_sum[EX_THREADS / 32];
  const KvView& c = a.c;
  const uint32_t chunk = blockIdx.x % a.exp_chunks, row = blockIdx.x / a.exp_chunks, h = row % a.heads, b = row / a.heads, g = h / a.group;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t cols = columns(a, b, false), first = chunk * EX_KEYS + threadIdx.x;
  if (chunk * EX_KEYS >= cols) return;
  const uint64_t at = (uint64_t)row * a.max_keys + first;
  const unsigned char* valid = a.valid + ((uint64_t)b * c.kv_heads + g) * a.valid_stride + first;
  bool in[EX_COLS];
  int32_t s[EX_COLS];
#pragma unroll
  for (int j = 0; j < EX_COLS; j++) {
    in[j] = first + j * EX_THREADS < cols && valid[j * EX_THREADS];
    s[j] = first + j * EX_THREADS < cols ? a.score[at + j * EX_THREADS] : 0;
  }
  int32_t best = INT32_MIN;
  const uint32_t used = (cols + a.chunk_keys - 1) / a.chunk_keys;
  for (uint32_t i = threadIdx.x; i < used; i += EX_THREADS) best = max(best, a.chunk_max[(uint64_t)row * a.chunks + i]);
  best = __reduce_max_sync(~0u, best);
  if (lane == 0) s_max[warp] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < EX_THREADS / 32; w++) best = max(best, s_max[w]);
  int64_t sum = 0;
  bool outside = false;
  int32_t x[EX_COLS], e[EX_COLS];
#pragma unroll
  for (int j = 0; j < EX_COLS; j++) {
    const int64_t d = in[j] ? (int64_t)s[j] - best : 0;
    outside |= d < a.exp_low;
    x[j] = (int32_t)max(d, (int64_t)a.exp_low);
    e[j] = __ldg(a.exp + (x[j] - a.exp_low));
  }
#pragma unroll
  for (int j = 0; j < EX_COLS; j++) {
    if (!in[j]) continue;
    if (e[j] < 0) { e[j] = 0; outside = true; }
    sum += e[j];
    if (a.exp_in) a.exp_in[at + j * EX_THREADS] = x[j];
    a.exp_out[at + j * EX_THREADS] = e[j];
  }
  if (outside) kv_flag(c, STATUS_KV_EXP);
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(~0u, sum, o);
  if (lane == 0) s_sum[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < EX_THREADS / 32; w++) sum += s_sum[w];
    atomicAdd(reinterpret_cast<unsigned long long*>(a.sum + row), (unsigned long long)sum);
  }
}

// ---- values ----------------------------------------------------------------------------------------
// sum_j o_j v_j exactly, on the same instruction.  o is at most 2^20: three unsigned digits base 256, which are
// the operand columns (3 per head); the rows are the bytes of v (v' = v + bias unsigned), so that
//   sum_j o_j v_j = sum_p,r 256^(p + r) (byte plane p of v' . digit r of o) - bias sum_j o_j.
// A warp takes 32 keys x 128 bytes of their rows: lane (g, t) loads 16 bytes of the 8 keys 8t .. 8t+7, and
// turning 4 keys x 4 bytes in registers (8 byte permutes) gives the A registers, keys along the instruction's
// inner dimension.  Sums of a chunk of at most 1024 keys stay far below 2^31.  The 8 bytes of digits that a lane
// needs for 32 keys lie together in shared memory.
// What bounds it: bytes of the values; 32 keys x 128 bytes cost a warp about 100 instructions of the 700 that
// an SM quarter issues while they arrive.
constexpr uint32_t VA_CHUNK = 1024;           // keys of a block at most
constexpr uint32_t VA_STRIDE = VA_CHUNK + 32; // bytes of a column's digits: eight columns on different banks
__host__ __device__ constexpr int va_tiles(int ht) { return (3 * ht + 7) / 8; }                   // instruction columns in eights
__host__ __device__ constexpr int va_threads(int ht) { return va_tiles(ht) > 2 ? 128 : 256; }     // by the registers of the sums
constexpr int VA_STAGES = 2;
constexpr size_t va_smem(int ht) {  // queues (later partial sums of 8 columns), digits, places of the keys
  return (size_t)va_threads(ht) / 32 * VA_STAGES * 4096 + (size_t)VA_STRIDE * 8 * va_tiles(ht) + VA_CHUNK * 8;
}

// bytes [key][plane] of 4 words -> words [plane] of 4 keys
__device__ __forceinline__ void turn4(uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t (&o)[4]) {
  const uint32_t ab0 = __byte_perm(a, b, 0x5140), ab1 = __byte_perm(a, b, 0x7362);
  const uint32_t cd0 = __byte_perm(c, d, 0x5140), cd1 = __byte_perm(c, d, 0x7362);
  o[0] = __byte_perm(ab0, cd0, 0x5410);
  o[1] = __byte_perm(ab0, cd0, 0x7632);
  o[2] = __byte_perm(ab1, cd1, 0x5410);
  o[3] = __byte_perm(ab1, cd1, 0x7632);
}

template <int EB, int HT>
__global__ void __launch_bounds__(va_threads(HT), 512 / va_threads(HT) - (va_tiles(HT) > 2 ? 1 : 0)) k_kv_values(AttendArgs a) {
  constexpr int NT = va_tiles(HT), THREADS = va_threads(HT);
  constexpr uint32_t ELEMS = 128 / EB;       // channels of a warp
  extern __shared__ uint4 s_dyn[];
  __shared__ unsigned long long s_total[HT];
  __shared__ int64_t s_sum[HT];
  __shared__ double s_inverse[HT];
  __shared__ uint32_t s_last;
  unsigned char* const s_digits = reinterpret_cast<unsigned char*>(s_dyn + THREADS / 32 * VA_STAGES * 256);
  int64_t* const s_at = reinterpret_cast<int64_t*>(s_digits + VA_STRIDE * 8 * NT);
  const KvView& c = a.c;
  const uint32_t D = c.head_dim, row_bytes = D * EB, segments = (row_bytes + 127) / 128;
  uint32_t x = blockIdx.x;
  const uint32_t tile = x % a.v_tiles;
  x /= a.v_tiles;
  const uint32_t part = x % a.v_parts;
  x /= a.v_parts;
  const uint32_t chunk = x % a.v_chunks, row = x / a.v_chunks, g = row % c.kv_heads, b = row / c.kv_heads;
  const uint32_t h0 = g * a.group + tile * HT, hn = min((uint32_t)HT, a.group - tile * HT);
  const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, gl = lane >> 2, t = lane & 3;
  const uint32_t n = kv_length(c, a.len, b, a.selected ? ~0ull : a.max_keys, false), cols = columns(a, b, false);
  const uint32_t first = chunk * a.v_chunk_keys, keys = min(cols, first + a.v_chunk_keys) - first;
  if (first >= cols) return;
  const uint64_t row0 = (uint64_t)b * a.heads + h0;
  const uint32_t wd = warp % a.v_split, wk = warp / a.v_split, groups = THREADS / 32 / a.v_split;
  const uint32_t segment = part * a.v_split + wd, byte = segment * 128 + gl * 16;
  const bool in_row = segment < segments && byte < row_bytes;
  const uint32_t padded = (keys + 31) & ~31u;
  for (uint32_t j = tid; j < padded; j += THREADS) {
    uint32_t slot = 0;
    const int32_t page = j < keys ? column_page(a, b, g, n, first + j, slot, false) : -1;
    s_at[j] = page >= 0 ? page * c.page_stride + g * c.head_stride + slot * c.slot_stride : -1;
  }
  if (tid < HT) {
    s_total[tid] = 0;
    s_sum[tid] = tid < hn ? a.sum[row0 + tid] : 0;
    s_inverse[tid] = s_sum[tid] > 0 ? 1.0 / (double)s_sum[tid] : 0.0;
  }
  __syncthreads();

  uint4* const queue = s_dyn + (uint64_t)warp * VA_STAGES * 256 + lane;
  auto fetch = [&](uint32_t k0, uint32_t stage) {
    if (k0 < padded) {
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const int64_t at = s_at[k0 + 8 * t + j];
        const bool there = in_row && at >= 0;
        copy_async(queue + (stage * 8 + j) * 32, there ? c.v + at + byte : c.v, there);
      }
    }
    copy_commit();
  };
  fetch(wk * 32, 0);
  fetch((wk + groups) * 32, 1);

  // the softmax of the chunk, while the first values are under way
  for (uint32_t j = tid; j < padded; j += THREADS) {
    const bool there = s_at[j] >= 0;
    int32_t e[HT];
#pragma unroll
    for (int h = 0; h < HT; h++) e[h] = there && h < hn ? a.exp_out[(row0 + h) * a.max_keys + first + j] : 0;
#pragma unroll
    for (int h = 0; h < HT; h++) {
      uint32_t o = 0;
      if (there && h < hn) {
        const int64_t sum = s_sum[h], top = ((int64_t)e[h] << a.soft_shift) + sum / 2;
        if (sum > 0) {
          // the quotient is at most 2^20: a 64-bit floating point estimate is off by one at most
          int64_t k = (int64_t)((double)top * s_inverse[h]);
          const int64_t r = top - k * sum;
          k += r < 0 ? -1 : r >= sum ? 1 : 0;
          o = (uint32_t)k;
        }
        if (a.softmax && part == 0) a.softmax[(row0 + h) * a.max_keys + first + j] = (int32_t)o;
      }
      s_digits[(3 * h) * VA_STRIDE + j] = (unsigned char)o;
      s_digits[(3 * h + 1) * VA_STRIDE + j] = (unsigned char)(o >> 8);
      s_digits[(3 * h + 2) * VA_STRIDE + j] = (unsigned char)(o >> 16);
      const uint32_t warp_sum = __reduce_add_sync(~0u, o);  // at most 32 x 2^20; whole warps: padded is a multiple of 32
      if (lane == 0 && warp_sum) atomicAdd(&s_total[h], (unsigned long long)warp_sum);
    }
#pragma unroll
    for (int k = 3 * HT; k < 8 * NT; k++) s_digits[k * VA_STRIDE + j] = 0;
  }
  __syncthreads();

  int32_t acc[8][NT][4];
#pragma unroll
  for (int m = 0; m < 8; m++)
#pragma unroll
    for (int k = 0; k < NT; k++) acc[m][k][0] = acc[m][k][1] = acc[m][k][2] = acc[m][k][3] = 0;
  uint32_t stage = 0;
#pragma unroll 1
  for (uint32_t k0 = wk * 32; k0 < padded; k0 += groups * 32) {
    copy_wait<VA_STAGES - 1>();
    uint4 v[8];
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = queue[(stage * 8 + j) * 32];
    uint2 d[NT];
#pragma unroll
    for (int k = 0; k < NT; k++) d[k] = *reinterpret_cast<const uint2*>(s_digits + (k * 8 + gl) * VA_STRIDE + k0 + 8 * t);
#pragma unroll
    for (int w = 0; w < 4; w++) {
      uint32_t p[4], r[4];
      auto word = [&](int j) { return w == 0 ? v[j].x : w == 1 ? v[j].y : w == 2 ? v[j].z : v[j].w; };
      turn4(word(0), word(1), word(2), word(3), p);
      turn4(word(4), word(5), word(6), word(7), r);
      p[3] ^= 0x80808080u;
      r[3] ^= 0x80808080u;
      if (EB == 2) { p[1] ^= 0x80808080u; r[1] ^= 0x80808080u; }
#pragma unroll
      for (int k = 0; k < NT; k++) {
        mma_u8u8(acc[2 * w][k], p[0], p[1], r[0], r[1], d[k].x, d[k].y);
        mma_u8u8(acc[2 * w + 1][k], p[2], p[3], r[2], r[3], d[k].x, d[k].y);
      }
    }
    fetch(k0 + 2 * groups * 32, stage);  // every register of this place has been used
    stage ^= 1;
  }
  copy_wait<0>();

  // weights of the byte planes in the lane; digits and the warps that dealt the keys through shared memory:
  // s_part[warp][column of eight][channel], eight columns at a time
  int64_t* s_part = reinterpret_cast<int64_t*>(s_dyn);
  const uint32_t outputs = a.v_split * ELEMS;  // channels of the block
  constexpr int MINE = (HT * THREADS / 32 * ELEMS + THREADS - 1) / THREADS;  // (head, channel) of a thread at most
  uint64_t mine[MINE];
#pragma unroll
  for (int i = 0; i < MINE; i++) mine[i] = 0;
#pragma unroll
  for (int k = 0; k < NT; k++) {
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; w++) {
#pragma unroll
      for (int half = 0; half < 2; half++) {
        const uint64_t a0 = (uint64_t)(int64_t)acc[2 * w][k][half] + ((uint64_t)(int64_t)acc[2 * w][k][2 + half] << 8);
        const uint64_t a1 = (uint64_t)(int64_t)acc[2 * w + 1][k][half] + ((uint64_t)(int64_t)acc[2 * w + 1][k][2 + half] << 8);
        int64_t* to = s_part + ((uint64_t)warp * 8 + 2 * t + half) * ELEMS;
        if (EB == 4) {
          to[gl * 4 + w] = (int64_t)(a0 + (a1 << 16));
        } else {
          to[gl * 8 + 2 * w] = (int64_t)a0;
          to[gl * 8 + 2 * w + 1] = (int64_t)a1;
        }
      }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < MINE; i++) {
      const uint32_t at = i * THREADS + tid, h = at / outputs, ch = at % outputs;
      if (h < hn) {
        for (uint32_t r = 0; r < 3; r++) {
          const uint32_t col = 3 * h + r;
          if (col / 8 != k) continue;
          uint64_t v = 0;
          for (uint32_t z = 0; z < groups; z++)
            v += (uint64_t)s_part[((uint64_t)(z * a.v_split + ch / ELEMS) * 8 + col % 8) * ELEMS + ch % ELEMS];
          mine[i] += v << (8 * r);
        }
      }
    }
  }
  const uint64_t bias = EB == 4 ? uint64_t(1) << 31 : uint64_t(1) << 15;
  const uint32_t used = (cols + a.v_chunk_keys - 1) / a.v_chunk_keys;
  const uint32_t ch0 = part * outputs;
  bool range = false;
  auto finish = [&](int64_t sum, uint64_t at) {
    const int64_t y = rdiv(sum, a.soft_shift);
    a.out[at] = saturate(y, INT32_MIN, INT32_MAX, range);
    if (a.out_rem) a.out_rem[at] = (int32_t)(uint32_t)((uint64_t)sum - ((uint64_t)y << a.soft_shift));
  };
#pragma unroll
  for (int i = 0; i < MINE; i++) {
    const uint32_t at = i * THREADS + tid, h = at / outputs, ch = ch0 + at % outputs;
    if (h < hn && ch < D) {
      const uint64_t v = mine[i] - bias * (uint64_t)s_total[h], to = (row0 + h) * D + ch;
      if (used == 1) finish((int64_t)v, to);
      else atomicAdd(reinterpret_cast<unsigned long long*>(a.acc + to), (unsigned long long)v);
    }
  }
  if (used > 1) {
    // the last of the row's blocks brings the sums to the output
    __threadfence();
    __syncthreads();
    if (tid == 0) s_last = atomicAdd(a.done + (((uint64_t)row * a.v_tiles + tile) * a.v_parts + part), 1u) == used - 1;
    __syncthreads();
    if (s_last) {
      __threadfence();
      for (uint32_t at = tid; at < hn * outputs; at += THREADS) {
        const uint32_t h = at / outputs, ch = ch0 + at % outputs;
        if (ch < D) finish(__ldcg(a.acc + (row0 + h) * D + ch), (row0 + h) * D + ch);
      }
    }
  }
  if (range) kv_flag(c, STATUS_KV_RANGE);
  if (chunk == 0 && part == 0 && tid < hn && a.sum[row0 + tid] == 0) kv_flag(c, STATUS_KV_EXP);
}

template <class K>
static int launch(grape_ctx* ctx, K kernel, const AttendArgs& a, uint64_t grid, uint32_t threads, size_t smem) {
  if (smem > 48 * 1024) GRAPE_CUDA_TRY(ctx, cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
  kernel<<<(uint32_t)grid, threads, smem, ctx->stream>>>(a);
  ctx->launches += 1;
  return GRAPE_OK;
}

template <int EB>
static int launch_scores(grape_ctx* ctx, const AttendArgs& a, uint32_t ht, uint64_t grid, uint32_t threads, size_t smem) {
  return launch(ctx, ht == 1 ? k_kv_scores<EB, 1> : ht == 2 ? k_kv_scores<EB, 2> : ht == 4 ? k_kv_scores<EB, 4> : k_kv_scores<EB, 8>, a, grid, threads,
                smem);
}

template <int EB>
static int launch_values(grape_ctx* ctx, const AttendArgs& a, uint32_t ht, uint64_t grid) {
  return launch(ctx, ht == 1 ? k_kv_values<EB, 1> : ht == 2 ? k_kv_values<EB, 2> : ht == 5 ? k_kv_values<EB, 5> : k_kv_values<EB, 8>, a, grid,
                va_threads(ht), va_smem(ht));
}

static int attend_launch(grape_ctx* ctx, const grape_kv_cache* cache, AttendArgs& a) {
  const uint64_t rows = (uint64_t)a.c.batch * a.heads, D = cache->head_dim, kv_rows = (uint64_t)a.c.batch * cache->kv_heads;
  const uint64_t all = a.selected ? (uint64_t)a.n_select * cache->page_size : (uint64_t)a.c.width * cache->page_size;
  const uint64_t cols = std::min(all, a.max_keys);
  const uint32_t row_bytes = (uint32_t)(D * cache->bits / 8), sms = (uint32_t)ctx->sm_count;

  // Scores: heads of a block (their columns are 8 times a key's bytes), warps that share a row of long keys
  // (eight 64-byte steps each at least), and keys of a block: 256 KB of them, fewer while that leaves the GPU
  // with under four blocks an SM.
  uint32_t ht = 1;
  while (ht < 8 && ht < a.group && (uint64_t)2 * ht * row_bytes * 8 <= SC_SMEM) ht *= 2;
  a.tiles = (a.group + ht - 1) / ht;
  const uint32_t blks = (row_bytes + 63) / 64, mt = sc_sixteens(ht);
  const size_t columns_bytes = (size_t)blks * ht * 512, queue_bytes = (size_t)sc_stages(ht) * mt * 1024, part_bytes = (size_t)2 * mt * ht * 64;
  // columns that leave room for one block an SM: 16 warps instead of 8, where their queues still fit
  const uint32_t threads = columns_bytes >= 48 * 1024 && columns_bytes + 16 * (queue_bytes + part_bytes) <= SC_SMEM_ALL ? 512 : 256;
  a.split = 1;
  while (a.split < threads / 32 && blks / (2 * a.split) >= 8) a.split *= 2;
  const size_t smem = columns_bytes + threads / 32 * (queue_bytes + (a.split > 1 ? part_bytes : 0));
  const uint32_t step = threads / 32 / a.split * 16 * mt;
  uint64_t keys = std::max<uint64_t>(step, (256 * 1024 / row_bytes + step - 1) / step * step);
  while (keys > step && kv_rows * a.tiles * ((cols + keys - 1) / keys) < 4ull * sms) keys = std::max<uint64_t>(step, keys / 2 / step * step);
  a.chunk_keys = (uint32_t)keys;
  const uint64_t chunks = (cols + keys - 1) / keys, exp_chunks = (cols + EX_KEYS - 1) / EX_KEYS;

  // Values: heads of a block (three columns each, in eights), 128-byte segments of a row dealt to the warps,
  // the rest of the warps share the keys.
  const uint32_t v_ht = a.group == 1 ? 1 : a.group == 2 ? 2 : a.group <= 5 ? 5 : 8;
  a.v_tiles = (a.group + v_ht - 1) / v_ht;
  const uint32_t segments = (row_bytes + 127) / 128, v_warps = va_threads(v_ht) / 32;
  a.v_split = 1;
  while (a.v_split < v_warps && a.v_split < segments) a.v_split *= 2;
  a.v_parts = (segments + a.v_split - 1) / a.v_split;
  const uint32_t v_step = v_warps / a.v_split * 32;
  uint64_t v_keys = VA_CHUNK;
  while (v_keys > v_step && kv_rows * a.v_tiles * a.v_parts * ((cols + v_keys - 1) / v_keys) < 4ull * sms) v_keys /= 2;
  a.v_chunk_keys = (uint32_t)v_keys;
  const uint64_t v_chunks = (cols + v_keys - 1) / v_keys;

  const uint64_t most = 0x7fffffffu;
  if (kv_rows * a.tiles * chunks > most || rows * exp_chunks > most || kv_rows * a.v_tiles * a.v_parts * v_chunks > most ||
      rows * D > (uint64_t(1) << 38))
    return kv_refuse(ctx, GRAPE_ERR_LIMIT, "too many rows and columns for one call");
  a.chunks = (uint32_t)chunks;
  a.exp_chunks = (uint32_t)exp_chunks;
  a.v_chunks = (uint32_t)v_chunks;
  const uint64_t dones = kv_rows * a.v_tiles * a.v_parts;
  a.done_per_row = (uint32_t)((uint64_t)a.v_tiles * a.v_parts);
  a.valid_stride = (cols + 15) & ~uint64_t(15);
  auto up = [](uint64_t n) { return (n + 255) & ~uint64_t(255); };
  const uint64_t b_max = up(rows * chunks * 4), b_acc = up(rows * D * 8), b_done = up(dones * 4), b_valid = up(kv_rows * a.valid_stride), b_sum = a.sum ? 0 : up(rows * 8);
  const uint64_t b_keys = up(rows * a.max_keys * 4);
  void* w = nullptr;
  if (int rc = kv_workspace(ctx, b_max + b_acc + b_done + b_valid + b_sum + (a.score ? 0 : b_keys) + (a.exp_out ? 0 : b_keys), &w)) return rc;
  char* p = reinterpret_cast<char*>(w);
  a.chunk_max = reinterpret_cast<int32_t*>(p);
  p += b_max;
  a.acc = reinterpret_cast<int64_t*>(p);
  p += b_acc;
  a.done = reinterpret_cast<uint32_t*>(p);
  p += b_done;
  a.valid = reinterpret_cast<unsigned char*>(p);
  p += b_valid;
  if (!a.sum) { a.sum = reinterpret_cast<int64_t*>(p); p += b_sum; }
  if (!a.score) { a.score = reinterpret_cast<int32_t*>(p); p += b_keys; }
  if (!a.exp_out) { a.exp_out = reinterpret_cast<int32_t*>(p); p += b_keys; }

  const uint64_t grid = kv_rows * a.tiles * chunks;
  if (int rc = cache->bits == 32 ? launch_scores<4>(ctx, a, ht, grid, threads, smem) : launch_scores<2>(ctx, a, ht, grid, threads, smem)) return rc;
  if (int rc = launch(ctx, k_kv_exp, a, rows * exp_chunks, EX_THREADS, 0)) return rc;
  if (int rc = cache->bits == 32 ? launch_values<4>(ctx, a, v_ht, dones * v_chunks) : launch_values<2>(ctx, a, v_ht, dones * v_chunks)) return rc;
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
  return attend_launch(ctx, cache, a);
} catch (const std::exception& e) {
  return kv_refuse(nullptr, GRAPE_ERR_NOMEM, "%s", e.what());
}
