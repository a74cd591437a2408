// Paged key-value cache of the decode step: appending tokens with their position rotation
// (grape_kv_append) and choosing pages by the bounds of their keys (grape_kv_select).
#include <algorithm>
#include <cstdio>
#include <exception>

#include "kv.cuh"

namespace grape {

static thread_local char g_kv_error[256];

int kv_refuse(grape_ctx* ctx, int code, const char* format, ...) {
  va_list args;
  va_start(args, format);
  vsnprintf(g_kv_error, sizeof g_kv_error, format, args);
  va_end(args);
  return fail(ctx, code, g_kv_error);
}

int kv_check_cache(grape_ctx* ctx, const grape_kv_cache* c, const int32_t* d_table, uint32_t width, uint32_t batch,
                   bool keys, bool values, bool bounds) {
  if (!c) return kv_refuse(ctx, GRAPE_ERR_INVALID, "cache is null");
  if ((keys && !c->d_k) || (values && !c->d_v)) return kv_refuse(ctx, GRAPE_ERR_INVALID, "cache without pages");
  if (bounds && !c->d_bounds) return kv_refuse(ctx, GRAPE_ERR_INVALID, "cache without bounds");
  if (c->bits != 16 && c->bits != 32) return kv_refuse(ctx, GRAPE_ERR_INVALID, "cache bits must be 16 or 32, not %u", c->bits);
  if (c->head_dim < 8 || c->head_dim > 4096 || c->head_dim % 8)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "head_dim must be a multiple of 8 up to 4096, not %u", c->head_dim);
  if (c->page_size < 1 || c->page_size > 4096) return kv_refuse(ctx, GRAPE_ERR_INVALID, "page_size must be 1 to 4096, not %u", c->page_size);
  if (c->kv_heads < 1 || c->kv_heads > 65535) return kv_refuse(ctx, GRAPE_ERR_INVALID, "kv_heads must be 1 to 65535, not %u", c->kv_heads);
  if (c->n_pages < 1 || c->n_pages > 0x7fffffffu) return kv_refuse(ctx, GRAPE_ERR_INVALID, "n_pages must be 1 to 2^31 - 1");
  if (c->page_stride % 8 || c->head_stride % 8 || c->slot_stride % 8)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "cache strides must be multiples of 8 elements");
  const uint64_t most = uint64_t(1) << 60;
  if (c->page_stride > most / c->n_pages || c->head_stride > most / c->kv_heads || c->slot_stride > most / c->page_size)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "cache strides too large");
  if ((c->n_pages > 1 && c->page_stride < c->head_dim) || (c->kv_heads > 1 && c->head_stride < c->head_dim) ||
      (c->page_size > 1 && c->slot_stride < c->head_dim))
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "cache strides smaller than head_dim");
  if (misaligned(c->d_k, 16) || misaligned(c->d_v, 16) || misaligned(c->d_bounds, 16))
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "cache pointers must be on 16 bytes");
  if (c->k_shift > 30 || c->v_shift > 30) return kv_refuse(ctx, GRAPE_ERR_INVALID, "cache shifts must be at most 30");
  if (batch && (!d_table || width < 1)) return kv_refuse(ctx, GRAPE_ERR_INVALID, "no page table");
  if ((uint64_t)width * c->page_size > 0x7fffffffu) return kv_refuse(ctx, GRAPE_ERR_LIMIT, "table_width * page_size must stay below 2^31");
  if (misaligned(d_table, 4)) return kv_refuse(ctx, GRAPE_ERR_INVALID, "page table must be on 4 bytes");
  return GRAPE_OK;
}

int kv_check_rows(grape_ctx* ctx, const char* what, const int32_t* d, uint64_t stride, uint64_t row) {
  if (!d) return kv_refuse(ctx, GRAPE_ERR_INVALID, "%s is null", what);
  if (misaligned(d, 16)) return kv_refuse(ctx, GRAPE_ERR_INVALID, "%s must be on 16 bytes", what);
  if (stride < row || stride % 4 || stride > (uint64_t(1) << 40))
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "row stride of %s must be a multiple of 4, at least %llu and at most 2^40", what, (unsigned long long)row);
  return GRAPE_OK;
}

KvView kv_view(grape_ctx* ctx, const grape_kv_cache* c, const int32_t* d_table, uint32_t width, uint32_t batch) {
  const int64_t e = c->bits / 8;
  KvView v;
  v.k = reinterpret_cast<char*>(c->d_k);
  v.v = reinterpret_cast<char*>(c->d_v);
  v.bounds = reinterpret_cast<char*>(c->d_bounds);
  v.page_stride = (int64_t)c->page_stride * e;
  v.head_stride = (int64_t)c->head_stride * e;
  v.slot_stride = (int64_t)c->slot_stride * e;
  v.n_pages = c->n_pages;
  v.page_size = c->page_size;
  v.kv_heads = c->kv_heads;
  v.head_dim = c->head_dim;
  v.by_page = FastDiv::of(c->page_size);
  v.table = d_table;
  v.width = width;
  v.batch = batch;
  v.status = ctx->d_status;
  return v;
}

int kv_workspace(grape_ctx* ctx, size_t bytes, void** out) {
  if (ctx->kv_work.empty() || ctx->kv_work.back().second < bytes) {
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    GRAPE_CUDA_TRY(ctx, cudaStreamIsCapturing(ctx->stream, &capture));
    if (capture != cudaStreamCaptureStatusNone)
      return kv_refuse(ctx, GRAPE_ERR_NOMEM, "the workspace has to grow to %zu bytes: make one such call outside the capture first", bytes);
    // twice the last block if there is room, so that what is kept adds up to less than the current one
    size_t want = ctx->kv_work.empty() ? size_t(4) << 20 : 2 * ctx->kv_work.back().second;
    if (want < bytes) want = bytes;
    ctx->kv_work.reserve(ctx->kv_work.size() + 1);
    void* p = nullptr;
    if (cudaMalloc(&p, want) != cudaSuccess) {
      cudaGetLastError();
      want = bytes;  // what the call needs may still be there
      if (cudaMalloc(&p, want) != cudaSuccess) {
        cudaGetLastError();
        return kv_refuse(ctx, GRAPE_ERR_NOMEM, "workspace of %zu bytes", want);
      }
    }
    ctx->kv_work.push_back({p, want});
  }
  *out = ctx->kv_work.back().first;
  return GRAPE_OK;
}

// ---- append ------------------------------------------------------------------------------------
// y = rdiv(a, s), rem = a - y 2^s with a = x 2^f or the rotated pair at the product of both scales.
// A streaming kernel: every input read once, every output written once, 16-byte accesses.  A block works
// on the tokens that ONE page receives, so that the page's bounds are a reduction inside the block and
// one plain read-modify-write: no atomics, and no order that could change them.
constexpr int AP_THREADS = 256;
// Sequences of a launch: every block looks through all of them for its own, so a batch of many times as many in one launch
// would cost their square (one token for each of 4096 and 262144 sequences: 0.12 and 302 ms, in launches of 1024 0.10 and 10).
constexpr uint32_t AP_BATCH = 1024;

struct AppendArgs {
  KvView c;
  const int32_t *start, *offsets;
  uint32_t tokens;
  const int32_t *cos, *sin;
  uint32_t positions, rot, rot_shift;
  uint32_t k_shift, v_shift;
  const int32_t *q, *k, *v;
  uint64_t q_stride, k_stride, v_stride;
  uint32_t heads;
  int32_t *q_out, *q_rem, *k_rem, *v_rem;
  uint32_t k_chunks, v_chunks;  // blockIdx.y: chunks of the keys' items, of the values', of the queries'
  FastDiv turned_items, plain_items;  // work items of a head: with rotation, without
  uint32_t lanes;               // threads of a block that share an item and deal the tokens out (power of two)
};

// An item is what one thread handles of a head for every token: 4 channels that lie together or, for the
// split pairing, two such groups dim/2 apart.
__host__ __device__ constexpr int ap_stages(bool interleaved) { return interleaved ? 8 : 6; }
constexpr size_t ap_smem(bool interleaved) { return (size_t)ap_stages(interleaved) * AP_THREADS * (interleaved ? 32 : 64); }

template <int EB, bool INTERLEAVED>
__global__ void __launch_bounds__(AP_THREADS, INTERLEAVED ? 3 : 2) k_kv_append(AppendArgs a) {
  __shared__ int s_b;
  constexpr int GROUPS = INTERLEAVED ? 1 : 2;  // of four channels that an item has at most
  extern __shared__ int4 s_queue[];  // [what][stage][thread]
  auto slot = [&](int what, uint32_t stage) {
    char* const mine = reinterpret_cast<char*>(s_queue + (what * ap_stages(INTERLEAVED) + stage) * AP_THREADS + threadIdx.x);
    // with neighbouring pairs a cosine or sine takes 8 bytes: both share the places of one 16-byte tensor
    return INTERLEAVED && what ? reinterpret_cast<char*>(s_queue + (ap_stages(true) + stage) * AP_THREADS) + (what - 1) * AP_THREADS * 8 + threadIdx.x * 8 : mine;
  };
  const KvView& c = a.c;
  const uint32_t unit = blockIdx.x, tid = threadIdx.x;
  // Units of a sequence begin at offsets[b] / page_size + 2 b: room for every page that its tokens can touch, and units
  // of its own as long as offsets do not fall.  A sequence whose rows do not lie in the call's has none.
  if (tid == 0) s_b = -1;
  __syncthreads();
  bool falls = false, outside = false;
  auto rows_of = [&](uint32_t b, int32_t& lo, int32_t& hi) {
    lo = __ldg(a.offsets + b);
    hi = __ldg(a.offsets + b + 1);
    falls |= hi < lo;
    return lo >= 0 && hi >= lo && (uint32_t)hi <= a.tokens;
  };
  auto has_unit = [&](uint32_t b, int32_t lo, int32_t hi) {  // lo / page_size + 2 b <= unit < hi / page_size + 2 b + 2
    const int64_t row = (int64_t)((int32_t)unit - 2 * (int32_t)b) * (int32_t)c.page_size;
    return lo < row + c.page_size && hi >= row - c.page_size;
  };
  for (uint32_t b = tid; b < c.batch; b += AP_THREADS) {
    int32_t lo, hi;
    const bool in = rows_of(b, lo, hi);
    outside |= !in;
    if (in && has_unit(b, lo, hi)) s_b = (int)b;
  }
  if (outside && unit == 0 && blockIdx.y == 0) kv_flag(c, STATUS_KV_PLACE);
  if (__syncthreads_or(falls)) {
    // of the sequences that claim the same rows the first has them; one warp finds the block's again
    if (tid == 0) s_b = -1;
    __syncthreads();
    int32_t taken = 0;
    for (uint32_t base = 0; tid < 32 && base < c.batch; base += 32) {
      int32_t lo = 0, hi = 0;
      const bool in = base + tid < c.batch && rows_of(base + tid, lo, hi);
      int32_t upto = in ? hi : 0;  // the largest end so far
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t before = __shfl_up_sync(~0u, upto, o);
        if ((int)tid >= o) upto = max(upto, before);
      }
      int32_t before = __shfl_up_sync(~0u, upto, 1);
      before = max(taken, tid ? before : 0);
      if (in && lo >= before && has_unit(base + tid, lo, hi)) s_b = (int)(base + tid);
      taken = max(taken, __shfl_sync(~0u, upto, 31));
    }
    __syncthreads();
  }
  if (s_b < 0) return;
  const uint32_t b = (uint32_t)s_b;
  const int64_t lo = __ldg(a.offsets + b), hi = __ldg(a.offsets + b + 1), start = __ldg(a.start + b);
  if (start < 0) {
    if (tid == 0) kv_flag(c, STATUS_KV_PLACE);
    return;
  }
  if (hi == lo || start > 0x7fffffff - (hi - lo)) {
    if (hi != lo && tid == 0) kv_flag(c, STATUS_KV_PLACE);
    return;
  }
  const uint32_t place = c.by_page.div((uint32_t)start) + (unit - (c.by_page.div((uint32_t)lo) + 2 * b));
  const int64_t page_first = (int64_t)place * c.page_size;
  int64_t p0 = max(start, page_first), p1 = min(start + (hi - lo), page_first + (int64_t)c.page_size);
  if (p0 >= p1) return;
  const int32_t page = kv_page(c, b, place);
  if (a.rot && p1 > (int64_t)a.positions) {
    p1 = a.positions;
    if (tid == 0) kv_flag(c, STATUS_KV_PLACE);
  }
  if (page < 0) {
    if (tid == 0) kv_flag(c, STATUS_KV_PLACE);
    return;
  }
  if (p0 >= p1) return;

  const uint32_t per_block = AP_THREADS / a.lanes;
  uint32_t chunk = blockIdx.y;
  const int kind = chunk < a.k_chunks ? 0 : chunk < a.k_chunks + a.v_chunks ? 1 : 2;  // keys, values, queries
  if (kind == 1) chunk -= a.k_chunks;
  if (kind == 2) chunk -= a.k_chunks + a.v_chunks;
  const uint32_t item = chunk * per_block + (tid & (per_block - 1)), lane = tid / per_block;
  const FastDiv& items = kind == 1 ? a.plain_items : a.turned_items;
  const uint32_t head = items.div(item), it = item - head * items.d, D = c.head_dim;
  const bool active = head < (kind == 2 ? a.heads : c.kv_heads);
  const uint32_t pairs = INTERLEAVED ? a.rot / 4 : a.rot / 8;  // items that are turned
  const bool turned = kind != 1 && it < pairs;
  const uint32_t ch = INTERLEAVED || kind == 1 ? 4 * it : turned ? 4 * it : a.rot + 4 * (it - pairs);
  const uint32_t ch2 = ch + a.rot / 2;
  const bool two = !INTERLEAVED && turned;
  const uint32_t shift = kind == 0 ? a.rot_shift + a.k_shift : kind == 1 ? a.v_shift : a.rot_shift;
  const uint32_t up = kind == 1 ? 0 : a.rot_shift;
  const uint32_t n_heads = kind == 2 ? a.heads : c.kv_heads;
  const bool wide = EB == 4 || kind == 2;  // int32 outputs
  const int64_t top = wide ? 0x7fffffffll : 0x7fffll;
  bool range = false;
  int32_t low[GROUPS][4], high[GROUPS][4];
#pragma unroll
  for (int w = 0; w < GROUPS; w++)
#pragma unroll
    for (int j = 0; j < 4; j++) {
      low[w][j] = 0x7fffffff;
      high[w][j] = -0x7fffffff - 1;
    }

  if (active) {
    // where this thread's first token lies in every tensor, and how far its next one is
    const uint32_t token0 = (uint32_t)(lo + (p0 - start)) + lane, turns = (uint32_t)(p1 - p0);
    uint32_t done = lane;
    const uint64_t in_row = kind == 0 ? a.k_stride : kind == 1 ? a.v_stride : a.q_stride, dense_row = (uint64_t)n_heads * D;
    const int32_t* in = (kind == 0 ? a.k : kind == 1 ? a.v : a.q) + token0 * in_row + (uint64_t)head * D + ch;
    int32_t* rem = kind == 0 ? a.k_rem : kind == 1 ? a.v_rem : a.q_rem;
    const bool with_rem = rem != nullptr;
    rem += with_rem ? token0 * dense_row + (uint64_t)head * D + ch : 0;
    char* out = kind == 2 ? reinterpret_cast<char*>(a.q_out + token0 * dense_row + (uint64_t)head * D + ch)
                          : (kind == 0 ? c.k : c.v) + page * c.page_stride + head * c.head_stride + (p0 + lane - page_first) * c.slot_stride + (int64_t)ch * EB;
    const uint64_t in_step = in_row * a.lanes, rem_step = dense_row * a.lanes, out_step = (kind == 2 ? dense_row * 4 : (uint64_t)c.slot_stride) * a.lanes;
    const uint32_t angle = a.rot / 2, angle_step = angle * a.lanes, at0 = INTERLEAVED ? ch / 2 : ch;
    const int32_t *cos = a.cos + (uint64_t)(p0 + lane) * angle + at0, *sin = a.sin + (uint64_t)(p0 + lane) * angle + at0;
    const uint32_t apart = a.rot / 2;  // of the two groups of a split pair

    const uint64_t half = (uint64_t(1) << shift) >> 1;
    const int32_t unit = (int32_t)(0u - (1u << shift));
    auto finish = [&](const int64_t (&x)[4], int32_t* rem_to, char* to, int which) {
      int32_t y[4], r[4];
      uint32_t over = 0;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        // both words of (x + half) >> shift; it fits 32 bits when the upper one is the lower one's sign
        const uint64_t sum = (uint64_t)x[j] + half;
        const uint32_t hi = (uint32_t)(sum >> 32);
        y[j] = (int32_t)__funnelshift_r((uint32_t)sum, hi, shift);
        r[j] = y[j] * unit + (int32_t)(uint32_t)(uint64_t)x[j];
        over |= (uint32_t)((int32_t)hi >> shift) ^ (uint32_t)(y[j] >> 31);
        if (!wide) over |= (uint32_t)(y[j] ^ (int32_t)(int16_t)y[j]);
      }
      if (over) {
#pragma unroll
        for (int j = 0; j < 4; j++) y[j] = saturate(rdiv(x[j], shift), -top - 1, top, range);
      }
      if (kind == 0) {
#pragma unroll
        for (int j = 0; j < 4; j++) {
          low[which][j] = min(low[which][j], y[j]);
          high[which][j] = max(high[which][j], y[j]);
        }
      }
      if (with_rem) __stcs(reinterpret_cast<int4*>(rem_to), make_int4(r[0], r[1], r[2], r[3]));
      if (wide) *reinterpret_cast<int4*>(to) = make_int4(y[0], y[1], y[2], y[3]);
      else *reinterpret_cast<short4*>(to) = make_short4((short)y[0], (short)y[1], (short)y[2], (short)y[3]);
    };
    // products of two int32; their sums wrap like unsigned ones
    auto turn = [](int32_t x0, int32_t x1, int32_t co, int32_t si, int64_t& y0, int64_t& y1) {
      y0 = (int64_t)((uint64_t)((int64_t)x0 * co) - (uint64_t)((int64_t)x1 * si));
      y1 = (int64_t)((uint64_t)((int64_t)x1 * co) + (uint64_t)((int64_t)x0 * si));
    };
    // The thread's own queue of copies runs AP_STAGES - 1 tokens ahead: what is under way costs no registers.
    constexpr int STAGES = ap_stages(INTERLEAVED);
    auto fetch = [&](uint32_t ahead, uint32_t stage) {  // `ahead` in the thread's turns from here
      if (done + ahead * a.lanes < turns) {
        const uint64_t n = ahead;
        copy_async<16>(slot(0, stage), in + n * in_step);
        if (turned) {
          if (GROUPS == 2) copy_async<16>(slot(1, stage), in + n * in_step + apart);
          copy_async<INTERLEAVED ? 8 : 16>(slot(GROUPS, stage), cos + n * angle_step);
          copy_async<INTERLEAVED ? 8 : 16>(slot(GROUPS + 1, stage), sin + n * angle_step);
        }
      }
      copy_commit();
    };
#pragma unroll 1
    for (int i = 0; i < STAGES - 1; i++) fetch(i, i);
    uint32_t stage = 0;
#pragma unroll 1
    for (; done < turns; done += a.lanes) {
      fetch(STAGES - 1, stage == 0 ? STAGES - 1 : stage - 1);  // into the place that was read a turn ago
      copy_wait<STAGES - 1>();
      const int4 x = *reinterpret_cast<const int4*>(slot(0, stage));
      int64_t y[4];
      if (!turned) {
        y[0] = (int64_t)((uint64_t)(int64_t)x.x << up);
        y[1] = (int64_t)((uint64_t)(int64_t)x.y << up);
        y[2] = (int64_t)((uint64_t)(int64_t)x.z << up);
        y[3] = (int64_t)((uint64_t)(int64_t)x.w << up);
        finish(y, rem, out, 0);
      } else if (INTERLEAVED) {
        const int2 co = *reinterpret_cast<const int2*>(slot(1, stage)), si = *reinterpret_cast<const int2*>(slot(2, stage));
        turn(x.x, x.y, co.x, si.x, y[0], y[1]);
        turn(x.z, x.w, co.y, si.y, y[2], y[3]);
        finish(y, rem, out, 0);
      } else {
        const int4 x2 = *reinterpret_cast<const int4*>(slot(1, stage)), co = *reinterpret_cast<const int4*>(slot(GROUPS, stage)),
                   si = *reinterpret_cast<const int4*>(slot(GROUPS + 1, stage));
        int64_t z[4];
        turn(x.x, x2.x, co.x, si.x, y[0], z[0]);
        turn(x.y, x2.y, co.y, si.y, y[1], z[1]);
        turn(x.z, x2.z, co.z, si.z, y[2], z[2]);
        turn(x.w, x2.w, co.w, si.w, y[3], z[3]);
        finish(y, rem, out, 0);
        finish(z, rem + apart, out + apart * (wide ? 4 : EB), GROUPS - 1);
      }
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      in += in_step;
      rem += rem_step;
      out += out_step;
      cos += angle_step;
      sin += angle_step;
    }
    copy_wait<0>();
  }
  if (range) kv_flag(c, STATUS_KV_RANGE);
  if (kind != 0 || !c.bounds) return;

  // bounds of the page: across the lanes that dealt the tokens out, then into the page's record
  // (its places of the queue are free: stages 2 w and 2 w + 1 of the first tensor take its group w)
  if (a.lanes > 1) {
#pragma unroll
    for (int w = 0; w < GROUPS; w++) {
      *reinterpret_cast<int4*>(slot(0, 2 * w)) = make_int4(low[w][0], low[w][1], low[w][2], low[w][3]);
      *reinterpret_cast<int4*>(slot(0, 2 * w + 1)) = make_int4(high[w][0], high[w][1], high[w][2], high[w][3]);
    }
    __syncthreads();
    if (lane != 0) return;
    for (uint32_t l = 1; l < a.lanes; l++) {
#pragma unroll
      for (int w = 0; w < GROUPS; w++) {
        const int4 m = reinterpret_cast<const int4*>(slot(0, 2 * w))[l * per_block], h = reinterpret_cast<const int4*>(slot(0, 2 * w + 1))[l * per_block];
        low[w][0] = min(low[w][0], m.x); low[w][1] = min(low[w][1], m.y);
        low[w][2] = min(low[w][2], m.z); low[w][3] = min(low[w][3], m.w);
        high[w][0] = max(high[w][0], h.x); high[w][1] = max(high[w][1], h.y);
        high[w][2] = max(high[w][2], h.z); high[w][3] = max(high[w][3], h.w);
      }
    }
  }
  if (!active) return;
  const bool fresh = p0 == page_first;
  for (int w = 0; w < GROUPS; w++) {
    if (w && !two) break;
    char* rec = c.bounds + (((int64_t)page * c.kv_heads + head) * 2 * D + (w ? ch2 : ch)) * EB;
    int32_t l[4], h[4];
#pragma unroll
    for (int j = 0; j < 4; j++) { l[j] = low[w][j]; h[j] = high[w][j]; }
    if (EB == 4) {
      int4 *pl = reinterpret_cast<int4*>(rec), *ph = reinterpret_cast<int4*>(rec + (int64_t)D * EB);
      if (!fresh) {
        const int4 ol = *pl, oh = *ph;
        l[0] = min(l[0], ol.x); l[1] = min(l[1], ol.y); l[2] = min(l[2], ol.z); l[3] = min(l[3], ol.w);
        h[0] = max(h[0], oh.x); h[1] = max(h[1], oh.y); h[2] = max(h[2], oh.z); h[3] = max(h[3], oh.w);
      }
      *pl = make_int4(l[0], l[1], l[2], l[3]);
      *ph = make_int4(h[0], h[1], h[2], h[3]);
    } else {
      short4 *pl = reinterpret_cast<short4*>(rec), *ph = reinterpret_cast<short4*>(rec + (int64_t)D * EB);
      if (!fresh) {
        const short4 ol = *pl, oh = *ph;
        l[0] = min(l[0], (int)ol.x); l[1] = min(l[1], (int)ol.y); l[2] = min(l[2], (int)ol.z); l[3] = min(l[3], (int)ol.w);
        h[0] = max(h[0], (int)oh.x); h[1] = max(h[1], (int)oh.y); h[2] = max(h[2], (int)oh.z); h[3] = max(h[3], (int)oh.w);
      }
      *pl = make_short4((short)l[0], (short)l[1], (short)l[2], (short)l[3]);
      *ph = make_short4((short)h[0], (short)h[1], (short)h[2], (short)h[3]);
    }
  }
}

// ---- select ------------------------------------------------------------------------------------
// bound = max over the group's heads of sum_d max(q_d lo_d, q_d hi_d) = sum_d q_d (q_d >= 0 ? hi_d : lo_d).
// LANES lanes take the two rows of four pages side by side, in 16-byte pieces: four pages' loads under way (one at a
// time reached 2.1 TB/s; eight, for one head, leave room for fewer warps: 48 us where four take 35), and four pages
// x four heads of sums to add up over the lanes, each step of which halves what a lane holds: 32 shuffles for
// 16 sums where one sum after the other takes 160.
// What bounds it: bytes of the bounds, fetched again for every four heads; a channel and head costs one select and one
// wide multiply-add.
constexpr int SB_THREADS = 128;
constexpr int SB_PAGES = 4;  // whose sums a lane holds at a time, for up to four heads

struct SelectArgs {
  KvView c;
  const int32_t* len;
  const int32_t* q;
  uint64_t q_stride;
  uint32_t heads, group;
  uint32_t n_select, recent;
  int32_t* selected;
  int64_t* bound;
  uint32_t chunks, chunk_pages;  // blocks of a row, pages of a block
};

// SPLIT: the block's warps share the channels of the same pages (and LANES is 32).
template <int EB, int LANES, int HEADS, bool SPLIT>
__global__ void __launch_bounds__(SB_THREADS) k_kv_bounds(SelectArgs a) {
  constexpr int WARPS = SB_THREADS / 32;
  extern __shared__ int4 s_q4[];
  __shared__ uint64_t s_part[SPLIT ? WARPS : 1][SB_PAGES * HEADS];
  const KvView& c = a.c;
  const uint32_t chunk = blockIdx.x % a.chunks, row = blockIdx.x / a.chunks, g = row % c.kv_heads, b = row / c.kv_heads;
  const uint32_t D = c.head_dim, vectors = D * EB / 16;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const uint32_t n = kv_length(c, a.len, b, ~0ull, chunk == 0 && threadIdx.x == 0);
  const uint32_t pages = c.by_page.div(n + c.page_size - 1);
  const uint32_t first = chunk * a.chunk_pages, last = min(pages, first + a.chunk_pages);
  if (first >= last) return;
  const int4* q = reinterpret_cast<const int4*>(a.q + (uint64_t)b * a.q_stride + (uint64_t)g * a.group * D);
  const uint32_t sub = threadIdx.x % LANES, mine = SPLIT ? 0 : threadIdx.x / LANES;
  constexpr uint32_t PER = (SPLIT ? 1 : SB_THREADS / LANES) * SB_PAGES;  // pages of the block's turn
  constexpr int NV = SB_PAGES * HEADS, LOG = NV == 16 ? 4 : NV == 8 ? 3 : 2;
  for (uint32_t h0 = 0; h0 < a.group; h0 += HEADS) {
    const uint32_t hn = min((uint32_t)HEADS, a.group - h0);
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < HEADS * D / 4; i += SB_THREADS)
      s_q4[i] = i < hn * D / 4 ? __ldg(q + (uint64_t)h0 * D / 4 + i) : make_int4(0, 0, 0, 0);
    __syncthreads();
    // whole warps run the loop: the shuffles below need every lane
    for (uint32_t base = first; base < last; base += PER) {
      const uint32_t i0 = base + mine * SB_PAGES;
      const int4* rows[SB_PAGES];
      uint32_t bad = 0;
#pragma unroll
      for (int p = 0; p < SB_PAGES; p++) {
        int32_t page = i0 + p < last ? kv_page(c, b, i0 + p) : 0;  // a page outside the cache reads page 0 and is dropped
        if (page < 0) {
          bad |= 1u << p;
          page = 0;
        }
        rows[p] = reinterpret_cast<const int4*>(c.bounds + ((int64_t)page * c.kv_heads + g) * 2 * D * EB);
      }
      uint64_t acc[NV];
#pragma unroll
      for (int k = 0; k < NV; k++) acc[k] = 0;
#pragma unroll 1
      for (uint32_t v = SPLIT ? threadIdx.x : sub; v < vectors; v += SPLIT ? SB_THREADS : LANES) {
        int4 lo[SB_PAGES], hi[SB_PAGES];
#pragma unroll
        for (int p = 0; p < SB_PAGES; p++) {
          lo[p] = __ldcs(rows[p] + v);
          hi[p] = __ldcs(rows[p] + vectors + v);
        }
#pragma unroll
        for (int h = 0; h < HEADS; h++) {
          constexpr int QV = EB == 4 ? 1 : 2;
#pragma unroll
          for (int k = 0; k < QV; k++) {
            const int4 q4 = s_q4[h * (D / 4) + v * QV + k];
            const int32_t qq[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
              const int32_t negative = qq[j] >> 31;  // all ones or none
#pragma unroll
              for (int p = 0; p < SB_PAGES; p++) {
                const int at = EB == 4 ? j : 2 * k + j / 2;
                const int32_t l = at == 0 ? lo[p].x : at == 1 ? lo[p].y : at == 2 ? lo[p].z : lo[p].w;
                const int32_t u = at == 0 ? hi[p].x : at == 1 ? hi[p].y : at == 2 ? hi[p].z : hi[p].w;
                int32_t x = (l & negative) | (u & ~negative);
                if (EB == 2) x = j & 1 ? x >> 16 : (int32_t)(int16_t)x;
                acc[p * HEADS + h] += (uint64_t)((int64_t)qq[j] * x);
              }
            }
          }
        }
      }
      // the sums over the lanes; a lane keeps the half of its values that its bit of the step names
      constexpr int STEPS = LANES == 32 ? 5 : LANES == 16 ? 4 : LANES == 8 ? 3 : 2;
      int held = NV;
#pragma unroll
      for (int s = 0; s < STEPS; s++) {
        const int o = LANES >> (s + 1);
        if (s < LOG) {
          held >>= 1;
          const bool upper = sub & o;
#pragma unroll
          for (int k = 0; k < NV / 2; k++) {
            if (k >= (NV >> (s + 1))) break;
            const uint64_t keep = upper ? acc[k + (NV >> (s + 1))] : acc[k], give = upper ? acc[k] : acc[k + (NV >> (s + 1))];
            acc[k] = keep + __shfl_xor_sync(~0u, give, o);
          }
        } else {
          acc[0] += __shfl_xor_sync(~0u, acc[0], o);
        }
      }
      // values page * HEADS + head: a lane holds NV >> min(STEPS, LOG) of them, from this one on
      constexpr int LEFT = STEPS >= LOG ? 1 : NV >> STEPS;
      uint32_t at = 0;
#pragma unroll
      for (int s = 0; s < (STEPS < LOG ? STEPS : LOG); s++)
        if (sub & (LANES >> (s + 1))) at += NV >> (s + 1);
      if (SPLIT) {
        __syncthreads();  // the turn before has been read
        s_part[threadIdx.x >> 5][at] = acc[0];
        __syncthreads();
        acc[0] = 0;
        for (int w = 0; w < WARPS; w++) acc[0] += s_part[w][at];
      }
      int64_t best = INT64_MIN;
#pragma unroll
      for (int k = 0; k < LEFT; k++)
        if (HEADS == 1 || (at + k) % HEADS < hn) best = max(best, (int64_t)acc[k]);
      // and the largest over the heads of a page that neighbouring lanes hold
#pragma unroll
      for (int k = 0; (1 << k) < HEADS; k++)
        if (LOG - k <= STEPS) best = max(best, __shfl_xor_sync(~0u, best, LANES >> (LOG - k)));
      const uint32_t p = at / HEADS, i = i0 + p;
      // lanes that hold the same value, and with SPLIT the warps: one of them writes
      const bool writes = at % HEADS == 0 && (STEPS <= LOG || sub % (LANES >> LOG) == 0) && (!SPLIT || threadIdx.x < 32);
      if (writes && i < last) {
        int64_t* to = a.bound + (uint64_t)row * c.width + i;
        if (bad >> p & 1) {
          best = INT64_MIN;
          kv_flag(c, STATUS_KV_PLACE);
        } else if (h0) {
          best = max(best, *to);
        }
        *to = best;
      }
    }
  }
}

// The `need` largest of a row's bounds by a radix search for the last one's value: per pass the 8 bits
// below those that are known are counted over the bounds that share them.  Bounds are taken relative to
// the least, so that the first pass spreads them over its bins.  Then one pass in the pages' order
// writes what is above that value, the first of what equals it, and the newest pages.
constexpr int PK_THREADS = 512, PK_HELD = 4;

__device__ __forceinline__ uint32_t block_sum_before(uint32_t flag, uint32_t* s_warp, uint32_t& total) {
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t votes = __ballot_sync(~0u, flag != 0);
  __syncthreads();
  if (lane == 0) s_warp[warp] = __popc(votes);
  __syncthreads();
  uint32_t before = 0;
  total = 0;
  for (uint32_t w = 0; w < PK_THREADS / 32; w++) {
    const uint32_t n = s_warp[w];
    if (w < warp) before += n;
    total += n;
  }
  return before + __popc(votes & ((1u << lane) - 1));
}

__global__ void __launch_bounds__(PK_THREADS) k_kv_pick(SelectArgs a) {
  __shared__ uint32_t s_bins[256], s_warp[PK_THREADS / 32], s_digit, s_left, s_count;
  __shared__ uint64_t s_low[PK_THREADS / 32], s_high[PK_THREADS / 32];
  const KvView& c = a.c;
  const uint32_t row = blockIdx.x, b = row / c.kv_heads, tid = threadIdx.x;
  const uint32_t n = kv_length(c, a.len, b, ~0ull, false);
  const uint32_t pages = c.by_page.div(n + c.page_size - 1);
  const uint32_t chosen = min(a.n_select, pages), newest = min(a.recent, pages);
  const uint32_t old = pages - newest, need = chosen - min(chosen, newest);
  int32_t* out = a.selected + (uint64_t)row * a.n_select;
  for (uint32_t i = tid; i < a.n_select; i += PK_THREADS)
    if (i >= chosen) out[i] = -1;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // for the bounds
  if (need >= old) {
    for (uint32_t i = tid; i < chosen; i += PK_THREADS) out[i] = (int32_t)i;
    return;
  }
  // the first PK_HELD turns' bounds stay in registers
  const int64_t* bound = a.bound + (uint64_t)row * c.width;
  uint64_t held[PK_HELD];
#pragma unroll
  for (int k = 0; k < PK_HELD; k++) held[k] = k * PK_THREADS + tid < old ? (uint64_t)bound[k * PK_THREADS + tid] ^ (uint64_t(1) << 63) : 0;
  auto for_old = [&](auto&& f) {
#pragma unroll
    for (int k = 0; k < PK_HELD; k++)
      if (k * PK_THREADS + tid < old) f(held[k]);
    for (uint32_t i = PK_HELD * PK_THREADS + tid; i < old; i += PK_THREADS) f((uint64_t)bound[i] ^ (uint64_t(1) << 63));
  };
  uint64_t low = ~0ull, high = 0;
  for_old([&](uint64_t k) {
    low = min(low, k);
    high = max(high, k);
  });
  for (int o = 16; o; o >>= 1) {
    low = min(low, __shfl_xor_sync(~0u, low, o));
    high = max(high, __shfl_xor_sync(~0u, high, o));
  }
  if ((tid & 31) == 0) { s_low[tid >> 5] = low; s_high[tid >> 5] = high; }
  __syncthreads();
  for (int w = 0; w < PK_THREADS / 32; w++) {
    low = min(low, s_low[w]);
    high = max(high, s_high[w]);
  }
  // known: the leading bits (of the difference to `low`) of the last bound that is taken; left: how many
  // of the bounds that begin with them are taken
  uint64_t known = 0;
  uint32_t left = need, bits = high == low ? 0 : 64 - __clzll((long long)(high - low));
  if (need == 0) bits = 0;
  while (bits) {
    const uint32_t w = min(8u, bits), shift = bits - w;
    __syncthreads();
    for (uint32_t i = tid; i < 256; i += PK_THREADS) s_bins[i] = 0;
    __syncthreads();
    for_old([&](uint64_t k) {
      const uint64_t d = k - low;
      if (bits == 64 || (d >> bits) == known) atomicAdd(&s_bins[(uint32_t)(d >> shift) & ((1u << w) - 1)], 1u);
    });
    __syncthreads();
    if (tid < 32) {
      // lane l holds bins 255-8l .. 248-8l: a scan from the largest digit down
      uint32_t sum = 0;
      for (int j = 0; j < 8; j++) sum += s_bins[255 - 8 * tid - j];
      uint32_t upto = sum;
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(~0u, upto, o);
        if ((int)tid >= o) upto += t;
      }
      uint32_t before = upto - sum;
      if (before < left && left <= upto) {
        for (int j = 0; j < 8; j++) {
          const uint32_t in_bin = s_bins[255 - 8 * tid - j];
          if (left <= before + in_bin) {
            s_digit = 255 - 8 * tid - j;
            s_left = left - before;
            s_count = in_bin;
            break;
          }
          before += in_bin;
        }
      }
    }
    __syncthreads();
    known = (known << w) | s_digit;
    left = s_left;
    bits = shift;
    if (s_count == left) break;  // the whole bin is taken: no need for the bits below
  }
  uint32_t written = 0, ties = 0;
  for (uint32_t base = 0; base < pages; base += PK_THREADS) {
    const uint32_t i = base + tid;
    bool above = i >= old && i < pages, tie = false;
    if (i < old) {
      const uint64_t d = ((uint64_t)bound[i] ^ (uint64_t(1) << 63)) - low, lead = d >> bits;
      above = need != 0 && lead > known;
      tie = need != 0 && lead == known;
    }
    uint32_t total;
    const uint32_t rank = block_sum_before(tie, s_warp, total);
    const bool take = above || (tie && ties + rank < left);
    ties += total;
    const uint32_t at = block_sum_before(take, s_warp, total);
    if (take) out[written + at] = (int32_t)i;
    written += total;
  }
}

// Units of work of a launch: the rows of its sequences are somewhere among the call's.
static uint64_t append_units(const grape_kv_cache* cache, uint32_t batch, uint32_t tokens) {
  return tokens / cache->page_size + 2ull * std::min(AP_BATCH, batch);
}

static int append_launch(grape_ctx* ctx, const grape_kv_cache* cache, AppendArgs& a, bool interleaved) {
  const uint32_t D = cache->head_dim, KV = cache->kv_heads;
  const uint32_t turned = interleaved ? D / 4 : a.rot / 8 + (D - a.rot) / 4;
  a.turned_items = FastDiv::of(turned);
  a.plain_items = FastDiv::of(D / 4);
  // Lanes that share an item deal a page's tokens out: more, smaller blocks, until there are eight
  // an SM or a lane would have fewer than eight tokens.
  const uint32_t batch = a.c.batch;
  const uint64_t units = append_units(cache, batch, a.tokens);
  const uint64_t items = (uint64_t)KV * turned + (uint64_t)KV * (D / 4) + (uint64_t)a.heads * turned;
  const uint64_t tokens_per_page = std::min<uint64_t>(cache->page_size, (a.tokens + batch - 1) / batch);
  a.lanes = 1;
  while (a.lanes < 4 && a.lanes * 16 <= tokens_per_page && units * items * a.lanes / AP_THREADS < (uint64_t)ctx->sm_count * 4 * 2) a.lanes *= 2;
  const uint64_t per = AP_THREADS / a.lanes;
  a.k_chunks = (uint32_t)(((uint64_t)KV * turned + per - 1) / per);
  a.v_chunks = (uint32_t)(((uint64_t)KV * (D / 4) + per - 1) / per);
  const uint64_t chunks = a.k_chunks + a.v_chunks + (a.q ? ((uint64_t)a.heads * turned + per - 1) / per : 0);
  if (chunks > 65535 || units > 0x7fffffffu) return kv_refuse(ctx, GRAPE_ERR_LIMIT, "too many heads or sequences for one call");
  const dim3 grid((uint32_t)units, (uint32_t)chunks);
  auto kernel = cache->bits == 32 ? (interleaved ? k_kv_append<4, true> : k_kv_append<4, false>) : (interleaved ? k_kv_append<2, true> : k_kv_append<2, false>);
  if (int rc = kv_allow_shared(ctx, kernel, ap_smem(interleaved))) return rc;
  for (uint32_t b = 0; b < batch; b += AP_BATCH) {
    a.c.batch = std::min(AP_BATCH, batch - b);
    kernel<<<grid, AP_THREADS, ap_smem(interleaved), ctx->stream>>>(a);
    ctx->launches += 1;
    GRAPE_CUDA_TRY(ctx, cudaGetLastError());
    a.start += AP_BATCH;
    a.offsets += AP_BATCH;
    a.c.table += (uint64_t)AP_BATCH * a.c.width;
  }
  return GRAPE_OK;
}

static int select_launch(grape_ctx* ctx, const grape_kv_cache* cache, SelectArgs& a) {
  const uint32_t D = cache->head_dim;
  const uint64_t rows = (uint64_t)a.c.batch * cache->kv_heads;
  if (!a.bound) {
    void* w = nullptr;
    if (int rc = kv_workspace(ctx, rows * a.c.width * sizeof(int64_t), &w)) return rc;
    a.bound = reinterpret_cast<int64_t*>(w);
  }
  const uint32_t vectors = D * cache->bits / 8 / 16;
  // Lanes of a page: its row's 16-byte pieces, a warp at most; from 128 pieces on the warps of a block share a page (119
  // pages of 4096 channels: 12.5 us, a warp a page 22.8).  A block takes up to four turns of its pages while that
  // leaves eight blocks an SM (16 x 2048 pages of 8 x 128 channels: 68 us, one turn 82, and one turn is what
  // fills the GPU from 476 pages of 8 heads: 15 us, a fixed 64 pages a block 16.6).  One head or two in a group have kernels of
  // their own: 4 x 2048 pages of 32 heads with 80 channels of 16 bits take 35 us, with three idle heads 57.
  const bool split = vectors >= SB_THREADS;
  const uint32_t lanes = vectors > 16 ? 32 : vectors > 8 ? 16 : vectors > 4 ? 8 : 4, heads = a.group == 1 ? 1 : a.group == 2 ? 2 : 4;
  const uint32_t turn = (split ? 1 : SB_THREADS / lanes) * SB_PAGES;
  uint32_t turns = 4;
  while (turns > 1 && rows * ((a.c.width + turn * turns - 1) / (turn * turns)) < (uint64_t)ctx->sm_count * 8) turns /= 2;
  a.chunk_pages = turn * turns;
  a.chunks = (a.c.width + a.chunk_pages - 1) / a.chunk_pages;
  if (rows * a.chunks > 0x7fffffffu) return kv_refuse(ctx, GRAPE_ERR_LIMIT, "too many pages for one call");
  const size_t smem = (size_t)heads * D * 4;
  auto pick = [&](auto k4, auto k2) { return cache->bits == 32 ? k4 : k2; };
  auto by_heads = [&](auto h) {
    constexpr int H = decltype(h)::value;
    return split         ? pick(k_kv_bounds<4, 32, H, true>, k_kv_bounds<2, 32, H, true>)
           : lanes == 32 ? pick(k_kv_bounds<4, 32, H, false>, k_kv_bounds<2, 32, H, false>)
           : lanes == 16 ? pick(k_kv_bounds<4, 16, H, false>, k_kv_bounds<2, 16, H, false>)
           : lanes == 8  ? pick(k_kv_bounds<4, 8, H, false>, k_kv_bounds<2, 8, H, false>)
                         : pick(k_kv_bounds<4, 4, H, false>, k_kv_bounds<2, 4, H, false>);
  };
  auto kernel = heads == 1   ? by_heads(std::integral_constant<int, 1>())
                : heads == 2 ? by_heads(std::integral_constant<int, 2>())
                             : by_heads(std::integral_constant<int, 4>());
  // The limit of 48 KB is for the queries and the kernel's own sums together: the widest head's need, for every width.
  if (int rc = kv_allow_shared(ctx, kernel, (size_t)heads * 4096 * 4)) return rc;
  kernel<<<(uint32_t)(rows * a.chunks), SB_THREADS, smem, ctx->stream>>>(a);
  GRAPE_CUDA_TRY(ctx, cudaGetLastError());  // no choice over bounds that were not made
  ctx->launches += 1;
  // the choice may begin while the last bounds are made; it waits for them on the device
  cudaLaunchAttribute attribute = {};
  attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((uint32_t)rows);
  config.blockDim = dim3(PK_THREADS);
  config.stream = ctx->stream;
  config.attrs = &attribute;
  config.numAttrs = 1;
  GRAPE_CUDA_TRY(ctx, cudaLaunchKernelEx(&config, k_kv_pick, a));
  ctx->launches += 1;
  GRAPE_CUDA_TRY(ctx, cudaGetLastError());
  return GRAPE_OK;
}

}  // namespace grape

using namespace grape;

extern "C" const char* grape_kv_error(void) { return g_kv_error; }

extern "C" int grape_kv_append(grape_ctx* ctx, const grape_kv_cache* cache, const int32_t* d_table, uint32_t table_width,
                               uint32_t batch, const int32_t* d_start, const int32_t* d_offsets, uint32_t tokens,
                               const grape_kv_rotation* rotation, const int32_t* d_q, uint64_t q_stride, uint32_t heads,
                               const int32_t* d_k, uint64_t k_stride, const int32_t* d_v, uint64_t v_stride,
                               int32_t* d_q_out, int32_t* d_q_rem, int32_t* d_k_rem, int32_t* d_v_rem) try {
  if (int rc = kv_check_cache(ctx, cache, d_table, table_width, batch, true, true, false)) return rc;
  const grape_kv_rotation none = {nullptr, nullptr, 0, 0, 0, 1};
  const grape_kv_rotation& r = rotation ? *rotation : none;
  if (r.interleaved > 1) return kv_refuse(ctx, GRAPE_ERR_INVALID, "rotation pairing must be 0 or 1, not %u", r.interleaved);
  if (r.dim % 8 || r.dim > cache->head_dim)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "rotation dim must be a multiple of 8 up to head_dim, not %u", r.dim);
  if (r.dim && (!r.d_cos || !r.d_sin || misaligned(r.d_cos, 16) || misaligned(r.d_sin, 16)))
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "rotation tables must be given, on 16 bytes");
  if (r.shift > 30 || r.shift + cache->k_shift > 30)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "rotation shift and key shift add up to more than 30");
  if (tokens > 0x7fffffffu || batch > 0x0fffffffu) return kv_refuse(ctx, GRAPE_ERR_LIMIT, "too many tokens or sequences");
  const uint64_t launches = ((uint64_t)batch + AP_BATCH - 1) / AP_BATCH;
  if (launches > 1 && launches * append_units(cache, batch, tokens) > (uint64_t(1) << 30))
    return kv_refuse(ctx, GRAPE_ERR_LIMIT, "too many sequences and tokens for one call");
  if (batch && (!d_start || !d_offsets || misaligned(d_start, 4) || misaligned(d_offsets, 4)))
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "start and offsets must be given, on 4 bytes");
  const uint64_t row = (uint64_t)cache->kv_heads * cache->head_dim;
  if (batch && tokens) {
    if (int rc = kv_check_rows(ctx, "keys", d_k, k_stride, row)) return rc;
    if (int rc = kv_check_rows(ctx, "values", d_v, v_stride, row)) return rc;
    if (d_q) {
      if (heads < 1 || heads > 65535) return kv_refuse(ctx, GRAPE_ERR_INVALID, "heads must be 1 to 65535, not %u", heads);
      if (int rc = kv_check_rows(ctx, "queries", d_q, q_stride, (uint64_t)heads * cache->head_dim)) return rc;
      if (!d_q_out) return kv_refuse(ctx, GRAPE_ERR_INVALID, "queries without an output");
    } else if (d_q_out || d_q_rem) {
      return kv_refuse(ctx, GRAPE_ERR_INVALID, "an output for queries that are not given");
    }
  }
  if (misaligned(d_q_out, 16) || misaligned(d_q_rem, 16) || misaligned(d_k_rem, 16) || misaligned(d_v_rem, 16))
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "outputs must be on 16 bytes");
  if (!ctx) return kv_refuse(ctx, GRAPE_ERR_INVALID, "null context");
  make_device_current(ctx);
  if (!batch || !tokens) return GRAPE_OK;
  AppendArgs a{};
  a.c = kv_view(ctx, cache, d_table, table_width, batch);
  a.start = d_start;
  a.offsets = d_offsets;
  a.tokens = tokens;
  a.cos = r.d_cos;
  a.sin = r.d_sin;
  a.positions = r.positions;
  a.rot = r.dim;
  a.rot_shift = r.shift;
  a.k_shift = cache->k_shift;
  a.v_shift = cache->v_shift;
  a.q = d_q;
  a.k = d_k;
  a.v = d_v;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.heads = d_q ? heads : 0;
  a.q_out = d_q_out;
  a.q_rem = d_q_rem;
  a.k_rem = d_k_rem;
  a.v_rem = d_v_rem;
  return append_launch(ctx, cache, a, r.interleaved != 0 || r.dim == 0);
} catch (const std::exception& e) {
  return kv_refuse(nullptr, GRAPE_ERR_NOMEM, "%s", e.what());
}

extern "C" int grape_kv_select(grape_ctx* ctx, const grape_kv_cache* cache, const int32_t* d_table, uint32_t table_width,
                               uint32_t batch, const int32_t* d_len, const int32_t* d_q, uint64_t q_stride, uint32_t heads,
                               uint32_t n_select, uint32_t recent, int32_t* d_selected, int64_t* d_bound) try {
  if (int rc = kv_check_cache(ctx, cache, d_table, table_width, batch, false, false, true)) return rc;
  if (heads < 1 || heads > 65535 || heads % cache->kv_heads)
    return kv_refuse(ctx, GRAPE_ERR_INVALID, "heads must be a multiple of kv_heads up to 65535, not %u", heads);
  if (n_select < 1 || n_select > (1u << 20)) return kv_refuse(ctx, GRAPE_ERR_INVALID, "n_select must be 1 to 2^20, not %u", n_select);
  if (recent > n_select) return kv_refuse(ctx, GRAPE_ERR_INVALID, "recent must be at most n_select, not %u", recent);
  if (batch) {
    if (int rc = kv_check_rows(ctx, "queries", d_q, q_stride, (uint64_t)heads * cache->head_dim)) return rc;
    if (!d_len || misaligned(d_len, 4)) return kv_refuse(ctx, GRAPE_ERR_INVALID, "lengths must be given, on 4 bytes");
    if (!d_selected || misaligned(d_selected, 4)) return kv_refuse(ctx, GRAPE_ERR_INVALID, "selected must be given, on 4 bytes");
  }
  if (misaligned(d_bound, 8)) return kv_refuse(ctx, GRAPE_ERR_INVALID, "bound must be on 8 bytes");
  if ((uint64_t)batch * cache->kv_heads > 0x7fffffffu) return kv_refuse(ctx, GRAPE_ERR_LIMIT, "too many sequences and heads for one call");
  if (!ctx) return kv_refuse(ctx, GRAPE_ERR_INVALID, "null context");
  make_device_current(ctx);
  if (!batch) return GRAPE_OK;
  SelectArgs a{};
  a.c = kv_view(ctx, cache, d_table, table_width, batch);
  a.len = d_len;
  a.q = d_q;
  a.q_stride = q_stride;
  a.heads = heads;
  a.group = heads / cache->kv_heads;
  a.n_select = n_select;
  a.recent = recent;
  a.selected = d_selected;
  a.bound = d_bound;
  return select_launch(ctx, cache, a);
} catch (const std::exception& e) {
  return kv_refuse(nullptr, GRAPE_ERR_NOMEM, "%s", e.what());
}
