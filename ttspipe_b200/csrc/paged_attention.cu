// Decode attention over a paged KV cache: one new token of each of n_seqs
// sequences against its own pages, with the rows' attention weights accumulated
// for a later eviction.
//
// Mathematics. Query head g of sequence b reads KV head h = g / groups. Over the
// rows j < lens[b] that take part (the mask's byte is not 0, the row's page is
// assigned)
//     s_j = scale * (q_g . k_j),  m = max s_j,  l = sum exp(s_j - m),
//     out_g = sum exp(s_j - m) v_j / l,
//     weight[h][j] += sum over the group's heads of exp(s_j - m) / l.
// A sequence without such a row (or whose scores are all -inf) gets zeros and adds
// nothing. Scores are kept in units of log2 (scale * log2 e folded in after the
// product), products and sums in fp32.
//
// What bounds it. A row of a KV head is 512 bytes and 4 * 128 * groups operations, so
// memory does: 64 sequences of 8192 rows (32 query and 8 KV heads, 2.1 GB) take 317 us,
// 6.8 TB/s, the rate of a plain copy on the same GPU, with the tensor pipe 15-18% busy.
// Keys and values go from global memory straight into MMA fragments: a lane reads the
// 16-byte pieces of a row that are its fragment once q's dimensions and v's are taken in
// that order (a sum does not mind), so there is no staging, no bank conflict and nothing to wait
// for but the loads; 3 CTAs of 4 warps an SM, each warp a tile of keys and values ahead, keep
// up to 96 KB of them requested. Few rows are latency: 1 x 19 rows 3.9 us, 1 x 2048 rows
// 7.4 us (about 1.0 to find the part, 1.7 for a tile a warp, 0.4 to join the warps, 1.1
// for the counter, 2.3 to join the parts).
//
// Work split. The unit of work is a tile of 16 rows of one (sequence, KV head): page
// sizes are multiples of 16, so a tile lies in one page. All tiles of all sequences and
// heads, in that order, and what each (sequence, head) costs besides, are one line that
// is cut into equal parts, one for each CTA, from the lengths on the device: ragged
// batches balance, and one captured graph serves every length. A (sequence, head) that
// lies in one CTA's part is finished there; one that several CTAs share is joined by the
// CTA that finishes it last (a counter of each (sequence, head), back at 0 afterwards),
// in the order of the parts, so results do not depend on timing.

#include "common.cuh"
#include "gemv_unit.cuh"
#include "kernels.cuh"

namespace nf4b {

namespace {

constexpr int kD = 128;
constexpr int kTile = PAGED_TILE;
constexpr int kJoin = 16;  // parts whose outputs a joining warp requests at once
// Parts times query heads from which a join is made in two steps: one CTA reads 512 bytes
// of each at 64 bytes a clock, a second step costs two more round trips. 16 heads on one,
// 65536 rows in 148 parts: 17.4 us in two steps, 28 in one; 8 heads to one, 111 parts: 31.3
// and 37; 16 heads, 33 parts: 13.4 and 11.9.
constexpr int kWide = 700;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Tiles of a sequence: its length is brought into [0, capacity].
__device__ __forceinline__ int seq_rows(const PagedAttnParams& p, int b) {
  const int n = p.lens[b];
  const int cap = p.max_pages * p.page_size;
  return n < 0 ? 0 : n > cap ? cap : n;
}

// The work of one (sequence, head) on the line: its tiles and what one costs besides
// (first loads, the joins of its warps and parts), in tiles; 0 where there are none.
__device__ __forceinline__ int seq_work(const PagedAttnParams& p, int b) {
  const int tiles = (seq_rows(p, b) + kTile - 1) / kTile;
  return tiles == 0 ? 0 : tiles + PAGED_SEQ_TILES;
}

// Where each sequence's work begins on the line, at the start of the kernels' dynamic
// shared memory: pre[b] = work of all (sequence < b, head), pre[n_seqs] the total, and
// each[b] = work of one head of sequence b.
struct Line {
  int* pre;
  int* each;
  __device__ __forceinline__ Line(uint8_t* smem, int n_seqs)
      : pre(reinterpret_cast<int*>(smem)), each(pre + n_seqs + 1) {}
  // Ends with a barrier.
  __device__ __forceinline__ void fill(const PagedAttnParams& p) {
    if (threadIdx.x < 32) {
      const int lane = threadIdx.x;
      int base = 0;
      for (int b0 = 0; b0 < p.n_seqs; b0 += 32) {
        const int b = b0 + lane;
        const int one = b < p.n_seqs ? seq_work(p, b) : 0;
        int t = one * p.n_kv;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
          const int o = __shfl_up_sync(0xffffffffu, t, off);
          if (lane >= off) t += o;
        }
        if (b < p.n_seqs) {
          pre[b + 1] = base + t;
          each[b] = one;
        }
        base += __shfl_sync(0xffffffffu, t, 31);
      }
      if (lane == 0) pre[0] = 0;
    }
    __syncthreads();
  }
  // The sequence of unit u < pre[n]: the last b with pre[b] <= u. By a whole warp, 32
  // places compared at a time.
  __device__ __forceinline__ int seq_of(int n, int u) const {
    const int lane = threadIdx.x & 31;
    int base = 0;
    for (int left = n; left > 1;) {
      const int step = (left + 31) >> 5, at = lane * step;
      base += (__popc(__ballot_sync(0xffffffffu, at < left && pre[base + at] <= u)) - 1) * step;
      left = min(step, n - base);
    }
    return base;
  }
};

constexpr size_t line_bytes(int n_seqs) { return (size_t)(2 * n_seqs + 1) * sizeof(int); }

// The number of parts: as many as CTAs, but PAGED_MIN_TILES units of work in each unless
// that puts several (sequence, head)s into one part while CTAs are left.
__device__ __forceinline__ int parts(const PagedAttnParams& p, int work, int ctas) {
  const int by_work = (work + PAGED_MIN_TILES - 1) / PAGED_MIN_TILES;
  return min(ctas, max(by_work, min(p.n_seqs * p.n_kv, work)));
}

// Part c of `work` units in n parts: its first unit, the earlier parts one longer where
// they do not come out even; and the part of a unit.
struct Parts {
  int each, longer;
  __device__ __forceinline__ Parts(int work, int n) : each(work / n), longer(work - work / n * n) {}
  __device__ __forceinline__ int first(int c) const { return c * each + min(c, longer); }
  __device__ __forceinline__ int of(int u) const {
    const int edge = longer * (each + 1);
    return u < edge ? u / (each + 1) : longer + (u - edge) / each;
  }
};

// One (sequence, head) part's running state in a warp. NT: tiles of eight query
// heads (groups <= 8: one, else two). o is O^T from the MMA: o[nt][j][.] holds
// dimensions d = (j / 4) * 64 + (lane / 4) * 8 + 2 (j % 4) + {0, 1} of heads
// 8 nt + 2 (lane % 4) + {0, 1}: [0] (d, head), [1] (d, head + 1), [2] (d + 1, head),
// [3] (d + 1, head + 1). m and l belong to head 8 nt + lane / 4; l is this lane's
// share of the sum. o and l are both kept times 2^kLift.
//
// The weights exp(s - m) enter the second product in 16 bits. Rounded once, each
// would be off by as much as the output's own rounding; so they enter twice, as the
// rounded value and as what rounding left (the MMA units idle otherwise: memory bounds
// this kernel), which leaves 2^-17. fp16 has no exponents for the small weights of
// many rows next to one large one, so there they are lifted by 2^14 (exact).
template <bool F16>
constexpr float kLift = F16 ? 14.f : 0.f;

template <int NT>
struct WarpState {
  float o[NT][8][4];
  float m[NT], l[NT];
};

// A join: the states of `parts` parts of a (sequence, head), from `first` on in steps of
// `step`, into its outputs, or (to >= 0) into the place of a part.
struct Join {
  int first, parts, step;
  int b, h, to;
  int c0, c1;  // its first and last part
};

// The warps' states of one (sequence, head) part, for the join inside the CTA.
template <int NT, int kWarps>
struct AttnShared {
  float o[kWarps][NT * 8][kD];
  float m[kWarps][NT * 8], l[kWarps][NT * 8];
  Join joins[2];  // what this CTA joins
  int n_joins, wide;
};

// Whether none of the four is infinite or NaN.
__device__ __forceinline__ bool finite4(const float (&x)[4]) {
  return (x[0] - x[0]) + (x[1] - x[1]) + ((x[2] - x[2]) + (x[3] - x[3])) == 0.f;
}

// The finished row of one query head, four dimensions to a lane.
template <bool F16>
__device__ __forceinline__ void store_out(const PagedAttnParams& p, size_t head, int lane, float m, float l,
                                          const float (&o)[4]) {
  const float r = l == 0.f ? 0.f : 1.f / l;
  uint2 w = make_uint2(0, 0);
  if (l != 0.f) w = make_uint2(pack_act2<F16>(o[0] * r, o[1] * r), pack_act2<F16>(o[2] * r, o[3] * r));
  *reinterpret_cast<uint2*>(p.out + head * kD + lane * 4) = w;
  if (lane == 0 && p.lse != nullptr) p.lse[head] = l == 0.f ? -INFINITY : m + log2f(l) - kLift<F16>;
}

// Where the state of part q of a (sequence, head) whose first part is c0 lies: a CTA
// shares at most its first and its last (sequence, head).
__device__ __forceinline__ int slot_of(int q, int c0) { return 2 * q + (q == c0 ? 1 : 0); }

// Up to kJoin parts of one (sequence, query head): their states (maximum, sum), one to a
// lane, and their outputs, four dimensions to a lane.
struct JoinPiece {
  float2 ml;
  float4 o[kJoin];
  int join, head;
  int n;      // parts; 0: nothing
  bool last;  // the last ones of this head
};

// The joins of a list of up to two. Each warp takes every kWarps-th query head, kJoin parts
// at a time, and requests the next ones before it adds up these (16 heads of 24 parts:
// 7 us, 10 when each waited for its own).
template <int kWarps, bool F16>
__device__ __forceinline__ void join_parts(const PagedAttnParams& p, const Join* joins, int n_joins) {
  const int lane = threadIdx.x & 31, G = p.groups;
  int i = threadIdx.x >> 5, q0 = 0;  // the next pieces: query head, first part
  JoinPiece x, next;
  x.n = 0;
  float M = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  do {
    next.n = 0;
    if (i < n_joins * G) {
      next.join = i / G;
      next.head = i % G;
      const Join j = joins[next.join];
      const int n = min(kJoin, j.parts - q0), q = j.first + q0 * j.step;
      const size_t at0 = (size_t)slot_of(q, j.c0) * G + next.head;  // the others are not c0
      const size_t at = (size_t)(2 * q) * G + next.head, step = (size_t)(2 * j.step) * G;
      next.ml = make_float2(-INFINITY, 0.f);
      if (lane < n) next.ml = __ldcg(&p.part_ml[lane == 0 ? at0 : at + lane * step]);
      const float4* from = reinterpret_cast<const float4*>(p.part_o + at * kD) + lane;
      next.o[0] = __ldcg(reinterpret_cast<const float4*>(p.part_o + at0 * kD) + lane);
#pragma unroll
      for (int k = 1; k < kJoin; ++k) {
        from += step * (kD / 4);
        if (k < n) next.o[k] = __ldcg(from);
      }
      next.n = n;
      next.last = q0 + kJoin >= j.parts;
      q0 = next.last ? 0 : q0 + kJoin;
      i += next.last ? kWarps : 0;
    }
    if (x.n) {
      // the sums so far are scaled to the new maximum
      float m = fmaxf(M, x.ml.x);
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
      const float mu = m == -INFINITY ? 0.f : m, old = exp2_fast(M - mu), f = exp2_fast(x.ml.x - mu);
      M = m;
      l = fmaf(l, old, f * x.ml.y);
#pragma unroll
      for (int d = 0; d < 4; ++d) o[d] *= old;
#pragma unroll
      for (int k = 0; k < kJoin; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
        if (k >= x.n) continue;
        o[0] = fmaf(fk, x.o[k].x, o[0]);
        o[1] = fmaf(fk, x.o[k].y, o[1]);
        o[2] = fmaf(fk, x.o[k].z, o[2]);
        o[3] = fmaf(fk, x.o[k].w, o[3]);
      }
      if (x.last) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
        const Join j = joins[x.join];
        if (j.to < 0) {
          store_out<F16>(p, (size_t)j.b * p.n_head + (size_t)j.h * G + x.head, lane, M == -INFINITY ? 0.f : M, l, o);
        } else {
          const size_t to = (size_t)j.to * G + x.head;
          *reinterpret_cast<float4*>(&p.part_o[to * kD + lane * 4]) = make_float4(o[0], o[1], o[2], o[3]);
          if (lane == 0) p.part_ml[to] = make_float2(M, l);
        }
        M = -INFINITY;
        l = o[0] = o[1] = o[2] = o[3] = 0.f;
      }
    }
    x = next;
  } while (x.n);
}

// An infinite value times the rest that rounding a weight left, which may be 0 or negative, is
// NaN, so the sums of dimensions with such values are wrong. Where a part ends with sums that are
// not finite under weights that are, a warp adds up the infinite and NaN values by themselves: of
// query head `head` and tiles t0 to t1, four dimensions to a lane, those of rows of weight 0
// (a score of -inf) as NaN, as 0 times them is. A dimension that has any gets that sum. Called, so that
// its code is not in the way of calls without such values (1 x 2048 rows: 7.3 us, 7.5 inline). With
// one such value a page 64 x 8192 rows take 1.3 ms instead of 0.32, with one in every row 3.5.
template <bool F16>
__device__ __noinline__ float4 sum_infinities(const PagedAttnParams& p, int b, int h, int head, int t0, int t1,
                                              float4 o) {
  constexpr int kRows = 4;  // of a tile at a time, where it has any; few registers, which are the caller's too
  const int lane = threadIdx.x & 31, tpp = p.page_size / kTile, rows = seq_rows(p, b);
  const int* table = p.table + (size_t)b * p.max_pages;
  const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + (size_t)b * p.max_pages * p.page_size;
  const uint2 q = reinterpret_cast<const uint2*>(p.q + ((size_t)b * p.n_head + (size_t)h * p.groups + head) * kD)[lane];
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  auto four = [](uint2 w, float (&x)[4]) {
    x[0] = act_lo<F16>(w.x), x[1] = act_hi<F16>(w.x), x[2] = act_lo<F16>(w.y), x[3] = act_hi<F16>(w.y);
  };
#pragma unroll 1
  for (int tile = t0; tile < t1; ++tile) {
    const int pg = table[tile / tpp];
    if (pg < 0 || pg >= p.n_pages) continue;
    const size_t row = (((size_t)pg * p.n_kv + h) * p.page_size + (size_t)(tile % tpp) * kTile) * kD;
    const uint2 *v = reinterpret_cast<const uint2*>(p.v + row) + lane, *k = reinterpret_cast<const uint2*>(p.k + row) + lane;
    uint32_t odd = 0;  // rows that take part and have such values
    {
      uint2 all[kTile];
#pragma unroll
      for (int r = 0; r < kTile; ++r) all[r] = v[r * (kD / 4)];
#pragma unroll
      for (int r = 0; r < kTile; ++r) {
        float x[4];
        four(all[r], x);
        const int j = tile * kTile + r;
        if (__any_sync(0xffffffffu, !finite4(x)) && j < rows && (mask == nullptr || mask[j] != 0)) odd |= 1u << r;
      }
    }
#pragma unroll 1
    for (; odd != 0; odd >>= kRows, v += kRows * (kD / 4), k += kRows * (kD / 4)) {
      float x[kRows][4], s[kRows];  // the values and a lane's share of each score
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        float y[4], z[4];
        four(v[r * (kD / 4)], x[r]);
        four(k[r * (kD / 4)], y);
        four(q, z);
        s[r] = y[0] * z[0] + y[1] * z[1] + (y[2] * z[2] + y[3] * z[3]);
      }
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        if (!(odd >> r & 1)) continue;
        bool none = false;
        if (__any_sync(0xffffffffu, !(fabsf(s[r] * p.scale_log2) < 0x1p100f))) {  // else the score is finite
#pragma unroll
          for (int off = 16; off > 0; off >>= 1) s[r] += __shfl_xor_sync(0xffffffffu, s[r], off);
          none = s[r] * p.scale_log2 == -INFINITY;
        }
#pragma unroll
        for (int d = 0; d < 4; ++d)
          if (!(x[r][d] - x[r][d] == 0.f)) sum[d] += none ? NAN : x[r][d];
      }
    }
  }
  return make_float4(sum[0] != 0.f ? sum[0] : o.x, sum[1] != 0.f ? sum[1] : o.y, sum[2] != 0.f ? sum[2] : o.z,
                     sum[3] != 0.f ? sum[3] : o.w);
}

template <int NT, int kWarps, bool F16>
__global__ void __launch_bounds__(kWarps * 32, NT == 1 && kWarps == 4 ? 3 : 1)
    paged_attention_kernel(const __grid_constant__ PagedAttnParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr int kThreads = kWarps * 32;
  using Shared = AttnShared<NT, kWarps>;
  Shared& sm = *reinterpret_cast<Shared*>(smem);
  Line line(smem + sizeof(Shared), p.n_seqs);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int G = p.groups;

  if (tid == 0) sm.n_joins = sm.wide = 0;
  pdl_wait();  // q, the new rows and the lengths come from earlier kernels
  line.fill(p);
  for (int b = blockIdx.x; b < p.n_seqs; b += gridDim.x)
    if (line.each[b] == 0)
      for (int i = tid; i < p.n_head * kD; i += kThreads) p.out[(size_t)b * p.n_head * kD + i] = 0;
  const int U = line.pre[p.n_seqs];
  const int N = parts(p, U, (int)gridDim.x);
  const int c = blockIdx.x;
  if (c >= N) return;
  const Parts cut(U, N);
  // Where this part and (odd lanes) the next one begin: sequence b, head h, tile t0 of it.
  // A (sequence, head) of up to PAGED_MIN_TILES tiles is not split (joining it would cost
  // more): a cut in it moves to its first tile.
  int u = min(cut.first(c + (lane & 1)), U - 1);
  int b = line.seq_of(p.n_seqs, __shfl_sync(0xffffffffu, u, 0));
  const int b1 = line.seq_of(p.n_seqs, __shfl_sync(0xffffffffu, u, 1));
  if (lane & 1) b = b1;
  const int from = u - line.pre[b];
  int h = from / line.each[b], t0 = from - h * line.each[b];
  if (line.each[b] <= PAGED_MIN_TILES + PAGED_SEQ_TILES) {
    u -= t0;
    t0 = 0;
  }
  const int u1 = c + 1 < N ? __shfl_sync(0xffffffffu, u, 1) : U;
  u = __shfl_sync(0xffffffffu, u, 0);
  b = __shfl_sync(0xffffffffu, b, 0);
  h = __shfl_sync(0xffffffffu, h, 0);
  t0 = __shfl_sync(0xffffffffu, t0, 0);
  const int tpp = p.page_size / kTile;

  auto advance = [&]() {  // to the next (sequence, head) with rows
    if (++h < p.n_kv) return;
    h = 0;
    do ++b;
    while (b < p.n_seqs && line.each[b] == 0);
  };

  for (; u < u1; t0 = 0) {
    const int work = line.each[b], T = work - PAGED_SEQ_TILES;
    const int t1 = min(T, t0 + (u1 - u));
    if (t0 >= T) {  // only the end of its work: nothing to do
      u += work - t0;
      advance();
      continue;
    }
    const int rows = seq_rows(p, b);
    const int* table = p.table + (size_t)b * p.max_pages;
    const uint8_t* mask = p.mask == nullptr ? nullptr : p.mask + (size_t)b * p.max_pages * p.page_size;
    float* scores = p.scores == nullptr ? nullptr : p.scores + (size_t)(u - t0) * G * kTile;

    // the group's queries as the A operand, dimensions in the order in which a
    // lane reads a key row: 16-byte pieces c * 4 + t
    uint4 qa[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = nt * 8 + g;
      const uint4* qr = reinterpret_cast<const uint4*>(p.q + ((size_t)b * p.n_head + (size_t)h * G + head) * kD);
#pragma unroll
      for (int cc = 0; cc < 4; ++cc) qa[nt][cc] = head < G ? qr[cc * 4 + t] : make_uint4(0, 0, 0, 0);
    }

    WarpState<NT> s;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      s.m[nt] = -INFINITY;
      s.l[nt] = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) s.o[nt][j][i] = 0.f;
    }

    // Keys and values of the next tile are requested as soon as this tile's have been
    // multiplied, its page is looked up one tile earlier still.
    uint4 kr[2][4], vr[4][2];
    int tile = t0 + warp;
    auto page_of = [&](int at) -> int {
      const int pg = at < t1 ? table[at / tpp] : 0;
      return pg < p.n_pages ? pg : -1;
    };
    auto row_of = [&](int at, int pg) -> size_t {
      return (((size_t)max(pg, 0) * p.n_kv + h) * p.page_size + (size_t)(at % tpp) * kTile) * (kD / 8);
    };
    auto load_k = [&](size_t row) {
      const uint4* kp = reinterpret_cast<const uint4*>(p.k) + row;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) kr[n][cc] = ld_stream_u4(kp + (n * 8 + g) * 16 + cc * 4 + t);
    };
    auto load_v = [&](size_t row) {
      const uint4* vp = reinterpret_cast<const uint4*>(p.v) + row;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int hh = 0; hh < 2; ++hh)
          vr[r][hh] = ld_stream_u4(vp + (2 * t + (r & 1) + (r >> 1) * 8) * 16 + hh * 8 + g);
    };
    int pg = page_of(tile), pg1 = page_of(tile + kWarps);
    size_t row = row_of(tile, pg);
    if (tile < t1) {
      load_k(row);
      load_v(row);
    }
    for (; tile < t1; tile += kWarps) {
      const int next = tile + kWarps, pg2 = page_of(next + kWarps);
      row = row_of(next, pg1);
      // the lane's four rows 2t, 2t + 1, 8 + 2t, 9 + 2t: which take part
      const bool full = pg >= 0 && (tile + 1) * kTile <= rows && mask == nullptr;
      bool see[4] = {true, true, true, true};
      if (!full) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int j = tile * kTile + 2 * t + (r & 1) + (r >> 1) * 8;
          see[r] = pg >= 0 && j < rows && (mask == nullptr || mask[j] != 0);
        }
      }
      float sc[2][4];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][i] = 0.f;
#pragma unroll
        for (int cc = 0; cc < 4; ++cc) {
          const uint4 q0 = qa[0][cc], q1 = NT == 1 ? make_uint4(0, 0, 0, 0) : qa[NT - 1][cc];
          mma_act<F16>(sc[n], q0.x, q1.x, q0.y, q1.y, kr[n][cc].x, kr[n][cc].y);
          mma_act<F16>(sc[n], q0.z, q1.z, q0.w, q1.w, kr[n][cc].z, kr[n][cc].w);
        }
      }
      if (next < t1) load_k(row);
      uint32_t ph[NT][2], pl[NT][2];  // P^T as the B operand: the rounded weights and what rounding left
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float x[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = see[r] ? sc[r >> 1][nt * 2 + (r & 1)] * p.scale_log2 : -INFINITY;
        if (scores != nullptr && nt * 8 + g < G) {
          float* sp = scores + ((size_t)tile * G + nt * 8 + g) * kTile + 2 * t;
          *reinterpret_cast<float2*>(sp) = make_float2(x[0], x[1]);
          *reinterpret_cast<float2*>(sp + 8) = make_float2(x[2], x[3]);
        }
        float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mnew = fmaxf(s.m[nt], mx);
        const float mu = mnew == -INFINITY ? 0.f : mnew;
        if (__any_sync(0xffffffffu, mnew > s.m[nt])) {
          const float f = exp2_fast(s.m[nt] - mu);
          const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
          s.l[nt] *= f;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            s.o[nt][j][0] *= f0;
            s.o[nt][j][1] *= f1;
            s.o[nt][j][2] *= f0;
            s.o[nt][j][3] *= f1;
          }
          s.m[nt] = mnew;
        }
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          e[r] = exp2_fast(x[r] - mu + kLift<F16>);
          s.l[nt] += e[r];
        }
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          ph[nt][n] = pack_act2<F16>(e[2 * n], e[2 * n + 1]);
          pl[nt][n] = pack_act2<F16>(e[2 * n] - act_lo<F16>(ph[nt][n]), e[2 * n + 1] - act_hi<F16>(ph[nt][n]));
        }
      }
      if (!full) {  // 0 * NaN of an unwritten row is NaN
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!see[r]) vr[r][0] = vr[r][1] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        const uint32_t* w0 = &vr[0][hh].x;
        const uint32_t* w1 = &vr[1][hh].x;
        const uint32_t* w2 = &vr[2][hh].x;
        const uint32_t* w3 = &vr[3][hh].x;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const uint32_t a0 = prmt(w0[w], w1[w], 0x5410u), a1 = prmt(w0[w], w1[w], 0x7632u);
          const uint32_t a2 = prmt(w2[w], w3[w], 0x5410u), a3 = prmt(w2[w], w3[w], 0x7632u);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_act<F16>(s.o[nt][hh * 4 + w], a0, a1, a2, a3, ph[nt][0], ph[nt][1]);
            mma_act<F16>(s.o[nt][hh * 4 + w], a0, a1, a2, a3, pl[nt][0], pl[nt][1]);
          }
        }
      }
      if (next < t1) load_v(row);
      pg = pg1;
      pg1 = pg2;
    }

    // the warps' states into shared memory
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      s.l[nt] += __shfl_xor_sync(0xffffffffu, s.l[nt], 1);
      s.l[nt] += __shfl_xor_sync(0xffffffffu, s.l[nt], 2);
      if (t == 0) {
        sm.m[warp][nt * 8 + g] = s.m[nt];
        sm.l[warp][nt * 8 + g] = s.l[nt];
      }
      if (nt * 8 + 2 * t < G) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int d = (j >> 2) * 64 + g * 8 + (j & 3) * 2;
          *reinterpret_cast<float2*>(&sm.o[warp][nt * 8 + 2 * t][d]) = make_float2(s.o[nt][j][0], s.o[nt][j][2]);
          *reinterpret_cast<float2*>(&sm.o[warp][nt * 8 + 2 * t + 1][d]) = make_float2(s.o[nt][j][1], s.o[nt][j][3]);
        }
      }
    }
    __syncthreads();
    // a warp joins the states of a query head, four dimensions to a lane
    const bool whole = t0 == 0 && t1 == T;
    const int slot = 2 * c + (t0 == 0 ? 1 : 0);
    const size_t head0 = (size_t)b * p.n_head + (size_t)h * G;
    for (int head = warp; head < G; head += kWarps) {
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, sm.m[w][head]);
      const float mu = M == -INFINITY ? 0.f : M;
      float l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2_fast(sm.m[w][head] - mu);
        const float4 x = *reinterpret_cast<const float4*>(&sm.o[w][head][lane * 4]);
        l = fmaf(f, sm.l[w][head], l);
        o[0] = fmaf(f, x.x, o[0]);
        o[1] = fmaf(f, x.y, o[1]);
        o[2] = fmaf(f, x.z, o[2]);
        o[3] = fmaf(f, x.w, o[3]);
      }
      if (__any_sync(0xffffffffu, l == l && !finite4(o))) {
        const float4 x = sum_infinities<F16>(p, b, h, head, t0, t1, make_float4(o[0], o[1], o[2], o[3]));
        o[0] = x.x, o[1] = x.y, o[2] = x.z, o[3] = x.w;
      }
      if (whole) {
        store_out<F16>(p, head0 + head, lane, mu, l, o);
      } else {
        *reinterpret_cast<float4*>(&p.part_o[((size_t)slot * G + head) * kD + lane * 4]) =
            make_float4(o[0], o[1], o[2], o[3]);
        if (lane == 0) p.part_ml[(size_t)slot * G + head] = make_float2(M, l);
      }
    }
    if (!whole) {
      // The CTAs whose parts hold this (sequence, head) are c0 to c1; the last one to come
      // here joins them. Where that is much (kWide), each kJoin of them are joined first
      // by the last of these, and the last of those joins the rest.
      const int c0 = cut.of(u - t0), c1 = cut.of(u - t0 + T - 1);
      const bool wide = (c1 - c0 + 1) * G >= kWide;
      const int first = wide ? c - (c - c0) % kJoin : c0, last = wide ? min(first + kJoin - 1, c1) : c1;
      __syncthreads();
      if (tid == 0) {
        int* counter = wide ? p.group_counters + slot_of(first, c0) : p.counters + b * p.n_kv + h;
        __threadfence();
        if (atomicAdd(counter, 1) == last - first) {
          __threadfence();
          *counter = 0;
          sm.joins[sm.n_joins++] = Join{first, last - first + 1, 1, b, h, wide ? slot_of(first, c0) : -1, c0, c1};
          if (wide) sm.wide = 1;
        }
      }
    }
    __syncthreads();  // the shared state is free again
    u += t1 == T ? work - t0 : t1 - t0;
    advance();
  }
  // joins after the main loop, at most two (so that their registers are not the loop's)
#pragma unroll 1
  for (bool again = true; again;) {
    again = sm.wide != 0;
    join_parts<kWarps, F16>(p, sm.joins, sm.n_joins);
    if (!again) break;
    __syncthreads();
    if (tid == 0) {  // joins of kJoin parts are parts themselves: the last of them joins these
      sm.wide = 0;
      int n = 0;
      for (int i = 0; i < sm.n_joins; ++i) {
        Join j = sm.joins[i];
        if (j.to < 0) continue;  // done
        const int groups = (j.c1 - j.c0) / kJoin + 1;
        __threadfence();
        int* counter = p.counters + j.b * p.n_kv + j.h;
        if (atomicAdd(counter, 1) != groups - 1) continue;
        __threadfence();
        *counter = 0;
        sm.joins[n++] = Join{j.c0, groups, kJoin, j.b, j.h, -1, j.c0, j.c1};
      }
      sm.n_joins = n;
    }
    __syncthreads();
  }
  pdl_launch_dependents();
}

// weight[row] += sum over the group's heads of 2^(score - lse), from the scores the
// attention kernel left (a row's weight needs the sum over all rows, which only the
// joins know). Four rows to a thread; a reduction instruction instead of a read and a
// write, so that sequences which share a page add up. Rows that take no part have the
// score -inf and receive 0, also where the sum of a head is NaN. Memory bounds it: 4 groups + 8 bytes a row and KV head,
// 20 us for 64 x 8192 rows (100 MB), about 4 us for small calls.
constexpr int kWThreads = 256;
constexpr int kWTiles = kWThreads / 4;  // tiles of one pass of a CTA

__global__ void __launch_bounds__(kWThreads) paged_weight_kernel(const __grid_constant__ PagedAttnParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  Line line(smem, p.n_seqs);
  pdl_wait();
  line.fill(p);
  const int U = line.pre[p.n_seqs], tpp = p.page_size / kTile, G = p.groups;
  const int i = (threadIdx.x & 3) * 4;
  // a warp takes eight units at a time, four lanes each
  for (long long u0 = (long long)blockIdx.x * kWTiles + (threadIdx.x >> 5) * 8; u0 < U;
       u0 += (long long)gridDim.x * kWTiles) {
    const int u = min((int)u0 + ((threadIdx.x & 31) >> 2), U);
    int b = line.seq_of(p.n_seqs, (int)u0);
    while (u < U && line.pre[b + 1] <= u) ++b;
    const int work = line.each[b], h = (u - line.pre[b]) / max(work, 1), tile = u - line.pre[b] - h * work;
    if (u == U || tile >= work - PAGED_SEQ_TILES) continue;
    const int pg = p.table[(size_t)b * p.max_pages + tile / tpp];
    const float* lse = p.lse + (size_t)b * p.n_head + (size_t)h * G;
    const float* sp = p.scores + (size_t)u * G * kTile + i;
    float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int head = 0; head < G; ++head) {
      const float4 x = __ldcs(reinterpret_cast<const float4*>(sp + head * kTile));
      const float L = lse[head] == -INFINITY ? INFINITY : lse[head];
      w.x += exp2_fast(x.x - L);
      w.y += exp2_fast(x.y - L);
      w.z += exp2_fast(x.z - L);
      w.w += exp2_fast(x.w - L);
    }
    if (pg < 0 || pg >= p.n_pages) continue;
    if (!(w.x == w.x && w.y == w.y && w.z == w.z && w.w == w.w)) {
      // a head whose sum is NaN (a visible score is NaN or +inf): the rows that take no part keep what they have
      const int n = seq_rows(p, b) - (tile * kTile + i);
      const uint8_t* mask =
          p.mask == nullptr ? nullptr : p.mask + (size_t)b * p.max_pages * p.page_size + tile * kTile + i;
      if (n <= 0 || (mask != nullptr && mask[0] == 0)) w.x = 0.f;
      if (n <= 1 || (mask != nullptr && mask[1] == 0)) w.y = 0.f;
      if (n <= 2 || (mask != nullptr && mask[2] == 0)) w.z = 0.f;
      if (n <= 3 || (mask != nullptr && mask[3] == 0)) w.w = 0.f;
    }
    float* out = p.weight + ((size_t)pg * p.n_kv + h) * p.page_size + (size_t)(tile % tpp) * kTile + i;
    asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(out), "f"(w.x), "f"(w.y), "f"(w.z), "f"(w.w)
                 : "memory");
  }
  pdl_launch_dependents();
}

template <typename K>
cudaError_t launch(K kernel, int grid, int threads, size_t smem, const PagedAttnParams& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

template <int NT, int kWarps, bool F16>
cudaError_t launch_attention(const PagedAttnParams& p, int grid, cudaStream_t stream) {
  constexpr size_t shared = sizeof(AttnShared<NT, kWarps>);
  auto kernel = paged_attention_kernel<NT, kWarps, F16>;
  static bool configured[64] = {};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) return cudaErrorInvalidDevice;
  if (!configured[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)(shared + line_bytes(PAGED_MAX_SEQS)));
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  return launch(kernel, grid, kWarps * 32, shared + line_bytes(p.n_seqs), p, stream);
}

long long most_work(int n_seqs, int n_kv, long long max_rows) {
  return (long long)n_seqs * n_kv * ((max_rows + kTile - 1) / kTile + PAGED_SEQ_TILES);
}

// Warps of a CTA: 8 where a join has many heads to share out (16 heads on one, 65536 rows:
// 17.4 us, 23 with 4) or where the whole cache is so small that a tile a warp is enough (1 x 2048
// rows: 7.5 us, 8.1 with 4); else 4, three CTAs on an SM.
int warps_for(long long work, int groups, int sms) { return groups > 8 || work <= 16LL * sms ? 8 : 4; }

// CTAs of a launch, all resident.
int grid_for(long long work, long long lists, int groups, int sms) {
  const long long by_work = (work + PAGED_MIN_TILES - 1) / PAGED_MIN_TILES, n = by_work > lists ? by_work : lists;
  const long long resident = (long long)sms * (warps_for(work, groups, sms) == 4 ? 3 : 1);
  const long long most = resident < PAGED_MAX_PARTS ? resident : PAGED_MAX_PARTS;
  return (int)(n < most ? n : most);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

void paged_attention_plan(int n_seqs, int n_head, int n_kv, long long max_rows, bool tracked, int sms,
                          PagedAttnPlan* plan) {
  const long long work = most_work(n_seqs, n_kv, max_rows);
  const int groups = n_head / n_kv;
  plan->grid = grid_for(work, (long long)n_seqs * n_kv, groups, sms);
  size_t at = PAGED_COUNTER_BYTES;
  plan->part_o = at;
  at += up256((size_t)2 * plan->grid * groups * kD * sizeof(float));
  plan->part_ml = at;
  at += up256((size_t)2 * plan->grid * groups * sizeof(float2));
  plan->lse = plan->scores = at;
  if (tracked) {
    at += up256((size_t)n_seqs * n_head * sizeof(float));
    plan->scores = at;
    at += up256((size_t)work * kTile * groups * sizeof(float));
  }
  plan->bytes = at;
}

cudaError_t launch_paged_attention(const PagedAttnParams& p, int grid, int sms, bool f16, cudaStream_t stream) {
  const long long work = most_work(p.n_seqs, p.n_kv, (long long)p.max_pages * p.page_size);
  cudaError_t e;
  if (p.groups > 8)
    e = f16 ? launch_attention<2, 8, true>(p, grid, stream) : launch_attention<2, 8, false>(p, grid, stream);
  else if (warps_for(work, p.groups, sms) == 8)
    e = f16 ? launch_attention<1, 8, true>(p, grid, stream) : launch_attention<1, 8, false>(p, grid, stream);
  else
    e = f16 ? launch_attention<1, 4, true>(p, grid, stream) : launch_attention<1, 4, false>(p, grid, stream);
  if (e != cudaSuccess || p.weight == nullptr) return e;
  const long long n = (work + kWTiles - 1) / kWTiles;
  return launch(paged_weight_kernel, (int)(n < 8LL * sms ? n : 8LL * sms), kWThreads,
                line_bytes(p.n_seqs), p, stream);
}

}  // namespace nf4b
