// The paged KV cache's other two operators: tokens entering their pages (q/k norm,
// rotary, scatter), and the eviction of the rows that were attended to least.

#include <limits.h>

#include "common.cuh"
#include "kernels.cuh"

namespace nf4b {

namespace {

constexpr int kD = 128;

// ---- write ------------------------------------------------------------------
// Half a warp for each head of a token, 16 bytes (four rotary pairs) to a lane; a warp
// takes kGroups times 2 kPairs heads of one token, so that the rotary row and the page are
// had once for all of them and the norm's reciprocal square root (fp64, one lane a head) once
// for each 2 kPairs. The arithmetic is
// qk_rope_kv_kernel's, rounding point for rounding point, so a row in a page has the bits it
// would have in a dense cache. (The norm's squares are exact in fp64. Their sum is taken in
// another order, which makes a difference past its 53rd bit at most, where values of a head are
// far apart, and is then rounded to 24: it shows for about one such head in 2^26.) 8188 tokens of 48 heads (202 MB) take 41 us with norm, 35 without: 4.9 and
// 5.8 TB/s, the norm bound by instruction issue (61% of all slots); one token 1.9 us, the launch.
constexpr int kWriteWarps = 4;

// Two fp32 numbers in one register pair: sm_100 multiplies and adds both at once, each
// rounded to nearest as by itself.
struct F2 {
  unsigned long long v;
};
__device__ __forceinline__ F2 f2(float x, float y) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpack(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}

// rsqrt_exact of common.cuh for a width of 128 with CUDA's fp64 rsqrt in place of a
// square root and a division. Both are within 2^-52 of 1 / sqrt(t), and that is nowhere so near
// the middle of two fp32 numbers: the rounded results agree for every fp32 t.
__device__ __forceinline__ float rsqrt_128(double ss, float eps) {
  const float t = __fadd_rn((float)(ss * (1.0 / 128)), eps);
  return (float)rsqrt((double)t);
}

template <int kPairs, int kGroups, bool F16>
__global__ void __launch_bounds__(kWriteWarps * 32, kPairs == 4 ? 7 : 1)
    paged_write_kernel(const __grid_constant__ PagedWriteParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31, half = lane >> 4, piece = lane & 15;
  const int heads = p.n_head + 2 * p.n_kv;
  constexpr int kSpan = 2 * kPairs * kGroups;
  const int spans = (heads + kSpan - 1) / kSpan;
  const unsigned item = blockIdx.x * kWriteWarps + (threadIdx.x >> 5);
  const int tok = (int)(item / spans);
  if (tok >= p.n_tokens) return;
  int first = (int)(item - (unsigned)tok * spans) * kSpan;
  const int end = min(heads, first + kSpan);
  const uint4* in = reinterpret_cast<const uint4*>(p.qkv + (size_t)tok * heads * kD) + piece;
  uint4 raw[kPairs], next[kPairs];
  auto load = [&](uint4 (&to)[kPairs], int head) {
#pragma unroll
    for (int u = 0; u < kPairs; ++u) {
      to[u] = make_uint4(0, 0, 0, 0);
      if (head + 2 * u < end) to[u] = ld_stream_u4(in + (head + 2 * u) * (kD / 8));
    }
  };
  load(raw, first + half);
  const int pos = p.positions[tok], row = p.rows[tok], seq = p.seqs == nullptr ? tok : p.seqs[tok];
  const bool turned = pos >= 0 && pos < p.freqs_rows;  // else the token is padding
  F2 c[2], sn[2], ns[2];  // cos, sin and -sin of pairs 2 i and 2 i + 1
  if (turned && first < p.n_head + p.n_kv) {
    float cs[8];
    const size_t at = (size_t)pos * kD + piece * 8;
    if (p.ftype == NF4B_F32) {
      const float4* f = reinterpret_cast<const float4*>(static_cast<const float*>(p.freqs) + at);
      *reinterpret_cast<float4*>(cs) = f[0];
      *reinterpret_cast<float4*>(cs + 4) = f[1];
    } else {
      const uint4 f = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.freqs) + at);
      const uint32_t w[4] = {f.x, f.y, f.z, f.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        cs[2 * i] = p.ftype == NF4B_F16 ? act_lo<true>(w[i]) : act_lo<false>(w[i]);
        cs[2 * i + 1] = p.ftype == NF4B_F16 ? act_hi<true>(w[i]) : act_hi<false>(w[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      c[i] = f2(cs[4 * i], cs[4 * i + 2]);
      sn[i] = f2(cs[4 * i + 1], cs[4 * i + 3]);
      ns[i] = f2(-cs[4 * i + 1], -cs[4 * i + 3]);
    }
  }
  long long slot = -1;  // the token's row in its page, of KV head 0
  if (end > p.n_head && turned && row >= 0 && row / p.page_size < p.max_pages && seq >= 0 &&
      seq < p.n_seqs) {
    const int pg = p.table[(size_t)seq * p.max_pages + row / p.page_size];
    if (pg >= 0 && pg < p.n_pages) slot = (long long)pg * p.n_kv * p.page_size + row % p.page_size;
  }
  uint4 nw = make_uint4(0, 0, 0, 0);
  int of = -1;  // whose norm weight nw is: 1 the queries', 0 the keys'
#pragma unroll 1
  for (;; first += 2 * kPairs) {
    const bool more = first + 2 * kPairs < end;
    if (more) load(next, first + 2 * kPairs + half);
    float r = 0.f;
    if (turned && p.qw != nullptr && first < p.n_head + p.n_kv) {
      double ss[kPairs];
#pragma unroll
      for (int u = 0; u < kPairs; ++u) {
        const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
        ss[u] = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const double x0 = act_lo<F16>(w[i]), x1 = act_hi<F16>(w[i]);
          ss[u] = fma(x0, x0, ss[u]);
          ss[u] = fma(x1, x1, ss[u]);
        }
      }
      // over the half warp; where there are four sums, lanes hand over those that others
      // finish: lane j ends with the sum of pair j % 4
      double mine = ss[0];
      if (kPairs == 4) {
        double two[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {  // lanes with bit 1 take pairs 2 and 3
          const bool up = lane & 2;
          const double keep = up ? ss[2 % kPairs + (i & (kPairs - 1))] : ss[i & (kPairs - 1)];
          const double give = up ? ss[i & (kPairs - 1)] : ss[2 % kPairs + (i & (kPairs - 1))];
          two[i] = keep + __shfl_xor_sync(0xffffffffu, give, 2);
        }
        const double keep = lane & 1 ? two[1] : two[0], give = lane & 1 ? two[0] : two[1];
        mine = keep + __shfl_xor_sync(0xffffffffu, give, 1);
        mine += __shfl_xor_sync(0xffffffffu, mine, 4);
        mine += __shfl_xor_sync(0xffffffffu, mine, 8);
      } else {
#pragma unroll
        for (int off = 8; off > 0; off >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, off);
      }
      r = rsqrt_128(mine, p.eps);
    }
#pragma unroll
    for (int u = 0; u < kPairs; ++u) {
      const int head = first + half + 2 * u;
      const float ru = __shfl_sync(0xffffffffu, r, (lane & 16) | u);
      if (head >= end) continue;
      const bool is_q = head < p.n_head, is_v = head >= p.n_head + p.n_kv;
      uint4 out = raw[u];
      if (!is_v && turned) {
        const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
        uint32_t o[4];
        if (p.qw != nullptr && of != (int)is_q) {
          of = is_q;
          nw = reinterpret_cast<const uint4*>(is_q ? p.qw : p.kw)[piece];
        }
        const uint32_t g[4] = {nw.x, nw.y, nw.z, nw.w};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          F2 x0 = f2(act_lo<F16>(w[2 * i]), act_lo<F16>(w[2 * i + 1]));
          F2 x1 = f2(act_hi<F16>(w[2 * i]), act_hi<F16>(w[2 * i + 1]));
          if (p.qw != nullptr) {
            const F2 rr = f2(ru, ru);
            const float2 y0 = unpack(mul2(mul2(x0, rr), f2(act_lo<F16>(g[2 * i]), act_lo<F16>(g[2 * i + 1]))));
            const float2 y1 = unpack(mul2(mul2(x1, rr), f2(act_hi<F16>(g[2 * i]), act_hi<F16>(g[2 * i + 1]))));
            const uint32_t a = pack_act2<F16>(y0.x, y1.x), b = pack_act2<F16>(y0.y, y1.y);  // the norm's rounding
            x0 = f2(act_lo<F16>(a), act_lo<F16>(b));
            x1 = f2(act_hi<F16>(a), act_hi<F16>(b));
          }
          const float2 z0 = unpack(add2(mul2(x0, c[i]), mul2(x1, ns[i])));
          const float2 z1 = unpack(add2(mul2(x1, c[i]), mul2(x0, sn[i])));
          o[2 * i] = pack_act2<F16>(z0.x, z1.x);
          o[2 * i + 1] = pack_act2<F16>(z0.y, z1.y);
        }
        out = make_uint4(o[0], o[1], o[2], o[3]);
      }
      if (is_q) {
        reinterpret_cast<uint4*>(p.q_out + ((size_t)tok * p.n_head + head) * kD)[piece] =
            turned ? out : make_uint4(0, 0, 0, 0);
      } else if (slot >= 0) {
        const size_t at = slot + (size_t)(head - p.n_head - (is_v ? p.n_kv : 0)) * p.page_size;
        reinterpret_cast<uint4*>((is_v ? p.v : p.k) + at * kD)[piece] = out;
        if (!is_v && piece == 0) {
          if (p.weight != nullptr) p.weight[at] = 0.f;
          if (p.position != nullptr) p.position[at] = pos;
        }
      }
    }
    if (!more) break;
#pragma unroll
    for (int u = 0; u < kPairs; ++u) raw[u] = next[u];
  }
  pdl_launch_dependents();
}

// ---- evict ------------------------------------------------------------------
// Of each (sequence, KV head) the first `left` = min(rows, budget) rows in this
// order stay: rows whose position is below `sink` or among the `recent` newest
// first, then by falling weight (NaN as -inf), equal ones by rising row. Rows at or
// past `left` that stay move, in order, into the rows below it that do not: there are
// equally many, the two sets are disjoint, and attention does not depend on the order
// of rows (the rotary is in the keys), so nothing else has to move.
// Rows without a page hold nothing. Below `left` they are no places: they count as kept where
// they are, before all others (there are at most `left` of them, and equal keys go by rising
// row), so as many rows stay as there are places with a page. From `left` on they come last,
// and rows with a page suffice: the places' own are as many.
//
// paged_select_kernel, one CTA or one cluster of CTAs a list, finds the smallest kept key
// digit by digit from the top (11, 11 and 10 bits, a histogram each) and lists the moves;
// paged_move_kernel makes them. 8 x 32768 rows halved (64 lists, 562 MB) take 130 us:
// about 27 to select, a chain of dependent steps (read, newest, three histograms, two
// counts), and 103 to move some 524,000 rows, 256 bytes of key and of value each between
// scattered places, at 5.2 TB/s of DRAM. 1 x 2048 rows are the chain alone, 9 us.
constexpr int kBins = 2048;

// Weights in rising order as unsigned integers; 0xFFFFFFFF (no weight maps there,
// NaN being taken as -inf) is for the protected rows and those below `left` without a page, 0
// for the others without one.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (!(w == w)) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 as 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Walks a list in groups of 128 rows, four consecutive ones (they lie in one page) to a
// lane; the page and the row in it are carried along instead of divided out.
struct Quads {
  const int32_t* table;
  int h, n_kv, n_pages, page_size, step_pages, step_rows;
  int row, page, at;
  __device__ __forceinline__ Quads(const PagedEvictParams& p, int b, int head, int first)
      : table(p.table + (size_t)b * p.max_pages), h(head), n_kv(p.n_kv), n_pages(p.n_pages), page_size(p.page_size),
        step_pages(128 / p.page_size), step_rows(128 % p.page_size), row(first), page(first / p.page_size),
        at(first % p.page_size) {}
  __device__ __forceinline__ void next() {
    row += 128;
    page += step_pages;
    at += step_rows;
    if (at >= page_size) {
      at -= page_size;
      ++page;
    }
  }
  // The pool row of `row`; -1 where its page is not assigned.
  __device__ __forceinline__ int pool() const {
    const int pg = table[page];
    return pg < 0 || pg >= n_pages ? -1 : (pg * n_kv + h) * page_size + at;
  }
};

__device__ __forceinline__ int warp_scan(int v, int lane) {  // inclusive
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const int o = __shfl_up_sync(0xffffffffu, v, off);
    if (lane >= off) v += o;
  }
  return v;
}

// Counts of digits that many rows may share (weight 0 of new rows, protected rows, a
// digit 0 below a common prefix) are kept by each thread and added once a warp: as
// single additions to one counter they would run one after another.
__device__ __forceinline__ void add_shared(int* to, int n, int lane) {
  n = __reduce_add_sync(0xffffffffu, n);
  if (lane == 0 && n != 0) atomicAdd(to, n);
}

__device__ __forceinline__ int* cluster_peer(int* p, unsigned rank) {  // the same place in another CTA of the cluster
  uint64_t out;
  asm("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
  return reinterpret_cast<int*>(out);
}

// A list belongs to a cluster of `size` CTAs, each with an equal share of its rows, and
// each warp of them with a run of that, kDeep groups of 128 rows at a time. kOnce: that is
// the whole run, and its keys stay in registers; longer runs are read again (from L2) for every
// step. The code is unrolled over the groups and runs once, so where a list is short its
// fetching costs as much as its work (1 x 2048 rows: 11.1 us with kDeep 4, 8.7 with 2).
template <int kThreads, int kDeep, bool kOnce>
__global__ void __launch_bounds__(kThreads, kThreads == 1024 ? 1 : 1024 / kThreads)
    paged_select_kernel(const __grid_constant__ PagedEvictParams p, int size) {
  __shared__ alignas(16) int hists[3][kBins];  // of each step; the first CTA's become the cluster's
  __shared__ int part[3][32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need, s_among, s_newest, s_sum[3];
  constexpr int kWarps = kThreads / 32, kMine = kBins / kThreads;
  pdl_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int list = blockIdx.x / size, rank = blockIdx.x - list * size;
  const int b = list / p.n_kv, h = list - b * p.n_kv;
  const int cap = p.max_pages * p.page_size;
  const int total = min(max(p.lens[b], 0), cap), left = min(total, p.budget);
  const bool all = total <= p.budget;
  const int run = (total + size * kWarps * 128 - 1) / (size * kWarps * 128) * 128;
  const int r0 = min(total, (rank * kWarps + warp) * run), r1 = min(total, r0 + run);  // this warp's rows
  if (tid == 0) {
    s_newest = INT_MIN;
    if (rank == 0 && h == 0) p.left[b] = left;
    if (rank == 0 && all) p.count[list] = 0;
  }
  auto sync = [&]() {
    if (size == 1) {
      __syncthreads();
    } else {
      __syncwarp();
      asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
  };
  for (int j = tid; j < 3 * kBins / 4; j += kThreads) reinterpret_cast<int4*>(hists)[j] = make_int4(0, 0, 0, 0);

  // a batch: kDeep groups of four rows of this lane
  int at[kDeep];  // their pool rows; -1 past the run and where no page is assigned
  float4 w[kDeep];
  int4 x[kDeep];
  uint4 k[kDeep];
  auto load = [&](Quads& q, bool weights) {
#pragma unroll
    for (int u = 0; u < kDeep; ++u, q.next()) at[u] = q.row < r1 ? q.pool() : -1;
#pragma unroll
    for (int u = 0; u < kDeep; ++u)
      if (at[u] >= 0) {
        x[u] = *reinterpret_cast<const int4*>(p.position + at[u]);
        if (weights) w[u] = *reinterpret_cast<const float4*>(p.weight + at[u]);
      }
  };
  // the weights and positions of the first rows into their output (rows that move
  // overwrite theirs afterwards)
  const bool copy_w = p.weight_out != p.weight, copy_p = p.position_out != p.position;
  auto copy = [&](int first) {
    if (!copy_w && !copy_p) return;
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const int i = first + u * 128;
      if (i >= left || at[u] < 0) continue;
      if (i + 4 <= left) {
        if (copy_w) *reinterpret_cast<float4*>(p.weight_out + at[u]) = w[u];
        if (copy_p) *reinterpret_cast<int4*>(p.position_out + at[u]) = x[u];
      } else {
        for (int j = 0; j < left - i; ++j) {
          if (copy_w) p.weight_out[at[u] + j] = p.weight[at[u] + j];
          if (copy_p) p.position_out[at[u] + j] = p.position[at[u] + j];
        }
      }
    }
  };
  if (kOnce) {
    Quads q(p, b, h, r0 + lane * 4);
    load(q, true);
    copy(r0 + lane * 4);
  }
  sync();

  if (!all && p.recent > 0) {
    int newest = INT_MIN;
    Quads q(p, b, h, r0 + lane * 4);
    for (int i0 = r0; i0 < r1; i0 += kDeep * 128) {
      if (!kOnce) load(q, false);
#pragma unroll
      for (int u = 0; u < kDeep; ++u) {
        if (at[u] < 0) continue;
        const int n = r1 - (i0 + u * 128 + lane * 4);  // at least one
        newest = max(newest, x[u].x);
        if (n > 1) newest = max(newest, x[u].y);
        if (n > 2) newest = max(newest, x[u].z);
        if (n > 3) newest = max(newest, x[u].w);
      }
    }
    newest = __reduce_max_sync(0xffffffffu, newest);
    if (lane == 0) atomicMax(&s_newest, newest);
    sync();
  }
  int newest = s_newest;
  if (!all && p.recent > 0)
    for (int r = 1; r < size; ++r) newest = max(newest, *cluster_peer(&s_newest, (rank + r) % size));
  // positions above this are among the newest (no position is above INT_MAX)
  const int guard = p.recent == 0 ? INT_MAX : newest < INT_MIN + p.recent ? INT_MIN : newest - p.recent;
  auto to_keys = [&](int first) {
    auto key = [&](float wt, int pos) -> uint32_t {
      return pos < p.sink || pos > guard ? 0xFFFFFFFFu : weight_key(wt);
    };
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      if (at[u] >= 0) {
        k[u] = make_uint4(key(w[u].x, x[u].x), key(w[u].y, x[u].y), key(w[u].z, x[u].z), key(w[u].w, x[u].w));
      } else {
        const int i = left - (first + u * 128);
        k[u] = make_uint4(i > 0 ? ~0u : 0u, i > 1 ? ~0u : 0u, i > 2 ? ~0u : 0u, i > 3 ? ~0u : 0u);
      }
    }
  };
  // f(u, i) for every group of the run, its first row i, with k[u] and at[u]
  auto each_batch = [&](auto f) {
    Quads q(p, b, h, r0 + lane * 4);
    for (int i0 = r0; i0 < r1; i0 += kDeep * 128) {
      if (!kOnce) {
        load(q, true);
        to_keys(i0 + lane * 4);
      }
      f(i0 + lane * 4);
    }
  };
  if (kOnce) to_keys(r0 + lane * 4);

  // the first digit's histogram
  const uint32_t kZero = weight_key(0.f);
  int zeros = 0, guarded = 0;
  each_batch([&](int first) {
    if (!kOnce) copy(first);
    if (all) return;
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const int i = first + u * 128;
      auto count = [&](uint32_t key, bool take) {
        if (!take) return;
        if (key == kZero)
          ++zeros;
        else if (key == 0xFFFFFFFFu)
          ++guarded;
        else
          atomicAdd(&hists[0][key >> 21], 1);
      };
      count(k[u].x, i < r1);
      count(k[u].y, i + 1 < r1);
      count(k[u].z, i + 2 < r1);
      count(k[u].w, i + 3 < r1);
    }
  });
  if (all) {  // the whole cluster returns
    pdl_launch_dependents();
    return;
  }
  add_shared(&hists[0][kZero >> 21], zeros, lane);
  add_shared(&hists[0][kBins - 1], guarded, lane);
  // the cluster's counts into the first CTA's histogram; few digits occur, so few have to go
  auto merge = [&](int* hist) {
    if (size > 1) {
      __syncthreads();
      if (rank > 0)
        for (int j = tid; j < kBins; j += kThreads)
          if (const int n = hist[j]) atomicAdd(cluster_peer(hist, 0) + j, n);
    }
    sync();
  };
  merge(hists[0]);

  // of one value a warp: the sum up to the warp before this one's, and of all
  auto warps_before = [&](const int* v, int* sum) -> int {
    const int upto = warp_scan(lane < kWarps ? v[lane] : 0, lane);
    *sum = __shfl_sync(0xffffffffu, upto, 31);
    return warp ? __shfl_sync(0xffffffffu, upto, warp - 1) : 0;
  };
  uint32_t prefix = 0;  // the smallest kept key's leading digits
  int need = left;      // rows that stay among those with these digits
#pragma unroll 1
  for (int step = 0; step < 3; ++step) {
    int* hist = hists[step];
    if (step > 0) {
      const int shift = step == 1 ? 10 : 0, up = step == 1 ? 21 : 10;
      const uint32_t mask = step == 1 ? 2047u : 1023u;
      int lowest = 0;
      each_batch([&](int first) {
#pragma unroll
        for (int u = 0; u < kDeep; ++u) {
          const int i = first + u * 128;
          auto count = [&](uint32_t key, bool take) {
            if (!take || (key >> up) != prefix) return;
            const uint32_t digit = (key >> shift) & mask;
            if (digit == 0)
              ++lowest;
            else
              atomicAdd(&hist[digit], 1);
          };
          count(k[u].x, i < r1);
          count(k[u].y, i + 1 < r1);
          count(k[u].z, i + 2 < r1);
          count(k[u].w, i + 3 < r1);
        }
      });
      __syncwarp();
      add_shared(&hist[0], lowest, lane);
      merge(hist);
    }
    // falling digits, kMine to a thread
    int n[kMine], sum = 0, all_of;
    const int* merged = (size > 1 ? cluster_peer(hist, 0) : hist) + kBins - kMine * (tid + 1);
#pragma unroll
    for (int j = 0; j < kMine; j += 2) {
      const int2 two = *reinterpret_cast<const int2*>(merged + j);
      n[kMine - 1 - j] = two.x;
      n[kMine - 2 - j] = two.y;
    }
#pragma unroll
    for (int j = 0; j < kMine; ++j) sum += n[j];
    const int mine = warp_scan(sum, lane);
    if (lane == 31) part[0][warp] = mine;
    __syncthreads();
    int above = warps_before(part[0], &all_of) + mine - sum;
#pragma unroll
    for (int j = 0; j < kMine; ++j) {
      if (above < need && need <= above + n[j]) {
        s_prefix = (prefix << (step == 2 ? 10 : 11)) | (uint32_t)(kBins - 1 - kMine * tid - j);
        s_need = need - above;
        s_among = n[j];
      }
      above += n[j];
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
    if (s_among == need) {  // all of them stay, whatever their other digits
      prefix <<= step == 0 ? 21 : step == 1 ? 10 : 0;
      break;
    }
  }

  // A key above prefix stays, and of the s_among ones from it on the first `need` do. Each
  // warp counts in its run, the counts are summed up, then it writes.
  const bool ties = s_among != need;  // some of the rows whose key is prefix go
  int gt[2] = {0, 0}, eq[2] = {0, 0};  // rows above prefix and with it, below `left` and from it on
  each_batch([&](int first) {
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const int i = first + u * 128;
      const uint32_t kk[4] = {k[u].x, k[u].y, k[u].z, k[u].w};
      const uint32_t low = (1u << min(max(left - i, 0), 4)) - 1u, in = (1u << min(max(r1 - i, 0), 4)) - 1u;
      uint32_t more = 0, same = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        more |= (kk[j] > prefix ? 1u : 0u) << j;
        same |= (kk[j] == prefix ? 1u : 0u) << j;
      }
      gt[0] += __popc(more & in & low);
      gt[1] += __popc(more & in & ~low);
      eq[0] += __popc(same & in & low);
      eq[1] += __popc(same & in & ~low);
    }
  });
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    gt[s] = __reduce_add_sync(0xffffffffu, gt[s]);
    eq[s] = __reduce_add_sync(0xffffffffu, eq[s]);
  }
  // of part[v] .. part[last], one value a warp: the sums up to this warp's, over the CTAs
  // before this one too, and of all
  auto before = [&](int v, int last, int* upto, int* of_all) {
    for (int j = v; j <= last; ++j) {
      upto[j - v] = warps_before(part[j], &of_all[j - v]);
      if (size > 1 && tid == 0) s_sum[j] = of_all[j - v];
    }
    if (size == 1) return;
    sync();
    for (int j = v; j <= last; ++j) {
      of_all[j - v] = 0;
      for (int r = 0; r < size; ++r) {
        const int theirs = *cluster_peer(&s_sum[j], r);
        if (r < rank) upto[j - v] += theirs;
        of_all[j - v] += theirs;
      }
    }
  };
  int eq_at = 0;
  if (ties) {
    if (lane == 0) part[0][warp] = eq[0] + eq[1];
    __syncthreads();
    int all_of;
    before(0, 0, &eq_at, &all_of);
    eq[1] = min(max(need - eq_at - eq[0], 0), eq[1]);
    eq[0] = min(max(need - eq_at, 0), eq[0]);
  }
  // a place that falls free below `left` and a row that moves down there are counted together
  if (lane == 0) {
    part[1][warp] = max(min(r1, left) - r0, 0) - gt[0] - eq[0];
    part[2][warp] = gt[1] + eq[1];
  }
  __syncthreads();
  int upto[2], of_all[2];  // equally many of both
  before(1, 2, upto, of_all);
  int hole_at = upto[0], out_at = upto[1];
  if (tid == 0 && rank == 0) p.count[list] = of_all[1];
  int32_t* to = p.to + (size_t)list * p.max_moves;
  int32_t* src = p.src + (size_t)list * p.max_moves;
  each_batch([&](int first) {
    uint32_t hole[kDeep], out[kDeep];  // a bit for each row
    int upto[kDeep];
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const int i = first + u * 128;
      const uint32_t kk[4] = {k[u].x, k[u].y, k[u].z, k[u].w};
      const uint32_t low = (1u << min(max(left - i, 0), 4)) - 1u, in = (1u << min(max(r1 - i, 0), 4)) - 1u;
      uint32_t kept = 0;
      if (ties) {
        uint32_t same = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) same |= (kk[j] == prefix ? 1u : 0u) << j;
        same &= in;
        const int n = __popc(same), before_me = warp_scan(n, lane);
        int left_of = need - (eq_at + before_me - n);  // how many of the equal rows from here on stay
        eq_at += __shfl_sync(0xffffffffu, before_me, 31);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (kk[j] > prefix || ((same >> j & 1) && left_of > 0)) kept |= 1u << j;
          left_of -= same >> j & 1;
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) kept |= (kk[j] >= prefix ? 1u : 0u) << j;
      }
      hole[u] = low & in & ~kept;
      out[u] = ~low & in & kept;
      upto[u] = warp_scan(__popc(hole[u]) + (__popc(out[u]) << 16), lane);
    }
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const int mine = upto[u] - (__popc(hole[u]) + (__popc(out[u]) << 16));
      const int sum = __shfl_sync(0xffffffffu, upto[u], 31);
      int hole_to = hole_at + (mine & 0xFFFF), out_to = out_at + (mine >> 16);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (hole[u] >> j & 1) to[hole_to++] = at[u] + j;
        if (out[u] >> j & 1) src[out_to++] = at[u] + j;
      }
      hole_at += sum & 0xFFFF;
      out_at += sum >> 16;
    }
  });
  if (size > 1) sync();  // no CTA leaves while another may read its sums
  pdl_launch_dependents();
}

constexpr int kMoveWarps = 8;
constexpr int kMoveRows = 8;  // rows that a warp has in flight
constexpr int kMovePiece = kMoveWarps * kMoveRows;

// Eight rows to a warp at a time: half of it copies the key rows, half the value rows,
// 16 bytes a lane; the next eight are looked up meanwhile. The lists' pieces of 64 rows
// are dealt out to the CTAs one list after another, so that lists of unequal length spread.
__global__ void __launch_bounds__(kMoveWarps * 32, 4)
    paged_move_kernel(const __grid_constant__ PagedEvictParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31, mine = (threadIdx.x >> 5) * kMoveRows + lane;
  const int lists = p.n_seqs * p.n_kv;
  for (int b = blockIdx.x * kMoveWarps * 32 + threadIdx.x; b < p.n_seqs; b += gridDim.x * kMoveWarps * 32)
    p.lens_out[b] = p.left[b];
  uint4* pool = reinterpret_cast<uint4*>(lane < 16 ? p.k : p.v) + (lane & 15);
  const int step_list = gridDim.x % lists, step_row = gridDim.x / lists * kMovePiece;
  int list = blockIdx.x % lists, row = blockIdx.x / lists * kMovePiece;
  auto fetch = [&](int& from, int& at) {  // the next rows of the warp, one to a lane
    from = at = -1;
    if (lane < kMoveRows && row + mine < p.max_moves && row + mine < p.count[list]) {
      from = p.src[(size_t)list * p.max_moves + row + mine];
      at = p.to[(size_t)list * p.max_moves + row + mine];
    }
    list += step_list;
    row += step_row;
    if (list >= lists) {
      list -= lists;
      row += kMovePiece;
    }
  };
  int from, at, from1, at1;
  bool more = row < p.max_moves;
  for (fetch(from, at); more; from = from1, at = at1) {
    more = row < p.max_moves;
    uint4 x[kMoveRows];
    float w;
    int pos;
    if (at >= 0) {
      w = p.weight[from];
      pos = p.position[from];
    }
#pragma unroll
    for (int j = 0; j < kMoveRows; ++j) {
      const int f = __shfl_sync(0xffffffffu, from, j);
      if (f >= 0) x[j] = ld_stream_u4(pool + (size_t)f * (kD / 8));  // no row is both read and written
    }
    fetch(from1, at1);
    if (at >= 0) {
      p.weight_out[at] = w;
      p.position_out[at] = pos;
    }
#pragma unroll
    for (int j = 0; j < kMoveRows; ++j) {
      const int t = __shfl_sync(0xffffffffu, at, j);
      if (t >= 0) __stcs(pool + (size_t)t * (kD / 8), x[j]);
    }
  }
  pdl_launch_dependents();
}

template <typename... A>
cudaError_t launch(void (*kernel)(A...), int grid, int threads, size_t smem, int cluster, cudaStream_t stream,
                   A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.dynamicSmemBytes = smem;
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

cudaError_t launch_paged_write(const PagedWriteParams& p, int sms, bool f16, cudaStream_t stream) {
  // 24 heads to a warp, eight at a time, once that gives the SMs some warps each (8188 tokens
  // of 48 heads with norm: 41 us, 45 with eight heads to a warp); until then two
  // (64 tokens: 2.6 us, 4.5 with eight)
  const int heads = p.n_head + 2 * p.n_kv;
  const bool many = (long long)p.n_tokens * heads >= 64LL * sms;
  const long long warps = (long long)p.n_tokens * (many ? (heads + 23) / 24 : (heads + 1) / 2);
  const int grid = (int)((warps + kWriteWarps - 1) / kWriteWarps);
  auto kernel = many ? (f16 ? paged_write_kernel<4, 3, true> : paged_write_kernel<4, 3, false>)
                     : (f16 ? paged_write_kernel<1, 1, true> : paged_write_kernel<1, 1, false>);
  return launch(kernel, grid, kWriteWarps * 32, 0, 1, stream, p);
}

void paged_evict_plan(int n_seqs, int n_kv, long long max_rows, int budget, PagedEvictPlan* plan) {
  const long long over = max_rows > budget ? max_rows - budget : 0;
  plan->max_moves = (int)(over < budget ? over : budget);
  size_t at = up256((size_t)n_seqs * n_kv * sizeof(int));
  plan->left = at;
  at += up256((size_t)n_seqs * sizeof(int));
  plan->to = at;
  at += up256((size_t)n_seqs * n_kv * plan->max_moves * sizeof(int32_t));
  plan->src = at;
  at += up256((size_t)n_seqs * n_kv * plan->max_moves * sizeof(int32_t));
  plan->bytes = at;
}

cudaError_t launch_paged_evict(const PagedEvictParams& p, int sms, cudaStream_t stream) {
  const int lists = p.n_seqs * p.n_kv, cap = p.max_pages * p.page_size;
  // Lists of up to 4096 rows: 8 rows to each of 256 or 512 threads (1 x 4096: 10.3 us, 12.7 with 16
  // rows). Longer ones: 1024 threads with 8 rows, in clusters of up to 8 CTAs, while every list's cluster
  // has SMs of its own (1 x 32768: 29 us, 34 with 16 rows); else 16 rows (8 x 32768: 130 us, 11
  // more with 8), up to 8192 of them to 512 threads (32 x 8192: 127 us, 139 with 1024). Past 131072
  // rows a cluster of 8 reads its list several times.
  auto cluster_for = [&](int rows) {
    int c = 1;
    while (c < 8 && cap > c * rows) c *= 2;
    return c;
  };
  const int c8 = cluster_for(8192), c16 = cluster_for(16384);
  cudaError_t e;
  if (cap <= 2048)
    e = launch(paged_select_kernel<256, 2, true>, lists, 256, 0, 1, stream, p, 1);
  else if (cap <= 4096)
    e = launch(paged_select_kernel<512, 2, true>, lists, 512, 0, 1, stream, p, 1);
  else if (cap <= c8 * 8192 && lists * c8 <= sms)
    e = launch(paged_select_kernel<1024, 2, true>, lists * c8, 1024, 0, c8, stream, p, c8);
  else if (cap <= 8192)
    e = launch(paged_select_kernel<512, 4, true>, lists, 512, 0, 1, stream, p, 1);
  else if (cap <= c16 * 16384)
    e = launch(paged_select_kernel<1024, 4, true>, lists * c16, 1024, 0, c16, stream, p, c16);
  else
    e = launch(paged_select_kernel<1024, 4, false>, lists * c16, 1024, 0, c16, stream, p, c16);
  if (e != cudaSuccess) return e;
  const long long want = (long long)lists * ((p.max_moves + kMovePiece - 1) / kMovePiece);
  const long long most = 4LL * sms;  // all resident
  return launch(paged_move_kernel, (int)(want < 1 ? 1 : want < most ? want : most), kMoveWarps * 32, 0, 1,
                stream, p);
}

}  // namespace nf4b
