// The paged KV cache's other two operators: tokens entering their pages (q/k norm,
// rotary, scatter), and the eviction of the rows that were attended to least.

#include "common.cuh"
#include "kernels.cuh"

namespace nf4b {

namespace {

constexpr int kD = 128;

// ---- write ------------------------------------------------------------------
// One warp for each head of each token, four dimensions to a lane (two rotary
// pairs). The arithmetic is qk_rope_kv_kernel's, rounding point for rounding point
// (the norm's sum of squares in fp64 is exact in any order), so a row in a page has
// the bits it would have in a dense cache.
constexpr int kWriteWarps = 8;

template <bool F16>
__global__ void __launch_bounds__(kWriteWarps * 32) paged_write_kernel(const __grid_constant__ PagedWriteParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int heads = p.n_head + 2 * p.n_kv;
  const long long total = (long long)p.n_tokens * heads;
  for (long long item = (long long)blockIdx.x * kWriteWarps + (threadIdx.x >> 5); item < total;
       item += (long long)gridDim.x * kWriteWarps) {
    const int tok = (int)(item / heads), head = (int)(item - (long long)tok * heads);
    const bool is_q = head < p.n_head, is_v = head >= p.n_head + p.n_kv;
    const int pos = p.positions[tok];
    const bool turned = pos >= 0 && pos < p.freqs_rows;  // else the token is padding
    const uint2 in = *reinterpret_cast<const uint2*>(p.qkv + item * kD + lane * 4);
    uint2 out = in;
    if (!is_v) {
      float x[4] = {act_lo<F16>(in.x), act_hi<F16>(in.x), act_lo<F16>(in.y), act_hi<F16>(in.y)};
      const uint16_t* w = is_q ? p.qw : p.kw;
      if (w != nullptr) {
        double ss = 0.0;
#pragma unroll
        for (int i = 0; i < 4; ++i) ss += (double)x[i] * (double)x[i];
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, off);
        const float r = rsqrt_exact(ss, kD, p.eps);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[i] = round_act<F16>(__fmul_rn(__fmul_rn(x[i], r), act2f<F16>(w[lane * 4 + i])));
      }
      if (turned) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          const long long fi = (long long)pos * kD + lane * 4 + i;
          const float c = load_freq(p.freqs, fi, p.ftype), sn = load_freq(p.freqs, fi + 1, p.ftype);
          y[i] = __fsub_rn(__fmul_rn(x[i], c), __fmul_rn(x[i + 1], sn));
          y[i + 1] = __fadd_rn(__fmul_rn(x[i + 1], c), __fmul_rn(x[i], sn));
        }
        out = make_uint2(pack_act2<F16>(y[0], y[1]), pack_act2<F16>(y[2], y[3]));
      } else {
        out = make_uint2(0, 0);
      }
    }
    if (is_q) {
      *reinterpret_cast<uint2*>(p.q_out + ((size_t)tok * p.n_head + head) * kD + lane * 4) = out;
      continue;
    }
    const int seq = p.seqs == nullptr ? tok : p.seqs[tok], row = p.rows[tok];
    if (!turned || row < 0 || row / p.page_size >= p.max_pages || seq < 0 || seq >= p.n_seqs) continue;
    const int pg = p.table[(size_t)seq * p.max_pages + row / p.page_size];
    if (pg < 0 || pg >= p.n_pages) continue;
    const int kh = head - p.n_head - (is_v ? p.n_kv : 0);
    const size_t at = ((size_t)pg * p.n_kv + kh) * p.page_size + row % p.page_size;
    *reinterpret_cast<uint2*>((is_v ? p.v : p.k) + at * kD + lane * 4) = out;
    if (!is_v && lane == 0) {
      if (p.weight != nullptr) p.weight[at] = 0.f;
      if (p.position != nullptr) p.position[at] = pos;
    }
  }
  pdl_launch_dependents();
}

// ---- evict ------------------------------------------------------------------
// Of each (sequence, KV head) the first `left` = min(rows, budget) rows in this
// order stay: rows whose position is below `sink` or among the `recent` newest
// first, then by falling weight (NaN as -inf), equal ones by rising row. Rows at or
// past `left` that stay move, in order, into the rows below it that do not: there are
// equally many, the two sets are disjoint, and attention does not depend on the order of rows
// (the rotary is in the keys), so nothing else has to move.
//
// paged_select_kernel finds the smallest kept key by four 8-bit steps from the top
// (a histogram each) and lists the moves; paged_move_kernel makes them.
constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;

// Weights in rising order as unsigned integers; 0xFFFFFFFF (no weight maps there,
// NaN being taken as -inf) is for the protected rows.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (!(w == w)) w = -INFINITY;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 as 0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct SelectView {
  const PagedEvictParams& p;
  int b, h;
  __device__ __forceinline__ long long slot(int row) const {  // -1: the row's page is not assigned
    const int pg = p.table[(size_t)b * p.max_pages + row / p.page_size];
    if (pg < 0 || pg >= p.n_pages) return -1;
    return ((long long)pg * p.n_kv + h) * p.page_size + row % p.page_size;
  }
};

__device__ __forceinline__ int block_reduce_max(int v, int* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = __reduce_max_sync(0xffffffffu, v);
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = __reduce_max_sync(0xffffffffu, red[lane]);
  __syncthreads();
  return v;
}

// Exclusive prefix of two counts packed in 16 bits each (at most 1024 of either), and their totals.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* red, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, x, off);
    if (lane >= off) x += o;
  }
  if (lane == 31) red[warp] = x;
  __syncthreads();
  uint32_t y = red[lane];
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t o = __shfl_up_sync(0xffffffffu, y, off);
    if (lane >= off) y += o;
  }
  const uint32_t before = warp ? __shfl_sync(0xffffffffu, y, warp - 1) : 0u;
  *total = __shfl_sync(0xffffffffu, y, 31);
  __syncthreads();
  return before + x - v;
}

__global__ void __launch_bounds__(kSelThreads) paged_select_kernel(const __grid_constant__ PagedEvictParams p) {
  __shared__ int hist[256];
  __shared__ int red[kSelWarps];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  static_assert(kSelWarps == 32, "the block reductions read one value a lane");
  pdl_wait();
  const int tid = threadIdx.x;
  const int b = blockIdx.x / p.n_kv, h = blockIdx.x - b * p.n_kv;
  const SelectView view{p, b, h};
  const int cap = p.max_pages * p.page_size;
  const int rows = min(max(p.lens[b], 0), cap), left = min(rows, p.budget);
  if (tid == 0) {
    p.count[blockIdx.x] = 0;
    if (h == 0) p.left[b] = left;
  }
  const bool copied = p.weight_out != p.weight || p.position_out != p.position;
  if (rows <= p.budget) {  // all stay
    if (copied)
      for (int i = tid; i < rows; i += kSelThreads) {
        const long long at = view.slot(i);
        if (at < 0) continue;
        p.weight_out[at] = p.weight[at];
        p.position_out[at] = p.position[at];
      }
    pdl_launch_dependents();
    return;
  }
  int newest = -1;
  if (p.recent > 0) {
    for (int i = tid; i < rows; i += kSelThreads) {
      const long long at = view.slot(i);
      if (at >= 0) newest = max(newest, p.position[at]);
    }
    newest = block_reduce_max(newest, red);
  }
  auto key = [&](int row) -> uint32_t {
    const long long at = view.slot(row);
    if (at < 0) return 0u;
    const int pos = p.position[at];
    if (pos < p.sink || (p.recent > 0 && (long long)pos > (long long)newest - p.recent)) return 0xFFFFFFFFu;
    return weight_key(p.weight[at]);
  };
  uint32_t prefix = 0;  // the smallest kept key's leading digits
  int need = left;      // rows of the remaining candidates that stay
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < rows; i += kSelThreads) {
      const uint32_t k = key(i);
      if (shift == 24 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255u], 1);
    }
    __syncthreads();
    if (tid < 32) {  // lane l: digits 255 - 8 l down to 248 - 8 l
      int n = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) n += hist[255 - tid * 8 - i];
      int x = n;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, x, off);
        if (tid >= off) x += o;
      }
      int above = x - n;
      if (above < need && need <= x) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int digit = 255 - tid * 8 - i;
          if (above < need && need <= above + hist[digit]) {
            s_prefix = (prefix << 8) | (uint32_t)digit;
            s_need = need - above;
          }
          above += hist[digit];
        }
      }
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
    __syncthreads();
  }
  // key > prefix stays; of those equal to it the first `need` do
  uint32_t* ured = reinterpret_cast<uint32_t*>(red);
  int equal = 0, holes = 0, moved = 0;
  int32_t* to = p.to + (size_t)blockIdx.x * p.max_moves;
  int32_t* src = p.src + (size_t)blockIdx.x * p.max_moves;
  for (int i0 = 0; i0 < rows; i0 += kSelThreads) {
    const int i = i0 + tid;
    const uint32_t k = i < rows ? key(i) : 0u;
    uint32_t total;
    const bool eq = i < rows && k == prefix;
    const int rank = equal + (int)block_scan(eq ? 1u : 0u, ured, &total);
    equal += (int)total;
    const bool kept = i < rows && (k > prefix || (eq && rank < need));
    const bool hole = i < left && !kept, out = i >= left && kept;
    const uint32_t at = block_scan((hole ? 1u : 0u) | (out ? 0x10000u : 0u), ured, &total);
    if (hole) to[holes + (int)(at & 0xFFFFu)] = i;
    if (out) src[moved + (int)(at >> 16)] = i;
    holes += (int)(total & 0xFFFFu);
    moved += (int)(total >> 16);
    if (copied && kept && i < left) {
      const long long s = view.slot(i);
      if (s >= 0) {
        p.weight_out[s] = p.weight[s];
        p.position_out[s] = p.position[s];
      }
    }
  }
  if (tid == 0) p.count[blockIdx.x] = moved;
  pdl_launch_dependents();
}

constexpr int kMoveWarps = 8;

// One warp a row: half of it copies the key row, half the value row, 16 bytes a lane.
__global__ void __launch_bounds__(kMoveWarps * 32) paged_move_kernel(const __grid_constant__ PagedEvictParams p) {
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int b = blockIdx.y / p.n_kv, h = blockIdx.y - b * p.n_kv;
  const SelectView view{p, b, h};
  if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0) p.lens_out[b] = p.left[b];
  const int n = p.count[blockIdx.y];
  const int32_t* to = p.to + (size_t)blockIdx.y * p.max_moves;
  const int32_t* src = p.src + (size_t)blockIdx.y * p.max_moves;
  for (int i = blockIdx.x * kMoveWarps + warp; i < n; i += gridDim.x * kMoveWarps) {
    const long long from = view.slot(src[i]), at = view.slot(to[i]);
    if (from < 0 || at < 0) continue;
    uint16_t* pool = lane < 16 ? p.k : p.v;
    reinterpret_cast<uint4*>(pool + at * kD)[lane & 15] = reinterpret_cast<const uint4*>(pool + from * kD)[lane & 15];
    if (lane == 0) {
      p.weight_out[at] = p.weight[from];
      p.position_out[at] = p.position[from];
    }
  }
  pdl_launch_dependents();
}

template <typename P>
cudaError_t launch(void (*kernel)(P), dim3 grid, int threads, const P& p, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

cudaError_t launch_paged_write(const PagedWriteParams& p, int sms, bool f16, cudaStream_t stream) {
  const long long items = (long long)p.n_tokens * (p.n_head + 2 * p.n_kv);
  const long long want = (items + kWriteWarps - 1) / kWriteWarps, most = 16LL * sms;
  return launch(f16 ? paged_write_kernel<true> : paged_write_kernel<false>, dim3((unsigned)(want < most ? want : most)),
                kWriteWarps * 32, p, stream);
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
  const int lists = p.n_seqs * p.n_kv;
  cudaError_t e = launch(paged_select_kernel, dim3((unsigned)lists), kSelThreads, p, stream);
  if (e != cudaSuccess) return e;
  long long x = (p.max_moves + kMoveWarps - 1) / kMoveWarps;
  const long long most = (8LL * sms + lists - 1) / lists;
  x = x > most ? most : x < 1 ? 1 : x;
  return launch(paged_move_kernel, dim3((unsigned)x, (unsigned)lists), kMoveWarps * 32, p, stream);
}

}  // namespace nf4b
