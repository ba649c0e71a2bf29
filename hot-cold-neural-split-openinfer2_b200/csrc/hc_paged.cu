// Paged 8-bit key/value cache: block tables and slot maps from request
// lengths, rotary positions, and the write of a step's keys and values.
//
// A page holds page_size tokens of every key-value head,
// [n_kv_heads][page_size][head_dim] e4m3 bytes, with one power-of-two scale
// per page and head: value = byte * scale.  e4m3 is a floating-point format,
// so a power of two costs no precision over absmax / 448; it makes the
// division exact (one rounding in all) and lets a page that grows be rescaled
// without a second rounding, except of values that fall among the format's
// subnormals.
#include <cooperative_groups.h>

#include <type_traits>

#include "hc_common.cuh"

namespace hcp {
using namespace hc;
namespace cg = cooperative_groups;

constexpr int MAX_REQ = 2048;           // requests of one step (their offsets sit in shared memory)
constexpr int MAX_ROWS = 1 << 30;       // rows of one call: 32-bit row indices step past the last one by a grid's width
constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_CL = 8;              // CTAs of a plan with many rows (one cluster)

// ---------------------------------------------------------------------------
// page plan
// ---------------------------------------------------------------------------
struct PlanArgs {
  const int32_t* starts;
  const int32_t* q_lens;
  int n_req;
  int32_t* tables;
  int64_t stride;
  int width;
  const int32_t* free_pages;
  int n_pages;
  int32_t* n_free;
  int page_size, n_rows;
  int32_t* cu_q;
  int32_t* kv_lens;
  int64_t* positions;
  int64_t* slots;
  int32_t* status;
};

// inclusive sums of two values over the block (1024 threads)
__device__ __forceinline__ void block_scan2(int64_t& a, int64_t& b, int64_t (*wsum)[2]) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
  if (lane == 31) {
    wsum[w][0] = a;
    wsum[w][1] = b;
  }
  __syncthreads();
  if (w == 0) {
    int64_t x = wsum[lane][0], y = wsum[lane][1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t p = __shfl_up_sync(0xffffffffu, x, o), q = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) {
        x += p;
        y += q;
      }
    }
    wsum[lane][0] = x;
    wsum[lane][1] = y;
  }
  __syncthreads();
  if (w > 0) {
    a += wsum[w - 1][0];
    b += wsum[w - 1][1];
  }
}

// first negative entry of row[lo..hi), whose filled entries form a prefix; hi if there is none
__device__ __forceinline__ int first_missing(const int32_t* row, int lo, int hi) {
  if (lo >= hi) return hi;
  const int32_t a = row[lo], b = row[hi - 1];
  if (a < 0) return lo;
  if (b >= 0) return hi;
  while (hi - lo > 1) {                 // row[lo] filled, row[hi - 1] missing
    const int mid = lo + (hi - lo) / 2;
    if (row[mid] < 0) hi = mid;
    else lo = mid;
  }
  return hi;
}

// largest i in [0, n) with first[i] <= x (first[0] = 0, ascending)
__device__ __forceinline__ int owner(const int32_t* first, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Every CTA of the cluster computes the same two prefix sums over the requests
// (new rows, pages to take), so nothing is exchanged; a cluster barrier keeps
// the tables and the free count unchanged until every CTA has read them.
// 8 n_req + 16 n_rows bytes, bound by latency (launch, lengths, scans, tables):
// 64 requests of one token 4.3 us in a graph, 256 prompts of 33,000 rows 10.4 us
// (in one CTA the rows alone took 24).
__global__ void __launch_bounds__(PLAN_THREADS) page_plan_kernel(const PlanArgs p) {
  __shared__ int32_t s_cu[MAX_REQ + 1], s_take[MAX_REQ + 1], s_first[MAX_REQ], s_start[MAX_REQ];
  __shared__ int64_t wsum[32][2];
  __shared__ int s_bad;
  cg::cluster_group cluster = cg::this_cluster();
  const int t = threadIdx.x, ncta = gridDim.x, cta = blockIdx.x;
  const int per = (p.n_req + PLAN_THREADS - 1) / PLAN_THREADS;       // 1 or 2 requests a thread
  const int n_free = *p.n_free;
  if (t == 0) s_bad = n_free < 0 || n_free > p.n_pages;
  __syncthreads();
  int64_t rows = 0, take = 0;
  bool bad = false;
  for (int i = 0; i < per; ++i) {
    const int r = t * per + i;
    if (r >= p.n_req) break;
    const int start = p.starts[r], q = p.q_lens[r];
    const int64_t end = (int64_t)start + q;
    int first = 0, miss = 0;
    if (start < 0 || q < 0 || end > (int64_t)p.width * p.page_size) {
      bad = true;
    } else {
      const int lo = start / p.page_size, hi = q ? ((int)end - 1) / p.page_size + 1 : lo;
      first = first_missing(p.tables + r * p.stride, lo, hi);
      miss = hi - first;
      rows += q;
      take += miss;
    }
    s_start[r] = start;
    s_first[r] = first;
    s_cu[r] = q;                      // lengths for now
    s_take[r] = miss;
  }
  if (bad) s_bad = 1;
  int64_t rows_in = rows, take_in = take;
  block_scan2(rows_in, take_in, wsum);
  const int64_t total_rows = wsum[31][0], total_take = wsum[31][1];
  bad = s_bad || total_rows > p.n_rows || total_take > n_free;
  if (!bad) {
    int64_t a = rows_in - rows, b = take_in - take;
    for (int i = 0; i < per; ++i) {
      const int r = t * per + i;
      if (r >= p.n_req) break;
      const int q = s_cu[r], m = s_take[r];
      s_cu[r] = (int32_t)a;
      s_take[r] = (int32_t)b;
      a += q;
      b += m;
    }
  }
  if (t == 0 && !bad) {
    s_cu[p.n_req] = (int32_t)total_rows;
    s_take[p.n_req] = (int32_t)total_take;
  }
  __syncthreads();
  if (ncta > 1) cluster.sync();       // every CTA has read what is written below
  const int lane0 = cta * PLAN_THREADS + t, lanes = ncta * PLAN_THREADS;
  if (bad) {                          // nothing allocated, no rows
    if (lane0 == 0 && p.status) atomicOr(p.status, HC_ERR_RANGE);
    for (int r = lane0; r <= p.n_req; r += lanes) {
      p.cu_q[r] = 0;
      if (r < p.n_req) p.kv_lens[r] = p.starts[r];
    }
    for (int i = lane0; i < p.n_rows; i += lanes) {
      p.positions[i] = -1;
      p.slots[i] = -1;
    }
    return;
  }
  for (int r = lane0; r <= p.n_req; r += lanes) {
    p.cu_q[r] = s_cu[r];
    if (r < p.n_req) p.kv_lens[r] = s_start[r] + s_cu[r + 1] - s_cu[r];
  }
  bool stray = false;
  for (int m = lane0; m < (int)total_take; m += lanes) {
    const int r = owner(s_take, p.n_req, m);
    const int32_t page = p.free_pages[n_free - 1 - m];
    stray |= page < 0 || page >= p.n_pages;
    p.tables[r * p.stride + s_first[r] + m - s_take[r]] = page;
  }
  for (int i = lane0; i < p.n_rows; i += lanes) {
    int64_t pos = -1, slot = -1;
    if (i < (int)total_rows) {
      const int r = owner(s_cu, p.n_req, i);
      const int at = s_start[r] + (i - s_cu[r]);
      const int pg = at / p.page_size;
      pos = at;
      const int32_t page = pg < s_first[r] ? p.tables[r * p.stride + pg]
                                           : p.free_pages[n_free - 1 - (s_take[r] + pg - s_first[r])];
      if (page < 0 || page >= p.n_pages) stray = true;
      else slot = (int64_t)page * p.page_size + at % p.page_size;
    }
    p.positions[i] = pos;
    p.slots[i] = slot;
  }
  if (stray && p.status) atomicOr(p.status, HC_ERR_RANGE);
  if (lane0 == 0) *p.n_free = n_free - (int)total_take;
}

struct ReleaseArgs {
  const uint8_t* done;
  int n_req;
  int32_t* tables;
  int64_t stride;
  int width;
  int32_t* free_pages;
  int n_pages;
  int32_t* n_free;
  int32_t* status;
};

// The pages of the finished requests go back onto the stack, request order
// then page order.  Their rows are read whole, by as many warps each as there
// are for so few rows: a search for the end of the prefix would miss a page
// behind a hole.  One CTA, bound by latency like the plan: a serving step
// releases a few requests.
__global__ void __launch_bounds__(PLAN_THREADS) page_release_kernel(const ReleaseArgs p) {
  __shared__ int32_t s_put[MAX_REQ], s_end[MAX_REQ], s_done[MAX_REQ];
  __shared__ int64_t wsum[32][2];
  __shared__ int s_bad;
  constexpr int WARPS = PLAN_THREADS / 32;
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int per = (p.n_req + PLAN_THREADS - 1) / PLAN_THREADS;
  const int n_free = *p.n_free;
  if (t == 0) s_bad = n_free < 0 || n_free > p.n_pages;
  // the finished requests, in order
  int64_t mine = 0, unused = 0;
  for (int i = 0; i < per; ++i) {
    const int r = t * per + i;
    if (r >= p.n_req) break;
    s_put[r] = s_end[r] = 0;
    mine += p.done[r] != 0;
  }
  int64_t upto = mine;
  block_scan2(upto, unused, wsum);
  const int n_done = (int)wsum[31][0];
  for (int i = 0, at = (int)(upto - mine); i < per; ++i) {
    const int r = t * per + i;
    if (r < p.n_req && p.done[r]) s_done[at++] = r;
  }
  __syncthreads();
  // filled entries of their rows, and where the last one ends
  int share = WARPS;                  // warps of a row
  while (share > 1 && share * n_done > WARPS) share /= 2;
  for (int i = w / share; i < n_done; i += WARPS / share) {
    const int r = s_done[i];
    const int32_t* row = p.tables + r * p.stride;
#pragma unroll 4
    for (unsigned at = w % share * 32; at < (unsigned)p.width; at += share * 32) {
      const int32_t page = at + lane < (unsigned)p.width ? row[at + lane] : -1;
      const uint32_t filled = __ballot_sync(0xffffffffu, page >= 0);
      if (page >= p.n_pages) s_bad = 1;
      if (lane == 0 && filled) {
        atomicAdd(&s_put[r], __popc(filled));
        atomicMax(&s_end[r], (int)(at + 32 - __clz(filled)));
      }
    }
  }
  __syncthreads();
  int64_t put = 0;
  for (int i = 0; i < per; ++i) {
    const int r = t * per + i;
    if (r >= p.n_req) break;
    if (s_put[r] != s_end[r]) s_bad = 1;                 // a hole
    put += s_put[r];
  }
  int64_t in = put;
  block_scan2(in, unused, wsum);
  const int64_t total = wsum[31][0];
  if (s_bad || n_free + total > p.n_pages) {             // or more pages than there are: nothing is released
    if (t == 0 && p.status) atomicOr(p.status, HC_ERR_RANGE);
    return;
  }
  int64_t a = in - put;
  for (int i = 0; i < per; ++i) {
    const int r = t * per + i;
    if (r >= p.n_req) break;
    const int n = s_put[r];
    s_put[r] = (int32_t)a;
    a += n;
  }
  __syncthreads();
  for (int m = t; m < (int)total; m += PLAN_THREADS) {
    const int r = owner(s_put, p.n_req, m);
    int32_t* at = p.tables + r * p.stride + m - s_put[r];
    p.free_pages[n_free + m] = *at;
    *at = -1;
  }
  if (t == 0) *p.n_free = n_free + (int)total;
}

// ---------------------------------------------------------------------------
// rotary positions
// ---------------------------------------------------------------------------
template <typename T>
struct Num;
template <>
struct Num<__half> {
  static __device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
  static __device__ __forceinline__ __half from_f(float x) { return __float2half_rn(x); }
};
template <>
struct Num<__nv_bfloat16> {
  static __device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
  static __device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }
};

// x c + y s for one output of a pair.  Queries: one fma, rounded.
template <typename T>
__device__ __forceinline__ T turn(T x, T y, float c, float s) {
  return Num<T>::from_f(fmaf(Num<T>::to_f(y), s, Num<T>::to_f(x) * c));
}
// Keys: the same to twice the precision (products split by fma, their sum by
// two-sum), rounded to fp32 and then to T, which equals the 64-bit value
// rounded so.  The 16-bit value decides the byte that the cache holds, which
// then depends on no order of operations.  Conversions to 64 bits and back run
// at a sixteenth of the fp32 rate here, so this costs half of what they do.
// Where fp32 does not hold the sum (or a product, under angles with a factor
// above 1) it stands uncorrected, infinite or NaN as for queries: its error
// terms are inf - inf.
__device__ __forceinline__ float turn_exact(float x, float y, float c, float s) {
  const float p = __fmul_rn(x, c), q = __fmul_rn(y, s);
  const float e = __fmaf_rn(x, c, -p), f = __fmaf_rn(y, s, -q);
  const float r = __fadd_rn(p, q), z = __fsub_rn(r, p);
  const float t = __fadd_rn(__fsub_rn(p, __fsub_rn(r, z)), __fsub_rn(q, z));
  return fabsf(r) < INFINITY ? __fadd_rn(r, __fadd_rn(t, __fadd_rn(e, f))) : r;
}
template <typename T>
__device__ __forceinline__ T turn_key(T x, T y, float c, float s) {
  return Num<T>::from_f(turn_exact(Num<T>::to_f(x), Num<T>::to_f(y), c, s));
}

struct RopeArgs {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int64_t q_row, q_head, k_row, k_head, qo_row, qo_head, ko_row, ko_head;
  const float* cos_t;
  const float* sin_t;
  int64_t table_rows;
  const int64_t* positions;
  int n_rows, nq, nk, dim, rot;       // nk: key heads rotated by rope_rows (0 where they go into the cache)
  int interleaved;
  int slots, rows_cta;                // heads of one row worked on at once; rows of a CTA (vector form)
  int32_t* status;
};

// position of a row: -1 for a row to leave alone (padding, or outside the tables)
__device__ __forceinline__ int64_t checked_pos(const int64_t* positions, int row, int64_t table_rows,
                                               int32_t* status) {
  const int64_t pos = positions[row];
  if (pos >= -1 && pos < table_rows) return pos;
  if (status) atomicOr(status, HC_ERR_RANGE);
  return -1;
}

// Vector form: a unit is 8 pairs (two 16-byte pieces of a head) or 16
// elements that pass through.  A thread keeps its unit's 8 angles and walks
// the row's heads with stride `slots`, four heads' loads in flight at a time.
// HBM-bound: each element read and written once; 8192 rows of 32 + 8 heads
// 34 us, 4.9 TB/s (51 us with one head's loads in flight at a time), one row
// 3.8 us.
template <typename T, bool KEY>
__device__ __forceinline__ void rope_unit(const uint4& av, const uint4& bv, T* dst, int a0, int b0, bool turned,
                                          bool interleaved, const float (&c)[8], const float (&s)[8]) {
  __align__(16) T a[8], b[8], x[8], y[8];
  *reinterpret_cast<uint4*>(a) = av;
  *reinterpret_cast<uint4*>(b) = bv;
  auto go = [](T u, T v, float cc, float ss) { return KEY ? turn_key<T>(u, v, cc, ss) : turn<T>(u, v, cc, ss); };
  if (!turned) {
    *reinterpret_cast<uint4*>(dst + a0) = av;
    *reinterpret_cast<uint4*>(dst + b0) = bv;
    return;
  }
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = go(a[2 * i], a[2 * i + 1], c[i], -s[i]);
      x[2 * i + 1] = go(a[2 * i + 1], a[2 * i], c[i], s[i]);
      y[2 * i] = go(b[2 * i], b[2 * i + 1], c[4 + i], -s[4 + i]);
      y[2 * i + 1] = go(b[2 * i + 1], b[2 * i], c[4 + i], s[4 + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = go(a[i], b[i], c[i], -s[i]);
      y[i] = go(b[i], a[i], c[i], s[i]);
    }
  }
  *reinterpret_cast<uint4*>(dst + a0) = *reinterpret_cast<const uint4*>(x);
  *reinterpret_cast<uint4*>(dst + b0) = *reinterpret_cast<const uint4*>(y);
}

constexpr int BATCH = 4;                // heads of a thread in flight
template <typename T, bool KEY>
__device__ __forceinline__ void rope_heads(const T* src, int64_t src_head, T* dst, int64_t dst_head, int heads,
                                           int slot, int slots, int a0, int b0, bool turned, bool interleaved,
                                           const float (&c)[8], const float (&s)[8]) {
  for (int h0 = slot; h0 < heads; h0 += BATCH * slots) {
    uint4 a[BATCH], b[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int h = min(h0 + k * slots, heads - 1);
      a[k] = *reinterpret_cast<const uint4*>(src + h * src_head + a0);
      b[k] = *reinterpret_cast<const uint4*>(src + h * src_head + b0);
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int h = h0 + k * slots;
      if (h < heads) rope_unit<T, KEY>(a[k], b[k], dst + h * dst_head, a0, b0, turned, interleaved, c, s);
    }
  }
}

template <typename T>
__device__ __forceinline__ void rope_rows_vec(const RopeArgs& p, int block) {
  const unsigned units = p.dim / 16, lanes = units * p.slots;
  const unsigned in = threadIdx.x / lanes, rest = threadIdx.x - in * lanes;
  const unsigned slot = rest / units, u = rest - slot * units;
  const int64_t row = (int64_t)block * p.rows_cta + in;
  if ((int)in >= p.rows_cta || row >= p.n_rows) return;
  const int64_t pos = checked_pos(p.positions, row, p.table_rows, p.status);
  if (pos < 0) return;
  const bool turned = (int)u < p.rot / 16;
  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = s[i] = 0.0f;
  if (turned) {
    const float4* cr = reinterpret_cast<const float4*>(p.cos_t + pos * (p.rot / 2) + 8 * u);
    const float4* sr = reinterpret_cast<const float4*>(p.sin_t + pos * (p.rot / 2) + 8 * u);
    *reinterpret_cast<float4*>(c) = __ldg(cr);
    *reinterpret_cast<float4*>(c + 4) = __ldg(cr + 1);
    *reinterpret_cast<float4*>(s) = __ldg(sr);
    *reinterpret_cast<float4*>(s + 4) = __ldg(sr + 1);
  }
  const bool pairs = p.interleaved || !turned;
  const int a0 = pairs ? 16 * u : 8 * u, b0 = pairs ? 16 * u + 8 : p.rot / 2 + 8 * u;
  const T* q = static_cast<const T*>(p.q) + row * p.q_row;
  T* qo = static_cast<T*>(p.q_out) + row * p.qo_row;
  if (turned || q != qo)
    rope_heads<T, false>(q, p.q_head, qo, p.qo_head, p.nq, slot, p.slots, a0, b0, turned, p.interleaved, c, s);
  const T* k = static_cast<const T*>(p.k) + row * p.k_row;
  T* ko = static_cast<T*>(p.k_out) + row * p.ko_row;
  if (p.nk && (turned || k != ko))
    rope_heads<T, true>(k, p.k_head, ko, p.ko_head, p.nk, slot, p.slots, a0, b0, turned, p.interleaved, c, s);
}

// Any rotary size, stride and alignment: a row a CTA, a thread per pair or
// passing element.  Bound by issue slots (74% busy) and 2-byte accesses: 8192
// rows of 32 + 8 heads with a rotary size of 90 take 105 us, 34 in the form above.
template <typename T>
__device__ __forceinline__ void rope_rows_any(const RopeArgs& p, int block) {
  const int64_t row = block;
  const int half = p.rot / 2, units = half + p.dim - p.rot, heads = p.nq + p.nk;
  const int64_t pos = checked_pos(p.positions, row, p.table_rows, p.status);
  if (pos < 0) return;
  for (unsigned it = threadIdx.x; it < (unsigned)(heads * units); it += blockDim.x) {
    const int h = it / (unsigned)units, u = it - (unsigned)(h * units);
    const bool key = h >= p.nq;
    const T* src = key ? static_cast<const T*>(p.k) + row * p.k_row + (h - p.nq) * p.k_head
                       : static_cast<const T*>(p.q) + row * p.q_row + h * p.q_head;
    T* dst = key ? static_cast<T*>(p.k_out) + row * p.ko_row + (h - p.nq) * p.ko_head
                 : static_cast<T*>(p.q_out) + row * p.qo_row + h * p.qo_head;
    if (u >= half) {
      dst[half + u] = src[half + u];
      continue;
    }
    const int i = p.interleaved ? 2 * u : u, j = p.interleaved ? 2 * u + 1 : u + half;
    const float c = __ldg(p.cos_t + pos * half + u), s = __ldg(p.sin_t + pos * half + u);
    const T a = src[i], b = src[j];
    dst[i] = key ? turn_key<T>(a, b, c, -s) : turn<T>(a, b, c, -s);
    dst[j] = key ? turn_key<T>(b, a, c, s) : turn<T>(b, a, c, s);
  }
}

constexpr int ROPE_THREADS = 256;

template <typename T, bool VEC>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(const RopeArgs p) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if constexpr (VEC) rope_rows_vec<T>(p, blockIdx.x);
  else rope_rows_any<T>(p, blockIdx.x);
}

// ---------------------------------------------------------------------------
// the write of a step's keys and values
// ---------------------------------------------------------------------------
constexpr int E_MIN = -40, E_MAX = 40;  // exponents of a page scale
constexpr float TOP_MAX = 448.0f * (1ll << E_MAX);      // the largest value that a page holds
constexpr int MANY = 16, FEW = 4;       // rows a warp holds at once
// Rows from which the queries get a launch of their own and a warp holds 16.  The host does not know the runs: prompts
// of 1024 rows and more gain (57 against 84 us at 6,444), single rows lose (1023 take 35 us, 1024 take 127).
constexpr int SPLIT_ROWS = 1024;
constexpr int APPEND_THREADS = 256;
constexpr int APPEND_WARPS = APPEND_THREADS / 32;

struct AppendArgs {
  uint8_t* pages[2];                  // keys, values
  float* scales[2];
  int n_pages, n_kv, page_size, page_log2;
  const void* src[2];
  int64_t src_row[2], src_head[2];
  const int64_t* slots;
  int n_rows;
  int seg;                            // rows a CTA looks for runs in
  int wpi;                            // warps of an item (one head's keys or values of a run)
  int beside;                         // runs beside the queries' kernel
  // rotation of the keys (fused form)
  const float* cos_t;
  const float* sin_t;
  int64_t table_rows;
  const int64_t* positions;
  int rot, interleaved;
  int32_t* status;
};

// exponent e of the smallest power of two with x <= 448 * 2^e, x >= 0 finite
__device__ __forceinline__ int scale_exponent(float x) {
  const uint32_t b = __float_as_uint(x);
  if (b < 0x00800000u) return E_MIN;                 // zero and subnormals
  // x = m 2^k with m in [1, 2); 448 = 1.75 * 2^8
  const int k = (int)(b >> 23) - 127;
  const int e = k - 8 + ((b & 0x007fffffu) > 0x00600000u ? 1 : 0);
  return max(E_MIN, min(E_MAX, e));
}
__device__ __forceinline__ float pow2f(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// e4m3 byte of x (finite, |x| at most 448 after saturation), round to nearest even
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  unsigned short r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// What a warp read of the rows from t0 on: lane l has row t0 + l.
struct Window {
  int t0;
  int64_t slot, pos;
};

// Writes one run (the consecutive rows that enter one page) of one head's keys
// or values: `wpi` warps, each with ROWS rows in registers (EL elements of a row
// per lane), so a run of up to ROWS wpi rows is read once and a longer one twice;
// the warps' largest values meet in shared memory.  The angles of a warp's rows
// come through shared memory, all copies in flight at once.  What bounds it is
// latency: the chain slot -> position -> angles and row -> scale (64 single rows
// 5.8 us, 6,444 rows of prompts in pages of 16 56 us in fp16 and 58 in bf16, 2.6
// TB/s with the queries; 74 us in pages of 64, 82 of 128).  With 16 rows a
// warp prompts have the most loads in flight (2 CTAs on an SM); 4 rows need half
// the registers, and a decode step's single rows have twice the CTAs.
// Rotary sizes that are not a multiple of 16, and unaligned rows, are read element
// by element: 64 single rows 7.3 us, the prompts 125.
// Every warp of the block calls it for the same run (`idle`: without an item).
template <typename T, int EL, int ROWS, bool VEC, bool ROPE>
__device__ __forceinline__ void append_run(const AppendArgs& p, int which, int head, int wi, bool idle, float* s_top,
                                           float* angles, const Window& win, int row0, int n, int64_t slot0) {
  constexpr int D = 32 * EL;
  const int lane = threadIdx.x & 31;
  const int64_t page = slot0 >> p.page_log2;
  const int lo = (int)slot0 & (p.page_size - 1);
  uint8_t* dst = p.pages[which] + (page * p.n_kv + head) * p.page_size * D;
  float* scale_at = p.scales[which] + page * p.n_kv + head;
  const T* src = static_cast<const T*>(p.src[which]) + head * p.src_head[which];
  const int64_t step = p.src_row[which];
  const float old = lo && !idle ? *scale_at : 0.0f;  // a run from the page's first row begins the page anew
  const int d0 = EL * lane, span = ROWS * p.wpi;
  if (idle) n = 0;

  auto load = [&](int row, T (&x)[EL]) {
    const T* at = src + row * step;
    if constexpr (VEC) {
      if constexpr (EL == 4) *reinterpret_cast<uint2*>(x) = __ldg(reinterpret_cast<const uint2*>(at + d0));
      else *reinterpret_cast<uint32_t*>(x) = __ldg(reinterpret_cast<const uint32_t*>(at + d0));
    } else {
#pragma unroll
      for (int e = 0; e < EL; ++e) x[e] = at[d0 + e];
    }
  };
  const int half = ROPE ? p.rot / 2 : 0;
  const bool second = ROPE && !p.interleaved && d0 >= half;
  // rotates a row that load() brought by the angles at `c` and c + half; every
  // lane of the warp takes part.  The other halves of its pairs are in this
  // lane, or `half` elements away in another.
  auto rotate = [&](const float* c, T (&x)[EL]) {
    T o[EL];
    if (!p.interleaved) {
      const int from = second ? lane - half / EL : lane + half / EL;
      if constexpr (EL == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(x);
        *reinterpret_cast<uint2*>(o) =
            make_uint2(__shfl_sync(0xffffffffu, v.x, from & 31), __shfl_sync(0xffffffffu, v.y, from & 31));
      } else {
        *reinterpret_cast<uint32_t*>(o) = __shfl_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(x), from & 31);
      }
      if (d0 >= p.rot) return;
      c += second ? d0 - half : d0;
#pragma unroll
      for (int e = 0; e < EL; ++e) x[e] = turn_key<T>(x[e], o[e], c[e], second ? c[half + e] : -c[half + e]);
    } else {
      if (d0 >= p.rot) return;
      c += d0 / 2;
#pragma unroll
      for (int e = 0; e < EL; ++e) o[e] = x[e];
#pragma unroll
      for (int e = 0; e < EL; ++e)
        x[e] = turn_key<T>(o[e], o[e ^ 1], c[e / 2], e & 1 ? c[half + e / 2] : -c[half + e / 2]);
    }
  };
  // the same for any rotary size and alignment
  auto rotate_any = [&](int row, int64_t pos, T (&x)[EL]) {
    const T* at = src + row * step;
#pragma unroll
    for (int e = 0; e < EL; ++e) {
      const int d = d0 + e;
      if (d >= p.rot) continue;
      const bool sec = p.interleaved ? (d & 1) : d >= half;
      const int pair = p.interleaved ? d >> 1 : sec ? d - half : d;
      const T mine = at[d], other = at[p.interleaved ? d ^ 1 : sec ? d - half : d + half];
      const float c = __ldg(p.cos_t + pos * half + pair), s = __ldg(p.sin_t + pos * half + pair);
      x[e] = turn_key<T>(mine, other, c, sec ? s : -s);
    }
  };
  // rows j0 .. of the run, all loads in flight before the first is used
  T x[ROWS][EL];
  auto load_chunk = [&](int j0) {
    const int m = n - j0, row = row0 + j0;
    int64_t pos = 0;
    if constexpr (ROPE) {
      if (which == 0) {
        const int at = row + min(lane & (ROWS - 1), m - 1), ahead = row - win.t0;
        if (ahead <= 32 - ROWS) pos = __shfl_sync(0xffffffffu, win.pos, (at - win.t0) & 31);
        else pos = p.positions[at];
        if constexpr (VEC) {                           // lane l copies piece l of a row's cosines and sines
          const bool sine = 4 * lane >= half;
          const float* table = sine ? p.sin_t + 4 * lane - half : p.cos_t + 4 * lane;
          const uint32_t to = smem_u32(angles) + 16 * lane;
#pragma unroll
          for (int j = 0; j < ROWS; ++j) {
            const int64_t at = __shfl_sync(0xffffffffu, pos, j);
            if (j < m && 2 * lane < half)
              asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(to + j * D * 4), "l"(table + at * half)
                           : "memory");
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      if (j < m) load(row + j, x[j]);
    if constexpr (ROPE) {
      if (which == 0) {
        if constexpr (VEC) {
          asm volatile("cp.async.wait_all;" ::: "memory");
          __syncwarp();
#pragma unroll
          for (int j = 0; j < ROWS; ++j)
            if (j < m) rotate(angles + j * D, x[j]);
          __syncwarp();
        } else {
#pragma unroll
          for (int j = 0; j < ROWS; ++j)
            if (j < m) rotate_any(row + j, __shfl_sync(0xffffffffu, pos, j), x[j]);
        }
      }
    }
  };
  // largest finite value of the run
  float top = 0.0f;
  bool odd = false;
  for (int j0 = ROWS * wi; j0 < n; j0 += span) {
    load_chunk(j0);
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      if (j0 + j < n) {
#pragma unroll
        for (int e = 0; e < EL; ++e) {
          const float a = fabsf(Num<T>::to_f(x[j][e]));
          if (a < INFINITY) top = fmaxf(top, a);
          else odd = true;
        }
      }
  }
  if constexpr (!std::is_same<T, __half>::value) odd |= top > TOP_MAX;       // saturates; no f16 value does
  if (__any_sync(0xffffffffu, odd) && lane == 0 && p.status) atomicOr(p.status, HC_ERR_RANGE);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) s_top[threadIdx.x >> 5] = top;
  __syncthreads();                                   // also: every warp has read the old scale
  if (idle) return;
  const int w0 = (int)(threadIdx.x >> 5) - wi;       // the item's first warp
  for (int k = 0; k < p.wpi; ++k) top = fmaxf(top, s_top[w0 + k]);
  const float need = pow2f(scale_exponent(top));
  const bool grown = need > old;
  const float now = grown ? need : old;
  const float inv = 1.0f / now;                      // exact: a power of two

  // the page's older rows at the larger scale
  if (lo && grown) {
    const float f = old * inv;
    for (int i = 32 * wi + lane; i < lo * D / 16; i += 32 * p.wpi) {
      uint4* at = reinterpret_cast<uint4*>(dst) + i;
      uint4 w = *at;
      uint32_t* ws = reinterpret_cast<uint32_t*>(&w);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t h0 = e4m3x2_to_f16x2(ws[k]), h1 = e4m3x2_to_f16x2(ws[k] >> 16);
        const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&h0));
        const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&h1));
        ws[k] = e4m3x2(a.x * f, a.y * f) | (e4m3x2(b.x * f, b.y * f) << 16);
      }
      *at = w;
    }
  }
  if (wi == 0 && lane == 0 && (grown || !lo)) *scale_at = now;
  for (int j0 = ROWS * wi; j0 < n; j0 += span) {
    if (n > span) load_chunk(j0);
#pragma unroll
    for (int j = 0; j < ROWS; ++j)
      if (j0 + j < n) {
        float f[EL];
#pragma unroll
        for (int e = 0; e < EL; ++e) {
          const float a = Num<T>::to_f(x[j][e]);
          f[e] = a != a ? 0.0f : a * inv;            // NaN is stored as 0; infinities saturate
        }
        uint8_t* at = dst + (int64_t)(lo + j0 + j) * D + d0;
        if constexpr (EL == 4) *reinterpret_cast<uint32_t*>(at) = e4m3x2(f[0], f[1]) | (e4m3x2(f[2], f[3]) << 16);
        else *reinterpret_cast<unsigned short*>(at) = (unsigned short)e4m3x2(f[0], f[1]);
      }
  }
}

// slot of row t; -1 for padding (negative slots, and in the fused form rows
// without a position in the tables); an index past the cache is flagged
template <bool ROPE>
__device__ __forceinline__ int64_t checked_slot(const AppendArgs& p, int t, bool flag) {
  const int64_t slot = p.slots[t];
  if (slot < 0) return -1;
  bool bad = slot >= (int64_t)p.n_pages * p.page_size;
  if constexpr (ROPE) {
    const int64_t pos = p.positions[t];
    if (pos == -1) return -1;
    bad = bad || pos < 0 || pos >= p.table_rows;
  }
  if (bad && flag && p.status) atomicOr(p.status, HC_ERR_RANGE);
  return bad ? -1 : slot;
}

// Runs that begin among rows [t0, t1), t1 - t0 <= 32: a row begins one unless
// the row before it lies in the same page.  Rows of a page that do not follow
// one another are flagged and left out.  The whole block works on one run.
template <typename T, int EL, int ROWS, bool VEC, bool ROPE>
__device__ __forceinline__ void append_rows(const AppendArgs& p, int t0, int t1, int item, int wi,
                                            float (*s_top)[APPEND_WARPS], float* angles) {
  const int lane = threadIdx.x & 31, which = item & 1;
  const bool idle = item >= 2 * p.n_kv, flag = item == 0 && wi == 0;
  const int head = idle ? 0 : item >> 1;
  // 32 rows' slots and positions at once: most runs need no second look
  Window win = {t0, -1, 0};
  const int mine = t0 + lane;
  if (mine < p.n_rows) {
    win.slot = checked_slot<ROPE>(p, mine, flag && mine < t1);
    if constexpr (ROPE) win.pos = p.positions[mine];
  }
  int64_t before = __shfl_up_sync(0xffffffffu, win.slot, 1);
  if (lane == 0) before = t0 ? checked_slot<ROPE>(p, t0 - 1, false) : -1;
  const bool same = win.slot >= 0 && before >= 0 && before >> p.page_log2 == win.slot >> p.page_log2;
  const bool begins = win.slot >= 0 && !same && mine < t1;
  if (same && before + 1 != win.slot && mine < t1 && flag && p.status) atomicOr(p.status, HC_ERR_RANGE);
  int turn = 0;
  for (uint32_t todo = __ballot_sync(0xffffffffu, begins); todo; todo &= todo - 1) {
    const int from = __ffs(todo) - 1, t = t0 + from;
    const int64_t first = __shfl_sync(0xffffffffu, win.slot, from);
    const int left = min(p.page_size - ((int)first & (p.page_size - 1)), p.n_rows - t);
    const uint32_t follow = __ballot_sync(0xffffffffu, lane >= from && win.slot == first + (lane - from)) >> from;
    int n = min(left, follow == 0xffffffffu ? 32 : __ffs(~follow) - 1);
    for (int base = n; n == base && base < left && base >= 32 - from; base += 32) {
      const int j = base + lane;
      const bool follows = j < left && checked_slot<ROPE>(p, t + j, false) == first + j;
      const uint32_t ok = __ballot_sync(0xffffffffu, follows);
      n += ok == 0xffffffffu ? 32 : __ffs(~ok) - 1;
    }
    append_run<T, EL, ROWS, VEC, ROPE>(p, which, head, wi, idle, s_top[turn ^= 1], angles, win, t, n, first);
  }
}

// n_append blocks write the cache, the others rotate the queries; the two kinds
// alternate over the grid, since one is bound by latency and the other by HBM.
template <typename T, int EL, int ROWS, bool VEC, bool ROPE>
__global__ void __launch_bounds__(APPEND_THREADS, ROWS == FEW ? 4 : 2)
    append_kernel(const AppendArgs p, const RopeArgs rope, unsigned n_append, unsigned groups) {
  const unsigned before = (unsigned)((uint64_t)blockIdx.x * n_append / gridDim.x);
  const unsigned upto = (unsigned)((uint64_t)(blockIdx.x + 1) * n_append / gridDim.x);
  if (upto > before) {
    extern __shared__ __align__(16) float s_angles[];                // [warp][ROWS][dim]
    __shared__ float s_top[2][APPEND_WARPS];
    const int w = threadIdx.x >> 5;
    const int item = (int)(before % groups) * (APPEND_WARPS / p.wpi) + w / p.wpi;
    const int t0 = (int)(before / groups) * p.seg;
    append_rows<T, EL, ROWS, VEC, ROPE>(p, t0, min(p.n_rows, t0 + p.seg), item, w % p.wpi, s_top,
                                  s_angles + w * ROWS * 32 * EL);
    if (p.beside) asm volatile("griddepcontrol.wait;" ::: "memory");   // the queries' kernel ends no later than this
    return;
  }
  if constexpr (ROPE) {
    if constexpr (VEC) rope_rows_vec<T>(rope, blockIdx.x - before);
    else rope_rows_any<T>(rope, blockIdx.x - before);
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
inline bool multiple(int64_t v, int64_t m) { return v % m == 0; }
inline bool aligned(const void* ptr, uintptr_t a) { return (reinterpret_cast<uintptr_t>(ptr) & (a - 1)) == 0; }
template <typename... P>
inline bool all_aligned(uintptr_t a, const P*... ptr) { return (aligned(ptr, a) && ...); }

int check_rope(const hc_rope_args* a, bool to_cache) {
  if (!a || !a->cos_t || !a->sin_t) return HC_ERR_ARG;
  if (a->n_rows != 0 && (!a->q || !a->q_out || !a->k || (!to_cache && !a->k_out) || !a->positions))
    return HC_ERR_ARG;
  if (a->n_rows < 0 || a->n_q_heads <= 0 || a->n_kv_heads <= 0 || a->head_dim <= 0 || a->rotary_dim <= 0 ||
      a->rotary_dim > a->head_dim || (a->rotary_dim & 1) || a->table_rows <= 0 ||
      (a->dtype != HC_F16 && a->dtype != HC_BF16) || a->interleaved < 0 || a->interleaved > 1)
    return HC_ERR_ARG;
  if (!aligned(a->q, 2) || !aligned(a->k, 2) || !aligned(a->q_out, 2) || !aligned(a->k_out, 2) ||
      !aligned(a->cos_t, 4) || !aligned(a->sin_t, 4) || !aligned(a->positions, 8))
    return HC_ERR_ARG;
  return a->n_rows > MAX_ROWS ? HC_ERR_UNSUPPORTED : HC_OK;
}

// The vector form wants 16-byte pieces throughout and whole units of 8 pairs.
bool rope_vec(const hc_rope_args* a, bool keys) {
  bool ok = multiple(a->rotary_dim, 16) && multiple(a->head_dim, 16) && a->head_dim <= 16 * ROPE_THREADS &&
            aligned(a->q, 16) && aligned(a->q_out, 16) &&
            multiple(a->q_row, 8) && multiple(a->q_head, 8) && multiple(a->q_out_row, 8) &&
            multiple(a->q_out_head, 8) && aligned(a->cos_t, 16) && aligned(a->sin_t, 16);
  if (keys)
    ok = ok && aligned(a->k, 16) && aligned(a->k_out, 16) && multiple(a->k_row, 8) && multiple(a->k_head, 8) &&
         multiple(a->k_out_row, 8) && multiple(a->k_out_head, 8);
  return ok;
}

RopeArgs rope_args(const hc_rope_args* a, bool keys, int32_t* status) {
  RopeArgs p;
  p.q = a->q;
  p.k = a->k;
  p.q_out = a->q_out;
  p.k_out = a->k_out;
  p.q_row = a->q_row;
  p.q_head = a->q_head;
  p.k_row = a->k_row;
  p.k_head = a->k_head;
  p.qo_row = a->q_out_row;
  p.qo_head = a->q_out_head;
  p.ko_row = a->k_out_row;
  p.ko_head = a->k_out_head;
  p.cos_t = a->cos_t;
  p.sin_t = a->sin_t;
  p.table_rows = a->table_rows;
  p.positions = a->positions;
  p.n_rows = a->n_rows;
  p.nq = a->n_q_heads;
  p.nk = keys ? a->n_kv_heads : 0;
  p.dim = a->head_dim;
  p.rot = a->rotary_dim;
  p.interleaved = a->interleaved;
  p.slots = 1;
  p.status = status;
  return p;
}

// Blocks of the rotation; sets how many heads of a row are worked on at once:
// all that a block has room for while rows are few, a quarter of them (each
// thread then has four heads' loads in flight) when rows fill the GPU.
int64_t rope_blocks(RopeArgs& p, bool vec) {
  p.rows_cta = 1;
  if (!vec) return p.n_rows;
  const int units = p.dim / 16, room = max(1, ROPE_THREADS / units);
  p.slots = min(room, max(p.nq, p.nk));
  if ((int64_t)p.n_rows * units * p.slots > 148 * 2048) p.slots = min(room, (max(p.nq, p.nk) + BATCH - 1) / BATCH);
  p.rows_cta = max(1, ROPE_THREADS / (units * p.slots));
  return (p.n_rows + p.rows_cta - 1) / p.rows_cta;
}

int check_pages(const hc_kv_pages* c) {
  if (!c || !c->k || !c->v || !c->k_scale || !c->v_scale) return HC_ERR_ARG;
  if (c->n_pages <= 0 || c->n_kv_heads <= 0) return HC_ERR_ARG;
  if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4))
    return HC_ERR_ARG;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return HC_ERR_UNSUPPORTED;
  if (c->head_dim != 64 && c->head_dim != 128) return HC_ERR_UNSUPPORTED;
  return HC_OK;
}

template <typename T, int ROWS>
int launch_append(AppendArgs& p, const hc_rope_args* rope, const hc_kv_pages* c, cudaStream_t stream) {
  RopeArgs ra = {};
  int64_t extra = 0;
  const int align = c->head_dim == 128 ? 4 : 2;      // elements a lane loads at once
  bool vec = aligned(p.src[0], 2 * align) && aligned(p.src[1], 2 * align) && multiple(p.src_row[0], align) &&
             multiple(p.src_row[1], align) && multiple(p.src_head[0], align) && multiple(p.src_head[1], align);
  if (rope) {
    vec = vec && rope_vec(rope, false);
    ra = rope_args(rope, false, p.status);
    extra = rope_blocks(ra, vec);
  }
  // Rows a CTA searches.  Few rows: one each, since in a decode step every row is a run (1,000 single rows take
  // 35 us so, 152 us with 16 rows a warp).  Many: up to a page, for which the CTAs do not outnumber the runs so much
  // (prompts of 6,444 rows: 57 us; 73 us when every eighth row has its CTAs).
  p.seg = ROWS == FEW ? 1 : max(1, min(min(32, c->page_size), p.n_rows / 256));
  // Warps of an item.  Many rows: enough to hold a whole page.  Few: a run may be one row or a page, and the host
  // does not know which; more warps shorten long runs and make single rows wait.  8 heads, with 1, 2, 4, 8 warps:
  // 64 single rows 5.3, 5.9, 6.3, 9.4 us, one run of 64 rows 33, 19, 11, 8; 500 single rows 14, 20, 31, 51, one
  // run of 400 44, 29, 22, 26.  So 8 while all of them fit twice over on the GPU, at least 2.
  p.wpi = c->page_size / ROWS;
  if constexpr (ROWS == FEW) {
    p.wpi = min(p.wpi, APPEND_WARPS);
    while (p.wpi > 2 && (int64_t)p.n_rows * 2 * p.n_kv * p.wpi > 148 * 16) p.wpi /= 2;
  }
  const int items = APPEND_WARPS / p.wpi;
  const int groups = (2 * p.n_kv + items - 1) / items;
  const int64_t n_append = (int64_t)((p.n_rows + p.seg - 1) / p.seg) * groups;
  // Few rows: one launch does both.  Many: the queries' rotation needs half of the registers that the write
  // does, and runs faster as a kernel of its own, which the write may run beside (6,444 rows of prompts with 32
  // query heads: 57 us, 84 in one launch).
  if (rope && ROWS == MANY) {
    if (vec) rope_kernel<T, true><<<(unsigned)extra, ROPE_THREADS, 0, stream>>>(ra);
    else rope_kernel<T, false><<<(unsigned)extra, ROPE_THREADS, 0, stream>>>(ra);
    if (cudaGetLastError() != cudaSuccess) return HC_ERR_CUDA;
    extra = 0;
    p.beside = 1;
  }
  if (n_append + extra > INT32_MAX) return HC_ERR_UNSUPPORTED;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(n_append + extra));
  cfg.blockDim = dim3(APPEND_THREADS);
  cfg.dynamicSmemBytes = rope && vec ? APPEND_WARPS * ROWS * c->head_dim * 4 : 0;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = p.beside ? 1 : 0;
  cudaError_t rc;
#define GO(EL, V, R)                                                                                          \
  rc = R && V ? cudaFuncSetAttribute(append_kernel<T, EL, ROWS, V, R>, cudaFuncAttributeMaxDynamicSharedMemorySize,  \
                                     (int)cfg.dynamicSmemBytes)                                               \
              : cudaSuccess;                                                                                  \
  if (rc == cudaSuccess)                                                                                      \
    rc = cudaLaunchKernelEx(&cfg, append_kernel<T, EL, ROWS, V, R>, p, ra, (unsigned)n_append, (unsigned)groups)
  if (c->head_dim == 128) {
    if (rope) {
      if (vec) { GO(4, true, true); }
      else { GO(4, false, true); }
    } else {
      if (vec) { GO(4, true, false); }
      else { GO(4, false, false); }
    }
  } else {
    if (rope) {
      if (vec) { GO(2, true, true); }
      else { GO(2, false, true); }
    } else {
      if (vec) { GO(2, true, false); }
      else { GO(2, false, false); }
    }
  }
#undef GO
  return rc == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

int launch_append(AppendArgs& p, int dtype, const hc_rope_args* rope, const hc_kv_pages* c, cudaStream_t stream) {
  if (p.n_rows < SPLIT_ROWS)
    return dtype == HC_F16 ? launch_append<__half, FEW>(p, rope, c, stream)
                           : launch_append<__nv_bfloat16, FEW>(p, rope, c, stream);
  return dtype == HC_F16 ? launch_append<__half, MANY>(p, rope, c, stream)
                         : launch_append<__nv_bfloat16, MANY>(p, rope, c, stream);
}

AppendArgs append_args(const hc_kv_pages* c, const void* k, int64_t k_row, int64_t k_head, const void* v,
                       int64_t v_row, int64_t v_head, const int64_t* slots, int32_t n_rows, int32_t* status) {
  AppendArgs p = {};
  p.pages[0] = c->k;
  p.pages[1] = c->v;
  p.scales[0] = c->k_scale;
  p.scales[1] = c->v_scale;
  p.n_pages = c->n_pages;
  p.n_kv = c->n_kv_heads;
  p.page_size = c->page_size;
  p.page_log2 = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  p.src[0] = k;
  p.src[1] = v;
  p.src_row[0] = k_row;
  p.src_row[1] = v_row;
  p.src_head[0] = k_head;
  p.src_head[1] = v_head;
  p.slots = slots;
  p.n_rows = n_rows;
  p.status = status;
  return p;
}

}  // namespace hcp

using namespace hcp;

extern "C" int hc_page_plan(const int32_t* starts, const int32_t* q_lens, int32_t n_requests, int32_t* tables,
                            int64_t table_stride, int32_t table_width, const int32_t* free_pages, int32_t n_pages,
                            int32_t* n_free, int32_t page_size, int32_t n_rows, int32_t* cu_q, int32_t* kv_lens,
                            int64_t* positions, int64_t* slots, int32_t* status, hc_stream_t stream) {
  if (!starts || !q_lens || !tables || !free_pages || !n_free || !cu_q || !kv_lens) return HC_ERR_ARG;
  if (n_rows < 0 || (n_rows && (!positions || !slots))) return HC_ERR_ARG;
  if (!all_aligned(4, starts, q_lens, tables, free_pages, n_free, cu_q, kv_lens, status) ||
      !all_aligned(8, positions, slots))
    return HC_ERR_ARG;
  if (n_requests <= 0 || table_width <= 0 || table_stride < table_width || n_pages <= 0 || page_size <= 0)
    return HC_ERR_ARG;
  if ((int64_t)table_width * page_size > INT32_MAX) return HC_ERR_ARG;
  if (n_requests > MAX_REQ || n_rows > MAX_ROWS) return HC_ERR_UNSUPPORTED;
  PlanArgs p = {starts, q_lens, n_requests, tables, table_stride, table_width, free_pages, n_pages, n_free,
                page_size, n_rows, cu_q, kv_lens, positions, slots, status};
  const int cl = n_rows > PLAN_THREADS ? PLAN_CL : 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cl);
  cfg.blockDim = dim3(PLAN_THREADS);
  cfg.stream = reinterpret_cast<cudaStream_t>(stream);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cl;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, page_plan_kernel, p) == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

extern "C" int hc_page_release(const uint8_t* done, int32_t n_requests, int32_t* tables, int64_t table_stride,
                               int32_t table_width, int32_t* free_pages, int32_t n_pages, int32_t* n_free,
                               int32_t* status, hc_stream_t stream) {
  if (!done || !tables || !free_pages || !n_free || !all_aligned(4, tables, free_pages, n_free, status))
    return HC_ERR_ARG;
  if (n_requests <= 0 || table_width <= 0 || table_stride < table_width || n_pages <= 0) return HC_ERR_ARG;
  if (n_requests > MAX_REQ) return HC_ERR_UNSUPPORTED;
  ReleaseArgs p = {done, n_requests, tables, table_stride, table_width, free_pages, n_pages, n_free, status};
  page_release_kernel<<<1, PLAN_THREADS, 0, reinterpret_cast<cudaStream_t>(stream)>>>(p);
  return cudaGetLastError() == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

extern "C" int hc_rope(const hc_rope_args* a, int32_t* status, hc_stream_t stream) {
  const int rc = check_rope(a, false);
  if (rc != HC_OK) return rc;
  if (!aligned(status, 4)) return HC_ERR_ARG;
  if (a->n_rows == 0) return HC_OK;
  const bool vec = rope_vec(a, true);
  RopeArgs p = rope_args(a, true, status);
  const int blocks = (int)rope_blocks(p, vec);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (a->dtype == HC_F16) {
    if (vec) rope_kernel<__half, true><<<blocks, ROPE_THREADS, 0, s>>>(p);
    else rope_kernel<__half, false><<<blocks, ROPE_THREADS, 0, s>>>(p);
  } else {
    if (vec) rope_kernel<__nv_bfloat16, true><<<blocks, ROPE_THREADS, 0, s>>>(p);
    else rope_kernel<__nv_bfloat16, false><<<blocks, ROPE_THREADS, 0, s>>>(p);
  }
  return cudaGetLastError() == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

extern "C" int hc_kv_append(const hc_kv_pages* cache, const void* k, int64_t k_row, int64_t k_head, const void* v,
                            int64_t v_row, int64_t v_head, const int64_t* slots, int32_t n_rows, int32_t dtype,
                            int32_t* status, hc_stream_t stream) {
  if (n_rows < 0 || (n_rows && (!k || !v || !slots)) || (dtype != HC_F16 && dtype != HC_BF16)) return HC_ERR_ARG;
  if (!all_aligned(2, k, v) || !aligned(slots, 8) || !aligned(status, 4)) return HC_ERR_ARG;
  if (n_rows > MAX_ROWS) return HC_ERR_UNSUPPORTED;
  const int rc = check_pages(cache);
  if (rc != HC_OK) return rc;
  if (n_rows == 0) return HC_OK;
  AppendArgs p = append_args(cache, k, k_row, k_head, v, v_row, v_head, slots, n_rows, status);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return launch_append(p, dtype, nullptr, cache, s);
}

extern "C" int hc_rope_append(const hc_rope_args* a, const hc_kv_pages* cache, const void* v, int64_t v_row,
                              int64_t v_head, const int64_t* slots, int32_t* status, hc_stream_t stream) {
  int rc = check_rope(a, true);
  if (rc != HC_OK) return rc;
  if ((a->n_rows && (!v || !slots)) || !aligned(v, 2) || !aligned(slots, 8) || !aligned(status, 4)) return HC_ERR_ARG;
  rc = check_pages(cache);
  if (rc != HC_OK) return rc;
  if (a->n_kv_heads != cache->n_kv_heads || a->head_dim != cache->head_dim) return HC_ERR_ARG;
  if (a->n_rows == 0) return HC_OK;
  AppendArgs p = append_args(cache, a->k, a->k_row, a->k_head, v, v_row, v_head, slots, a->n_rows, status);
  p.cos_t = a->cos_t;
  p.sin_t = a->sin_t;
  p.table_rows = a->table_rows;
  p.positions = a->positions;
  p.rot = a->rotary_dim;
  p.interleaved = a->interleaved;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return launch_append(p, a->dtype, a, cache, s);
}
