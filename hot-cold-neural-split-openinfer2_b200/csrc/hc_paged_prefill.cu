// Paged attention of many rows (prompts) on the tcgen05 tensor cores.
//
// One CTA takes 256 rows (token, query head) of one request and key-value
// head, as two groups of 128, and walks the request's keys 64 at a time:
//   S = Q K^T   128 x 64 per group, accumulated in TMEM, two buffers a group
//   P = 2^(S - m), f16, written over S in TMEM by the group's four warps (a
//       thread has a row, so its maximum and sum need no exchange)
//   O += P V    accumulated in TMEM, A operand P from TMEM
// e4m3 keys and values become f16 (exactly) in shared memory, 128 keys a tile
// and two tiles deep: four warps load a tile's bytes into registers, convert,
// and store the operand layout; each conversion serves 256 rows.  With two
// score buffers a group's softmax runs on without waiting for its products,
// and the tensor cores always have the other group's to do.
//
// Few tiles over long contexts would leave SMs idle, so a tile's keys are cut
// into pieces no longer than an SM's average share of all keys (and than
// MIN_PIECE); the pieces of a cut tile leave partial softmaxes, which a second
// kernel joins.
//
// What bounds it: the latency of a half's chain (score barrier, TMEM loads,
// maximum, exponentials, TMEM stores, barrier), which two softmax warps a
// scheduler do not cover.  No resource is busy all the time: at dim 128 the tensor
// pipe 43%, the exponentials' 44%, issue slots 45%; at dim 64 26, 53 and 44%.  A
// prompt of 4096 tokens, 32 / 8 heads of 128: 155 to 157 us in a graph, 880
// TFLOP/s, 164 as a call among others (the products alone need 86 us).  Pieces of
// 33 to 1500 tokens behind up to 8000, 16 / 2 heads of 64: 160 us, of which 45 are
// products and 62 exponentials; their 220 unequal units on 148 SMs leave a tail.
// 16 tokens of 4 heads a group behind 30,000 keys 57 us, 1.6 ms if their keys are
// not cut.  A converted tile serves 256 rows: 8 converter warps at 96 registers
// took 167 us for the prompt, tiles converted 64 keys at a time 164.
//
// Page scales: a key's scale joins the factor of its 16 score columns, a
// value's scale enters as log2 in the exponent (see hc_paged_attn.cu).
//
// Operand layouts (128-byte swizzle, 8-row atoms of 1024 bytes): Q and K are
// K-major, rows of 64 f16 per 16 KB block; V has the same image, read MN-major
// (dims contiguous).  TMEM: S of group x and buffer b at column 128 x + 64 b (P
// over its first 32 columns), O at 256 + 128 x.  Each group's products are
// issued by a thread of its own (one thread spent 2000 cycles on the 24 MMAs of
// 64 keys, which take 1250) and run in the order it issues them, so a buffer is
// written again without a wait for the product that read it.
#include "hc_paged_attn.cuh"

namespace hca8 {

constexpr int CONVERTERS = 4;          // warps
constexpr int MMA_WARP = 8 + CONVERTERS;                // two, one for each group
constexpr int SCALE_WARP = MMA_WARP + 2;
constexpr int PF_THREADS = 32 * (SCALE_WARP + 1);       // and 8 softmax warps
constexpr int GROUP_ROWS = 128;
constexpr int ROWS = 2 * GROUP_ROWS;
constexpr int KT = 128;                // keys per converted tile
constexpr int HALF = 64;               // keys per score buffer
constexpr int MIN_PIECE = 16;          // halves of a piece at least: beginning one costs about four
constexpr int SLICES = KT / 16;        // 16-key slices: no page is smaller
constexpr uint32_t PF_TRIES = 1u << 22; // a wait gives up after so many tries (each suspends for a while)

template <int D>
struct Layout {
  static constexpr int BLOCKS = D / 64;                  // 64-dim blocks of a row
  static constexpr int BLOCK = KT * 128;                 // bytes of a block of 128 rows
  static constexpr int TILE = BLOCKS * BLOCK;
  static constexpr int Q = 0;                            // two groups
  static constexpr int K = 2 * TILE;                     // two stages
  static constexpr int V = 4 * TILE;                     // two stages
  static constexpr int BYTES = 6 * TILE + 1024;          // + alignment
};

__device__ __forceinline__ uint64_t sw128_desc(uint32_t addr, uint32_t lbo, uint32_t sbo) {
  // start >> 4 [0,14), LBO >> 4 [16,30), SBO >> 4 [32,46), version 1 at [46,48), 128-byte swizzle (2) at [61,64)
  return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)((lbo >> 4) & 0x3FFFu) << 16) |
         ((uint64_t)((sbo >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16: f16 operands, fp32 accumulator, M = 128
__host__ __device__ constexpr uint32_t pf_idesc(int n, int b_mn) {
  return (1u << 4) | ((uint32_t)b_mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
// generic stores to shared memory (this thread's, and others' it has synchronised with) before the tensor cores' reads
__device__ __forceinline__ void fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define R4(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
// 32 columns of this thread's TMEM lane; the values are there after tmem_wait_ld
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : R4(v, 0), R4(v, 4), R4(v, 8), R4(v, 12), R4(v, 16), R4(v, 20), R4(v, 24), R4(v, 28)
      : "r"(addr)
      : "memory");
}
// 16 columns, with the wait
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15}, [%16];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : R4(v, 0), R4(v, 4), R4(v, 8), R4(v, 12)
      : "r"(addr)
      : "memory");
}
#undef R4
#define X4(v, i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3])
// every load so far has arrived; v names the registers, so that nothing that reads them moves ahead of it
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : X4(v, 0), X4(v, 4), X4(v, 8), X4(v, 12), X4(v, 16), X4(v, 20), X4(v, 24), X4(v, 28)
               :
               : "memory");
}
#undef X4
#define W4(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16};" ::"r"(addr),
      W4(v, 0), W4(v, 4), W4(v, 8), W4(v, 12)
      : "memory");
}
#undef W4
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// two fp32 lanes in one instruction
__device__ __forceinline__ uint64_t pair2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Bounded wait, kept short: the roles' loops share the instruction caches.
__device__ __forceinline__ bool wait_on(uint64_t* bar, uint32_t parity) {
#pragma unroll 1
  for (uint32_t n = 0; n < PF_TRIES; ++n)
    if (mbar_try_wait(bar, parity)) return true;
  return false;
}

struct Bars {
  uint64_t k_full[2], v_full[2];       // converters -> MMA
  uint64_t k_free[2], v_free[2];       // MMA -> converters
  uint64_t s_full[2][2];               // MMA -> group: the buffer's scores are complete
  uint64_t p_full[2][2];               // group -> MMA: the buffer's weights are written
  uint64_t o_done[2];                  // MMA -> group: a half's product is in O
  uint64_t done[2];                    // MMA -> group: all products are
  uint64_t meta[4];                    // scale warp -> groups: a tile's scales
  uint64_t drain[2];
  uint64_t q_full[2];                  // group -> MMA: its queries are in place
};

// Shared by the roles of one CTA.
struct Slice {
  float k, lv, iv;                     // key scale, log2 and reciprocal of the value scale
};

// factor of a slice's scores; never 0, which would make NaN of a masked score
__device__ __forceinline__ float factor(float k, float fac) { return fmaxf(k * fac, 1e-37f); }
// Columns past `last` are not seen.
__device__ __forceinline__ void mask_row(uint32_t (&s)[2][32], int last) {
#pragma unroll
  for (int c = 0; c < HALF; ++c)
    if (c > last) s[c >> 5][c & 31] = 0xff800000u;
}
// The largest exponent (base 2, scales applied) of this thread's row of a half.
__device__ __forceinline__ float row_max(const uint32_t (&s)[2][32], const Slice* sl, float fac) {
  float top = -INFINITY;
#pragma unroll
  for (int q = 0; q < HALF / 16; ++q) {
    float x[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) x[c] = __uint_as_float(s[q >> 1][16 * (q & 1) + c]);
    const float a = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), max3(x[6], x[7], x[8]));
    const float b = max3(max3(x[9], x[10], x[11]), max3(x[12], x[13], x[14]), x[15]);
    top = fmaxf(top, fmaf(fmaxf(a, b), factor(sl[q].k, fac), sl[q].lv));
  }
  return top;
}
// P = 2^(s - m) in f16 over the first half of the row's scores; returns l plus the row's share of the denominator.
__device__ __forceinline__ float row_weights(uint32_t at_s, const uint32_t (&s)[2][32], const Slice* sl, float fac,
                                             float m, float l) {
#pragma unroll
  for (int q = 0; q < HALF / 32; ++q) {
    uint32_t pk[16];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const Slice& k = sl[2 * q + hf];
      const float f = factor(k.k, fac), d = k.lv - m;
      const uint64_t f2 = pair2(f, f), d2 = pair2(d, d);
      uint64_t sum = 0;
#pragma unroll
      for (int c = 0; c < 16; c += 2) {
        float a, b;
        unpair2(fma2(pair2(__uint_as_float(s[q][16 * hf + c]), __uint_as_float(s[q][16 * hf + c + 1])), f2, d2), a, b);
        a = ex2(a);
        b = ex2(b);
        sum = add2(sum, pair2(a, b));
        pk[8 * hf + c / 2] = pack2<__half>(a, b);
      }
      float a, b;
      unpair2(sum, a, b);
      l = fmaf(a + b, k.iv, l);
    }
    tmem_st16(at_s + 16 * q, pk);
  }
  return l;
}
// one lane of a converged warp; the compiler then keeps the products' operands in uniform registers
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(p));
  return p != 0;
}

template <typename T, int D>
__global__ void __launch_bounds__(PF_THREADS, 1) paged_prefill_kernel(const AttnParams p) {
  using L = Layout<D>;
  extern __shared__ uint8_t raw[];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  __shared__ Bars bar;
  __shared__ Slice meta[4][SLICES];    // a tile's slot is written again four tiles later: no reader is left by then
  __shared__ uint32_t s_tmem;
  __shared__ int2 s_pre[MAX_REQ + 1];  // pieces and slots for partials before each request
  __shared__ int64_t s_wsum[PF_THREADS / 32];
  __shared__ int s_piece;
  __shared__ Req s_req[KEPT_REQ];
  const int t = threadIdx.x, lane = t & 31, w = __shfl_sync(0xffffffffu, t >> 5, 0);
  const uint32_t smem = (smem_u32(raw) + 1023) & ~1023u;

  // The step's work in halves sets the piece length; with it, the pieces of each request.  Where offsets go back the
  // requests (each in range by itself) may claim more rows than there are: the grid, the slots and the 32-bit sums
  // below, which hold for n_rows rows, would not do, and none of these requests is served.
  auto too_many = [&]() {
    int64_t claimed = 0;
#pragma unroll 1
    for (int r = 0; r < p.n_req; ++r) claimed += request(p, r, false).q_len;
    return claimed > p.n_rows;
  };
  auto tiles_of = [&](const Req& x) { return (x.q_len * p.g + ROWS - 1) / ROWS; };
  auto halves_of = [](int kv) { return (kv + HALF - 1) / HALF; };
  auto piece_of = [&](int64_t halves) {                 // even
    const uint64_t share = ((uint64_t)halves + p.sms - 1) / (unsigned)p.sms;
    return (int)min((uint64_t)(1 << 28), max((uint64_t)MIN_PIECE, share + (share & 1)));
  };
  auto units_of = [&](const Req& x, int piece) {        // pieces << 32 | slots
    const int cuts = max(1, (halves_of(x.kv) + piece - 1) / piece), n = tiles_of(x) * p.nkv * cuts;
    return ((int64_t)n << 32) + (cuts > 1 ? n : 0);
  };
  auto scan = [&](int64_t v) {                          // inclusive, over the warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  if (p.n_req <= 32) {                                  // a request a lane, one barrier
    if (w == 0) {
      Req x = {0, 0, 0};
      if (lane < p.n_req) s_req[lane] = x = request(p, lane, blockIdx.x == 0);
      const bool back = __any_sync(0xffffffffu, lane < p.n_req && p.cu_q[lane + 1] < p.cu_q[lane]) && too_many();
      int64_t sum = (int64_t)tiles_of(x) * p.nkv * halves_of(x.kv);
#pragma unroll
      for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      const int piece = piece_of(sum);
      const int64_t upto = scan(lane < p.n_req ? units_of(x, piece) : 0);
      s_pre[lane + 1] = make_int2(back ? -1 : (int)(upto >> 32), (int)upto);
      if (lane == 0) s_pre[0] = make_int2(0, 0), s_piece = piece;
    }
    __syncthreads();
  } else {
    const int per = (p.n_req + PF_THREADS - 1) / PF_THREADS;
    auto mine = [&](int i) {
      const int r = t * per + i;
      return p.n_req <= KEPT_REQ ? s_req[r] : request(p, r, false);
    };
    const int count = max(0, min(per, p.n_req - t * per));
    int64_t sum = 0;
    bool back = false;
    for (int i = 0; i < count; ++i) {
      const Req x = request(p, t * per + i, blockIdx.x == 0);
      if (p.n_req <= KEPT_REQ) s_req[t * per + i] = x;
      sum += (int64_t)tiles_of(x) * p.nkv * halves_of(x.kv);
      back |= p.cu_q[t * per + i + 1] < p.cu_q[t * per + i];
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_wsum[w] = sum;
    back = __syncthreads_or(back) && too_many();
    sum = 0;
    for (int k = 0; k < PF_THREADS / 32; ++k) sum += s_wsum[k];
    __syncthreads();
    const int piece = piece_of(sum);
    int64_t own = 0;
    for (int i = 0; i < count; ++i) own += units_of(mine(i), piece);
    const int64_t upto = scan(own);
    if (lane == 31) s_wsum[w] = upto;
    if (t == 0) s_pre[0] = make_int2(0, 0), s_piece = piece;
    __syncthreads();
    int64_t at = upto - own;
    for (int k = 0; k < w; ++k) at += s_wsum[k];
    for (int i = 0; i < count; ++i) {
      at += units_of(mine(i), piece);
      s_pre[t * per + i + 1] = make_int2(back ? -1 : (int)(at >> 32), (int)at);
    }
    __syncthreads();
  }
  const int piece = s_piece, all = s_pre[p.n_req].x;
  const bool over = (unsigned)all > gridDim.x;          // -1: none is served
  if (blockIdx.x == 0 && t == 0) {
    p.pf_cuts[0] = make_int4(over ? 0 : s_pre[p.n_req].y, 0, 0, 0);
    if (over && p.status) atomicOr(p.status, HC_ERR_RANGE);
  }
  if (over) return;
  // later tiles see more keys: they start first
  const int unit = all - 1 - (int)blockIdx.x;
  if (unit < 0) return;
  int r = 0;
  for (int b = p.n_req; b - r > 1;) {
    const int mid = (r + b) / 2;
    if (s_pre[mid].x <= unit) r = mid;
    else b = mid;
  }
  const Req x = p.n_req <= KEPT_REQ ? s_req[r] : request(p, r, false);
  const unsigned cuts = max(1, (halves_of(x.kv) + piece - 1) / piece);
  const unsigned in = unit - s_pre[r].x;               // (tile, key-value head, piece)
  const int cut = in % cuts, h = in / cuts % p.nkv, row0 = (int)(in / cuts / p.nkv) * ROWS;
  const int slot = s_pre[r].y + (int)in;
  const int n_here = min(ROWS, x.q_len * p.g - row0);
  const int lim_last = x.kv - x.q_len + (row0 + n_here - 1) / p.g;       // last key that any row sees
  const int tile_half = lim_last < 0 ? 0 : lim_last / HALF + 1;          // halves of the tile
  const int n_cut = max(1, (tile_half + piece - 1) / piece);             // pieces that have any
  const bool split = n_cut > 1;
  if (cuts > 1 && t == 0) {
    p.pf_cuts[1 + 2 * slot] = make_int4(row0, n_here, x.q0, h);
    p.pf_cuts[2 + 2 * slot] = make_int4(split && cut == 0 ? n_cut : 0, 0, 0, 0);
  }
  if (cut >= n_cut) return;
  // from here on keys count from the piece's first
  const int key_first = cut * piece * HALF;
  const int n_half = min(tile_half - cut * piece, piece), n_tiles = (n_half + 1) / 2;
  const int behind = x.kv - x.q_len - key_first, lim_hi = min(lim_last - key_first, n_half * HALF - 1);
  const int32_t* table = p.tables + (int64_t)r * p.t_stride + (key_first >> p.page_log2);
  const bool two = n_here > GROUP_ROWS;

  if (w == MMA_WARP) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (t == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.k_full[i], CONVERTERS);
      mbar_init(&bar.v_full[i], CONVERTERS);
      mbar_init(&bar.k_free[i], two ? 2 : 1);           // both issuers
      mbar_init(&bar.v_free[i], two ? 2 : 1);
      mbar_init(&bar.drain[i], 1);
      mbar_init(&bar.q_full[i], GROUP_ROWS);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&bar.s_full[i][b], 1);
        mbar_init(&bar.p_full[i][b], GROUP_ROWS);
      }
      mbar_init(&bar.o_done[i], 1);
      mbar_init(&bar.done[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bar.meta[i], 1);
    mbar_fence_init();
  }

  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, s_tmem, 0);
  bool ok = true;

  if (w < 8) {
    // ---- softmax: group g2, one row a thread --------------------------------
    const int g2 = w >> 2;
    if (g2 == 0 || two) {
      // this thread's row; queries and outputs move LPR lanes to a row, RPI rows an instruction
      constexpr int LPR = D / 8, RPI = 32 / LPR;
      const int c = lane % LPR, row = t & (GROUP_ROWS - 1);
      const uint32_t q_tile = smem + L::Q + g2 * L::TILE;
      int lim = -1;
      int64_t q_at = -1, out_at = -1, lse_at = 0;
      if (t < n_here) {
        const int tok = (row0 + t) / p.g, head = h * p.g + (row0 + t) - tok * p.g;
        lim = behind + tok;
        q_at = (int64_t)(x.q0 + tok) * p.q_row + head * p.q_head;
        out_at = (int64_t)(x.q0 + tok) * p.o_row + head * p.o_head;
        lse_at = (int64_t)(x.q0 + tok) * p.nq + head;
      }
      // the factor stays positive (a maximum is taken before it is applied); the sign goes to the query
      const float sign = p.scale2 < 0.0f ? -1.0f : 1.0f;
      float fac = fabsf(p.scale2);
      const bool q_vec = (reinterpret_cast<uintptr_t>(p.q) & 15) == 0 && p.q_row % 8 == 0 && p.q_head % 8 == 0;
      auto spot = [&](int to) {                         // of piece c of row `to` in the operand tile
        return q_tile + to * 128 + (c / 8) * L::BLOCK + (((c % 8) ^ (to & 7)) << 4);
      };
      auto place_query = [&](int i, uint4 v) {          // converts and stores pieces of rows RPI i ..
        const uint32_t e[4] = {v.x, v.y, v.z, v.w};
        uint32_t f[4];
        float up = sign;
        if constexpr (!std::is_same<T, __half>::value) {         // bf16: a power of two brings a row into f16's range
          float top = 0.0f;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float2 a = unpack2<T>(e[k]);
            top = max3(top, fabsf(a.x), fabsf(a.y));
          }
#pragma unroll
          for (int o = 1; o < LPR; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const int k = min(126, 135 - (int)(__float_as_uint(top) >> 23));       // top * 2^k in [2^8, 2^9)
          up *= __uint_as_float((uint32_t)(k + 127) << 23);
          const int mine = __shfl_sync(0xffffffffu, k, (lane % RPI) * LPR);      // to the thread that has the row
          if (lane / RPI == i) fac *= __uint_as_float((uint32_t)(127 - mine) << 23);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 a = unpack2<T>(e[k]);
          f[k] = pack2<__half>(a.x * up, a.y * up);
        }
        sts16(spot(32 * (w & 3) + RPI * i + lane / LPR), f[0], f[1], f[2], f[3]);
      };
      if (q_vec && std::is_same<T, __half>::value && sign > 0.0f) {              // f16 as it is: straight into the tile
#pragma unroll 4
        for (int i = 0; i < 32 / RPI; ++i) {
          const int src = RPI * i + lane / LPR;
          const int64_t at = __shfl_sync(0xffffffffu, q_at, src);
          const T* q = static_cast<const T*>(p.q) + (at >= 0 ? at : 0) + 8 * c;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(spot(32 * (w & 3) + src)), "l"(q),
                       "r"(at >= 0 ? 16 : 0)
                       : "memory");
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
      } else if (q_vec) {
        uint4 v[32 / RPI];
#pragma unroll
        for (int i = 0; i < 32 / RPI; ++i) {
          const int64_t at = __shfl_sync(0xffffffffu, q_at, RPI * i + lane / LPR);
          v[i] = make_uint4(0u, 0u, 0u, 0u);
          if (at >= 0) v[i] = __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + at + 8 * c));
        }
#pragma unroll
        for (int i = 0; i < 32 / RPI; ++i) place_query(i, v[i]);
      } else {
#pragma unroll 1
        for (int i = 0; i < 32 / RPI; ++i) {
          const int64_t at = __shfl_sync(0xffffffffu, q_at, RPI * i + lane / LPR);
          uint32_t e[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
          if (at >= 0) {
            const unsigned short* q = reinterpret_cast<const unsigned short*>(static_cast<const T*>(p.q) + at + 8 * c);
#pragma unroll
            for (int k = 0; k < 8; ++k) e[k] = __ldg(q + k);
          }
          place_query(i, make_uint4(e[0] | (e[1] << 16), e[2] | (e[3] << 16), e[4] | (e[5] << 16),
                                    e[6] | (e[7] << 16)));
        }
      }
      fence_proxy();
      mbar_arrive(&bar.q_full[g2]);

      const uint32_t at_s = tmem + ((uint32_t)(w & 3) << 21) + 128 * g2, at_o = at_s + 256;
      const int lim_first = behind + (row0 + GROUP_ROWS * g2) / p.g;
      float m = M_NONE, l = 0.0f;
      for (int i = 0; i < n_half; ++i) {
        const int b = i & 1, j = i >> 1;
        if (b == 0) ok = ok && wait_on(&bar.meta[j & 3], (j >> 2) & 1);
        ok = ok && wait_on(&bar.s_full[g2][b], j & 1);
        if (!__all_sync(0xffffffffu, ok)) break;
        fence_after();
        const Slice* sl = meta[j & 3] + (HALF / 16) * b;
        const bool masked = i * HALF + HALF - 1 > lim_first;
        const int last = lim - i * HALF;                // columns past it are not seen
        const uint32_t at = at_s + HALF * b;
        uint32_t s[2][32];
        tmem_ld32(at, s[0]);
        tmem_ld32(at + 32, s[1]);
        tmem_wait_ld(s[0]);
        tmem_wait_ld(s[1]);
        if (masked) mask_row(s, last);
        const float top = row_max(s, sl, fac);
        if (__any_sync(0xffffffffu, top > m + W_MAX)) {
          const float m1 = fmaxf(m, top - W_REF), keep = ex2(m - m1);
          m = m1;
          l *= keep;
          if (i > 0) {
            ok = wait_on(&bar.o_done[g2], (i - 1) & 1);
            if (!__all_sync(0xffffffffu, ok)) break;
            fence_after();
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 16) {
              uint32_t o[16];
              tmem_ld16(at_o + c0, o);
#pragma unroll
              for (int c = 0; c < 16; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * keep);
              tmem_st16(at_o + c0, o);
            }
          }
        }
        l = row_weights(at, s, sl, fac, m, l);
        tmem_wait_st();
        fence_before();
        mbar_arrive(&bar.p_full[g2][b]);
      }
      uint32_t s[32];
      if (n_tiles > 0) {
        ok = ok && wait_on(&bar.done[g2], 0);
        ok = __all_sync(0xffffffffu, ok);
        fence_after();
      }
      if (split) {                                      // a partial: [D / 4][256 rows] of four dims, then m and l
        float* part = p.pf_part + (int64_t)slot * (ROWS * (D + 2));
#pragma unroll 1
        for (int c0 = 0; c0 < D; c0 += 32) {
          if (!ok) break;
          tmem_ld32(at_o + c0, s);
          tmem_wait_ld(s);
#pragma unroll
          for (int c = 0; c < 32; c += 4)
            reinterpret_cast<uint4*>(part)[(c0 + c) / 4 * ROWS + t] = make_uint4(s[c], s[c + 1], s[c + 2], s[c + 3]);
        }
        part[ROWS * D + t] = m;
        part[ROWS * D + ROWS + t] = l;
      } else {
      // The warp's 32 rows go through its part of the query tile (no product reads it any more), so that a
      // store instruction writes whole rows.
      const float inv = l > 0.0f ? __frcp_rn(l) : l;    // no key: 0, and NaN stays NaN
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        if (n_tiles > 0 && ok) {
          tmem_ld32(at_o + c0, s);
          tmem_wait_ld(s);
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) s[c] = 0u;
        }
#pragma unroll
        for (int c = 0; c < 32; c += 8) {
          uint32_t o[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            o[k] = l == 0.0f ? 0u
                             : pack2<T>(__uint_as_float(s[c + 2 * k]) * inv, __uint_as_float(s[c + 2 * k + 1]) * inv);
          const int x = (c0 + c) / 8;
          sts16(q_tile + row * 128 + (x / 8) * L::BLOCK + (((x % 8) ^ (row & 7)) << 4), o[0], o[1], o[2], o[3]);
        }
      }
      __syncwarp();
#pragma unroll 4
      for (int i = 0; i < 32 / RPI; ++i) {
        const int src = RPI * i + lane / LPR, n = 32 * (w & 3) + src;
        const int64_t at = __shfl_sync(0xffffffffu, out_at, src);
        uint4 v;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "r"(q_tile + n * 128 + (c / 8) * L::BLOCK + (((c % 8) ^ (n & 7)) << 4))
                     : "memory");
        if (at < 0) continue;
        T* out = static_cast<T*>(p.out) + at + 8 * c;
        if ((reinterpret_cast<uintptr_t>(out) & 15) == 0) {
          *reinterpret_cast<uint4*>(out) = v;
        } else {
          const uint32_t e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll 1
          for (int k = 0; k < 4; ++k) {
            const uint32_t u = k == 0 ? e[0] : k == 1 ? e[1] : k == 2 ? e[2] : e[3];
            const T* pair = reinterpret_cast<const T*>(&u);
            out[2 * k] = pair[0];
            out[2 * k + 1] = pair[1];
          }
        }
      }
      if (out_at >= 0 && p.lse) p.lse[lse_at] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * LN2;
      }
    }
  } else if (w < MMA_WARP) {
    // ---- converters: e4m3 pages -> f16 operand tiles -------------------------
    constexpr int PIECES = D / 16;                      // 16-byte pieces of a key row
    constexpr int KEYS = 32 * CONVERTERS / PIECES;      // keys that the threads cover at once
    constexpr int N = KT / KEYS;                        // pieces per thread
    const int ct = t - 256, piece = ct % PIECES, key0 = ct / PIECES;
    uint4 kr[N], vr[N];
    // Page of the slice that holds a key.  Keys behind lim_hi read the page of
    // lim_hi: their bytes are replaced before they are converted.
    auto page_of = [&](int key) { return __ldg(table + (min(key, lim_hi) >> p.page_log2)); };
    // A thread's pieces lie in N slices; it reads their pages itself, a tile
    // ahead: shuffles between the loads made each wait for the one before.
    // Every load is unconditional, from an address inside the pool.
    const uint32_t page_bytes = (uint32_t)D << p.page_log2, in_page = ((uint32_t)1 << p.page_log2) - 1;
    int pg[N];
    auto pages = [&](int j) {
#pragma unroll
      for (int i = 0; i < N; ++i) pg[i] = page_of(j * KT + key0 + KEYS * i);
    };
    auto load = [&](const uint8_t* pool, int j, uint4 (&v)[N]) {
      const uint8_t* base = pool + 16 * piece;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const uint32_t head = (uint32_t)((unsigned)pg[i] < (unsigned)p.n_pages ? pg[i] : 0) * p.nkv + h;
        const uint32_t key = (uint32_t)(j * KT + key0 + KEYS * i) & in_page;
        v[i] = __ldg(reinterpret_cast<const uint4*>(base + (uint64_t)head * page_bytes + key * D));
      }
    };
    // pieces of tile j without a page or behind lim_hi become zeros
    uint32_t lost = 0, lost_next = 0;                   // pieces whose page is not in the pool
    auto lose = [&]() {
      lost_next = 0;
#pragma unroll
      for (int i = 0; i < N; ++i) lost_next |= (unsigned)pg[i] < (unsigned)p.n_pages ? 0u : 1u << i;
    };
    auto blank = [&](int j, uint4 (&v)[N]) {
      if (j + 1 < n_tiles && !__any_sync(0xffffffffu, lost != 0)) return;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (((lost >> i) & 1) || j * KT + key0 + KEYS * i > lim_hi) v[i] = make_uint4(0u, 0u, 0u, 0u);
    };
    auto store = [&](uint32_t dst, const uint4 (&v)[N]) {
      // a lane's two 16-byte halves in an order that spreads eight lanes over all banks
      const int flip = D == 128 ? piece >> 2 : 0;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int kk = key0 + KEYS * i;
        uint32_t f[8];
        const uint32_t wv[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f[2 * k] = e4m3x2_to_f16x2(wv[k]);
          f[2 * k + 1] = e4m3x2_to_f16x2(wv[k] >> 16);
        }
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const int half = hf ^ flip, c = 2 * piece + half;
          const uint32_t at = dst + (c / 8) * L::BLOCK + kk * 128 + (((c % 8) ^ (kk & 7)) << 4);
          if (half) sts16(at, f[4], f[5], f[6], f[7]);
          else sts16(at, f[0], f[1], f[2], f[3]);
        }
      }
      __syncwarp();
    };
    // The next tile's bytes are loaded while this one's are converted.  The
    // issuers order these stores before their products: a proxy fence here
    // would wait for the loads in flight.
    if (n_tiles > 0) {
      pages(0);
      load(p.kp, 0, kr);
      load(p.vp, 0, vr);
      lose();
      lost = lost_next;
      pages(1);
    }
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j & 1;
      if (j >= 2) ok = ok && wait_on(&bar.k_free[st], ((j >> 1) - 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) break;
      blank(j, kr);
      store(smem + L::K + st * L::TILE, kr);
      if (lane == 0) mbar_arrive(&bar.k_full[st]);      // after store()'s __syncwarp
      if (j + 1 < n_tiles) {
        load(p.kp, j + 1, kr);
        lose();
      }
      if (j >= 2) ok = ok && wait_on(&bar.v_free[st], ((j >> 1) - 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) break;
      blank(j, vr);
      store(smem + L::V + st * L::TILE, vr);
      if (lane == 0) mbar_arrive(&bar.v_full[st]);
      if (j + 1 < n_tiles) {
        load(p.vp, j + 1, vr);
        lost = lost_next;
        pages(j + 2);
      }
    }
  } else if (w == SCALE_WARP) {
    // ---- scales: lane l has slice l of a tile; pages and scales run ahead ------
    const int key = (lane & (SLICES - 1)) * 16;
    auto page_of = [&](int j) { return __ldg(table + (min(j * KT + key, lim_hi) >> p.page_log2)); };
    auto head_of = [&](int page) { return (int64_t)((unsigned)page < (unsigned)p.n_pages ? page : 0) * p.nkv + h; };
    int at = -1, next = -1;
    float ks = 0.0f, vs = 1.0f;
    if (n_tiles > 0) {
      at = page_of(0);
      next = page_of(1);
      ks = __ldg(p.ks + head_of(at));
      vs = __ldg(p.vs + head_of(at));
    }
    for (int j = 0; j < n_tiles; ++j) {
      Slice mine = {0.0f, -INFINITY, 0.0f};             // no page: no weight
      if ((unsigned)at < (unsigned)p.n_pages) {
        const float b = fmaxf(vs, VS_MIN);
        mine.k = ks;
        mine.lv = __log2f(b);
        mine.iv = __frcp_rn(b);
      } else if (j * KT + key <= lim_hi && p.status) {
        atomicOr(p.status, HC_ERR_RANGE);
      }
      if (j + 1 < n_tiles) {
        at = next;
        ks = __ldg(p.ks + head_of(at));
        vs = __ldg(p.vs + head_of(at));
        next = page_of(j + 2);
      }
      // the stage's keys are used up, so every reader of the slot is past it
      if (j >= 2) ok = ok && wait_on(&bar.k_free[j & 1], ((j >> 1) - 1) & 1);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (lane < SLICES) meta[j & 3][lane] = mine;
      __syncwarp();
      if (lane == 0) mbar_arrive(&bar.meta[j & 3]);
    }
  } else if (n_tiles > 0) {
    // ---- MMA: one thread a group ----------------------------------------------
    // Half i uses buffer i % 2 and stage (i / 2) % 2.  The loops stay rolled:
    // unrolled over the stages, the issuers' code pushed the other roles' out of
    // the instruction caches.
    if (elect_one() && (w == MMA_WARP || two)) {
      constexpr uint32_t id_s = pf_idesc(HALF, 0), id_o = pf_idesc(D, 1);
      const int g2 = w - MMA_WARP;
      const uint32_t t_s = tmem + 128 * g2, t_o = t_s + 256;
      const uint64_t d_q = sw128_desc(smem + L::Q + g2 * L::TILE, 16, 1024);
      const uint64_t d_k = sw128_desc(smem + L::K, 16, 1024), d_v = sw128_desc(smem + L::V, L::BLOCK, 1024);
      auto place = [](int i) {                          // of half i among the two stages, in descriptor units
        return (uint64_t)((((i >> 1) & 1) * L::TILE + (i & 1) * (HALF * 128)) >> 4);
      };
      auto scores = [&](int i) {
        uint64_t a = d_q, b = d_k + place(i);
        const uint32_t d = t_s + HALF * (i & 1);
#pragma unroll
        for (int e = 0; e < D / 64; ++e) {
#pragma unroll
          for (int k = 0; k < 4; ++k) mma_ss(d, a + 2 * k, b + 2 * k, id_s, e + k);
          a += L::BLOCK >> 4;
          b += L::BLOCK >> 4;
        }
        mma_commit(&bar.s_full[g2][i & 1]);
      };
      ok = wait_on(&bar.q_full[g2], 0) && wait_on(&bar.k_full[0], 0);
      if (ok) {
        fence_proxy();
        fence_after();
        scores(0);
        if (n_half > 1) scores(1);
        mma_commit(&bar.k_free[0]);
#pragma unroll 1
        for (int i = 0; i < n_half; ++i) {
          const int st = (i >> 1) & 1;
          const bool more = i + 2 < n_half;
          if ((i & 1) == 0) {
            ok = wait_on(&bar.v_full[st], (i >> 2) & 1);
            if (more) ok = ok && wait_on(&bar.k_full[st ^ 1], ((i + 2) >> 2) & 1);
            fence_proxy();
          }
          ok = ok && wait_on(&bar.p_full[g2][i & 1], st);
          if (!ok) break;
          fence_after();
          const uint64_t b = d_v + place(i);
#pragma unroll
          for (int e = 0; e < HALF / 16; ++e)
            mma_ts(t_o, t_s + HALF * (i & 1) + 8 * e, b + 128 * e, id_o, i + e);
          mma_commit(&bar.o_done[g2]);
          if (i & 1) mma_commit(&bar.v_free[st]);
          if (more) {
            scores(i + 2);
            if (i & 1) mma_commit(&bar.k_free[st ^ 1]);
          }
        }
        if (ok) mma_commit(&bar.done[g2]);
      }
      // every product that was issued has completed before the CTA gives up its memory
      mma_commit(&bar.drain[g2]);
      wait_on(&bar.drain[g2], 0);
    }
  }
  if (!ok && p.status) atomicOr(p.status, HC_ERR_TIMEOUT);
  fence_before();
  __syncthreads();
  fence_after();
  if (w == MMA_WARP)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// Joins the pieces of the tiles that were cut: a thread has a row and 16 dims.
template <typename T, int D>
__global__ void __launch_bounds__(ROWS) paged_prefill_join_kernel(const AttnParams p) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int t = threadIdx.x, slots = p.pf_cuts[0].x;
  for (int slot = blockIdx.x; slot < slots; slot += gridDim.x) {
    const int n = p.pf_cuts[2 + 2 * slot].x;
    const int4 tile = p.pf_cuts[1 + 2 * slot];           // first row, rows, first token, key-value head
    if (n == 0 || t >= tile.y) continue;
    const int64_t stride = ROWS * (D + 2);
    const float* part = p.pf_part + slot * stride;
    float M = M_NONE, L = 0.0f;
    for (int k = 0; k < n; ++k) M = fmaxf(M, part[k * stride + ROWS * D + t]);
    float a[16];
#pragma unroll
    for (int c = 0; c < 16; ++c) a[c] = 0.0f;
#pragma unroll 2
    for (int k = 0; k < n; ++k) {
      const float* q = part + k * stride;
      const float f = ex2(q[ROWS * D + t] - M);
      L = fmaf(q[ROWS * D + ROWS + t], f, L);
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4 v = reinterpret_cast<const float4*>(q)[(4 * blockIdx.y + c) * ROWS + t];
        // a piece that the row sees nothing of has f = 0; its sums are finite, as the cache holds no NaN
        a[4 * c] = fmaf(v.x, f, a[4 * c]);
        a[4 * c + 1] = fmaf(v.y, f, a[4 * c + 1]);
        a[4 * c + 2] = fmaf(v.z, f, a[4 * c + 2]);
        a[4 * c + 3] = fmaf(v.w, f, a[4 * c + 3]);
      }
    }
    const float inv = L > 0.0f ? __frcp_rn(L) : L;
    const int tok = tile.z + (tile.x + t) / p.g, head = tile.w * p.g + (tile.x + t) % p.g;
    T* out = static_cast<T*>(p.out) + (int64_t)tok * p.o_row + head * p.o_head + 16 * blockIdx.y;
    uint32_t o[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) o[c] = L == 0.0f ? 0u : pack2<T>(a[2 * c] * inv, a[2 * c + 1] * inv);
    if ((reinterpret_cast<uintptr_t>(out) & 15) == 0) {
      reinterpret_cast<uint4*>(out)[0] = make_uint4(o[0], o[1], o[2], o[3]);
      reinterpret_cast<uint4*>(out)[1] = make_uint4(o[4], o[5], o[6], o[7]);
    } else {
      const T* e = reinterpret_cast<const T*>(o);
#pragma unroll
      for (int c = 0; c < 16; ++c) out[c] = e[c];
    }
    if (p.lse && blockIdx.y == 0)
      p.lse[(int64_t)tok * p.nq + head] = L == 0.0f ? -INFINITY : (M + __log2f(L)) * LN2;
  }
}

// Slots for partials: a request that is cut has under twice its work over the piece length, and a piece is at
// least an SM's share of all work.
constexpr int MAX_SMS = 148, MAX_SLOTS = 2 * MAX_SMS;

int64_t prefill_workspace(int head_dim) {
  return 16 * (1 + 2 * MAX_SLOTS) + (int64_t)MAX_SLOTS * ROWS * (head_dim + 2) * 4;
}

template <typename T, int D>
int launch_pf(AttnParams p, void* workspace, int sms, cudaStream_t stream) {
  using L = Layout<D>;
  p.sms = min(sms, MAX_SMS);
  p.pf_cuts = static_cast<int4*>(workspace);
  p.pf_part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + 16 * (1 + 2 * MAX_SLOTS));
  if (cudaFuncSetAttribute(paged_prefill_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::BYTES) !=
      cudaSuccess)
    return HC_ERR_CUDA;
  // the lengths are on the device: as many pieces as any lengths of these rows can need
  const int64_t tiles = ((int64_t)p.n_rows * p.g + ROWS - 1) / ROWS + min(p.n_req, p.n_rows);
  const int64_t pieces = tiles * p.nkv + p.sms;
  if (pieces > INT32_MAX) return HC_ERR_UNSUPPORTED;
  paged_prefill_kernel<T, D><<<(unsigned)pieces, PF_THREADS, L::BYTES, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return HC_ERR_CUDA;
  // no length that the tables hold is cut
  if (((int64_t)p.width << p.page_log2) <= MIN_PIECE * HALF) return HC_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(MAX_SMS / 2, D / 16);
  cfg.blockDim = dim3(ROWS);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_prefill_join_kernel<T, D>, p) == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

int launch_prefill(const AttnParams& p, int dtype, int head_dim, void* workspace, int sms, cudaStream_t stream) {
  if (dtype == HC_F16)
    return head_dim == 128 ? launch_pf<__half, 128>(p, workspace, sms, stream)
                           : launch_pf<__half, 64>(p, workspace, sms, stream);
  return head_dim == 128 ? launch_pf<__nv_bfloat16, 128>(p, workspace, sms, stream)
                         : launch_pf<__nv_bfloat16, 64>(p, workspace, sms, stream);
}

}  // namespace hca8
