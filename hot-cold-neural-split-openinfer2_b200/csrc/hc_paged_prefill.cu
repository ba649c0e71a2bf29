// Paged attention of many rows (prompts) on the tcgen05 tensor cores.
//
// One CTA takes 256 rows (token, query head) of one request and key-value
// head, as two groups of 128, and walks the request's keys 128 at a time:
//   S = Q K^T   128 x 128 per group, accumulated in TMEM
//   P = 2^(S - m), f16, written over S in TMEM by the group's four warps (a
//       thread has a row, so its maximum and sum need no exchange)
//   O += P V    accumulated in TMEM, A operand P from TMEM
// e4m3 keys and values become f16 (exactly) in shared memory; four warps load
// a tile's bytes into registers one tile ahead, convert, and store the operand
// layout.  The groups alternate: while one group's softmax runs, the tensor
// cores work on the other's two products, and each conversion serves 256 rows.
//
// Page scales: a key's scale joins the factor of its 16 score columns, a
// value's scale enters as log2 in the exponent (see hc_paged_attn.cu).
//
// Operand layouts (128-byte swizzle, 8-row atoms of 1024 bytes): Q and K are
// K-major, rows of 64 f16 per 16 KB block; V has the same image, read MN-major
// (dims contiguous).  TMEM: S of group x at column 128 x (P over its first 64
// columns), O at 256 + 128 x.
#include "hc_paged_attn.cuh"

namespace hca8 {

constexpr int PF_THREADS = 416;        // 8 softmax warps, 4 converter warps, 1 MMA warp
constexpr int GROUP_ROWS = 128;
constexpr int ROWS = 2 * GROUP_ROWS;
constexpr int KT = 128;                // keys per tile
constexpr int SLICES = KT / 16;        // 16-key slices: no page is smaller
constexpr uint64_t PF_WAIT_NS = 2000000000ull;

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
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

#define R4(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
// 32 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : R4(v, 0), R4(v, 4), R4(v, 8), R4(v, 12), R4(v, 16), R4(v, 20), R4(v, 24), R4(v, 28)
      : "r"(addr)
      : "memory");
}
#undef R4
#define W4(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
      "%14, %15, %16};" ::"r"(addr),
      W4(v, 0), W4(v, 4), W4(v, 8), W4(v, 12)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(addr),
      W4(v, 0), W4(v, 4), W4(v, 8), W4(v, 12), W4(v, 16), W4(v, 20), W4(v, 24), W4(v, 28)
      : "memory");
}
#undef W4
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

struct Bars {
  uint64_t k_full[2], v_full[2];       // converters -> MMA
  uint64_t k_free[2], v_free[2];       // MMA -> converters
  uint64_t s_full[2];                  // MMA -> group: S of the next tile (and every earlier product) is complete
  uint64_t p_full[2];                  // group -> MMA: P is written
  uint64_t done[2];                    // MMA -> group: all products complete
  uint64_t meta[4];                    // converters -> groups: a tile's scales
  uint64_t drain;
};

// Shared by the roles of one CTA.
struct Slice {
  float k, lv, iv;                     // key scale, log2 and reciprocal of the value scale
};

template <typename T, int D>
__global__ void __launch_bounds__(PF_THREADS, 1) paged_prefill_kernel(const AttnParams p) {
  using L = Layout<D>;
  extern __shared__ uint8_t raw[];
  __shared__ Bars bar;
  __shared__ Slice meta[4][SLICES];    // a tile's slot is written again four tiles later: no reader is left by then
  __shared__ uint32_t s_tmem;
  __shared__ int s_pre[MAX_REQ + 1];
  __shared__ int s_wsum[PF_THREADS / 32];
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const uint32_t smem = (smem_u32(raw) + 1023) & ~1023u;

  // tiles before each request
  const int per = (p.n_req + PF_THREADS - 1) / PF_THREADS;
  int sum = 0;
  for (int i = 0; i < per; ++i) {
    const int r = t * per + i;
    if (r >= p.n_req) break;
    sum += (request(p, r, blockIdx.x == 0).q_len * p.g + ROWS - 1) / ROWS;
    s_pre[r + 1] = sum;
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) s_wsum[w] = inc;
  if (t == 0) s_pre[0] = 0;
  __syncthreads();
  int base = inc - sum, total = 0;
  for (int k = 0; k < PF_THREADS / 32; ++k) {
    if (k < w) base += s_wsum[k];
    total += s_wsum[k];
  }
  for (int i = 0; i < per; ++i) {
    const int r = t * per + i;
    if (r >= p.n_req) break;
    s_pre[r + 1] += base;
  }
  __syncthreads();
  // later tiles see more keys: they start first
  const int h = blockIdx.x % p.nkv, tile = total - 1 - blockIdx.x / p.nkv;
  if (tile < 0) return;
  int r = 0;
  for (int b = p.n_req; b - r > 1;) {
    const int mid = (r + b) / 2;
    if (s_pre[mid] <= tile) r = mid;
    else b = mid;
  }
  const Req x = request(p, r, false);
  const int row0 = (tile - s_pre[r]) * ROWS;
  const int n_here = min(ROWS, x.q_len * p.g - row0);
  const int behind = x.kv - x.q_len;
  const int lim_hi = behind + (row0 + n_here - 1) / p.g;         // last key that any row sees
  const int n_tiles = lim_hi < 0 ? 0 : lim_hi / KT + 1;
  const bool two = n_here > GROUP_ROWS;

  if (w == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (t == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bar.k_full[i], 4);
      mbar_init(&bar.v_full[i], 4);
      mbar_init(&bar.k_free[i], 1);
      mbar_init(&bar.v_free[i], 1);
      mbar_init(&bar.s_full[i], 1);
      mbar_init(&bar.p_full[i], GROUP_ROWS);
      mbar_init(&bar.done[i], 1);
    }
    for (int i = 0; i < 4; ++i) mbar_init(&bar.meta[i], 1);
    mbar_init(&bar.drain, 1);
    mbar_fence_init();
  }

  // queries: a thread has a row
  float fac = 0.0f;
  int lim = -1;
  int64_t out_at = -1, lse_at = 0;
  if (w < 8) {
    float v[8];
    const bool live = t < n_here;
    const T* q = static_cast<const T*>(p.q);
    if (live) {
      const int tok = (row0 + t) / p.g, head = h * p.g + (row0 + t) % p.g;
      lim = behind + tok;
      q += (int64_t)(x.q0 + tok) * p.q_row + head * p.q_head;
      out_at = (int64_t)(x.q0 + tok) * p.o_row + head * p.o_head;
      lse_at = (int64_t)(x.q0 + tok) * p.nq + head;
    }
    const bool vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0;
    auto load8 = [&](int e) {
      if (!live) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.0f;
      } else if (vec) {
        const uint4 a = __ldg(reinterpret_cast<const uint4*>(q + e));
        const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = unpack2<T>(aw[k]);
          v[2 * k] = f.x;
          v[2 * k + 1] = f.y;
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = load_f<T>(q + e + k);
      }
    };
    // the factor stays positive (a maximum is taken before it is applied); the sign goes to the query
    float up = p.scale2 < 0.0f ? -1.0f : 1.0f;
    fac = fabsf(p.scale2);
    if constexpr (!std::is_same<T, __half>::value) {
      float top = 0.0f;
      for (int e = 0; e < D; e += 8) {
        load8(e);
#pragma unroll
        for (int k = 0; k < 8; ++k) top = fmaxf(top, fabsf(v[k]));
      }
      const int k = min(126, 135 - (int)(__float_as_uint(top) >> 23));     // top * 2^k in [2^8, 2^9)
      up *= __uint_as_float((uint32_t)(k + 127) << 23);
      fac *= __uint_as_float((uint32_t)(127 - k) << 23);
    }
    const int row = t & (GROUP_ROWS - 1);
    const uint32_t dst = smem + L::Q + (t >> 7) * L::TILE + row * 128;
#pragma unroll
    for (int e = 0; e < D; e += 8) {
      load8(e);
      const int c = e / 8;
      sts16(dst + (c / 8) * L::BLOCK + (((c % 8) ^ (row & 7)) << 4), pack2<__half>(v[0] * up, v[1] * up),
            pack2<__half>(v[2] * up, v[3] * up), pack2<__half>(v[4] * up, v[5] * up),
            pack2<__half>(v[6] * up, v[7] * up));
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = s_tmem;
  bool ok = true;

  if (w < 8) {
    // ---- softmax: group g2, one row a thread --------------------------------
    const int g2 = w >> 2;
    if (g2 == 0 || two) {
      const uint32_t at_s = tmem + ((uint32_t)(w & 3) << 21) + 128 * g2, at_o = at_s + 256;
      const int lim_first = behind + (row0 + GROUP_ROWS * g2) / p.g;
      float m = M_NONE, l = 0.0f;
      uint32_t s[32];
      for (int j = 0; j < n_tiles; ++j) {
        ok = ok && mbar_wait(&bar.meta[j & 3], (j >> 2) & 1, PF_WAIT_NS);
        ok = ok && mbar_wait(&bar.s_full[g2], j & 1, PF_WAIT_NS);
        if (!__all_sync(0xffffffffu, ok)) break;
        fence_after();
        const Slice* sl = meta[j & 3];
        const bool masked = j * KT + KT - 1 > lim_first;
        const int last = lim - j * KT;                  // columns past it are not seen
        float top = -INFINITY;
#pragma unroll
        for (int c0 = 0; c0 < KT; c0 += 32) {
          tmem_ld32(at_s + c0, s);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            float mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 16; ++c) {
              float v = __uint_as_float(s[16 * hf + c]);
              if (masked && c0 + 16 * hf + c > last) v = -INFINITY;
              mx = fmaxf(mx, v);
            }
            const Slice& q = sl[c0 / 16 + hf];
            top = fmaxf(top, fmaf(mx, q.k * fac, q.lv));
          }
        }
        if (__any_sync(0xffffffffu, top > m + 8.0f)) {
          const float m1 = fmaxf(m, top), keep = ex2(m - m1);
          m = m1;
          l *= keep;
          if (j > 0) {                                  // S of this tile is complete, so the products before it are
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += 32) {
              tmem_ld32(at_o + c0, s);
#pragma unroll
              for (int c = 0; c < 32; ++c) s[c] = __float_as_uint(__uint_as_float(s[c]) * keep);
              tmem_st32(at_o + c0, s);
            }
          }
        }
#pragma unroll
        for (int c0 = 0; c0 < KT; c0 += 32) {
          tmem_ld32(at_s + c0, s);
          uint32_t pk[16];
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            const Slice& q = sl[c0 / 16 + hf];
            const float f = q.k * fac, d = q.lv - m;
            float part = 0.0f;
#pragma unroll
            for (int c = 0; c < 16; c += 2) {
              float a = ex2(fmaf(__uint_as_float(s[16 * hf + c]), f, d));
              float b = ex2(fmaf(__uint_as_float(s[16 * hf + c + 1]), f, d));
              if (masked) {
                if (c0 + 16 * hf + c > last) a = 0.0f;
                if (c0 + 16 * hf + c + 1 > last) b = 0.0f;
              }
              part += a + b;
              pk[8 * hf + c / 2] = pack2<__half>(a, b);
            }
            l = fmaf(part, q.iv, l);
          }
          tmem_st16(at_s + c0 / 2, pk);
        }
        tmem_wait_st();
        fence_before();
        mbar_arrive(&bar.p_full[g2]);
      }
      if (n_tiles > 0) {
        ok = ok && mbar_wait(&bar.done[g2], 0, PF_WAIT_NS);
        ok = __all_sync(0xffffffffu, ok);
        fence_after();
      }
      T* out = static_cast<T*>(p.out) + out_at;
      const bool vec = (reinterpret_cast<uintptr_t>(out) & 15) == 0;
      const float inv = l > 0.0f ? __frcp_rn(l) : l;    // no key: 0, and NaN stays NaN
#pragma unroll 1
      for (int c0 = 0; c0 < D; c0 += 32) {
        if (n_tiles > 0 && ok) {
          tmem_ld32(at_o + c0, s);
        } else {
#pragma unroll
          for (int c = 0; c < 32; ++c) s[c] = 0u;
        }
        if (out_at >= 0) {
#pragma unroll
          for (int c = 0; c < 32; c += 8) {
            uint32_t o[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              o[k] = l == 0.0f ? 0u
                               : pack2<T>(__uint_as_float(s[c + 2 * k]) * inv, __uint_as_float(s[c + 2 * k + 1]) * inv);
            if (vec) {
              *reinterpret_cast<uint4*>(out + c0 + c) = make_uint4(o[0], o[1], o[2], o[3]);
            } else {
              const T* e = reinterpret_cast<const T*>(o);
#pragma unroll
              for (int k = 0; k < 8; ++k) out[c0 + c + k] = e[k];
            }
          }
        }
      }
      if (out_at >= 0 && p.lse) p.lse[lse_at] = l == 0.0f ? -INFINITY : (m + __log2f(l)) * LN2;
    }
  } else if (w < 12) {
    // ---- converters: e4m3 pages -> f16 operand tiles -------------------------
    constexpr int PIECES = D / 16;                      // 16-byte pieces of a key row
    constexpr int KEYS = 128 / PIECES;                  // keys that the 128 threads cover at once
    constexpr int N = KT / KEYS;                        // pieces per thread
    const int ct = t - 256, piece = ct % PIECES, key0 = ct / PIECES;
    uint4 kr[N], vr[N];
    // a lane's page and scales of slice `lane` of a tile
    auto page_of = [&](int j) {
      int page = -1;
      const int key = j * KT + (lane & (SLICES - 1)) * 16;
      if (key <= lim_hi) {
        page = __ldg(p.tables + (int64_t)r * p.t_stride + (key >> p.page_log2));
        if (page < 0 || page >= p.n_pages) {
          if (p.status) atomicOr(p.status, HC_ERR_RANGE);
          page = -1;
        }
      }
      return page;
    };
    auto load = [&](const uint8_t* pool, int j, int page, uint4 (&v)[N]) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int kk = key0 + KEYS * i, key = j * KT + kk;
        const int pg = __shfl_sync(0xffffffffu, page, kk / 16);
        v[i] = make_uint4(0u, 0u, 0u, 0u);
        if (pg >= 0 && key <= lim_hi)
          v[i] = __ldg(reinterpret_cast<const uint4*>(
              pool + ((((int64_t)pg * p.nkv + h) << p.page_log2) + (key & ((1 << p.page_log2) - 1))) * D + 16 * piece));
      }
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
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    };
    int page = -1;
    if (n_tiles > 0) {
      page = page_of(0);
      load(p.kp, 0, page, kr);
      load(p.vp, 0, page, vr);
    }
    for (int j = 0; j < n_tiles; ++j) {
      const int st = j & 1;
      Slice mine = {0.0f, 0.0f, 0.0f};
      if (w == 8 && lane < SLICES && page >= 0) {
        const float a = __ldg(p.ks + (int64_t)page * p.nkv + h);
        const float b = fmaxf(__ldg(p.vs + (int64_t)page * p.nkv + h), 1e-30f);
        mine.k = a;
        mine.lv = __log2f(b);
        mine.iv = __frcp_rn(b);
      } else if (page < 0) {
        mine.lv = -INFINITY;                            // no page: no weight
      }
      const int next = j + 1 < n_tiles ? page_of(j + 1) : -1;
      if (j >= 2) ok = ok && mbar_wait(&bar.k_free[st], ((j >> 1) - 1) & 1, PF_WAIT_NS);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (w == 8 && lane < SLICES) meta[j & 3][lane] = mine;
      store(smem + L::K + st * L::TILE, kr);
      if (lane == 0) {                                  // after store()'s __syncwarp
        if (w == 8) mbar_arrive(&bar.meta[j & 3]);
        mbar_arrive(&bar.k_full[st]);
      }
      if (j + 1 < n_tiles) load(p.kp, j + 1, next, kr);
      if (j >= 2) ok = ok && mbar_wait(&bar.v_free[st], ((j >> 1) - 1) & 1, PF_WAIT_NS);
      if (!__all_sync(0xffffffffu, ok)) break;
      store(smem + L::V + st * L::TILE, vr);
      if (lane == 0) mbar_arrive(&bar.v_full[st]);
      if (j + 1 < n_tiles) load(p.vp, j + 1, next, vr);
      page = next;
    }
  } else if (n_tiles > 0) {
    // ---- MMA: one thread issues -----------------------------------------------
    if (lane == 0) {
      constexpr uint32_t id_s = pf_idesc(KT, 0), id_o = pf_idesc(D, 1);
      auto scores = [&](int g2, int j) {
        const uint32_t q = smem + L::Q + g2 * L::TILE, k = smem + L::K + (j & 1) * L::TILE;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
          const uint32_t at = (i / 4) * L::BLOCK + (i % 4) * 32;
          mma_ss(tmem + 128 * g2, sw128_desc(q + at, 16, 1024), sw128_desc(k + at, 16, 1024), id_s, i > 0);
        }
      };
      auto values = [&](int g2, int j) {
        const uint32_t v = smem + L::V + (j & 1) * L::TILE;
#pragma unroll
        for (int i = 0; i < KT / 16; ++i)
          mma_ts(tmem + 256 + 128 * g2, tmem + 128 * g2 + 8 * i, sw128_desc(v + 2048 * i, L::BLOCK, 1024), id_o,
                 j > 0 || i > 0);
      };
      ok = mbar_wait(&bar.k_full[0], 0, PF_WAIT_NS);
      if (ok) {
        fence_after();
        scores(0, 0);
        mma_commit(&bar.s_full[0]);
        if (two) {
          scores(1, 0);
          mma_commit(&bar.s_full[1]);
        }
        mma_commit(&bar.k_free[0]);
        for (int j = 0; j < n_tiles && ok; ++j) {
          const bool more = j + 1 < n_tiles;
          ok = mbar_wait(&bar.v_full[j & 1], (j >> 1) & 1, PF_WAIT_NS);
          if (more) ok = ok && mbar_wait(&bar.k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, PF_WAIT_NS);
          for (int g2 = 0; g2 < (two ? 2 : 1) && ok; ++g2) {
            ok = mbar_wait(&bar.p_full[g2], j & 1, PF_WAIT_NS);
            if (!ok) break;
            fence_after();
            values(g2, j);
            if (more) {
              scores(g2, j + 1);
              mma_commit(&bar.s_full[g2]);
            } else {
              mma_commit(&bar.done[g2]);
            }
          }
          if (!ok) break;
          mma_commit(&bar.v_free[j & 1]);
          if (more) mma_commit(&bar.k_free[(j + 1) & 1]);
        }
      }
      // every product that was issued has completed before the CTA gives up its memory
      mma_commit(&bar.drain);
      mbar_wait(&bar.drain, 0, PF_WAIT_NS);
    }
  }
  if (!ok && p.status) atomicOr(p.status, HC_ERR_TIMEOUT);
  fence_before();
  __syncthreads();
  fence_after();
  if (w == 12)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

template <typename T, int D>
int launch_pf(const AttnParams& p, cudaStream_t stream) {
  using L = Layout<D>;
  if (cudaFuncSetAttribute(paged_prefill_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, L::BYTES) !=
      cudaSuccess)
    return HC_ERR_CUDA;
  // the lengths are on the device: as many tiles as any lengths of these rows can need
  const int64_t tiles = ((int64_t)p.n_rows * p.g + ROWS - 1) / ROWS + min(p.n_req, p.n_rows);
  if (tiles * p.nkv > INT32_MAX) return HC_ERR_UNSUPPORTED;
  paged_prefill_kernel<T, D><<<(unsigned)(tiles * p.nkv), PF_THREADS, L::BYTES, stream>>>(p);
  return cudaGetLastError() == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

int launch_prefill(const AttnParams& p, int dtype, int head_dim, cudaStream_t stream) {
  if (dtype == HC_F16)
    return head_dim == 128 ? launch_pf<__half, 128>(p, stream) : launch_pf<__half, 64>(p, stream);
  return head_dim == 128 ? launch_pf<__nv_bfloat16, 128>(p, stream) : launch_pf<__nv_bfloat16, 64>(p, stream);
}

}  // namespace hca8
