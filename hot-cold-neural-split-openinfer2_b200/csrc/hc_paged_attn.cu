// Causal attention of a step's rows over the paged 8-bit cache.
//
// The query heads that share a key-value head and a request's new tokens are
// the rows of one problem: row n is token n / g, head n % g (g query heads per
// key-value head).  A work item is (request, key-value head, tile of RT rows);
// its keys are taken 16 at a time (a chunk), and the chunks of all items form
// one list that is cut into equal contiguous shares, one per CTA.  Ragged
// lengths and few long requests then load every SM alike.  An item that a cut
// divides leaves one partial softmax per share in the workspace; a second,
// programmatically launched kernel joins those.
//
// Softmax over keys j with page scales ks, vs:
//   s_j = scale ks_j (q . k_j),  out = sum_j e^{s_j} vs_j v_j / sum_j e^{s_j}
// where k_j, v_j are the raw e4m3 numbers (exact in f16).  In base 2, with
// t_j = s_j log2(e) + log2(vs_j) and a running reference m: p_j = 2^{t_j - m}
// is the weight of v_j and p_j / vs_j its share of the denominator, so the
// value scale costs nothing.  p is rounded to f16 for the product: relative
// 2^-11, like the output, down to 2^-25 of the row's largest weight, and by
// 2^-36 of that one at most below (W_REF in hc_paged_attn.cuh); a row of many
// small weights beside one large one needs that room.
//
// Bound by HBM, each cached byte read once (in a graph; 32 / 8 heads of 128): 4
// requests of 60,000 to 131,000 keys 134 to 141 us by the run (5.5 to 5.8 TB/s; a
// copy of this loop that only loads takes 132); 64 requests of 100 to 8000 keys
// 96 to 99 us (5.4 to 5.6 TB/s).  With 9 to 16 rows an item (NT = 2) the latter
// take 129 us: 232 registers leave two CTAs an SM, and with them a third fewer
// loads in flight (HBM at 53% of its peak, 70% with NT = 1).  Three CTAs of four
// warps on an SM; two, eight warps each, were slower, and so were shares of a
// half or a quarter of this length (more items are cut).
#include "hc_paged_attn.cuh"

namespace hca8 {

constexpr int CHUNK = 16;              // keys per chunk; no page is smaller
constexpr int THREADS = 128;
constexpr int WARPS = THREADS / 32;
constexpr int STAGES = 3;              // chunks in flight per warp
constexpr int ITEM_COST = 16;          // what beginning an item costs, in chunks
// Rows of a request and head that these kernels take: two MMA columns of 8.  64 requests of 100 to 8000 keys with
// 16 rows take 129 us here; with 20 rows the tiles of hc_paged_prefill.cu take 276 us, with 64 rows 280.
constexpr int SMALL = 16;
constexpr int MIN_SHARE = 2 * WARPS;   // units of a share at least

__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
// d[16x8] += a[16x16] b[16x8], f16 operands, fp32 sums
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// Byte offset of 16-byte piece x of key row `key` in a chunk of [16][D] bytes.
// The pieces are permuted by the key so that the fragment reads below touch
// every bank once (D = 128) or twice (values at D = 64).
template <int D>
__device__ __forceinline__ uint32_t piece_at(int key, int x) {
  return D == 128 ? key * 128 + ((x ^ (key & 7)) << 4) : key * 64 + ((x ^ ((key >> 1) & 3)) << 4);
}

template <typename T, int D, int NT>
struct Cfg {
  static constexpr int RT = 8 * NT;                            // rows of an item
  static constexpr int RING = WARPS * STAGES * CHUNK * D * 2;  // bytes
  static constexpr int PART = RT * (D + 2);                    // floats of one partial
};

// four dims of one output row from its sums
template <typename T>
__device__ __forceinline__ void write_row(const AttnParams& p, int tok, int head, int d, float M, float L, float a0,
                                          float a1, float a2, float a3) {
  const float inv = L > 0.0f ? __frcp_rn(L) : L;                     // no key: 0, and NaN stays NaN
  T* out = static_cast<T*>(p.out) + (int64_t)tok * p.o_row + head * p.o_head + d;
  const uint32_t w0 = pack2<T>(a0 * inv, a1 * inv), w1 = pack2<T>(a2 * inv, a3 * inv);
  if ((reinterpret_cast<uintptr_t>(out) & 7) == 0) {
    *reinterpret_cast<uint2*>(out) = make_uint2(w0, w1);
  } else {
    const T* a = reinterpret_cast<const T*>(&w0);
    const T* b = reinterpret_cast<const T*>(&w1);
    out[0] = a[0];
    out[1] = a[1];
    out[2] = b[0];
    out[3] = b[1];
  }
  if (p.lse && d == 0) p.lse[(int64_t)tok * p.nq + head] = L == 0.0f ? -INFINITY : (M + __log2f(L)) * LN2;
}

// MMA shapes: S^T[16 keys][8 rows] = K Q^T and O^T[16 dims][8 rows] += V^T P^T,
// so 8 rows fill an MMA's N and keys or dims its M.  Both inner dimensions may
// be permuted freely as long as the two operands agree: lane (i, c) = (lane / 4,
// lane % 4) takes dims [D/4 c, D/4 (c + 1)) of keys i, i + 8 and dims [D/8 i,
// D/8 (i + 1)) of values 2c, 2c + 1, 2c + 8, 2c + 9, each contiguous in a row.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 3 : 2) paged_attn_kernel(const AttnParams p) {
  using C = Cfg<T, D, NT>;
  constexpr int RT = C::RT;
  constexpr int KS = D / 16;           // k steps of S, also m tiles of O
  constexpr int KW = D / 16;           // words of a key row per lane
  constexpr int VW = D / 32;           // words of a value row per lane
  extern __shared__ __align__(16) uint8_t ring[];
  int64_t* s_pre = reinterpret_cast<int64_t*>(ring + C::RING);       // [n_req + 1]
  __shared__ int64_t s_wsum[WARPS];
  __shared__ Req s_req[KEPT_REQ];
  __shared__ float s_m[WARPS][RT], s_l[WARPS][RT];
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  const int i8 = lane >> 2, c4 = lane & 3;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // chunks before each request
  const int per = (p.n_req + THREADS - 1) / THREADS;
  int64_t sum = 0;
  for (int i = 0; i < per; ++i) {
    const int r = t * per + i;
    if (r >= p.n_req) break;
    const Req x = request(p, r, blockIdx.x == 0);
    if (p.n_req <= KEPT_REQ) s_req[r] = x;
    const int64_t tiles = (x.q_len * p.g + RT - 1) / RT;
    sum += tiles * p.nkv * (ITEM_COST + max(1, (x.kv + CHUNK - 1) / CHUNK));
    s_pre[r + 1] = sum;
  }
  int64_t inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) s_wsum[w] = inc;
  if (t == 0) s_pre[0] = 0;
  __syncthreads();
  int64_t base = inc - sum, total = 0;
#pragma unroll
  for (int k = 0; k < WARPS; ++k) {
    if (k < w) base += s_wsum[k];
    total += s_wsum[k];
  }
  for (int i = 0; i < per; ++i) {
    const int r = t * per + i;
    if (r >= p.n_req) break;
    s_pre[r + 1] += base;
  }
  __syncthreads();
  const int parts = (int)max((int64_t)1, min((int64_t)gridDim.x, total / MIN_SHARE));
  const int cta = blockIdx.x;
  if (cta >= parts || total == 0) {
    if (t == 0) p.cuts[2 * cta] = make_int4(0, 0, 0, 0);
    return;
  }
  const int64_t lo = (int64_t)((uint64_t)total * cta / parts), hi = (int64_t)((uint64_t)total * (cta + 1) / parts);
  if (t == 0) p.cuts[2 * cta] = make_int4(0, 0, 0, 0);

  const uint32_t my_ring = smem_u32(ring) + w * (STAGES * CHUNK * D * 2);
  int64_t u = lo;
  while (u < hi) {
    // the item that holds unit u: ITEM_COST units, then its chunks
    int r = 0;
    for (int b = p.n_req; b - r > 1;) {
      const int mid = (r + b) / 2;
      if (s_pre[mid] <= u) r = mid;
      else b = mid;
    }
    const Req x = p.n_req <= KEPT_REQ ? s_req[r] : request(p, r, false);
    const int n_chunks = max(1, (x.kv + CHUNK - 1) / CHUNK);
    const int rows = x.q_len * p.g, tiles = (rows + RT - 1) / RT;
    const uint64_t off = (uint64_t)(u - s_pre[r]);
    const uint32_t span = n_chunks + ITEM_COST;
    const int item = (int)(off / span), pos = (int)(off - (uint64_t)item * span) - ITEM_COST;
    const int c0 = max(0, pos), c1 = (int)min((int64_t)n_chunks, pos + (hi - u));
    u += c1 - pos;
    if (c1 <= c0) continue;            // the share ends before the item's first chunk
    const int h = item / tiles, row0 = (item % tiles) * RT;
    const int n_here = min(RT, rows - row0);
    // key index of the last key that the first and the last row see
    const int behind = x.kv - x.q_len;
    const int lim_lo = behind + row0 / p.g, lim_hi = behind + (row0 + n_here - 1) / p.g;
    const int c_end = min(c1, lim_hi < 0 ? 0 : lim_hi / CHUNK + 1);

    // This warp's chunks: c0 + w + WARPS k, k < count.  Lane k % 32 holds chunk
    // k's place in the pools (in chunks; NONE without a page), its key scale
    // and the logarithm and reciprocal of its value scale; two sets, for the
    // even and odd 32 chunks.  The first loads start before anything else.
    const int count = c_end > c0 + w ? (c_end - c0 - w + WARPS - 1) / WARPS : 0;
    uint32_t at_[2];
    float sk[2], sl[2], si[2];
    auto load_places = [&](int batch, int set) {
      const int k = batch * 32 + lane;
      uint32_t at = NONE;
      if (k < count) {
        const int key = (c0 + w + WARPS * k) * CHUNK;
        const int page = __ldg(p.tables + (int64_t)r * p.t_stride + (key >> p.page_log2));
        if (page < 0 || page >= p.n_pages) {
          if (p.status) atomicOr(p.status, HC_ERR_RANGE);
        } else {
          at = (uint32_t)(((((int64_t)page * p.nkv + h) << p.page_log2) + (key & ((1 << p.page_log2) - 1))) / CHUNK);
        }
      }
      if (set) at_[1] = at;
      else at_[0] = at;
    };
    auto load_scales = [&](int set) {
      const uint32_t at = set ? at_[1] : at_[0];
      float a = 0.0f, b = 1.0f;
      if (at != NONE) {
        const uint32_t head = at >> (p.page_log2 - 4);           // page * nkv + h
        a = __ldg(p.ks + head);
        b = fmaxf(__ldg(p.vs + head), VS_MIN);
      }
      const float lb = __log2f(b), ib = __frcp_rn(b);
      if (set) sk[1] = a, sl[1] = lb, si[1] = ib;
      else sk[0] = a, sl[0] = lb, si[0] = ib;
    };
    auto issue = [&](int k) {
      const uint32_t at = __shfl_sync(0xffffffffu, (k >> 5) & 1 ? at_[1] : at_[0], k & 31);
      if (k < count && at != NONE) {
        const uint32_t dst = my_ring + (k % STAGES) * (CHUNK * D * 2);
        const uint8_t* ksrc = p.kp + (uint64_t)at * (CHUNK * D) + lane * 16;
        const uint8_t* vsrc = p.vp + (uint64_t)at * (CHUNK * D) + lane * 16;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const int b = (j * 32 + lane) * 16;
          const uint32_t s = piece_at<D>(b / D, (b % D) / 16);
          cp16(dst + s, ksrc + j * 512);
          cp16(dst + CHUNK * D + s, vsrc + j * 512);
        }
      }
      cp_commit();
    };
    load_places(0, 0);
#pragma unroll
    for (int k = 0; k < STAGES - 1; ++k) issue(k);

    // this lane's part of its query row(s), in f16, and the rows' factors
    uint32_t qf[NT][KS][2];
    float fac[NT][2];
    int lim[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int n = nt * 8 + i8;
      float v[D / 4];
#pragma unroll
      for (int e = 0; e < D / 4; ++e) v[e] = 0.0f;
      if (n < n_here) {
        const int tok = (row0 + n) / p.g, head = h * p.g + (row0 + n) % p.g;
        const T* q = static_cast<const T*>(p.q) + (int64_t)(x.q0 + tok) * p.q_row + head * p.q_head + (D / 4) * c4;
        if ((reinterpret_cast<uintptr_t>(q) & 15) == 0) {
#pragma unroll
          for (int e = 0; e < D / 4; e += 8) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(q + e));
            const uint32_t aw[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const float2 f = unpack2<T>(aw[k]);
              v[e + 2 * k] = f.x;
              v[e + 2 * k + 1] = f.y;
            }
          }
        } else {
#pragma unroll
          for (int e = 0; e < D / 4; ++e) v[e] = load_f<T>(q + e);
        }
      }
      float f = p.scale2;
      if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
        // bf16: a power of two per row brings it into f16's range
        float top = 0.0f;
#pragma unroll
        for (int e = 0; e < D / 4; ++e) top = fmaxf(top, fabsf(v[e]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const int k = min(126, 135 - (int)(__float_as_uint(top) >> 23));     // top * 2^k in [2^8, 2^9)
        const float up = __uint_as_float((uint32_t)(k + 127) << 23);
#pragma unroll
        for (int e = 0; e < D / 4; ++e) v[e] *= up;
        f *= __uint_as_float((uint32_t)(127 - k) << 23);
      }
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        qf[nt][s][0] = pack2<__half>(v[4 * s], v[4 * s + 1]);
        qf[nt][s][1] = pack2<__half>(v[4 * s + 2], v[4 * s + 3]);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        fac[nt][e] = __shfl_sync(0xffffffffu, f, (2 * c4 + e) * 4);
        const int m = nt * 8 + 2 * c4 + e;
        lim[nt][e] = m < n_here ? behind + (row0 + m) / p.g : -1;
      }
    }

    float m[NT][2], l[NT][2], o[NT][KS][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        m[nt][e] = M_NONE;
        l[nt][e] = 0.0f;
      }
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[nt][k][e] = 0.0f;
    }

    load_places(1, 1);
    load_scales(0);
    load_scales(1);
    for (int k = 0; k < count; ++k) {
      cp_wait<STAGES - 2>();
      __syncwarp();
      issue(k + STAGES - 1);
      const int set = (k >> 5) & 1;
      const uint32_t at = __shfl_sync(0xffffffffu, set ? at_[1] : at_[0], k & 31);
      const float kscale = __shfl_sync(0xffffffffu, set ? sk[1] : sk[0], k & 31);
      const float lv = __shfl_sync(0xffffffffu, set ? sl[1] : sl[0], k & 31);
      const float iv = __shfl_sync(0xffffffffu, set ? si[1] : si[0], k & 31);
      const int key0 = (c0 + w + WARPS * k) * CHUNK;
      if ((k & 31) == 31) {
        load_places((k >> 5) + 2, set);
        load_scales(set);
      }
      if (at == NONE) continue;
      const uint32_t kb = my_ring + (k % STAGES) * (CHUNK * D * 2), vb = kb + CHUNK * D;

      // S^T
      uint32_t kw[2][KW];
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int j = 0; j < KW / 4; ++j) {
          const uint4 v = lds128(kb + piece_at<D>(i8 + 8 * e, (KW / 4) * c4 + j));
          kw[e][4 * j] = v.x;
          kw[e][4 * j + 1] = v.y;
          kw[e][4 * j + 2] = v.z;
          kw[e][4 * j + 3] = v.w;
        }
      float s[NT][4], s1[NT][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[nt][e] = s1[nt][e] = 0.0f;
#pragma unroll
      for (int j = 0; j < KS; ++j) {
        const uint32_t a0 = e4m3x2_to_f16x2(kw[0][j]), a2 = e4m3x2_to_f16x2(kw[0][j] >> 16);
        const uint32_t a1 = e4m3x2_to_f16x2(kw[1][j]), a3 = e4m3x2_to_f16x2(kw[1][j] >> 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
          mma16816(j & 1 ? s1[nt] : s[nt], a0, a1, a2, a3, qf[nt][j][0], qf[nt][j][1]);
      }

      // weights
      const bool masked = key0 + CHUNK - 1 > lim_lo;
      bool over = false;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = fmaf(s[nt][e] + s1[nt][e], fac[nt][e & 1] * kscale, lv);
          if (masked && key0 + i8 + (e >> 1) * 8 > lim[nt][e & 1]) v = -INFINITY;
          s[nt][e] = v;
          over |= v > m[nt][e & 1] + W_MAX;
        }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = fmaxf(s[nt][e], s[nt][e + 2]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            top = fmaxf(top - W_REF, m[nt][e]);
            const float keep = ex2(m[nt][e] - top);
            m[nt][e] = top;
            l[nt][e] *= keep;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
              o[nt][j][e] *= keep;
              o[nt][j][e + 2] *= keep;
            }
          }
      }
      uint32_t pb[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[nt][e] = ex2(s[nt][e] - m[nt][e & 1]);
          l[nt][e & 1] = fmaf(s[nt][e], iv, l[nt][e & 1]);
        }
        pb[nt][0] = transpose8x8(pack2<__half>(s[nt][0], s[nt][1]));
        pb[nt][1] = transpose8x8(pack2<__half>(s[nt][2], s[nt][3]));
      }

      // O^T
      uint32_t vw[4][VW];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int key = 2 * c4 + (e & 1) + (e >> 1) * 8;
        if constexpr (D == 128) {
          const uint4 v = lds128(vb + piece_at<D>(key, i8));
          vw[e][0] = v.x;
          vw[e][1] = v.y;
          vw[e][2] = v.z;
          vw[e][3] = v.w;
        } else {
          const uint2 v = lds64(vb + piece_at<D>(key, i8 >> 1) + 8 * (i8 & 1));
          vw[e][0] = v.x;
          vw[e][1] = v.y;
        }
        if (key0 + CHUNK - 1 > lim_hi && key0 + key > lim_hi) {      // a weight of 0 times a NaN is not 0
#pragma unroll
          for (int j = 0; j < VW; ++j) vw[e][j] = 0u;
        }
      }
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        const uint32_t x0 = __byte_perm(vw[0][j], vw[1][j], 0x5140), x1 = __byte_perm(vw[0][j], vw[1][j], 0x7362);
        const uint32_t y0 = __byte_perm(vw[2][j], vw[3][j], 0x5140), y1 = __byte_perm(vw[2][j], vw[3][j], 0x7362);
        const uint32_t f0 = e4m3x2_to_f16x2(x0), f1 = e4m3x2_to_f16x2(x0 >> 16);
        const uint32_t f2 = e4m3x2_to_f16x2(y0), f3 = e4m3x2_to_f16x2(y0 >> 16);
        const uint32_t g0 = e4m3x2_to_f16x2(x1), g1 = e4m3x2_to_f16x2(x1 >> 16);
        const uint32_t g2 = e4m3x2_to_f16x2(y1), g3 = e4m3x2_to_f16x2(y1 >> 16);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          mma16816(o[nt][2 * j], f0, f1, f2, f3, pb[nt][0], pb[nt][1]);
          mma16816(o[nt][2 * j + 1], g0, g1, g2, g3, pb[nt][0], pb[nt][1]);
        }
      }
    }
    cp_wait<0>();
    __syncwarp();

    // the warps' partials, joined in shared memory (each in its own part of the ring)
    float* mine = reinterpret_cast<float*>(ring + w * (STAGES * CHUNK * D * 2));
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float sum_l = l[nt][e];
        sum_l += __shfl_xor_sync(0xffffffffu, sum_l, 4);
        sum_l += __shfl_xor_sync(0xffffffffu, sum_l, 8);
        sum_l += __shfl_xor_sync(0xffffffffu, sum_l, 16);
        const int row = nt * 8 + 2 * c4 + e;
        if (i8 == 0) {
          s_m[w][row] = m[nt][e];
          s_l[w][row] = sum_l;
        }
        float* at = mine + row * D + (D / 8) * i8;
#pragma unroll
        for (int j = 0; j < KS; j += 2)
          *reinterpret_cast<float4*>(at + 2 * j) =
              make_float4(o[nt][j][e], o[nt][j][e + 2], o[nt][j + 1][e], o[nt][j + 1][e + 2]);
      }
    __syncthreads();
    const bool whole = c0 == 0 && c1 == n_chunks;
    float* part = p.part + (int64_t)(2 * cta + (c0 == 0 ? 1 : 0)) * C::PART;
    for (int e = t; e < RT * D / 4; e += THREADS) {
      const int row = e / (D / 4), d = (e % (D / 4)) * 4;
      float M = s_m[0][row];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) M = fmaxf(M, s_m[k][row]);
      float L = 0.0f, a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
#pragma unroll
      for (int k = 0; k < WARPS; ++k) {
        const float f = ex2(s_m[k][row] - M);
        const float4 v = *reinterpret_cast<const float4*>(ring + k * (STAGES * CHUNK * D * 2) + (row * D + d) * 4);
        L = fmaf(s_l[k][row], f, L);
        a0 = fmaf(v.x, f, a0);
        a1 = fmaf(v.y, f, a1);
        a2 = fmaf(v.z, f, a2);
        a3 = fmaf(v.w, f, a3);
      }
      if (whole) {
        if (row < n_here)
          write_row<T>(p, x.q0 + (row0 + row) / p.g, h * p.g + (row0 + row) % p.g, d, M, L, a0, a1, a2, a3);
      } else {
        *reinterpret_cast<float4*>(part + row * D + d) = make_float4(a0, a1, a2, a3);
        if (d == 0) {
          part[RT * D + row] = M;
          part[RT * D + RT + row] = L;
        }
      }
    }
    if (!whole && c0 == 0 && t == 0) {
      // the item's first piece: the pieces of CTAs cta .. last belong to it
      const int last = (int)(((uint64_t)(u + n_chunks - c1) * parts - 1) / (uint64_t)total);
      p.cuts[2 * cta] = make_int4(r, h, row0, last - cta + 1);
      p.cuts[2 * cta + 1] = make_int4(n_here, x.q0, 0, 0);
    }
    __syncthreads();
  }
}

// Joins the pieces of the items that the shares' borders divide, in the order
// of the shares: two rows a CTA, 32 lanes of four dims each, the pieces dealt
// to groups of lanes whose sums meet in shared memory.  Launched ahead of the
// pieces' end; it adds 1 to 2 us, all of it latency.
constexpr int JOIN_ROWS = 2;
template <typename T, int D, int NT>
__global__ void __launch_bounds__(THREADS) paged_join_kernel(const AttnParams p) {
  using C = Cfg<T, D, NT>;
  constexpr int RT = C::RT;
  constexpr int LANES = D / 4, GROUPS = THREADS / (LANES * JOIN_ROWS);
  __shared__ float s_acc[GROUPS][JOIN_ROWS][LANES][6];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int cta = blockIdx.x;
  const int4 cut = p.cuts[2 * cta];             // request, head, first row, pieces
  const int4 rest = p.cuts[2 * cta + 1];        // rows, first token
  const int n = cut.w;
  const int row = blockIdx.y * JOIN_ROWS + (threadIdx.x / LANES) % JOIN_ROWS, d = (threadIdx.x % LANES) * 4;
  if (n == 0 || blockIdx.y * JOIN_ROWS >= rest.x) return;
  const int grp = threadIdx.x / (LANES * JOIN_ROWS);
  // piece 0 is the last of its share (slot 1), the others are the first of theirs
  const float* first = p.part + (int64_t)(2 * cta + 1) * C::PART;
  const float* others = p.part + (int64_t)(2 * cta) * C::PART;
  // running maximum, four pieces' loads at a time
  float M = M_NONE, L = 0.0f, a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
  for (int k0 = grp; k0 < n; k0 += 4 * GROUPS) {
    float pm[4], pl[4];
    float4 v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = k0 + e * GROUPS;
      const float* q = k ? others + (int64_t)k * 2 * C::PART : first;
      pm[e] = M_NONE, pl[e] = 0.0f, v[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (k < n) {
        pm[e] = q[RT * D + row];
        pl[e] = q[RT * D + RT + row];
        v[e] = *reinterpret_cast<const float4*>(q + row * D + d);
      }
    }
    const float M1 = fmaxf(fmaxf(fmaxf(pm[0], pm[1]), fmaxf(pm[2], pm[3])), M), keep = ex2(M - M1);
    M = M1, L *= keep, a0 *= keep, a1 *= keep, a2 *= keep, a3 *= keep;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float f = ex2(pm[e] - M);
      L = fmaf(pl[e], f, L);
      a0 = fmaf(v[e].x, f, a0);
      a1 = fmaf(v[e].y, f, a1);
      a2 = fmaf(v[e].z, f, a2);
      a3 = fmaf(v[e].w, f, a3);
    }
  }
  float* mine = s_acc[grp][(threadIdx.x / LANES) % JOIN_ROWS][threadIdx.x % LANES];
  mine[0] = L, mine[1] = a0, mine[2] = a1, mine[3] = a2, mine[4] = a3, mine[5] = M;
  __syncthreads();
  if (grp != 0 || row >= rest.x) return;
#pragma unroll
  for (int k = 1; k < GROUPS; ++k) {
    const float* o = s_acc[k][(threadIdx.x / LANES) % JOIN_ROWS][threadIdx.x % LANES];
    const float M1 = fmaxf(M, o[5]), f = ex2(M - M1), g = ex2(o[5] - M1);
    M = M1, L = L * f + o[0] * g, a0 = a0 * f + o[1] * g, a1 = a1 * f + o[2] * g, a2 = a2 * f + o[3] * g;
    a3 = a3 * f + o[4] * g;
  }
  write_row<T>(p, rest.y + (cut.z + row) / p.g, cut.y * p.g + (cut.z + row) % p.g, d, M, L, a0, a1, a2, a3);
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return 0;
  return n;
}
constexpr int MAX_GRID = 444;          // workspace sizing: 3 CTAs on each of a B200's 148 SMs

int64_t workspace_need(int head_dim) { return MAX_GRID * 32ll + 2ll * MAX_GRID * 16 * (head_dim + 2) * 4; }
bool tiled(int64_t rows) { return rows > SMALL; }

template <typename T, int D, int NT>
int launch(AttnParams& p, void* workspace, cudaStream_t stream) {
  using C = Cfg<T, D, NT>;
  const int grid = min(sm_count() * (NT == 1 ? 3 : 2), MAX_GRID);      // resident CTAs: registers bound them
  if (grid <= 0) return HC_ERR_CUDA;
  p.cuts = static_cast<int4*>(workspace);
  p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + MAX_GRID * 32);
  const int smem = C::RING + (p.n_req + 1) * 8;
  if (cudaFuncSetAttribute(paged_attn_kernel<T, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) !=
      cudaSuccess)
    return HC_ERR_CUDA;
  paged_attn_kernel<T, D, NT><<<grid, THREADS, smem, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return HC_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, C::RT / JOIN_ROWS);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_join_kernel<T, D, NT>, p) == cudaSuccess ? HC_OK : HC_ERR_CUDA;
}

template <typename T>
int launch_typed(AttnParams& p, int head_dim, int rows, void* workspace, cudaStream_t stream) {
  // rows of the largest request and head: 8 fill one MMA's columns (64 requests as above 99 us), more take two
  // (129 us).  A step that holds both, or prompts beside single tokens, runs its small requests on the latter too.
  if (head_dim == 128)
    return rows <= 8 ? launch<T, 128, 1>(p, workspace, stream) : launch<T, 128, 2>(p, workspace, stream);
  return rows <= 8 ? launch<T, 64, 1>(p, workspace, stream) : launch<T, 64, 2>(p, workspace, stream);
}

inline bool aligned(const void* ptr, uintptr_t a) { return (reinterpret_cast<uintptr_t>(ptr) & (a - 1)) == 0; }

}  // namespace hca8

using namespace hca8;

extern "C" int64_t hc_paged_attn_workspace_bytes(int32_t n_requests, int32_t n_rows, int32_t n_q_heads,
                                                 int32_t n_kv_heads, int32_t head_dim) {
  if (n_requests <= 0 || n_rows < 0 || n_q_heads <= 0 || n_kv_heads <= 0 || (head_dim != 64 && head_dim != 128))
    return -1;
  const int64_t rows = (int64_t)n_rows * (n_q_heads / n_kv_heads);
  return workspace_need(head_dim) + (tiled(rows) ? prefill_workspace(head_dim) : 0);
}

extern "C" int hc_paged_attn(const hc_attn_args* a, const hc_kv_pages* c, void* workspace, int64_t workspace_bytes,
                             int32_t* status, hc_stream_t stream) {
  if (!a || !c || !a->tables || !a->cu_q || !a->kv_lens) return HC_ERR_ARG;
  if (a->n_rows != 0 && (!a->q || !a->out)) return HC_ERR_ARG;
  if (!c->k || !c->v || !c->k_scale || !c->v_scale || c->n_pages <= 0 || c->n_kv_heads <= 0) return HC_ERR_ARG;
  if (a->n_requests <= 0 || a->n_rows < 0 || a->max_q < 0 || a->n_q_heads <= 0 ||
      a->n_q_heads % c->n_kv_heads || a->table_width <= 0 || a->table_stride < a->table_width ||
      (a->dtype != HC_F16 && a->dtype != HC_BF16) || !(fabsf(a->scale) < INFINITY))
    return HC_ERR_ARG;
  if (a->q_row < 0 || a->q_head < 0 || a->out_row < 0 || a->out_head < 0) return HC_ERR_ARG;
  if (!aligned(a->q, 2) || !aligned(a->out, 2) || !aligned(a->lse, 4) || !aligned(c->k, 16) || !aligned(c->v, 16) ||
      !aligned(a->tables, 4) || !aligned(c->k_scale, 4) || !aligned(c->v_scale, 4) || !aligned(a->cu_q, 4) ||
      !aligned(a->kv_lens, 4) || !aligned(status, 4))
    return HC_ERR_ARG;
  if (c->page_size != 16 && c->page_size != 32 && c->page_size != 64 && c->page_size != 128)
    return HC_ERR_UNSUPPORTED;
  if ((c->head_dim != 64 && c->head_dim != 128) || a->n_q_heads / c->n_kv_heads > 16 || a->n_requests > MAX_REQ)
    return HC_ERR_UNSUPPORTED;
  if ((int64_t)a->table_width * c->page_size > INT32_MAX) return HC_ERR_ARG;
  if ((int64_t)a->n_rows * (a->n_q_heads / c->n_kv_heads) > 1 << 30) return HC_ERR_UNSUPPORTED;   // rows are int32
  if (a->n_rows == 0) return HC_OK;
  if (!workspace || !aligned(workspace, 16) ||
      workspace_bytes <
          hc_paged_attn_workspace_bytes(a->n_requests, a->n_rows, a->n_q_heads, c->n_kv_heads, c->head_dim))
    return HC_ERR_ARG;
  AttnParams p = {};
  p.q = a->q;
  p.out = a->out;
  p.lse = a->lse;
  p.q_row = a->q_row;
  p.q_head = a->q_head;
  p.o_row = a->out_row;
  p.o_head = a->out_head;
  p.tables = a->tables;
  p.t_stride = a->table_stride;
  p.width = a->table_width;
  p.cu_q = a->cu_q;
  p.kv_lens = a->kv_lens;
  p.n_req = a->n_requests;
  p.n_rows = a->n_rows;
  p.nq = a->n_q_heads;
  p.nkv = c->n_kv_heads;
  p.g = a->n_q_heads / c->n_kv_heads;
  p.scale2 = a->scale * LOG2E;
  p.kp = c->k;
  p.vp = c->v;
  p.ks = c->k_scale;
  p.vs = c->v_scale;
  p.n_pages = c->n_pages;
  p.page_log2 = c->page_size == 16 ? 4 : c->page_size == 32 ? 5 : c->page_size == 64 ? 6 : 7;
  p.status = status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  // Up to SMALL rows of a request and head the keys are split over the GPU; more fill the tensor cores' tiles.
  const int64_t rows = (int64_t)min(a->max_q, a->n_rows) * p.g;
  p.rows_from = 0;
  p.rows_to = INT32_MAX;
  if (tiled(rows)) {
    const int sms = sm_count();
    if (sms <= 0) return HC_ERR_CUDA;
    p.rows_from = SMALL + 1;
    const int rc = launch_prefill(p, a->dtype, c->head_dim,
                                  static_cast<uint8_t*>(workspace) + workspace_need(c->head_dim), sms, s);
    if (rc != HC_OK) return rc;
    p.rows_from = 0;
    p.rows_to = SMALL + 1;
  }
  return a->dtype == HC_F16 ? launch_typed<__half>(p, c->head_dim, (int)min(rows, (int64_t)64), workspace, s)
                            : launch_typed<__nv_bfloat16>(p, c->head_dim, (int)min(rows, (int64_t)64), workspace, s);
}
