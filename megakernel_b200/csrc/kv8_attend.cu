// Attention over the paged 8-bit cache (megakernel_kv8_attend).
#include "paged.cuh"
#include "tc_ptx.cuh"

#ifndef ATT_FILL
#define ATT_FILL 3
#endif

namespace mkp {

struct Attend {
  const void* q;
  void* out;
  float* lse;
  const int* kv_lens;
  long long q_row, q_head;
  int q_heads, causal, window;
  float scale;   // log2(e) x the softmax scale
  int bf16;      // q and out: bf16, else f16
  int* status;
};

// ---- warp-level pieces ---------------------------------------------------------------

// D[16x8] += A[16x16] B[16x8], f16 in, fp32 accumulate.
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two codes (the low or the high half of w) -> f16x2, exactly: e4m3 and the
// whole numbers to 127 are f16 values.
template <class F> __device__ __forceinline__ void expand(uint32_t w, uint32_t& lo, uint32_t& hi);
template <> __device__ __forceinline__ void expand<E4M3>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi) : "r"(w));
}
// 0x6400 + b is the f16 value 1024 + b for a byte b; codes are biased by 128.
template <> __device__ __forceinline__ void expand<I8>(uint32_t w, uint32_t& lo, uint32_t& hi) {
  const uint32_t u = w ^ 0x80808080u;
  const __half2 bias = __half2half2(__ushort_as_half((unsigned short)0x6480));   // 1152
  uint32_t x = __byte_perm(u, 0x64646464u, 0x4140), y = __byte_perm(u, 0x64646464u, 0x4342);
  const __half2 a = __hsub2(*reinterpret_cast<__half2*>(&x), bias);
  const __half2 b = __hsub2(*reinterpret_cast<__half2*>(&y), bias);
  lo = *reinterpret_cast<const uint32_t*>(&a);
  hi = *reinterpret_cast<const uint32_t*>(&b);
}

// Bits 7 of the bytes of w that are e4m3 NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

__device__ __forceinline__ float load_q(const void* q, long long i, bool bf16) {
  return bf16 ? __bfloat162float(((const __nv_bfloat16*)q)[i]) : __half2float(((const __half*)q)[i]);
}
__device__ __forceinline__ void store_out(void* o, long long i, float v, bool bf16) {
  if (bf16) ((__nv_bfloat16*)o)[i] = __float2bfloat16_rn(v);
  else ((__half*)o)[i] = __float2half_rn(v);
}

// The word at p's place in the shared memory of block `rank` of the cluster.
__device__ __forceinline__ float remote_f32(const float* p, uint32_t rank) {
  uint32_t at;
  float v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(mk::smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ uint64_t policy_evict_normal() {
  uint64_t pol;
  asm volatile("createpolicy.fractional.L2::evict_normal.b64 %0, 1.0;" : "=l"(pol));
  return pol;
}

constexpr int kStages = 2;
constexpr int kWarps = 4;
constexpr int kStageBytes = 8192;      // K and V codes of one step
constexpr uint32_t kWaitLimit = 1u << 22;
constexpr float kNone = -1e30f;        // running reference of a row that has seen nothing
constexpr float kSlack = 5.f;          // weights may reach 2^kSlack before the reference moves

// Bounded wait; each probe may itself suspend for a while.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity) {
  for (uint32_t i = 0; i < kWaitLimit; ++i)
    if (mk::mbar_try_wait(bar, parity)) return true;
  return false;
}

template <int D, int NT, int MW>
constexpr int rows_smem() {
  constexpr int ring = (kWarps / MW) * kStages * kStageBytes, parts = kWarps * 8 * NT * D * 4;
  return ring > parts ? ring : parts;
}

// 8 x 8 f16 matrix, lane (g, t) holding row g, columns 2 t and 2 t + 1 -> its transpose.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// ---- attention of few rows per sequence -------------------------------------------------
//
// Work item: (8 NT MW rows of one sequence and kv head, counting a row once per
// query head of the group; the positions split over the S blocks of a cluster
// and their warps).  MW warps that hold 8 NT rows each share a stream of steps
// of TS positions; the 4 / MW such groups of a block, and the blocks of the
// cluster, take every (4 / MW) S-th step.
//
// The codes of a step, contiguous in a page, arrive by bulk copies in a ring
// per group (K 4 KB and V 4 KB a stage): nothing of the stream passes through
// registers before it is used.  Both products have the positions or the head
// dimension as the 16 rows of an m16n8k16 f16 product and the query rows as
// its 8 columns, fp32 accumulation:
//   S^T [positions x rows] = K Q^T,   O^T [dims x rows] += V^T P^T,
// so that 8 rows (a decode step of 8 query heads per kv head) waste nothing.
// The order of the head dimension in the first product and of the output's
// rows in the second is free, so a lane reads 16 consecutive bytes of K (its
// part of four k-steps) and D / 8 consecutive bytes of V from each of four
// positions; the code bytes become f16 in registers, exactly.  q is brought to
// 2^14 by a power of two per row (bf16 values fit f16 then, 2^-39 of the row's
// largest lost at most).
//
// Softmax per row relative to a running reference m: p = 2^(s - m), l = sum p,
// fp32.  m moves to the maximum only when some p would pass 2^5 (one vote per
// 32 positions), so most steps have no exchange between lanes at all.  The
// scale of a K page multiplies the scores, that of a V page the weights:
// w = 2^10 p scale / vref, vref the largest V scale so far, goes into the second
// product in f16: 11 bits down to 2^-29 of the row's largest, an absolute 2^-35
// below that (at p scale / vref alone it was 2^-25, which rows with one
// dominant position showed).  The sum l takes the unrounded p.
template <class F, int P, int D, int NT, int MW>
__global__ void __launch_bounds__(kWarps * 32, D == 64 || NT == 1 ? 3 : 2) attend_rows_kernel(const Cache c, const Attend a) {
  constexpr int TS = kStageBytes / 2 / D, kSub = TS > P ? TS / P : 1, kGroups = kWarps / MW;
  constexpr int kSubRows = TS / kSub;               // positions of a step in one page
  constexpr int kBatch = 32 / kSub;                 // steps whose pages the lanes hold
  constexpr int R = 8 * NT;                         // rows of a warp
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t s_full[kGroups * kStages], s_empty[kGroups * kStages];
  __shared__ float s_m[kWarps][R], s_l[kWarps][R], s_v[kWarps], s_top[MW * R], s_sum[MW * R];
  __shared__ int s_nan;

  uint32_t rank, split;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(split));
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int mw = warp % MW, grp = warp / MW;
  const int group = a.q_heads / c.kv_heads;
  const int cta = blockIdx.x / split, h = cta % c.kv_heads, item = cta / c.kv_heads;

  // sequence b owns the items from starts[b] group / (R MW) + b on
  auto key = [&](int i) { return (int)((long long)__ldg(c.starts + i) * group / (R * MW)) + i; };
  const int b = warp_search(c.seqs, item, key);
  const int r0 = __ldg(c.starts + b), r1 = __ldg(c.starts + b + 1), first = __ldg(c.first + b);
  if (r0 < 0 || r1 < r0 || r1 > c.rows || first > (1 << 30)) {
    report(a.status, MK_ERR_INVALID_ARG);
    return;   // the whole cluster: every block of it has this item
  }
  const int n = r1 - r0, m0 = (item - key(b)) * R * MW;
  if (m0 < 0 || m0 >= n * group) return;
  const int valid = min(n * group - m0, R * MW);
  int len = a.kv_lens ? __ldg(a.kv_lens + b) : first + n;
  if (len > c.table_width * P) {
    report(a.status, MK_ERR_CAPACITY);
    len = c.table_width * P;
  }
  // what the row of index m sees: [lo, hi)
  auto sees = [&](int m, int& lo, int& hi) {
    const int pos = first + m / group;
    lo = hi = 0;
    if (m < n * group && pos >= 0) {
      hi = max(a.causal ? min(len, pos + 1) : len, 0);
      lo = a.window ? max(pos - a.window + 1, 0) : 0;
    }
  };
  int lo_all, hi_all, lo_max, hi_min;
  sees(m0 + valid - 1, lo_max, hi_all);
  sees(m0, lo_all, hi_min);
  const int begin = lo_all / TS * TS;
  const int all_steps = hi_all > begin ? (hi_all - begin + TS - 1) / TS : 0;
  const int stride = (int)split * kGroups, my = (int)rank * kGroups + grp;
  const int steps = all_steps > my ? (all_steps - my - 1) / stride + 1 : 0;

  if (threadIdx.x == 0) {
    s_nan = 0;
    for (int i = 0; i < kGroups * kStages; ++i) {
      mk::mbar_init(&s_full[i], kSub);
      mk::mbar_init(&s_empty[i], MW);
    }
    mk::fence_mbar_init();
  }
  __syncthreads();

  // Pages of kBatch steps, one per lane: id (-1: not wanted, or reported) and
  // scales (a K scale of 0 marks a page that is not there).
  struct Page { int id; float ks, vs; };
  auto pages_from = [&](int step) {
    Page p{-1, 0.f, 0.f};
    const int st = step + lane / kSub;
    const int pos = begin + (st * stride + my) * TS + (lane % kSub) * kSubRows;
    if (st < steps && pos < hi_all && pos + kSubRows > lo_all) {
      p.id = page_id(c, b, pos / P, a.status);
      if (p.id >= 0) {
        const float* sc = c.scales + p.id * c.scale_stride + h;
        p.ks = fmaxf(__ldg(sc), 1.17549435e-38f);
        p.vs = __ldg(sc + c.kv_heads);
      }
    }
    return p;
  };
  Page cur = pages_from(0), nxt = pages_from(kBatch);
  int base = 0;
  uint8_t* ring = smem + grp * kStages * kStageBytes;
  // Codes that no other item reads do not stay in the L2 cache.
  const uint64_t policy = n * group <= R * MW ? mk::policy_evict_first() : policy_evict_normal();
  // The lanes that hold the pages of step st copy their part of it.
  auto fetch = [&](int st) {
    const int id = st - base < kBatch ? cur.id : nxt.id;
    if (st < steps && lane / kSub == (st - base) % kBatch) {
      uint64_t* bar = &s_full[grp * kStages + st % kStages];
      const int sub = lane % kSub;
      mk::mbar_arrive_expect_tx(bar, id >= 0 ? 2 * kSubRows * D : 0);
      if (id >= 0) {
        const int pos = begin + (st * stride + my) * TS + sub * kSubRows;
        uint8_t* dst = ring + st % kStages * kStageBytes + sub * kSubRows * D;
        const uint8_t* k = c.codes + id * c.page_stride + ((long long)h * P + pos % P) * D;
        mk::bulk_g2s(dst, k, kSubRows * D, bar, policy);
        mk::bulk_g2s(dst + TS * D, k + (long long)c.kv_heads * P * D, kSubRows * D, bar, policy);
      }
    }
  };
  if (mw == 0)
    for (int i = 0; i < kStages; ++i) fetch(i);

  // q fragments, row 8 nt + g of this warp: k-step j holds dimensions
  // 64 (j / 4) + 16 t + 4 (j % 4) + {0, 1 | 2, 3}.  rq, lo, hi: rows 2 t and
  // 2 t + 1, whose scores this lane will hold.
  uint32_t q[NT][D / 16][2];
  float rq[NT][2];
  int lo[NT][2], hi[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    const int m = m0 + mw * R + 8 * nt + g;
    const bool real = m < n * group;
    const long long at = real ? (long long)(r0 + m / group) * a.q_row + (h * group + m % group) * a.q_head : 0;
    float v[D / 4];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < D / 4; ++i) {
      v[i] = real ? load_q(a.q, at + i / 16 * 64 + 16 * t + i % 16, a.bf16) : 0.f;
      top = fmaxf(top, fabsf(v[i]));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // power of two that brings the largest to [2^14, 2^15)
    const int ex = min(max((int)(__float_as_uint(top) >> 23), 30), 240);
    const float up = __uint_as_float((uint32_t)(127 + 127 + 14 - ex) << 23);
#pragma unroll
    for (int j = 0; j < D / 16; ++j) {
      q[nt][j][0] = pack_f16(v[4 * j] * up, v[4 * j + 1] * up);
      q[nt][j][1] = pack_f16(v[4 * j + 2] * up, v[4 * j + 3] * up);
    }
    const float back = a.scale * __uint_as_float((uint32_t)(ex - 14) << 23);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      rq[nt][e] = __shfl_sync(0xffffffffu, back, 4 * (2 * t + e));
      sees(m0 + mw * R + 8 * nt + 2 * t + e, lo[nt][e], hi[nt][e]);
    }
  }

  float o[NT][D / 16][4] = {};
  float m[NT][2], l[NT][2], vref = 0.f, iv = 0.f;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
    for (int e = 0; e < 2; ++e) m[nt][e] = kNone, l[nt][e] = 0.f;
  bool alive = true;
  int nan_seen = 0, failed = 0;
  for (int st = 0; st < steps; ++st) {
    if (st - base == kBatch) {
      base += kBatch;
      cur = nxt;
      nxt = pages_from(base + kBatch);
    }
    float ks[kSub], vs[kSub];
    float vmax = vref;
    bool whole = true;
#pragma unroll
    for (int i = 0; i < kSub; ++i) {
      const int src = (st - base) * kSub + i;
      ks[i] = __shfl_sync(0xffffffffu, cur.ks, src);
      vs[i] = __shfl_sync(0xffffffffu, cur.vs, src);
      whole = whole && ks[i] > 0.f;
      vmax = fmaxf(vmax, vs[i]);
    }
    if (vmax > vref) {
      const float r = vref / vmax;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
#pragma unroll
          for (int x = 0; x < 4; ++x) o[nt][i][x] *= r;
      vref = vmax;
      iv = 1024.f / vmax;
    }
    const int pos = begin + (st * stride + my) * TS;
    whole = whole && pos >= lo_max && pos + TS <= hi_min;
    if (!wait_bar(&s_full[grp * kStages + st % kStages], (st / kStages) & 1)) {
      alive = false;
      failed = st;
      break;
    }
    const uint8_t* kb = ring + st % kStages * kStageBytes;
    const uint8_t* vb = kb + TS * D;

#pragma unroll
    for (int half = 0; half < TS / 32; ++half) {   // 32 positions
      float s[2][NT][4];
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const uint8_t* k0 = kb + (half * 32 + mt * 16 + g) * D + 16 * t;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) s[mt][nt][0] = s[mt][nt][1] = s[mt][nt][2] = s[mt][nt][3] = 0.f;
#pragma unroll
        for (int d = 0; d < D / 64; ++d) {
          const uint4 x = *reinterpret_cast<const uint4*>(k0 + d * 64);
          const uint4 y = *reinterpret_cast<const uint4*>(k0 + d * 64 + 8 * D);
          const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t ka[4];
            expand<F>(xs[j], ka[0], ka[2]);
            expand<F>(ys[j], ka[1], ka[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(s[mt][nt], ka, q[nt][d * 4 + j][0], q[nt][d * 4 + j][1]);
          }
        }
      }
      float f[2][NT][2];
      bool over = false;
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int i = (half * 32 + mt * 16) / kSubRows;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
          for (int e = 0; e < 2; ++e) f[mt][nt][e] = fmaxf(rq[nt][e] * ks[i], 1.17549435e-38f);   // -inf x 0 would be NaN
          if (!whole) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int j = pos + half * 32 + mt * 16 + g + 8 * (x >> 1);
              if (ks[i] == 0.f || j < lo[nt][x & 1] || j >= hi[nt][x & 1]) s[mt][nt][x] = -INFINITY;
            }
          }
#pragma unroll
          for (int x = 0; x < 4; ++x) over = over || fmaf(s[mt][nt][x], f[mt][nt][x & 1], -m[nt][x & 1]) > kSlack;
        }
      }
      if (__any_sync(0xffffffffu, over)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float top = m[nt][e];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
              top = fmaxf(top, fmaxf(s[mt][nt][e], s[mt][nt][2 + e]) * f[mt][nt][e]);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float keep = ex2(m[nt][e] - top);
            m[nt][e] = top;
            l[nt][e] *= keep;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) {
              o[nt][i][e] *= keep;
              o[nt][i][2 + e] *= keep;
            }
          }
      }
#pragma unroll
      for (int mt = 0; mt < 2; ++mt) {
        const int at = half * 32 + mt * 16, i = at / kSubRows;
        const float rv = vs[i] * iv;
        uint32_t pb[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float p[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            p[x] = ex2(fmaf(s[mt][nt][x], f[mt][nt][x & 1], -m[nt][x & 1]));
            l[nt][x & 1] += p[x];
          }
          pb[nt][0] = transpose8(pack_f16(p[0] * rv, p[1] * rv));
          pb[nt][1] = transpose8(pack_f16(p[2] * rv, p[3] * rv));
        }
        uint32_t v[4][D / 32];   // positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int row = at + 2 * t + (x & 1) + 8 * (x >> 1);
          const uint8_t* vp = vb + row * D + g * (D / 8);
          if constexpr (D == 64) {
            const uint2 u = *reinterpret_cast<const uint2*>(vp);
            v[x][0] = u.x; v[x][1] = u.y;
          } else {
            const uint4 u = *reinterpret_cast<const uint4*>(vp);
            v[x][0] = u.x; v[x][1] = u.y; v[x][2] = u.z; v[x][3] = u.w;
          }
          if (!whole) {
            // What no row sees may hold anything: its codes count as 0.  A NaN
            // that only some rows see is taken out here and put back at the end.
            const bool dead = ks[i] == 0.f || pos + row >= hi_all || pos + row < lo_all;
#pragma unroll
            for (int y = 0; y < D / 32; ++y) {
              if (dead) v[x][y] = 0;
              if constexpr (F::kTopExp == 8) {
                const uint32_t bad = nan_bytes(v[x][y]);
                if (bad) {
                  nan_seen = 1;
                  v[x][y] &= ~((bad >> 7) * 0xffu);
                }
              }
            }
          }
        }
#pragma unroll
        for (int y = 0; y < D / 32; ++y) {
          // byte pairs of two positions; dimensions 4 y + {0, 1} and {2, 3} of this lane
          uint32_t va[4], vc[4];
          expand<F>(__byte_perm(v[0][y], v[1][y], 0x5140), va[0], va[1]);
          expand<F>(__byte_perm(v[2][y], v[3][y], 0x5140), va[2], va[3]);
          expand<F>(__byte_perm(v[0][y], v[1][y], 0x7362), vc[0], vc[1]);
          expand<F>(__byte_perm(v[2][y], v[3][y], 0x7362), vc[2], vc[3]);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(o[nt][2 * y], va, pb[nt][0], pb[nt][1]);
            mma_f16(o[nt][2 * y + 1], vc, pb[nt][0], pb[nt][1]);
          }
        }
      }
    }
    __syncwarp();
    if constexpr (MW > 1) {
      if (lane == 0) mk::mbar_arrive(&s_empty[grp * kStages + st % kStages]);
      if (mw == 0) {
        if (st + kStages < steps && !wait_bar(&s_empty[grp * kStages + st % kStages], (st / kStages) & 1)) {
          alive = false;
          failed = st + 1;
          break;
        }
        fetch(st + kStages);
      }
    } else {
      fetch(st + kStages);
    }
  }
  if (!alive) {
    // Leave no copy in flight: the block's shared memory is given away at its
    // end.  (Waits are bounded; a copy that never lands is reported.)
    report(a.status, MK_ERR_TIMEOUT);
    for (int i = 0; i < kStages; ++i)
      if (failed + i < steps) wait_bar(&s_full[grp * kStages + (failed + i) % kStages], ((failed + i) / kStages) & 1);
  }
  if (nan_seen) s_nan = 1;

  // ---- join the warps, then the blocks of the cluster
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float x = l[nt][e];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (g == 0) {
        s_m[warp][8 * nt + 2 * t + e] = m[nt][e];
        s_l[warp][8 * nt + 2 * t + e] = x;
      }
    }
  if (lane == 0) s_v[warp] = vref * (1.f / 1024.f);
  __syncthreads();   // the ring is free
  float* part = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int i = 0; i < D / 16; i += 2)   // dimensions (D / 8) g + 2 i .. + 3 of row 2 t + e
        *reinterpret_cast<float4*>(part + (warp * R + 8 * nt + 2 * t + e) * D + (D / 8) * g + 2 * i) =
            make_float4(o[nt][i][e], o[nt][i][2 + e], o[nt][i + 1][e], o[nt][i + 1][2 + e]);
  __syncthreads();
  for (int i = threadIdx.x; i < valid * D; i += kWarps * 32) {
    const int r = i / D, w0 = r / R;   // warps w0, w0 + MW, ... hold row r
    float top = kNone, sum = 0.f, acc = 0.f;
#pragma unroll
    for (int x = 0; x < kGroups; ++x) top = fmaxf(top, s_m[w0 + x * MW][r % R]);
#pragma unroll
    for (int x = 0; x < kGroups; ++x) {
      const int w = w0 + x * MW;
      const float f = ex2(s_m[w][r % R] - top);
      sum += f * s_l[w][r % R];
      acc += f * s_v[w] * part[(w * R + r % R) * D + i % D];
    }
    part[(w0 * R + r % R) * D + i % D] = acc;
    if (i % D == 0) {
      s_top[r] = top;
      s_sum[r] = sum;
    }
  }
  if (split > 1) mk::cluster_sync_all();
  else __syncthreads();
  const int nan_any = s_nan;
  // block `rank` finishes every split-th run of 32 elements
  for (int i = threadIdx.x; i < valid * D; i += kWarps * 32) {
    if ((i >> 5) % (int)split != (int)rank) continue;
    const int r = i / D, d = i % D;
    float top = s_top[r], sum = s_sum[r], acc = part[i];   // rows of warps 0 .. MW - 1 lie in order
    int bad = nan_any;
    if (split > 1) {
      top = kNone;
      for (uint32_t k = 0; k < split; ++k) top = fmaxf(top, remote_f32(&s_top[r], k));
      sum = acc = 0.f;
      for (uint32_t k = 0; k < split; ++k) {
        const float f = ex2(remote_f32(&s_top[r], k) - top);
        sum += f * remote_f32(&s_sum[r], k);
        acc += f * remote_f32(&part[i], k);
        bad |= __float_as_int(remote_f32(reinterpret_cast<const float*>(&s_nan), k));
      }
    }
    float v = sum == 0.f ? 0.f : acc / sum;   // nothing seen: 0
    if (bad) {
      // NaN codes of positions that this row sees and another row of the item does not
      int rlo, rhi;
      sees(m0 + r, rlo, rhi);
      for (int j = rlo; j < rhi; ++j) {
        if (j >= lo_max + TS && j < hi_min - TS) j = hi_min - TS;   // whole steps kept theirs
        const int id = page_id(c, b, j / P, nullptr);
        if (id < 0) continue;
        const uint8_t code = c.codes[id * c.page_stride + ((long long)(c.kv_heads + h) * P + j % P) * D + d];
        if (F::kTopExp == 8 && (code & 127) == 127) v = __int_as_float(0x7fffffff);
      }
    }
    const long long at = (long long)(r0 + (m0 + r) / group) * a.q_heads + h * group + (m0 + r) % group;
    store_out(a.out, at * D + d, v, a.bf16);
    if (a.lse && d == 0) a.lse[at] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
  }
  if (split > 1) mk::cluster_sync_all();   // peers have read this block's shared memory
}

int cache_of(const mk_kv8* m, Cache* c);

template <class F, int P, int D, int NT, int MW>
static int launch_rows(const Cache& c, const Attend& a, cudaStream_t stream) {
  const int group = a.q_heads / c.kv_heads;
  const long long items = (long long)c.rows * group / (8 * NT * MW) + c.seqs;
  const long long most = (long long)c.table_width * P;
  // Blocks per item: until the grid fills the GPU ATT_FILL times over, but no
  // more than one step of each group of warps per block at full capacity.
  int split = 1;
  while (split < 8 && items * c.kv_heads * split < 148 * ATT_FILL && most > (long long)split * (kWarps / MW) * (kStageBytes / 2 / D)) split *= 2;
  const long long blocks = items * c.kv_heads * split;
  if (blocks > 0x7fffffffLL) return MK_ERR_INVALID_ARG;
  auto kernel = &attend_rows_kernel<F, P, D, NT, MW>;
  constexpr int bytes = rows_smem<D, NT, MW>();
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return MK_ERR_CUDA;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(kWarps * 32);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim = {(unsigned)split, 1, 1};
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, c, a) == cudaSuccess ? MK_OK : MK_ERR_CUDA;
}

template <class F, int P, int D>
static int launch(const Cache& c, const Attend& a, cudaStream_t stream) {
  // rows of a sequence, once per query head of the group, on average
  const long long per = ((long long)c.rows * (a.q_heads / c.kv_heads) + c.seqs - 1) / c.seqs;
  if (per <= 8) return launch_rows<F, P, D, 1, 1>(c, a, stream);
  if (per <= 16) return launch_rows<F, P, D, 2, 1>(c, a, stream);
  if (per <= 32) return launch_rows<F, P, D, 2, 2>(c, a, stream);
  return launch_rows<F, P, D, 2, 4>(c, a, stream);
}

}  // namespace mkp

using namespace mkp;

extern "C" int megakernel_kv8_attend(const mk_kv8* cache, const void* d_q, long long q_row, long long q_head,
                                     int q_heads, int type, float sm_scale, int causal, int window,
                                     const int* d_kv_lens, void* d_out, float* d_lse, int* d_status, void* stream) {
  Cache c;
  const int rc = cache_of(cache, &c);
  if (rc != MK_OK) return rc;
  if (type != MK_TYPE_BF16 && type != MK_TYPE_F16) return MK_ERR_INVALID_ARG;
  if (q_heads < 1 || q_heads % c.kv_heads || q_heads > 65535 || window < 0 || !(sm_scale > 0.f))
    return MK_ERR_INVALID_ARG;
  if (c.rows == 0) return MK_OK;
  if (c.seqs == 0) return MK_ERR_INVALID_ARG;
  if (!d_q || !d_out || ((uintptr_t)d_q & 15) || ((uintptr_t)d_out & 15) || q_row % 8 || q_head % 8 || q_row < 0 ||
      q_head < 0)
    return MK_ERR_INVALID_ARG;
  const Attend a{d_q, d_out, d_lse, d_kv_lens, q_row, q_head, q_heads, causal, window,
                 sm_scale * 1.4426950408889634f, type == MK_TYPE_BF16, d_status};
  auto with_d = [&](auto f, auto p) {
    using F = decltype(f);
    constexpr int P = decltype(p)::value;
    return cache->head_dim == 64 ? launch<F, P, 64>(c, a, (cudaStream_t)stream)
                                 : launch<F, P, 128>(c, a, (cudaStream_t)stream);
  };
  auto with_p = [&](auto f) {
    if (cache->page_size == 16) return with_d(f, std::integral_constant<int, 16>{});
    if (cache->page_size == 32) return with_d(f, std::integral_constant<int, 32>{});
    return with_d(f, std::integral_constant<int, 64>{});
  };
  return cache->format == MK_KV8_E4M3 ? with_p(E4M3{}) : with_p(I8{});
}
