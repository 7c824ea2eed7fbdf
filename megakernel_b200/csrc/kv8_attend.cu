// Attention over the paged 8-bit cache (megakernel_kv8_attend).
#include "paged.cuh"

namespace mkp {

struct Attend {
  const void* q;
  void* out;
  float* lse;
  const int* kv_lens;
  long long q_row, q_head;
  int q_heads, causal, window;
  float scale;   // log2(e) x the softmax scale
  int* status;
};

// One block of four warps per (row, query head); each warp walks every fourth
// position with a running maximum and sum, and the four are joined at the end.
template <class T, class F, int P, int D>
__global__ void __launch_bounds__(128) attend_simple_kernel(const Cache c, const Attend a) {
  constexpr int kPer = D / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int row = blockIdx.x, hq = blockIdx.y, group = a.q_heads / c.kv_heads, h = hq / group;
  const int b = warp_search(c.seqs, row, [&](int i) { return __ldg(c.starts + i); });
  const int r0 = __ldg(c.starts + b), r1 = __ldg(c.starts + b + 1), first = __ldg(c.first + b);
  int lo = 0, hi = 0;
  if (r0 < 0 || r1 < r0 || r1 > c.rows || first > (1 << 30)) {
    report(a.status, MK_ERR_INVALID_ARG);
  } else if (row >= r0 && row < r1) {
    const int pos = first + row - r0;
    int len = a.kv_lens ? __ldg(a.kv_lens + b) : first + r1 - r0;
    if (len > c.table_width * P) {
      report(a.status, MK_ERR_CAPACITY);
      len = c.table_width * P;
    }
    if (pos >= 0) {
      hi = a.causal ? min(len, pos + 1) : len;
      lo = a.window ? max(pos - a.window + 1, 0) : 0;
    }
  }
  float q[kPer], acc[kPer] = {};
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    q[i] = Elem<T>::to_f32(((const T*)a.q)[row * a.q_row + hq * a.q_head + lane * kPer + i]) * a.scale;
  float m = -INFINITY, l = 0.f;
  for (int j = lo + warp; j < hi; j += 4) {
    const int id = page_id(c, b, j / P, a.status);
    if (id < 0) continue;
    const uint8_t* kp = c.codes + id * c.page_stride + (long long)h * P * D + (j % P) * D + lane * kPer;
    const uint8_t* vp = kp + (long long)c.kv_heads * P * D;
    const float* sc = c.scales + id * c.scale_stride + h;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) s += q[i] * F::decode(kp[i]);
    s = mk::warp_sum(s) * sc[0];
    const float top = fmaxf(m, s), w = exp2f(s - top), keep = exp2f(m - top);
    l = l * keep + w;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = acc[i] * keep + w * sc[c.kv_heads] * F::decode(vp[i]);
    m = top;
  }
  __shared__ float s_m[4], s_l[4], s_acc[4][D];
#pragma unroll
  for (int i = 0; i < kPer; ++i) s_acc[warp][lane * kPer + i] = acc[i];
  if (lane == 0) {
    s_m[warp] = m;
    s_l[warp] = l;
  }
  __syncthreads();
  const float top = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float w[4], sum = 0.f;
  for (int i = 0; i < 4; ++i) {
    w[i] = s_l[i] > 0.f ? exp2f(s_m[i] - top) : 0.f;
    sum += w[i] * s_l[i];
  }
  for (int d = threadIdx.x; d < D; d += 128) {
    float o = 0.f;
    for (int i = 0; i < 4; ++i) o += w[i] * s_acc[i][d];
    ((T*)a.out)[((long long)row * a.q_heads + hq) * D + d] = Elem<T>::from_f32(sum > 0.f ? o / sum : 0.f);
  }
  if (a.lse && threadIdx.x == 0)
    a.lse[(long long)row * a.q_heads + hq] = sum > 0.f ? (top + log2f(sum)) * 0.6931471805599453f : -INFINITY;
}

int cache_of(const mk_kv8* m, Cache* c);

template <class T, class F, int P, int D>
static int launch(const Cache& c, const Attend& a, cudaStream_t stream) {
  attend_simple_kernel<T, F, P, D><<<dim3((unsigned)c.rows, (unsigned)a.q_heads), 128, 0, stream>>>(c, a);
  return cudaGetLastError() == cudaSuccess ? MK_OK : MK_ERR_CUDA;
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
                 sm_scale * 1.4426950408889634f, d_status};
  auto run = [&](auto t, auto f, auto p, auto d) {
    return launch<decltype(t), decltype(f), decltype(p)::value, decltype(d)::value>(c, a, (cudaStream_t)stream);
  };
  auto with_d = [&](auto t, auto f, auto p) {
    return cache->head_dim == 64 ? run(t, f, p, std::integral_constant<int, 64>{})
                                 : run(t, f, p, std::integral_constant<int, 128>{});
  };
  auto with_p = [&](auto t, auto f) {
    if (cache->page_size == 16) return with_d(t, f, std::integral_constant<int, 16>{});
    if (cache->page_size == 32) return with_d(t, f, std::integral_constant<int, 32>{});
    return with_d(t, f, std::integral_constant<int, 64>{});
  };
  auto with_f = [&](auto t) { return cache->format == MK_KV8_E4M3 ? with_p(t, E4M3{}) : with_p(t, I8{}); };
  return type == MK_TYPE_BF16 ? with_f(__nv_bfloat16{}) : with_f(__half{});
}
