// Rotary positions with one or several axes on queries and keys.
//
// Bytes bound it: every element is read and written once.  A CTA takes a few
// tokens and computes their cosines and sines once into shared memory (64-bit
// angles, rope.cuh).  A thread then keeps one place of one token -- two
// 8-element chunks, the halves of 8 pairs, with their cosines and sines in
// registers -- and goes through the heads with it, four heads' loads ahead of
// the four it works on; the first four leave before the angles are computed.
// 2 x 6,011 tokens of 28 + 4 heads of 128 in bf16 (197 MB): 38.5 us, 5.1 TB/s
// (78 % of the copy rate); two heads in flight and more CTAs an SM, 38.9-41.6
// us; eight heads, 57 us.
#include "rope.cuh"

namespace wnw {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 8;  // tokens of a CTA at most

// eight consecutive elements, rounded to the type
template <typename T>
__device__ inline void store8(T* p, const float (&f)[8]) {
  uint4 u;
  T* t = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = DT<T>::from_f(f[i]);
  *reinterpret_cast<uint4*>(p) = u;
}
template <>
__device__ inline void store8<float>(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

struct RotarySide {
  const void* x;
  void* y;
  int64_t sb, sh, sn, ob, oh, on;
  int heads;
};

template <typename T>
__global__ void __launch_bounds__(kRotThreads, 2)
    rotary_kernel(RotarySide q, RotarySide k, const wnw_rope rope, int D, int64_t tokens, int64_t total, int per_cta,
                  int inverse, int32_t* err) {
  constexpr int UN = sizeof(T) == 4 ? 2 : 4, W = sizeof(T) / 2;  // heads in flight, 16-byte words a chunk
  extern __shared__ float2 cs[];  // [8 pairs of a place][tokens of the CTA][places that turn]
  const int half = rope.rot / 2, turned = rope.rot / 16;
  const int64_t t0 = int64_t(blockIdx.x) * per_cta;
  const int nt = static_cast<int>(min(int64_t(per_cta), total - t0));
  const int duos = D / 16;  // places of a token
  const int places = duos * per_cta;
  const int duo = threadIdx.x % duos, lt = threadIdx.x / duos % per_cta, h0 = threadIdx.x / places;
  const int step = kRotThreads / places;
  const bool work = h0 < step && lt < nt;
  const int64_t t = t0 + (work ? lt : 0);
  const int64_t b = t / tokens, n = t - b * tokens;
  const bool turn = duo < turned;
  const int da = turn ? 8 * duo : rope.rot + 16 * (duo - turned);
  const int db = turn ? da + half : da + 8;
  const T* xq = static_cast<const T*>(q.x) + b * q.sb + n * q.sn;
  const T* xk = static_cast<const T*>(k.x) + b * k.sb + n * k.sn;
  T* yq = static_cast<T*>(q.y) + b * q.ob + n * q.on;
  T* yk = static_cast<T*>(k.y) + b * k.ob + n * k.on;
  const int heads = q.heads + k.heads;  // query heads, then key heads

  uint4 u[UN][W], v[UN][W];
  auto load = [&](int h) {
#pragma unroll
    for (int i = 0; i < UN; ++i, h += step)
      if (h < heads) {
        const T* x = h < q.heads ? xq + h * q.sh : xk + (h - q.heads) * k.sh;
#pragma unroll
        for (int w = 0; w < W; ++w) {
          u[i][w] = __ldcs(reinterpret_cast<const uint4*>(x + da) + w);
          v[i][w] = __ldcs(reinterpret_cast<const uint4*>(x + db) + w);
        }
      }
  };
  if (work) load(h0);  // on their way while the angles are computed
  // the tokens' positions, then each thread's pair of dimensions for them
  __shared__ double s_pos[4 * kRotTokens];
  if (threadIdx.x < rope.num_axes * nt) {
    const int64_t tt = t0 + threadIdx.x % nt, bb = tt / tokens;
    s_pos[threadIdx.x] = rope_pos(rope, threadIdx.x / nt, bb, tt - bb * tokens);
  }
  const int rows = min(nt, kRotThreads / half);
  const int e = threadIdx.x % half;
  RopePair rp{0, 0.0};
  if (threadIdx.x < rows * half) rp = rope_pair(rope, e, err);
  __syncthreads();
  if (threadIdx.x < rows * half) {
#pragma unroll 2
    for (int l = threadIdx.x / half; l < nt; l += rows) {
      float2 c = rope_turn_of(rope, s_pos[rp.axis * nt + l] * rp.freq);
      if (inverse) c.y = -c.y;
      cs[((e & 7) * per_cta + l) * turned + (e >> 3)] = c;
    }
  }
  __syncthreads();
  if (!work) return;
  float2 c[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) c[e] = turn ? cs[(e * per_cta + lt) * turned + duo] : make_float2(1.f, 0.f);
#pragma unroll 1
  for (int h = h0; h < heads;) {
    uint4 cu[UN][W], cv[UN][W];
#pragma unroll
    for (int i = 0; i < UN; ++i)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        cu[i][w] = u[i][w];
        cv[i][w] = v[i][w];
      }
    const int hc = h;
    h += UN * step;
    load(h);
#pragma unroll
    for (int i = 0; i < UN; ++i) {
      const int hh = hc + i * step;
      if (hh >= heads) break;
      float fu[8], fv[8];
#pragma unroll
      for (int w = 0; w < W; ++w) {
        unpack16<T>(cu[i][w], fu + 8 / W * w);
        unpack16<T>(cv[i][w], fv + 8 / W * w);
      }
      if (turn) {
#pragma unroll
        for (int e = 0; e < 8; ++e) rope_turn(fu[e], fv[e], c[e], fu[e], fv[e]);
      }
      T* y = hh < q.heads ? yq + hh * q.oh : yk + (hh - q.heads) * k.oh;
      store8<T>(y + da, fu);
      store8<T>(y + db, fv);
    }
  }
}

template <typename T>
static wnw_status launch_rotary(const wnw_rotary_args* a, cudaStream_t s) {
  RotarySide q{a->q, a->q_out, a->q_stride_b, a->q_stride_h, a->q_stride_n, a->qo_stride_b, a->qo_stride_h,
               a->qo_stride_n, a->num_q_heads};
  RotarySide k{a->k, a->k_out, a->k_stride_b, a->k_stride_h, a->k_stride_n, a->ko_stride_b, a->ko_stride_h,
               a->ko_stride_n, a->num_kv_heads};
  const int64_t total = int64_t(a->batch) * a->tokens;
  // tokens of a CTA: doubled while the grid has more than three CTAs an SM
  // (then it has 1.5 at least) and each place a thread
  int per = 1;
  while (per < kRotTokens && total > int64_t(per) * 3 * sm_count() && 2 * per * (a->head_dim / 16) <= kRotThreads) per *= 2;
  const size_t smem = sizeof(float2) * per * (a->rope.rot / 2);
  const int64_t grid = (total + per - 1) / per;
  WNW_CHECK_ARG(grid < (int64_t(1) << 31), "too many tokens");
  rotary_kernel<T><<<static_cast<unsigned>(grid), kRotThreads, smem, s>>>(q, k, a->rope, a->head_dim, a->tokens, total,
                                                                          per, a->inverse, a->err);
  WNW_CUDA_TRY(cudaGetLastError());
  return WNW_OK;
}

static bool strides_ok(int64_t b, int64_t h, int64_t n, int elems) {
  return b % elems == 0 && h % elems == 0 && n % elems == 0;
}

}  // namespace wnw

extern "C" wnw_status wnw_rotary(const wnw_rotary_args* a, void* stream) {
  using namespace wnw;
  WNW_CHECK_ARG(a != nullptr, "null args");
  WNW_CHECK_ARG(a->head_dim >= 16 && a->head_dim <= 512 && a->head_dim % 16 == 0,
                "head_dim %d: a multiple of 16 up to 512", a->head_dim);
  WNW_CHECK_ARG(a->batch >= 0 && a->tokens >= 0 && a->num_q_heads >= 0 && a->num_kv_heads >= 0, "negative size");
  WNW_CHECK_ARG(a->err != nullptr, "null error word");
  const int64_t heads = int64_t(a->num_q_heads) + a->num_kv_heads;
  if (a->batch == 0 || a->tokens == 0 || heads == 0) return WNW_OK;
  WNW_CHECK_ARG((a->num_q_heads == 0 || (a->q && a->q_out)) && (a->num_kv_heads == 0 || (a->k && a->k_out)),
                "null pointer argument");
  const int e16 = a->dtype == WNW_F32 ? 4 : 8;
  WNW_CHECK_ARG(a->num_q_heads == 0 || (aligned16(a->q) && aligned16(a->q_out) &&
                                        strides_ok(a->q_stride_b, a->q_stride_h, a->q_stride_n, e16) &&
                                        strides_ok(a->qo_stride_b, a->qo_stride_h, a->qo_stride_n, e16)),
                "q and its output need 16-byte aligned rows");
  WNW_CHECK_ARG(a->num_kv_heads == 0 || (aligned16(a->k) && aligned16(a->k_out) &&
                                         strides_ok(a->k_stride_b, a->k_stride_h, a->k_stride_n, e16) &&
                                         strides_ok(a->ko_stride_b, a->ko_stride_h, a->ko_stride_n, e16)),
                "k and its output need 16-byte aligned rows");
  WNW_CHECK_ARG(heads * a->head_dim <= (1 << 26), "too many heads");
  const wnw_status st = check_rope(a->rope, a->head_dim);
  if (st != WNW_OK) return st;
  WNW_CHECK_ARG(a->rope.rot > 0, "rotation of no dimensions");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (a->dtype) {
    case WNW_F32: return launch_rotary<float>(a, s);
    case WNW_F16: return launch_rotary<__half>(a, s);
    case WNW_BF16: return launch_rotary<__nv_bfloat16>(a, s);
    default: set_error("unknown dtype %d", a->dtype); return WNW_ERR_UNSUPPORTED;
  }
}

extern "C" wnw_status wnw_rotary_step(const wnw_rotary_args* a, const void* q, void* q_out, const void* k, void* k_out,
                                      const void* positions, void* stream) {
  using namespace wnw;
  WNW_CHECK_ARG(a != nullptr, "null args");
  wnw_rotary_args b = *a;
  b.q = q;
  b.q_out = q_out;
  b.k = k;
  b.k_out = k_out;
  b.rope.pos = positions;
  return wnw_rotary(&b, stream);
}
