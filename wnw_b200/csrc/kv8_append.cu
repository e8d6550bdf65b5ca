// Append to the paged 8-bit cache: keys rotated on the way, full blocks
// quantised, the unfinished block kept in 16 bits; the same tokens' queries
// rotated beside.
//
// A prompt's append (16-bit rows in, 8-bit codes out) takes 24.4 us for 15,064
// tokens of 8 heads, 3.8 TB/s (58 % of the copy rate).  The key CTAs' chains are
// its length: alone they take 22 us, 17 without angles, the values 14; 60 % of
// the issue slots are used while SMs are busy, 46 % over the launch.  A decoded
// token's append is latency: 3.3 us.
// One CTA takes one 32-token block of one or more kv heads of a
// sample, and of those the keys, the values or the queries: three short chains
// side by side instead of one after another, and only keys and queries need
// angles.
// Keys: a thread has a quarter of one token's row, loads it a head ahead,
// turns it (the block's cosines and sines lie in shared memory, computed once
// a CTA) and writes its codes straight into the record.
// Values are held transposed: the rows of the next head come into shared
// memory by asynchronous copies, and transposing matrix loads (ldmatrix.trans)
// with the tokens' rows in an order of our choice give a lane eight
// consecutive tokens of one dimension, so their codes leave as 8 bytes a lane,
// 256 a warp.
#include <algorithm>
#include <climits>

#include "kv8.cuh"
#include "mma.cuh"
#include "rope.cuh"

namespace wnw {

constexpr int kApThreads = 128;
constexpr int kApWarps = 4;
constexpr int kApHeads = 32;  // heads of a CTA at most

struct AppendParams {
  wnw_kv8_append_args a;
  int heads_per_cta, groups;  // kv heads of a CTA, groups of that many
  int page_shift;
};

// the larger magnitudes of two packed pairs of 16-bit numbers (NaN wins; the
// sign bits are not used)
template <typename T>
__device__ __forceinline__ uint32_t max_mag2(uint32_t m, uint32_t x);
template <>
__device__ __forceinline__ uint32_t max_mag2<__nv_bfloat16>(uint32_t m, uint32_t x) {
  uint32_t d;
  asm("max.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(m), "r"(x));
  return d;
}
template <>
__device__ __forceinline__ uint32_t max_mag2<__half>(uint32_t m, uint32_t x) {
  uint32_t d;
  asm("max.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(d) : "r"(m), "r"(x));
  return d;
}
// of a warp's pairs: the largest magnitude's bits (NaN above infinity)
__device__ __forceinline__ uint32_t warp_mag(uint32_t m) {
  return __reduce_max_sync(0xffffffffu, max(m & 0x7fffu, (m >> 16) & 0x7fffu));
}

// one 16-bit number's bits as fp32
template <typename T>
__device__ __forceinline__ float half_bits_to_f(uint32_t h) {
  const uint16_t u = static_cast<uint16_t>(h);
  return DT<T>::to_f(*reinterpret_cast<const T*>(&u));
}

// Two fp32 numbers in one register pair: both products in one instruction.
// Sums stay single: the compiler joins paired products and sums into paired
// fused ones, which round once where rope_turn and the codes round twice
struct F2 {
  uint64_t v;
};
__device__ __forceinline__ F2 f2(float a, float b) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 f2_mul(F2 a, F2 b) {
  float2 r;
  asm("{\n\t.reg .b64 p;\n\tmul.rn.f32x2 p, %2, %3;\n\tmov.b64 {%0, %1}, p;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "l"(a.v), "l"(b.v));
  return r;
}

template <int CODE>
__device__ inline uint32_t code4(float a, float b, float c, float d, F2 inv) {
  const float2 x = f2_mul(f2(a, b), inv), y = f2_mul(f2(c, d), inv);
  if constexpr (CODE == WNW_KV8_E4M3) {
    uint32_t w;
    asm("{\n\t.reg .b16 lo, hi;\n\tcvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n\t"
        "cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n\tmov.b32 %0, {lo, hi};\n\t}"
        : "=r"(w)
        : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
    return w;
  } else {
    // 1.5 x 2^23 + x: the nearest integer (halves to even) is the low byte;
    // |x| is at most 127 and a few units in the last place
    auto q = [](float x) { return __float_as_uint(__fadd_rn(x, 12582912.f)); };
    return __byte_perm(__byte_perm(q(x.x), q(x.y), 0x0040), __byte_perm(q(y.x), q(y.y), 0x0040), 0x5410);
  }
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// the two chunks of a place (8 pairs), turned in place, two pairs at a time
// with rope_turn's roundings; c: two pairs' cosines, then their sines, a word,
// every fourth word
template <typename T>
__device__ __forceinline__ void turn_place(uint4 (&w)[2], const float4* c) {
  float u[8], v[8];
  unpack16<T>(w[0], u);
  unpack16<T>(w[1], v);
  uint32_t* a = reinterpret_cast<uint32_t*>(&w[0]);
  uint32_t* b = reinterpret_cast<uint32_t*>(&w[1]);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float4 c2 = c[4 * e];
    const F2 co = f2(c2.x, c2.y), si = f2(c2.z, c2.w);
    const F2 x = f2(u[2 * e], u[2 * e + 1]), y = f2(v[2 * e], v[2 * e + 1]);
    const float2 xc = f2_mul(x, co), ys = f2_mul(y, si), yc = f2_mul(y, co), xs = f2_mul(x, si);
    a[e] = pack2<T>(__fsub_rn(xc.x, ys.x), __fsub_rn(xc.y, ys.y));
    b[e] = pack2<T>(__fadd_rn(yc.x, xs.x), __fadd_rn(yc.y, xs.y));
  }
}

template <int D>
struct ApSmem {
  static constexpr int kRow = 2 * D + 16;         // a value row, padded against bank conflicts
  static constexpr int kStage = kKv8Block * kRow;
  static constexpr int kCsRow = D / 2 * 8 + 64;   // a token's cosines and sines
  static constexpr int kBytes = 2 * kStage > kKv8Block * kCsRow ? 2 * kStage : kKv8Block * kCsRow;
};

// what a CTA works on
enum { kApKeys = 0, kApValues = 1, kApQueries = 2 };

// The order in which a launch's CTAs start.  Those of queries, keys and values
// side by side (in blockIdx.x) for long appends with queries: 777 tokens of 4
// samples 17.8 us, 18.3 in the other order, 1,841 of 3 16.8 and 19.7.  All
// queries, then all keys, then all values (in blockIdx.z), the longest chains
// first, for the others: a prompt without queries 24.4 us, 27.5 side by side;
// few CTAs with queries 5.8 and 7.0
template <int RESIDENT>
__host__ __device__ inline bool append_mixed(const wnw_kv8_append_args& a) {
  return RESIDENT > 4 && a.q != nullptr;
}

template <typename T, int D, int CODE, int RESIDENT>
__global__ void __launch_bounds__(kApThreads, RESIDENT) kv8_append_kernel(const __grid_constant__ AppendParams p) {
  using Rec = Kv8Rec<D>;
  using Sm = ApSmem<D>;
  constexpr int DPT = D / 64;  // places (pairs of 8-element chunks) a thread has of a key row
  constexpr int VG = D / 32;   // groups of 8 value dimensions a warp has
  const wnw_kv8_append_args& a = p.a;
  const wnw_kv8_store& st = a.store;
  extern __shared__ __align__(128) uint8_t smem[];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.y;
  // queries, keys, values: the longest chains start first
  const bool mixed = append_mixed<RESIDENT>(a);  // see append_mixed
  const int block = mixed ? blockIdx.x / 3 : blockIdx.x;
  const int part = mixed ? blockIdx.x - 3 * block : blockIdx.z / p.groups;
  const int role = a.q == nullptr ? part : part == 0 ? kApQueries : part - 1;
  const int h0 = (mixed ? blockIdx.z : blockIdx.z - part * p.groups) * p.heads_per_cta;
  const int nh = min(p.heads_per_cta, a.num_kv_heads - h0);
  const int half = a.rope.rot / 2;
  const int turned = a.rope.rot / 16;
  const int row = tid >> 2, quarter = tid & 3;  // the thread's token of the block and its part of a row

  pdl_wait();
  pdl_launch_dependents();
  const int64_t start = a.starts ? a.starts[b] : 0;
  const int count = a.counts ? a.counts[b] : a.tokens;
  if (count <= 0 || start < 0 || start + count > a.tokens || count > a.max_count) {
    if (count != 0 && tid == 0 && blockIdx.x == 0 && blockIdx.z == 0) atomicOr(st.err, WNW_DEVERR_BAD_INDEX);
    return;
  }

  // A CTA's items: of each head the block number blockIdx.x behind its length;
  // where the tail slot that the first block's earlier tokens are read from is
  // the one that the last block's tokens are written to, the first block's CTA
  // does the last block too, afterwards.  A lane looks a head's length and page
  // up, so that no head waits for its own, and leaves what is to be done in one
  // word of four:
  //   x  the call's token at the block's row 0 (were it new)
  //   y  the record of a full block
  //   z  head | the new tokens' rows [lo, hi) << 8, 16 | tail slot << 24
  __shared__ int4 s_item[2 * kApHeads];
  __shared__ int s_items;
  __shared__ uint32_t s_mag[2][kApWarps];
  if (warp == 0) {
    int L = 0, end = 0, rec = 0, jb[2] = {-1, -1};
    if (lane < nh) {
      const int seg = b * a.num_kv_heads + h0 + lane;
      L = a.seg_len[seg];
      const int64_t end64 = int64_t(L) + count;
      if (L < 0 || end64 > (int64_t(st.max_pages) << p.page_shift) * kKv8Block) {
        if (block == 0 && role == 0) atomicOr(st.err, L < 0 ? WNW_DEVERR_BAD_INDEX : WNW_DEVERR_CAPACITY);
      } else {
        end = static_cast<int>(end64);
        const int j0 = L / kKv8Block, j = j0 + block, jl = end / kKv8Block;
        const bool clash = role != kApQueries && (L % kKv8Block) != 0 && (end % kKv8Block) != 0 && jl - j0 >= 2 &&
                           ((jl - j0) & 1) == 0;
        // (numbers of blocks: a block behind the last one may begin beyond 31 bits)
        if (j <= (end - 1) / kKv8Block && !(clash && j == jl)) jb[0] = j;
        if (clash && j == j0) jb[1] = jl;
        if (jb[0] >= 0 && j < jl && role != kApQueries) {
          const int page = __ldg(st.page_table + int64_t(seg) * st.max_pages + (j >> p.page_shift));
          if (page < 0 || page >= st.num_pages) {
            atomicOr(st.err, WNW_DEVERR_BAD_INDEX);
            jb[0] = -1;
          }
          rec = (page << p.page_shift) + (j & (st.page_blocks - 1));
        }
      }
    }
    __syncwarp();
    const uint32_t has0 = __ballot_sync(0xffffffffu, jb[0] >= 0), has1 = __ballot_sync(0xffffffffu, jb[1] >= 0);
    const uint32_t below = (1u << lane) - 1;
    int at = __popc(has0 & below) + __popc(has1 & below);
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      if (jb[pass] < 0) continue;
      const int r0 = jb[pass] * kKv8Block;
      s_item[at++] = make_int4(static_cast<int>(start) + r0 - L, rec,
                               lane | max(0, L - r0) << 8 | min(kKv8Block, end - r0) << 16 | (jb[pass] & 1) << 24, 0);
    }
    if (lane == 0) s_items = __popc(has0) + __popc(has1);
  }
  __syncwarp();
  __syncthreads();
  const int items = s_items;
  struct Item {
    int src, rec, head, lo, hi, slot;
  };
  auto item = [&](int i) {
    const int4 t = s_item[i];
    return Item{t.x, t.y, t.z & 255, t.z >> 8 & 255, t.z >> 16 & 255, t.z >> 24};
  };
  auto record = [&](const Item& t) { return static_cast<uint8_t*>(st.pool) + int64_t(t.rec) * Rec::kStride; };
  auto tail_slot = [&](const Item& t) { return (int64_t(b) * a.num_kv_heads + h0 + t.head) * 2 + t.slot; };
  // of all threads' magnitudes: the block's scale (a NaN or an infinity makes
  // it, so the block, NaN).  `par` alternates from call to call: one barrier
  // then keeps a call's reads ahead of the next but one's writes
  auto scale_of = [&](uint32_t m, int par) {
    m = warp_mag(m);
    if (lane == 0) s_mag[par][warp] = m;
    __syncwarp();
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kApWarps; ++w) m = max(m, s_mag[par][w]);
    const float f = half_bits_to_f<T>(m);
    const float s = __fmul_rn(f, 1.f / kv8_top<CODE>());
    return !(f < INFINITY) ? __int_as_float(0x7fffffff) : s < 1.17549435e-38f ? 1.17549435e-38f : s;
  };
  auto code8 = [](const uint4& w, float by) {
    const F2 inv = f2(by, by);
    float f[8];
    unpack16<T>(w, f);
    return make_uint2(code4<CODE>(f[0], f[1], f[2], f[3], inv), code4<CODE>(f[4], f[5], f[6], f[7], inv));
  };

  if (role == kApValues) {
    // an item's rows on their way into a stage; 16-byte chunk c of row r lies at
    // chunk c ^ 2 (r / 8): the matrix loads below take rows 8 apart together
    auto at_chunk = [](int r, int c) { return r * Sm::kRow + ((c ^ (2 * (r >> 3))) << 4); };
    constexpr int SR = kApThreads / (D / 8);  // rows a step of the CTA
    const int fr = tid / (D / 8), fc = tid % (D / 8);
    const T* v0 = static_cast<const T*>(a.v) + b * a.v_stride_b + h0 * a.v_stride_h + fr * a.v_stride_n + 8 * fc;
    auto fetch = [&](int i, int stage) {
      const Item t = item(i);
      uint8_t* dst = smem + stage * Sm::kStage;
      const T* from = v0 + t.head * a.v_stride_h + t.src * a.v_stride_n;
      if (t.lo == 0 && t.hi == kKv8Block) {
#pragma unroll
        for (int k = 0; k < D / 32; ++k, from += SR * a.v_stride_n)
          cp_async16(smem_u32(dst) + at_chunk(fr + k * SR, fc), from);
      } else {
        const uint16_t* tv = static_cast<const uint16_t*>(st.tail_v) + tail_slot(t) * D * kKv8Block;
#pragma unroll 1
        for (int r = fr; r < kKv8Block; r += SR, from += SR * a.v_stride_n) {
          if (r >= t.lo && r < t.hi) {
            cp_async16(smem_u32(dst) + at_chunk(r, fc), from);
          } else if (r < t.lo && t.hi == kKv8Block) {
            alignas(16) uint16_t e[8];
#pragma unroll
            for (int d = 0; d < 8; ++d) e[d] = tv[(8 * fc + d) * kKv8Block + r];
            *reinterpret_cast<uint4*>(dst + at_chunk(r, fc)) = *reinterpret_cast<const uint4*>(e);
          }
        }
      }
      cp_async_commit();
      __syncwarp();
    };
    if (items > 0) fetch(0, 0);
#pragma unroll 1
    for (int i = 0; i < items; ++i) {
      const int at = i & 1;
      cp_async_wait<0>();
      __syncthreads();  // everybody's rows of this stage are there, the other one is read
      if (i + 1 < items) fetch(i + 1, at ^ 1);
      const Item t = item(i);
      const int lo = t.lo, hi = t.hi;
      // this lane's values: dimension 8 (VG warp + c) + lane / 4, tokens 8 (lane % 4) ... + 7
      uint4 v[VG];
      uint32_t m = 0;
      const int r = 8 * ((lane & 7) >> 1) + 2 * (lane >> 3) + (lane & 1);  // the row this lane addresses
      const uint32_t from = smem_u32(smem + at * Sm::kStage);
      const int d0 = 8 * warp * VG + (lane >> 2), t0 = 8 * (lane & 3);
#pragma unroll
      for (int c = 0; c < VG; ++c) {
        ldsm_x4_t(from + at_chunk(r, warp * VG + c), v[c].x, v[c].y, v[c].z, v[c].w);
        m = max_mag2<T>(max_mag2<T>(max_mag2<T>(max_mag2<T>(m, v[c].x), v[c].y), v[c].z), v[c].w);
      }
      if (hi == kKv8Block) {
        const float s = scale_of(m, at);
        const float inv = __frcp_rn(s);
        uint8_t* out = record(t);
#pragma unroll
        for (int c = 0; c < VG; ++c)
          *reinterpret_cast<uint2*>(out + kKv8Block * D + (d0 + 8 * c) * kKv8Block + t0) = code8(v[c], inv);
        if (tid < 3) reinterpret_cast<float*>(out + Rec::kCodes)[1 + tid] = tid == 0 ? s : 0.f;
      } else {  // the unfinished block's new rows
        uint16_t* tv = static_cast<uint16_t*>(st.tail_v) + (tail_slot(t) * D + d0) * kKv8Block + t0;
#pragma unroll
        for (int c = 0; c < VG; ++c) {
          const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
          if (lo <= t0 && t0 + 8 <= hi) {
            *reinterpret_cast<uint4*>(tv + 8 * c * kKv8Block) = v[c];
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (t0 + e >= lo && t0 + e < hi)
                tv[8 * c * kKv8Block + e] = static_cast<uint16_t>(e & 1 ? w[e / 2] >> 16 : w[e / 2]);
          }
        }
      }
      __syncwarp();
    }
    return;
  }

  // ---- keys and queries
  int dk[DPT][2];  // the dimensions of the thread's chunks
  bool turn[DPT];
#pragma unroll
  for (int x = 0; x < DPT; ++x) {
    const int duo = 4 * x + quarter;  // (neighbouring threads' chunks side by side)
    turn[x] = duo < turned;
    dk[x][0] = turn[x] ? 8 * duo : a.rope.rot + 16 * (duo - turned);
    dk[x][1] = turn[x] ? 8 * duo + half : dk[x][0] + 8;
  }
  // cosines and sines: pair e of token r; pairs two a word, a place's four
  // words 64 bytes apart, neighbouring threads' words side by side.  A thread
  // computes one pair's for some of the rows, from the block's positions
  const int ae = half ? tid % half : 0, arow = half ? tid / half : 0, astep = half ? kApThreads / half : 1;
  uint8_t* cs_mine;
  {
    const int duo = ae >> 3, w = (ae & 7) >> 1;
    cs_mine = smem + ((duo / 4 * 4 + w) * 4 + duo % 4) * 16 + (ae & 1) * 4;
  }
  __shared__ double s_pos[4][kKv8Block];
  RopePair rp{0, 0.0};
  if (half && arow < astep) rp = rope_pair(a.rope, ae, st.err);
  int have = INT_MIN;  // the table's row r is token r + have of the call
  auto positions = [&](const Item& t) {
    if (half && warp < a.rope.num_axes && lane >= t.lo && lane < t.hi)
      s_pos[warp][lane] = rope_pos(a.rope, warp, b, t.src + lane);
    __syncwarp();
  };
  auto angles = [&](const Item& t) {
    const int lo = t.lo, hi = t.hi;
    __syncthreads();  // the last table is read, the positions are there
    if (arow < astep) {
      constexpr int UN = 4;  // chains of dependent 64-bit operations side by side
#pragma unroll 1
      for (int r = lo + arow; r < hi; r += UN * astep) {
        float2 c[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) c[u] = rope_turn_of(a.rope, s_pos[rp.axis][min(r + u * astep, hi - 1)] * rp.freq);
#pragma unroll
        for (int u = 0; u < UN; ++u)
          if (r + u * astep < hi) {
            float* to = reinterpret_cast<float*>(cs_mine + (r + u * astep) * Sm::kCsRow);
            to[0] = c[u].x;
            to[2] = c[u].y;
          }
      }
    }
    __syncwarp();
    __syncthreads();
    have = t.src;
  };
  const float4* cs = reinterpret_cast<const float4*>(smem + row * Sm::kCsRow + quarter * 16);
  struct Row {
    uint4 c[DPT][2];
  };

  if (role == kApKeys) {
    const T* k0 = static_cast<const T*>(a.k) + b * a.k_stride_b + h0 * a.k_stride_h + row * a.k_stride_n;
    auto fetch = [&](int i, Row& w) {
      const Item t = item(i);
      const T* kr = k0 + t.head * a.k_stride_h + t.src * a.k_stride_n;
      bool there = row >= t.lo && row < t.hi;
      if (row < t.lo && t.hi == kKv8Block) {
        there = true;
        kr = static_cast<const T*>(st.tail_k) + (tail_slot(t) * kKv8Block + row) * D;
      }
      if (there) {
#pragma unroll
        for (int x = 0; x < DPT; ++x)
#pragma unroll
          for (int y = 0; y < 2; ++y) w.c[x][y] = __ldcs(reinterpret_cast<const uint4*>(kr + dk[x][y]));
      }
      __syncwarp();
    };
    Row x, ahead;
    if (items > 0) {
      fetch(0, ahead);
      positions(item(0));
    }
    int par = 0;
#pragma unroll 1
    for (int i = 0; i < items; ++i) {
      x = ahead;
      if (i + 1 < items) fetch(i + 1, ahead);
      const Item t = item(i);
      if (half && t.src != have) {
        if (have != INT_MIN) {
          __syncthreads();  // the last positions are read
          positions(t);
        }
        angles(t);
      }
      const bool fresh = row >= t.lo && row < t.hi;
      uint32_t m = 0;
#pragma unroll
      for (int y = 0; y < DPT; ++y) {
        if (fresh && turn[y]) turn_place<T>(x.c[y], cs + 16 * y);  // rounded to the type, as the model's keys
#pragma unroll
        for (int z = 0; z < 2; ++z)
          m = max_mag2<T>(max_mag2<T>(max_mag2<T>(max_mag2<T>(m, x.c[y][z].x), x.c[y][z].y), x.c[y][z].z), x.c[y][z].w);
      }
      __syncwarp();
      if (t.hi == kKv8Block) {
        const float s = scale_of(m, par);
        par ^= 1;
        const float inv = __frcp_rn(s);
        uint8_t* out = record(t);
        uint2 kc[DPT][2];
#pragma unroll
        for (int y = 0; y < DPT; ++y)
#pragma unroll
          for (int z = 0; z < 2; ++z) kc[y][z] = code8(x.c[y][z], inv);
        auto k_at = [&](int d) { return out + (d >> 6) * kKv8Block * 64 + row * 64 + (d & 63); };
#pragma unroll
        for (int y = 0; y < DPT; ++y)
#pragma unroll
          for (int z = 0; z < 2; ++z) *reinterpret_cast<uint2*>(k_at(dk[y][z])) = kc[y][z];
        if (tid == 0) *reinterpret_cast<float*>(out + Rec::kCodes) = s;
      } else if (fresh) {  // the unfinished block's new rows
        T* tk = static_cast<T*>(st.tail_k) + (tail_slot(t) * kKv8Block + row) * D;
#pragma unroll
        for (int y = 0; y < DPT; ++y) {
          *reinterpret_cast<uint4*>(tk + dk[y][0]) = x.c[y][0];
          *reinterpret_cast<uint4*>(tk + dk[y][1]) = x.c[y][1];
        }
      }
      __syncwarp();
      // (the earlier tokens of a first block were read before its barrier, the
      // last block's are written behind it)
    }
    return;
  }

#pragma unroll 1
  for (int i = 0; i < items; ++i) {
    const Item t = item(i);
    const int per_kv = row >= t.lo && row < t.hi ? a.group : 0;  // this thread's query heads
    const int64_t n = t.src + row, h = int64_t(h0 + t.head) * a.group;
    const T* x = static_cast<const T*>(a.q) + b * a.q_stride_b + h * a.q_stride_h + n * a.q_stride_n;
    T* y = static_cast<T*>(a.q_out) + b * a.qo_stride_b + h * a.qo_stride_h + n * a.qo_stride_n;
    constexpr int UN = RESIDENT > 4 ? 1 : 2;  // heads ahead of those worked on
    Row w[UN];
    auto load = [&](int g) {
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        if (g + k < per_kv) {
#pragma unroll
          for (int z = 0; z < DPT; ++z)
#pragma unroll
            for (int e = 0; e < 2; ++e) w[k].c[z][e] = __ldcs(reinterpret_cast<const uint4*>(x + dk[z][e]));
        }
        x += a.q_stride_h;
      }
    };
    load(0);
    __syncwarp();
    if (t.src != have) {
      if (have != INT_MIN) __syncthreads();  // the last positions are read
      positions(t);
      angles(t);
    }
#pragma unroll 1
    for (int g = 0; g < per_kv; g += UN) {
      Row u[UN];
#pragma unroll
      for (int k = 0; k < UN; ++k) u[k] = w[k];
      load(g + UN);
#pragma unroll
      for (int k = 0; k < UN; ++k) {
        if (g + k >= per_kv) break;
#pragma unroll
        for (int z = 0; z < DPT; ++z) {
          if (turn[z]) turn_place<T>(u[k].c[z], cs + 16 * z);
#pragma unroll
          for (int e = 0; e < 2; ++e) *reinterpret_cast<uint4*>(y + dk[z][e]) = u[k].c[z][e];
        }
        y += a.qo_stride_h;
      }
    }
  }
}

template <typename T, int D, int CODE, int RESIDENT>
static wnw_status launch_append(const wnw_kv8_append_args* a, int blocks, cudaStream_t s) {
  AppendParams p;
  p.a = *a;
  p.page_shift = 0;
  while ((1 << p.page_shift) < a->store.page_blocks) ++p.page_shift;
  // Heads of one CTA share its look-ups and angles: as many as leave the
  // device full.  15,064 tokens, 8 heads: 24.4 us with all heads in a CTA (942
  // CTAs), a fifth more with four; 777 tokens of 4 samples, 4 heads: 17.8 us
  // with one, a fifth more with two.  Single tokens are all latency: their CTAs
  // go out in one wave (32 of 8 heads: 3.7 us with two heads a CTA, 4.8 in 768
  // CTAs)
  const int64_t wave = int64_t(RESIDENT) * sm_count();
  const int roles = a->q ? 3 : 2;
  const int most = std::min(a->num_kv_heads, kApHeads);
  auto ctas = [&](int h) { return int64_t(blocks) * a->batch * ((a->num_kv_heads + h - 1) / h) * roles; };
  int hpc = 1;
  while (hpc < most && (RESIDENT == 4 ? ctas(hpc) > wave : ctas(std::min(most, 2 * hpc)) >= wave))
    hpc = std::min(most, 2 * hpc);
  p.heads_per_cta = hpc;
  const int groups = p.groups = (a->num_kv_heads + hpc - 1) / hpc;
  WNW_CHECK_ARG(a->batch <= 65535 && groups <= 21845, "batch or heads beyond 65,535");
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  const bool mixed = append_mixed<RESIDENT>(*a);
  cfg.gridDim = mixed ? dim3(3 * blocks, a->batch, groups) : dim3(blocks, a->batch, roles * groups);
  cfg.blockDim = dim3(kApThreads, 1, 1);
  cfg.dynamicSmemBytes = ApSmem<D>::kBytes;
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  WNW_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv8_append_kernel<T, D, CODE, RESIDENT>, p));
  return WNW_OK;
}

// Single tokens and appends of few CTAs: four CTAs an SM with all the registers
// they like (30 tokens of 3 samples, 8 heads and 64 query heads: 6.2 us, 6.7 the
// other way; a single token 3.3 and 3.7).  Others: six CTAs an SM, eight at
// head_dim 64 (777 tokens of 4 samples at head_dim 128: 17.8 us, 21.4 with
// four; 15,064 tokens of 8 heads at head_dim 64: 15.5 us, 17.3 with six; at
// head_dim 128 seven and eight take 28 and 32 us instead of 24.4)
template <typename T, int D, int CODE>
static wnw_status append_size(const wnw_kv8_append_args* a, cudaStream_t s) {
  const int blocks = (kKv8Block - 1 + a->max_count + kKv8Block - 1) / kKv8Block;
  const int64_t ctas = int64_t(blocks) * a->batch * a->num_kv_heads * (a->q ? 3 : 2);
  return blocks == 1 || ctas <= 2 * sm_count() ? launch_append<T, D, CODE, 4>(a, blocks, s)
                                               : launch_append<T, D, CODE, D == 64 ? 8 : 6>(a, blocks, s);
}

template <typename T, int D>
static wnw_status append_code(const wnw_kv8_append_args* a, cudaStream_t s) {
  return a->store.code == WNW_KV8_E4M3 ? append_size<T, D, WNW_KV8_E4M3>(a, s) : append_size<T, D, WNW_KV8_INT8>(a, s);
}

template <typename T>
static wnw_status append_dim(const wnw_kv8_append_args* a, cudaStream_t s) {
  return a->store.head_dim == 64 ? append_code<T, 64>(a, s) : append_code<T, 128>(a, s);
}

}  // namespace wnw

extern "C" wnw_status wnw_kv8_append(const wnw_kv8_append_args* a, void* stream) {
  using namespace wnw;
  WNW_CHECK_ARG(a != nullptr, "null args");
  wnw_status st = check_kv8_store(a->store);
  if (st != WNW_OK) return st;
  WNW_CHECK_ARG(a->batch > 0 && a->num_kv_heads > 0 && int64_t(a->batch) * a->num_kv_heads == a->store.num_segs,
                "batch %d x kv heads %d is not the store's %d segments", a->batch, a->num_kv_heads,
                a->store.num_segs);
  WNW_CHECK_ARG(a->tokens >= 0 && a->max_count >= 0 && a->max_count <= a->tokens && a->tokens < (1 << 30),
                "max_count %d of %d tokens", a->max_count, a->tokens);
  WNW_CHECK_ARG(a->seg_len != nullptr, "null lengths");
  if (a->max_count == 0) return WNW_OK;
  WNW_CHECK_ARG(a->counts != nullptr || a->max_count == a->tokens, "max_count without counts");
  WNW_CHECK_ARG(a->counts != nullptr || a->starts == nullptr, "starts without counts");
  WNW_CHECK_ARG(a->k && a->v && aligned16(a->k) && aligned16(a->v), "k and v must be given, 16-byte aligned");
  WNW_CHECK_ARG(((a->k_stride_b | a->k_stride_h | a->k_stride_n | a->v_stride_b | a->v_stride_h | a->v_stride_n) & 7) == 0,
                "k and v strides must be multiples of 8 elements");
  if (a->q != nullptr) {
    WNW_CHECK_ARG(a->rope.rot > 0, "queries are taken to be rotated: a rotation is needed");
    WNW_CHECK_ARG(a->group >= 1 && a->group <= 1024, "group %d", a->group);
    WNW_CHECK_ARG(a->q_out && aligned16(a->q) && aligned16(a->q_out) &&
                      ((a->q_stride_b | a->q_stride_h | a->q_stride_n | a->qo_stride_b | a->qo_stride_h |
                        a->qo_stride_n) & 7) == 0,
                  "q and its output need 16-byte aligned rows");
  }
  st = check_rope(a->rope, a->store.head_dim);
  if (st != WNW_OK) return st;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->store.dtype == WNW_F16 ? append_dim<__half>(a, s) : append_dim<__nv_bfloat16>(a, s);
}

extern "C" wnw_status wnw_kv8_append_step(const wnw_kv8_append_args* a, const void* k, const void* v,
                                          const int32_t* seg_len, const int32_t* starts, const int32_t* counts,
                                          const void* positions, const void* q, void* q_out, void* stream) {
  using namespace wnw;
  WNW_CHECK_ARG(a != nullptr, "null args");
  wnw_kv8_append_args b = *a;
  b.k = k;
  b.v = v;
  b.seg_len = seg_len;
  b.starts = starts;
  b.counts = counts;
  b.rope.pos = positions;
  b.q = q;
  b.q_out = q_out;
  return wnw_kv8_append(&b, stream);
}
