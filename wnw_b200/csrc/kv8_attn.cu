// Decode attention over the paged 8-bit cache: one query token a segment.
//
// Per segment (kv head of a sample) and its G <= 8 query heads
//   s_tg = scale * k_scale[block(t)] * (q_g . code(k_t))
//   o_g  = sum_t 2^(s_tg - m_g) v_scale[block(t)] code(v_t) / sum_t 2^(s_tg - m_g)
// in base 2, with an online maximum m_g.  It is bound by the codes' bytes:
// every block's record (4 KB of keys, 4 KB of values at head_dim 128, both
// scales behind them) is read once, by one bulk copy.
//
// Division of work: the blocks of all segments form one line, cut evenly
// over the grid's warps (148 CTAs of 8 warps) from the lengths on the device,
// so ragged batches and one long sequence both fill every SM, and nothing is
// planned on the host.  A warp streams its stretch through three records of
// shared memory of its own (197 KB an SM, all of it in flight at the start).
// Where the line passes from one segment to the next inside a warp, the warp
// writes the finished segment itself; pieces that several warps have of a
// segment are merged through shared memory, each warp a slice of the output,
// and parts of several CTAs through `partials`, slice by slice, by the last
// warp to arrive, in the line's order: results repeat bit for bit.
//
// Products: q is brought to [2^15, 2^16) per head by a power of two and held
// in fp16: exact for fp16 models, for bf16 ones down to 2^-32 of the head's
// largest dimension (11 bits, bf16's 8 fit; what fp16 cannot hold below that
// is under 2^-40 of it).  Codes become fp16 exactly, so the first product
// rounds in its fp32 accumulation only.  The second takes the probabilities
// of full blocks as two fp16 terms, 22 bits, so outputs are as near as with
// fp32 ones (one term, 2^-11 of each, is as much as an fp16 output's own
// rounding and an eighth of a bf16 one's; it was 1 to 3 % faster: two requests
// of 120k tokens 85.4 us, one of 15k 14.6).  They are held 2^14 above the
// running maximum's, so that what fp16 loses stays under 2^-39 of it
// (unscaled, 255 equal tokens 17 nats under a first one of value zero
// vanished); the values' scale takes the 2^14 back.  The unfinished block's
// are two terms of its type: 16 bits in bf16, 2^-8 of its output's rounding (a
// third term cost calls of a few tokens 3 to 5 %).  Both products run as
// m16n8k16 tensor-core ones with the head group as n: a query token has G
// rows only, the tensor pipe is busy 23 to 29 % of the time and its shape does
// not bound.  The value scale is applied to each block's product in fp32.
//
// Measured (e4m3, bf16, head_dim 128, groups of 4, 6,547 GB/s copy rate): two
// requests of 120k tokens 86.6 us = 5.7 TB/s of codes (87 %); 32 ragged
// requests of 6k tokens in int8, groups of 7, 48.3 us = 4.9 TB/s (SMs reach
// the end of their stretches up to 10 us apart); one request of 15k tokens
// 15.1 us, of which about 4 pass before the first record lands and 6 in the
// merge and its arrivals; 32 segments of 40 tokens 8 us, 3 segments of 9
// tokens, which nothing merges, 3.3.  With `fresh` the time ahead of the
// records hides behind the append (81.3, 44.2, 12.9 and 6.8 us).  The 16-bit
// kernel takes 154.7, 83.5 and 16.9 us for the first three lengths.
#include <atomic>
#include <type_traits>

#include "kv8.cuh"
#include "mma.cuh"

namespace wnw {

constexpr int kK8Threads = 256;
constexpr int kK8Warps = 8;
constexpr float kK8Log2e = 1.4426950408889634f;
constexpr float kK8Ln2 = 0.6931471805599453f;
constexpr float kK8Up = 16384.f, kK8Down = 1.f / 16384.f;  // fp16 probabilities are held 2^14 up

template <int D>
constexpr int k8_stages() {
  return D == 128 ? 3 : 6;
}

// a piece: output [G][D], maxima [G], sums [G], padded to 16 bytes; one a warp
// lies beside the stages, its other one in its stages, which are done by then
template <int D>
__host__ __device__ constexpr int k8_piece_floats(int G) {
  return G * D + (2 * G + 3) / 4 * 4;
}
// a CTA's part of a segment in `partials`: output, then maximum and sum, of each column of 4
__host__ __device__ constexpr int k8_part_floats(int cols) { return 6 * cols; }
template <int D>
constexpr int k8_smem_bytes(int G) {
  return kK8Warps * (k8_stages<D>() * Kv8Rec<D>::kUsed + 4 * k8_piece_floats<D>(G));
}

struct K8Params {
  wnw_kv8_attn_args a;
  int page_shift;
};

// four codes (one word) as two fp16 pairs: bytes 0, 1 and bytes 2, 3
template <int CODE>
__device__ __forceinline__ void codes_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (CODE == WNW_KV8_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  } else {
    // 0x6400 + u is 1024 + u in fp16: u = code + 128, so 1152 brings it back
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const uint32_t off = 0x64806480u;  // 1152, 1152
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(lo) : "r"(a), "r"(off));
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(hi) : "r"(b), "r"(off));
  }
}

__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}

// the line of blocks: a segment's length counts ceil(rows / 32) units, an
// empty one counts one (somebody has to write its zeros)
__device__ __forceinline__ int seg_units(int len) { return len <= 0 ? 1 : (len - 1) / kKv8Block + 1; }

// U units over NT warps: warp i starts at floor(i U / NT), in 32 bits
struct K8Line {
  int base, rem, NT;
  __device__ __forceinline__ int start(int i) const { return i * base + (i * rem) / NT; }
  // the warp that holds unit x
  __device__ __forceinline__ int warp_of(int x) const {
    const int U = base * NT + rem;
    int i = min(NT - 1, static_cast<int>(static_cast<float>(x) * (static_cast<float>(NT) / static_cast<float>(U))));
    while (start(i) > x) --i;
    while (start(i + 1) <= x) ++i;
    return i;
  }
};

template <typename T>
__device__ __forceinline__ void store4(T* p, float4 v) {
  uint2 u;
  u.x = pack2<T>(v.x, v.y);
  u.y = pack2<T>(v.z, v.w);
  *reinterpret_cast<uint2*>(p) = u;
}

// v += f x, s += f l
__device__ __forceinline__ void fma4(float4& v, const float4& x, float l, float f, float& s) {
  v.x = fmaf(x.x, f, v.x);
  v.y = fmaf(x.y, f, v.y);
  v.z = fmaf(x.z, f, v.z);
  v.w = fmaf(x.w, f, v.w);
  s = fmaf(l, f, s);
}

// column i (4 outputs) of a finished segment
template <typename T, int D>
__device__ __forceinline__ void k8_write(const wnw_kv8_attn_args& a, int seg, int i, float m, float l, float4 v) {
  const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
  const int64_t at = static_cast<int64_t>(seg) * a.group;
  store4<T>(static_cast<T*>(a.out) + at * D + 4 * i, make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv));
  if (a.lse != nullptr && 4 * i % D == 0) a.lse[at + 4 * i / D] = (m + log2f(l)) * kK8Ln2;
}

template <typename T, int D, int CODE>
__global__ void __launch_bounds__(kK8Threads, 1) kv8_attn_kernel(const __grid_constant__ K8Params p) {
  using Rec = Kv8Rec<D>;
  constexpr int ST = k8_stages<D>();
  constexpr int NS = D / 16;
  constexpr int NW = kK8Warps;
  const wnw_kv8_attn_args& a = p.a;
  const wnw_kv8_store& st = a.store;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[NW][ST];
  __shared__ int s_scan[NW];
  __shared__ int s_seg[NW], s_first[NW];  // the segment a warp starts in, and that segment's first unit
  // the pieces a warp leaves to be merged: e = 0 began before the warp's
  // stretch, e = 1 goes on behind it; their segment's first and end unit
  __shared__ int s_pseg[NW][2], s_pfirst[NW][2], s_pend[NW][2];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int G = a.group;
  const int S = st.num_segs;
  const int PF = k8_piece_floats<D>(G);
  const int cap = (st.max_pages << p.page_shift) * kKv8Block;
  uint8_t* my_stage = smem + warp * ST * Rec::kUsed;
  float* heads_area = reinterpret_cast<float*>(smem + NW * ST * Rec::kUsed);
  auto piece_ptr = [&](int w, int e) -> float* {  // [output G x D][maxima G][sums G]
    return e == 0 ? heads_area + w * PF : reinterpret_cast<float*>(smem + w * ST * Rec::kUsed);
  };
  // a length beyond the page table or below zero is refused (see rows_of): what fits is attended
  auto len_of = [&](int s) { return min(max(0, __ldg(a.seg_len + s)), cap); };
  if (lane == 0) {
#pragma unroll
    for (int i = 0; i < ST; ++i) mbar_init(&bars[warp][i], 1);
    fence_mbar_init();
    s_pseg[warp][0] = s_pseg[warp][1] = -1;
  }
  // `fresh` tokens may still be on their way in (a.fresh >= 0): lengths, page
  // table and the blocks before them are read ahead of the wait, so that the
  // records stream while the append that precedes this launch finishes
  const bool early = a.fresh >= 0;
  if (!early) {
    pdl_wait();
    pdl_launch_dependents();
  }

  // ---- where this warp's stretch of the line begins: the segment it starts
  // in, and that segment's first unit.  Up to 256 segments every warp sums all
  // lengths for itself (eight a lane, no barrier: a barrier and a look at
  // shared memory each are a tenth of a short call); beyond, the CTA does
  const int w0 = blockIdx.x * NW;
  K8Line line;
  int starts, my_seg = 0, my_first = 0;
  // units of segments [lo, hi), those before them over the scope, the total
  const bool alone = S <= 8 * 32;
  const int scope = alone ? 32 : kK8Threads, rank = alone ? lane : tid;
  const int per = (S + scope - 1) / scope;
  const int c0 = min(S, rank * per), c1 = min(S, c0 + per);
  int mine = 0;
  for (int s = c0; s < c1; ++s) mine += seg_units(len_of(s));
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  int before = incl - mine, U = __shfl_sync(0xffffffffu, incl, 31);
  if (!alone) {
    if (lane == 31) s_scan[warp] = incl;
    __syncthreads();
    U = 0;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if (w < warp) before += s_scan[w];
      U += s_scan[w];
    }
  }
  line.NT = min(static_cast<int>(gridDim.x) * NW, (U + NW - 1) / NW * NW);  // warps at work
  line.base = U / line.NT;
  line.rem = U - line.base * line.NT;
  if (w0 >= line.NT) return;  // (nothing read or written that the kernel before may be writing)
  starts = line.start(w0 + min(lane, NW));  // lane w: where warp w starts
  // the thread whose segments hold unit x finds the one
  auto find = [&](int x, int& seg, int& first) {
    int f = before, s = c0;
    for (;;) {
      const int n = seg_units(len_of(s));
      if (x < f + n) break;
      f += n;
      ++s;
    }
    seg = s;
    first = f;
  };
  if (alone) {
    const int x = __shfl_sync(0xffffffffu, starts, warp);
    const bool here = x >= before && x < before + mine;
    if (here) find(x, my_seg, my_first);
    __syncwarp();
    // (a warp without units may start behind the line: it has no segment)
    const uint32_t who = __ballot_sync(0xffffffffu, here);
    const int from = who ? __ffs(who) - 1 : 0;
    my_seg = __shfl_sync(0xffffffffu, my_seg, from);
    my_first = __shfl_sync(0xffffffffu, my_first, from);
  } else {
    uint32_t hits = 0;  // the warps that start in this thread's segments
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const int x = __shfl_sync(0xffffffffu, starts, w);
      hits |= (x >= before && x < before + mine ? 1u : 0u) << w;
    }
    for (; hits != 0; hits &= hits - 1) {
      const int w = __ffs(hits) - 1;
      find(line.start(w0 + w), s_seg[w], s_first[w]);
    }
    __syncwarp();
    __syncthreads();
    my_seg = s_seg[warp];
    my_first = s_first[warp];
  }
  const int X0 = __shfl_sync(0xffffffffu, starts, 0), X1 = __shfl_sync(0xffffffffu, starts, NW);
  const int x0 = __shfl_sync(0xffffffffu, starts, warp), x1 = __shfl_sync(0xffffffffu, starts, warp + 1);

  if (x0 < x1) {
    auto rows_of = [&](int s) {
      const int len = __ldg(a.seg_len + s);
      if ((len < 0 || len > cap) && lane == 0) atomicOr(st.err, len < 0 ? WNW_DEVERR_BAD_INDEX : WNW_DEVERR_CAPACITY);
      return min(max(0, len), cap);
    };
    // the query rows of the segment at hand (loaded behind the first copies'
    // issue: ahead of it they cost ragged batches 5 %)
    uint4 qraw[D / 64][2];
    auto load_q = [&](int seg) {
      const T* qs = static_cast<const T*>(a.q) + (static_cast<int64_t>(seg) * G + gid) * D + 16 * tig;
#pragma unroll
      for (int j = 0; j < D / 64; ++j)
#pragma unroll
        for (int v = 0; v < 2; ++v)
          qraw[j][v] = gid < G ? *reinterpret_cast<const uint4*>(qs + 64 * j + 8 * v) : make_uint4(0u, 0u, 0u, 0u);
    };
    // ---- producer: walks the stretch ahead of the consumer, full blocks only
    int ps = my_seg, pf = my_first, px = x0;
    int plen = rows_of(ps);
    int pend = pf + seg_units(plen), pfull = plen / kKv8Block;
    int rec_b0 = 0, rec_n = 0, rec = -1;  // lane i: the record of block rec_b0 + i
    int issued = 0, used = 0;
    uint32_t there = 0;  // bit i: stage i holds a record (its page exists)
    bool waited = !early;
    auto produce = [&]() {  // issues the next full block's copy, if the stretch has one
      for (;;) {
        if (px >= x1) return;
        if (px >= pend) {
          pf = pend;
          ++ps;
          plen = rows_of(ps);
          pend = pf + seg_units(plen);
          pfull = plen / kKv8Block;
          rec_b0 = rec_n = 0;
          continue;
        }
        const int b = px - pf;
        if (!waited && b < pfull && b >= (plen - a.fresh) / kKv8Block) return;  // perhaps not there yet
        ++px;
        if (b >= pfull) continue;  // the unfinished block
        if (b >= rec_b0 + rec_n) {
          rec_b0 = b;
          rec_n = 32;
          const int bi = b + lane;
          rec = -1;
          if (bi < pfull) {
            const int page =
                __ldg(st.page_table + static_cast<int64_t>(ps) * st.max_pages + (bi >> p.page_shift));
            if (page >= 0 && page < st.num_pages)
              rec = (page << p.page_shift) + (bi & (st.page_blocks - 1));
            else
              atomicOr(st.err, WNW_DEVERR_BAD_INDEX);
          }
        }
        const int r = __shfl_sync(0xffffffffu, rec, b - rec_b0);
        const int sg = issued % ST;
        there = (there & ~(1u << sg)) | (r >= 0 ? 1u << sg : 0u);  // no such page: the block counts as absent
        if (lane == 0) {
          if (r >= 0) {
            mbar_arrive_expect_tx(&bars[warp][sg], Rec::kUsed);
            bulk_g2s(my_stage + sg * Rec::kUsed, static_cast<const uint8_t*>(st.pool) + r * Rec::kStride, Rec::kUsed,
                     &bars[warp][sg]);
          } else {
            mbar_arrive(&bars[warp][sg]);
          }
        }
        ++issued;
        return;
      }
    };
#pragma unroll 1
    for (int i = 0; i < ST; ++i) produce();
    if (early) {
      pdl_wait();
      pdl_launch_dependents();
      waited = true;
#pragma unroll 1
      while (issued < ST && px < x1) produce();
    }

    // ---- consumer
    int cseg = my_seg, cf = my_first;
    for (int x = x0; x < x1;) {
      const int len = len_of(cseg);
      const int n = seg_units(len);
      const int nfull = len / kKv8Block, left = len - nfull * kKv8Block;
      const int xe = min(cf + n, x1);
      load_q(cseg);
      const bool began = x == cf, ends = xe == cf + n;
      // q as the B operand, dimensions in the order in which a lane's 16-byte
      // loads of the keys bring them: pair (4j + u) holds 64j + 16 tig + 4u + {0, 1}, {2, 3}
      uint32_t qb[NS][2];
      float fac;
      {
        uint32_t mx = 0;
        float qf[D / 4];
#pragma unroll
        for (int j = 0; j < D / 64; ++j)
#pragma unroll
          for (int v = 0; v < 2; ++v) unpack16<T>(qraw[j][v], qf + 16 * j + 8 * v);
#pragma unroll
        for (int e = 0; e < D / 4; ++e) mx = max(mx, __float_as_uint(qf[e]) & 0x7fffffffu);
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // (an infinity or a NaN comes through as it is; the factor back stays a normal number)
        const int e = mx >= 0x7f800000u || mx == 0 ? 0 : min(120, 142 - static_cast<int>(mx >> 23));
        const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
        fac = a.scale * kK8Log2e * __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
        for (int j = 0; j < D / 64; ++j)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float* f = qf + 16 * j + 4 * u;
            qb[4 * j + u][0] = pack2<__half>(f[0] * up, f[1] * up);
            qb[4 * j + u][1] = pack2<__half>(f[2] * up, f[3] * up);
          }
      }
      // the two heads of a lane's accumulators
      const float fac0 = __shfl_sync(0xffffffffu, fac, 8 * tig), fac1 = __shfl_sync(0xffffffffu, fac, 8 * tig + 4);
      float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
      float o[NS][4];
#pragma unroll
      for (int u = 0; u < NS; ++u) o[u][0] = o[u][1] = o[u][2] = o[u][3] = 0.f;

      // token of row `gid` of row group r (0..3): with it the transposed
      // probabilities of groups (0, 1), (2, 3) are the B operands of the two
      // 16-token steps in which a lane's 8 value bytes lie in order
      const int tok = 8 * (gid >> 1) + (gid & 1);

      // scores -> probabilities times `up` (fp32, in sc), the running state, al0 / al1.  (2^14 is not
      // taken into the exponent: beyond 2^24 a score less 14 is not that)
      auto softmax = [&](float (&sc)[2][4], float& al0, float& al1, float up) {
        float mx0 = fmaxf(fmaxf(sc[0][0], sc[0][2]), fmaxf(sc[1][0], sc[1][2]));
        float mx1 = fmaxf(fmaxf(sc[0][1], sc[0][3]), fmaxf(sc[1][1], sc[1][3]));
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
          mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, off));
          mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, off));
        }
        mx0 = fmaxf(mx0, m0);
        mx1 = fmaxf(mx1, m1);
        const float b0 = mx0 == -INFINITY ? 0.f : mx0, b1 = mx1 == -INFINITY ? 0.f : mx1;
        al0 = ex2(m0 - b0);
        al1 = ex2(m1 - b1);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sc[i][0] = ex2(sc[i][0] - b0);
          sc[i][1] = ex2(sc[i][1] - b1);
          sc[i][2] = ex2(sc[i][2] - b0);
          sc[i][3] = ex2(sc[i][3] - b1);
        }
        m0 = mx0;
        m1 = mx1;
        l0 = l0 * al0 + ((sc[0][0] + sc[0][2]) + (sc[1][0] + sc[1][2]));
        l1 = l1 * al1 + ((sc[0][1] + sc[0][3]) + (sc[1][1] + sc[1][3]));
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][e] *= up;
      };

      __syncwarp();
      if (ends && left > 0) {
        // ---- the unfinished block, 16-bit rows straight from global memory:
        // first, while the stretch's first copies are on their way
        const int64_t slot = static_cast<int64_t>(cseg) * 2 + (nfull & 1);
        const T* tk = static_cast<const T*>(st.tail_k) + slot * kKv8Block * D + 16 * tig;
        const T* tv = static_cast<const T*>(st.tail_v) + slot * kKv8Block * D;
        const float f0 = a.scale * kK8Log2e;
        float sc[2][4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[i][e] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const uint4 z = make_uint4(0u, 0u, 0u, 0u);
            const uint4 qv = qraw[j][v];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              const int ta = tok + 4 * i, tb = ta + 2;
              const uint4 ra = ta < left ? *reinterpret_cast<const uint4*>(tk + ta * D + 64 * j + 8 * v) : z;
              const uint4 rb = tb < left ? *reinterpret_cast<const uint4*>(tk + tb * D + 64 * j + 8 * v) : z;
              mma16816<T>(sc[i], ra.x, rb.x, ra.y, rb.y, qv.x, qv.y);
              mma16816<T>(sc[i], ra.z, rb.z, ra.w, rb.w, qv.z, qv.w);
            }
          }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const bool va = tok + 4 * i < left, vb = tok + 4 * i + 2 < left;
          sc[i][0] = va ? sc[i][0] * f0 : -INFINITY;
          sc[i][1] = va ? sc[i][1] * f0 : -INFINITY;
          sc[i][2] = vb ? sc[i][2] * f0 : -INFINITY;
          sc[i][3] = vb ? sc[i][3] * f0 : -INFINITY;
        }
        // probabilities as two terms of the type (8 + 8 bits for bf16, whose
        // range needs no 2^14; 11 + 11 for fp16)
        constexpr bool kHalf = std::is_same<T, __half>::value;
        float al0, al1;
        softmax(sc, al0, al1, kHalf ? kK8Up : 1.f);
        uint32_t pb[4], pr[4];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const float p0 = sc[i][2 * y], p1 = sc[i][2 * y + 1];
            const float h0 = DT<T>::to_f(DT<T>::from_f(p0)), h1 = DT<T>::to_f(DT<T>::from_f(p1));
            pb[2 * i + y] = movm_t(pack2<T>(h0, h1));
            pr[2 * i + y] = movm_t(pack2<T>(p0 - h0, p1 - h1));
          }
        uint32_t keep[4];  // tokens 8 tig + {0, 1}, {2, 3}, ...: what lies behind the last one is not read as numbers
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int t = 8 * tig + 2 * r;
          keep[r] = (t < left ? 0xffffu : 0u) | (t + 1 < left ? 0xffff0000u : 0u);
        }
#pragma unroll
        for (int u = 0; u < NS; ++u) {
          uint4 va = *reinterpret_cast<const uint4*>(tv + (16 * u + gid) * kKv8Block + 8 * tig);
          uint4 vc = *reinterpret_cast<const uint4*>(tv + (16 * u + 8 + gid) * kKv8Block + 8 * tig);
          va.x &= keep[0], va.y &= keep[1], va.z &= keep[2], va.w &= keep[3];
          vc.x &= keep[0], vc.y &= keep[1], vc.z &= keep[2], vc.w &= keep[3];
          mma16816<T>(o[u], va.x, vc.x, va.y, vc.y, pb[0], pb[1]);
          mma16816<T>(o[u], va.z, vc.z, va.w, vc.w, pb[2], pb[3]);
          mma16816<T>(o[u], va.x, vc.x, va.y, vc.y, pr[0], pr[1]);
          mma16816<T>(o[u], va.z, vc.z, va.w, vc.w, pr[2], pr[3]);
          if constexpr (kHalf) o[u][0] *= kK8Down, o[u][1] *= kK8Down, o[u][2] *= kK8Down, o[u][3] *= kK8Down;
        }
      }
      const int xb = min(xe, cf + nfull);
      for (; x < xb; ++x) {
        const int sg = used % ST;
        mbar_wait(&bars[warp][sg], (used / ST) & 1, st.err);
        __syncwarp();
        ++used;
        const uint8_t* rec_p = my_stage + sg * Rec::kUsed;
        if ((there >> sg) & 1u) {
          const float2 scl = *reinterpret_cast<const float2*>(rec_p + Rec::kCodes);
          const uint32_t kb = smem_u32(rec_p) + tok * 64 + 16 * tig;
          const uint32_t vb = smem_u32(rec_p) + kKv8Block * D + gid * kKv8Block + 8 * tig;
          float sc[2][4];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < D / 64; ++j) {
              const uint4 ra = lds128(kb + j * kKv8Block * 64 + (4 * i) * 64);      // group 2i: tokens tok + 4i
              const uint4 rb = lds128(kb + j * kKv8Block * 64 + (4 * i + 2) * 64);  // group 2i + 1
              const uint32_t wa[4] = {ra.x, ra.y, ra.z, ra.w}, wb[4] = {rb.x, rb.y, rb.z, rb.w};
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                uint32_t a0, a1, a2, a3;
                codes_to_half<CODE>(wa[u], a0, a2);
                codes_to_half<CODE>(wb[u], a1, a3);
                mma16816<__half>(c, a0, a1, a2, a3, qb[4 * j + u][0], qb[4 * j + u][1]);
              }
            }
            const float k0 = fac0 * scl.x, k1 = fac1 * scl.x;
            sc[i][0] = c[0] * k0;
            sc[i][1] = c[1] * k1;
            sc[i][2] = c[2] * k0;
            sc[i][3] = c[3] * k1;
          }
          float al0, al1;
          softmax(sc, al0, al1, kK8Up);
          // (a block of values below 2^-103 loses bits of its scale here)
          const float vs = scl.y * kK8Down;
          uint32_t pb[4], pr[4];  // probabilities, and what their rounding left
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const uint32_t w = pack2<__half>(sc[i][2 * y], sc[i][2 * y + 1]);
              const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w));
              pb[2 * i + y] = movm_t(w);
              pr[2 * i + y] = movm_t(pack2<__half>(sc[i][2 * y] - h.x, sc[i][2 * y + 1] - h.y));
            }
#pragma unroll
          for (int u = 0; u < NS; ++u) {
            const uint2 va = lds64(vb + 16 * u * kKv8Block);
            const uint2 vc = lds64(vb + (16 * u + 8) * kKv8Block);
            float c[4] = {0.f, 0.f, 0.f, 0.f};
            uint32_t a0, a1, a2, a3;
            codes_to_half<CODE>(va.x, a0, a2);
            codes_to_half<CODE>(vc.x, a1, a3);
            mma16816<__half>(c, a0, a1, a2, a3, pb[0], pb[1]);
            mma16816<__half>(c, a0, a1, a2, a3, pr[0], pr[1]);
            codes_to_half<CODE>(va.y, a0, a2);
            codes_to_half<CODE>(vc.y, a1, a3);
            mma16816<__half>(c, a0, a1, a2, a3, pb[2], pb[3]);
            mma16816<__half>(c, a0, a1, a2, a3, pr[2], pr[3]);
            o[u][0] = fmaf(vs, c[0], o[u][0] * al0);
            o[u][1] = fmaf(vs, c[1], o[u][1] * al1);
            o[u][2] = fmaf(vs, c[2], o[u][2] * al0);
            o[u][3] = fmaf(vs, c[3], o[u][3] * al1);
          }
        }
        __syncwarp();  // the stage is read
        produce();
      }
      x = xe;
      // ---- the stretch leaves the segment
#pragma unroll
      for (int off = 4; off < 32; off <<= 1) {
        l0 += __shfl_xor_sync(0xffffffffu, l0, off);
        l1 += __shfl_xor_sync(0xffffffffu, l1, off);
      }
      const int g0 = 2 * tig, g1 = g0 + 1;
      if (began && ends) {
        const float i0 = l0 > 0.f || l0 != l0 ? 1.f / l0 : 0.f, i1 = l1 > 0.f || l1 != l1 ? 1.f / l1 : 0.f;
        T* out = static_cast<T*>(a.out) + static_cast<int64_t>(cseg) * G * D;
#pragma unroll
        for (int u = 0; u < NS; ++u) {
          const int d0 = 16 * u + gid, d1 = d0 + 8;
          if (g0 < G) {
            out[g0 * D + d0] = DT<T>::from_f(o[u][0] * i0);
            out[g0 * D + d1] = DT<T>::from_f(o[u][2] * i0);
          }
          if (g1 < G) {
            out[g1 * D + d0] = DT<T>::from_f(o[u][1] * i1);
            out[g1 * D + d1] = DT<T>::from_f(o[u][3] * i1);
          }
        }
        if (a.lse != nullptr && gid == 0) {
          if (g0 < G) a.lse[static_cast<int64_t>(cseg) * G + g0] = (m0 + log2f(l0)) * kK8Ln2;
          if (g1 < G) a.lse[static_cast<int64_t>(cseg) * G + g1] = (m1 + log2f(l1)) * kK8Ln2;
        }
      } else {
        const int e = began ? 1 : 0;  // (the last piece's stages are done: every copy has been waited for)
        float* po = piece_ptr(warp, e);
        float* pm = po + G * D;
        if (gid == 0) {
          if (g0 < G) {
            pm[g0] = m0;
            pm[G + g0] = l0;
          }
          if (g1 < G) {
            pm[g1] = m1;
            pm[G + g1] = l1;
          }
        }
#pragma unroll
        for (int u = 0; u < NS; ++u) {
          const int d0 = 16 * u + gid, d1 = d0 + 8;
          if (g0 < G) {
            po[g0 * D + d0] = o[u][0];
            po[g0 * D + d1] = o[u][2];
          }
          if (g1 < G) {
            po[g1 * D + d0] = o[u][1];
            po[g1 * D + d1] = o[u][3];
          }
        }
        if (lane == 0) {
          s_pseg[warp][e] = cseg;
          s_pfirst[warp][e] = cf;
          s_pend[warp][e] = cf + n;
        }
      }
      __syncwarp();
      cf += n;
      ++cseg;
    }
  }
  if (early) pdl_wait();  // (a warp without units: it may write below)
  __syncwarp();
  __syncthreads();

  // ---- merges.  Every warp takes a slice of the output columns (4 outputs
  // each) of every run of pieces of one segment, and from here on works alone:
  // nothing below waits for another warp.  Lane 2 w + e holds warp w's piece e
  const int cw = G * D / (4 * NW);  // columns of a slice
  const int col = warp * cw + lane;
  int pseg = -1, pfirst = 0, pend = 0;
  if (lane < 2 * NW) {
    pseg = s_pseg[lane >> 1][lane & 1];
    pfirst = s_pfirst[lane >> 1][lane & 1];
    pend = s_pend[lane >> 1][lane & 1];
  }
  const uint32_t same = __match_any_sync(0xffffffffu, pseg);
  uint32_t runs = __ballot_sync(0xffffffffu, pseg >= 0 && (same & ((1u << lane) - 1)) == 0);
  // segments shared with other CTAs: from before, on behind
  int sh_seg[2] = {-1, -1}, sh_first = 0, sh_end[2] = {0, 0};
  const int cols = NW * cw;
  const int64_t PS = k8_part_floats(cols);
  for (; runs != 0; runs &= runs - 1) {
    const int lead = __ffs(runs) - 1;
    const uint32_t members = __shfl_sync(0xffffffffu, same, lead);
    const int seg = __shfl_sync(0xffffffffu, pseg, lead);
    const int first = __shfl_sync(0xffffffffu, pfirst, lead), end = __shfl_sync(0xffffffffu, pend, lead);
    const bool whole = first >= X0 && end <= X1;
    if (!whole) {
      if (first < X0) {
        sh_seg[0] = seg, sh_first = first, sh_end[0] = end;
      } else {
        sh_seg[1] = seg, sh_end[1] = end;
      }
    }
    if (lane < cw) {
      const int g = 4 * col / D;
      float m[NW], l[NW];
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const uint32_t has = members >> (2 * w) & 3u;
        const float* pc = piece_ptr(w, has >> 1) + G * D + g;
        m[w] = has ? pc[0] : -INFINITY;
        l[w] = has ? pc[G] : 0.f;
        mx = fmaxf(mx, m[w]);
      }
      const float bs = mx == -INFINITY ? 0.f : mx;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float ls = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const uint32_t has = members >> (2 * w) & 3u;
        if (has) fma4(v, reinterpret_cast<const float4*>(piece_ptr(w, has >> 1))[col], l[w], ex2(m[w] - bs), ls);
      }
      if (whole) {
        k8_write<T, D>(a, seg, col, mx, ls, v);
      } else {
        float* part = a.partials + (2 * static_cast<int64_t>(blockIdx.x) + (first < X0 ? 0 : 1)) * PS;
        reinterpret_cast<float4*>(part)[col] = v;
        reinterpret_cast<float2*>(part + 4 * cols)[col] = make_float2(mx, ls);
      }
    }
    __syncwarp();
  }
  if (sh_seg[0] < 0 && sh_seg[1] < 0) return;
  // the CTAs that hold a part of a shared segment: those of its first and its
  // last unit, and all between; of a slice's warps the last to arrive merges
  int ca[2], cb[2];
  ca[0] = sh_seg[0] >= 0 ? line.warp_of(sh_first) / NW : 0;
  ca[1] = blockIdx.x;
#pragma unroll
  for (int e = 0; e < 2; ++e) cb[e] = sh_seg[e] >= 0 ? line.warp_of(sh_end[e] - 1) / NW : 0;
  bool last = false;
  if (lane < 2) {
    const int seg = lane ? sh_seg[1] : sh_seg[0];
    if (seg >= 0) {
      int32_t* cnt = a.counters + static_cast<int64_t>(seg) * WNW_KV8_COUNTER_STRIDE + warp;
      last = atom_add_acq_rel_gpu(cnt, 1) == (lane ? cb[1] - ca[1] : cb[0] - ca[0]);
      if (last) *cnt = 0;
    }
  }
  const uint32_t lasts = __ballot_sync(0xffffffffu, last);
  __syncwarp();  // what lanes 0 and 1 acquired orders the other lanes' loads of partials too (a vote orders no memory)
#pragma unroll 1
  for (int e = 0; e < 2; ++e) {
    if (!(lasts >> e & 1u)) continue;
    const int c_first = e ? ca[1] : ca[0], np = (e ? cb[1] : cb[0]) - c_first + 1;
    // partial c: a CTA's from-before part, but the first CTA's on-behind part.
    // Lane groups take the partials in turn, twelve at a time in flight
    const float* base = a.partials + 2 * static_cast<int64_t>(c_first) * PS;
    const int groups = 32 / cw, grp = lane / cw, i = warp * cw + lane - grp * cw;
    float m = -INFINITY, l = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int PRE = 12;
    if (grp < groups) {
#pragma unroll 1
      for (int c0 = grp; c0 < np; c0 += PRE * groups) {
        float2 pm[PRE];
        float4 pv[PRE];
        float mx = m;
#pragma unroll
        for (int u = 0; u < PRE; ++u) {
          const int c = c0 + u * groups;
          pm[u] = make_float2(-INFINITY, 0.f);
          if (c < np) {
            const float* pc = base + (2 * static_cast<int64_t>(c) + (c == 0 ? 1 : 0)) * PS;
            pv[u] = __ldcg(reinterpret_cast<const float4*>(pc) + i);
            pm[u] = __ldcg(reinterpret_cast<const float2*>(pc + 4 * cols) + i);
          }
        }
#pragma unroll
        for (int u = 0; u < PRE; ++u) mx = fmaxf(mx, pm[u].x);
        const float bs = mx == -INFINITY ? 0.f : mx;
        const float f = ex2(m - bs);
        v.x *= f, v.y *= f, v.z *= f, v.w *= f, l *= f;
#pragma unroll
        for (int u = 0; u < PRE; ++u)
          if (c0 + u * groups < np) fma4(v, pv[u], pm[u].y, ex2(pm[u].x - bs), l);
        m = mx;
      }
    }
    __syncwarp();
    for (int q = 1; q < groups; ++q) {  // the groups' states, in order
      const int from = (lane + q * cw) & 31;
      const float qm = __shfl_sync(0xffffffffu, m, from), ql = __shfl_sync(0xffffffffu, l, from);
      const float4 qv = make_float4(__shfl_sync(0xffffffffu, v.x, from), __shfl_sync(0xffffffffu, v.y, from),
                                    __shfl_sync(0xffffffffu, v.z, from), __shfl_sync(0xffffffffu, v.w, from));
      if (grp == 0) {
        const float mx = fmaxf(m, qm), bs = mx == -INFINITY ? 0.f : mx;
        const float f = ex2(m - bs);
        v.x *= f, v.y *= f, v.z *= f, v.w *= f, l *= f;
        fma4(v, qv, ql, ex2(qm - bs), l);
        m = mx;
      }
      __syncwarp();
    }
    if (grp == 0) k8_write<T, D>(a, e ? sh_seg[1] : sh_seg[0], i, m, l, v);
    __syncwarp();
  }
}

template <typename T, int D, int CODE>
static wnw_status launch_kv8(const wnw_kv8_attn_args* a, cudaStream_t s) {
  static std::atomic<uint64_t> configured{0};
  {
    const wnw_status st = raise_smem_limit(configured, kv8_attn_kernel<T, D, CODE>, k8_smem_bytes<D>(8));
    if (st != WNW_OK) return st;
  }
  K8Params p;
  p.a = *a;
  p.page_shift = 0;
  while ((1 << p.page_shift) < a->store.page_blocks) ++p.page_shift;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(sm_count(), 1, 1);
  cfg.blockDim = dim3(kK8Threads, 1, 1);
  cfg.dynamicSmemBytes = k8_smem_bytes<D>(a->group);
  cfg.stream = s;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  WNW_CUDA_TRY(cudaLaunchKernelEx(&cfg, kv8_attn_kernel<T, D, CODE>, p));
  return WNW_OK;
}

template <typename T, int D>
static wnw_status attn_code(const wnw_kv8_attn_args* a, cudaStream_t s) {
  return a->store.code == WNW_KV8_E4M3 ? launch_kv8<T, D, WNW_KV8_E4M3>(a, s) : launch_kv8<T, D, WNW_KV8_INT8>(a, s);
}
template <typename T>
static wnw_status attn_dim(const wnw_kv8_attn_args* a, cudaStream_t s) {
  return a->store.head_dim == 64 ? attn_code<T, 64>(a, s) : attn_code<T, 128>(a, s);
}

}  // namespace wnw

extern "C" wnw_status wnw_kv8_attn_scratch(int head_dim, int group, int64_t* partial_floats) {
  using namespace wnw;
  WNW_CHECK_ARG(partial_floats != nullptr, "null pointer argument");
  WNW_CHECK_ARG((head_dim == 64 || head_dim == 128) && group >= 1 && group <= 8, "head_dim %d, group %d", head_dim,
                group);
  *partial_floats = int64_t(2) * sm_count() * k8_part_floats(group * head_dim / 4);
  return WNW_OK;
}

extern "C" wnw_status wnw_kv8_attn(const wnw_kv8_attn_args* a, void* stream) {
  using namespace wnw;
  WNW_CHECK_ARG(a != nullptr, "null args");
  const wnw_status st = check_kv8_store(a->store);
  if (st != WNW_OK) return st;
  WNW_CHECK_ARG(a->group >= 1 && a->group <= 8, "group %d (1..8)", a->group);
  WNW_CHECK_ARG(a->q && a->seg_len && a->out && a->partials && a->counters, "null pointer argument");
  WNW_CHECK_ARG(aligned16(a->q) && aligned16(a->out) && aligned16(a->partials), "q, out and partials must be 16-byte aligned");
  WNW_CHECK_ARG(a->scale == a->scale, "scale is NaN");
  WNW_CHECK_ARG(a->fresh >= -1, "fresh %d: -1 or a number of tokens", a->fresh);
  WNW_CHECK_ARG(int64_t(a->store.num_segs) * (int64_t(a->store.max_pages) * a->store.page_blocks + 1) < (int64_t(1) << 31),
                "2^31 blocks or more over all segments' page tables");
  int64_t need = 0;
  const wnw_status s2 = wnw_kv8_attn_scratch(a->store.head_dim, a->group, &need);
  if (s2 != WNW_OK) return s2;
  if (a->partial_floats < need) {
    set_error("partials hold %lld floats, %lld needed", static_cast<long long>(a->partial_floats),
              static_cast<long long>(need));
    return WNW_ERR_CAPACITY;
  }
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return a->store.dtype == WNW_F16 ? attn_dim<__half>(a, s) : attn_dim<__nv_bfloat16>(a, s);
}

extern "C" wnw_status wnw_kv8_attn_step(const wnw_kv8_attn_args* a, const void* q, const int32_t* seg_len, void* out,
                                        float* lse, int fresh, void* stream) {
  using namespace wnw;
  WNW_CHECK_ARG(a != nullptr, "null args");
  wnw_kv8_attn_args b = *a;
  b.q = q;
  b.seg_len = seg_len;
  b.out = out;
  b.lse = lse;
  b.fresh = fresh;
  return wnw_kv8_attn(&b, stream);
}
