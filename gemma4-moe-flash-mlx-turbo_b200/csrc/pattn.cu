// Attention over the pages of a cache: every row of a step (a decode token, a
// few, a whole prompt) against the positions that its window and the first
// `sinks` positions leave visible.
//   s_j = scale q . k_j,  out = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)
// with the running maximum m and sum of the online softmax in fp32.
//
// Two kernels share the rows of a step:
//   paged_attn_split_kernel  sequences with at most 8 (row, head) pairs to a kv
//                            head: decodes.  Bound by the pages' bytes.
//   paged_attn_rows_kernel   the others, a CTA per (row, head).
#include <algorithm>
#include <cmath>
#include <mutex>
#include "pattn.cuh"

namespace fmoe {
namespace pa {

// ---------------------------------------------------------------------------
// few rows: split over the keys
//
// The pages' bytes are what a decode costs, so the work is cut by them: all
// (sequence, kv head) items' keys form one line of granules of 16 positions (a
// granule never leaves its page), and every CTA takes the same length of it,
// whatever the sequences' lengths are.  A warp owns every NW-th granule of its
// CTA's part and keeps its own ring of cp.async copies, running maximum, sum
// and output, so that nothing in the loop waits for another warp and the copies
// run on across the ends of items.  At the end of an item its warps' results
// are joined in shared memory; an item that lies in several CTAs goes to
// scratch, and the CTA that arrives last joins the parts, in the order of the
// keys, so that the result does not depend on who that is.
//
// One granule, with the 8 columns being the item's (row, head) pairs:
//   S^T [16 keys x 8]   = K  [16 x D] Q^T    mma m16n8k16, A = K  (ldmatrix)
//   O^T [D x 8]        += V^T [D x 16] P^T   mma m16n8k16, A = V^T (ldmatrix.trans)
// The weights P are rounded to bf16 for the second product (the sum of the
// weights is kept of the unrounded ones, in fp32).  The maximum that the weights
// refer to is moved only when a score passes it by 2^8: fp32 sums lose nothing
// by it, and O is rescaled a few times per item at most.
//
// 4-bit rows are never unpacked to memory: a code is or-ed into the mantissa of
// bf16 128 (exact), and with the group's (s, b) of the key
//   q . k = sum_g s_g (q . (128 + c))_g + (b_g - 128 s_g) (sum of q)_g
// V's s goes into the weights, v = s (c - 8) + (b + 8 s), and what does not
// depend on the dim is summed apart in fp32.

template <int D_, int BITS_>
struct Few {
  static constexpr int D = D_, BITS = BITS_, NG = D / 64;
  // A warp's output is D / 2 registers, a bf16 piece of 512 dims 16 KB: four
  // warps there, so that a ring holds three pieces.
  static constexpr int NW = D == 512 && BITS == 16 ? 4 : 8, NT = 32 * NW;
  static constexpr int CODES = BITS == 16 ? 32 * D : 8 * D;  // a granule's rows of K or V
  static constexpr int PIECE = CODES + (BITS == 4 ? D : 0);  // and its (scale, bias) pairs
  static constexpr int NP = BITS == 16 ? 3 : D == 256 ? 10 : 5;  // pieces in a warp's ring
  static constexpr int OS = D + 4;                               // row stride of a joined output, floats
  static constexpr int MW = D == 256 || BITS == 4 ? 2 : 1;       // warps that hand over their output at a time
  static constexpr int MAXSEG = 32;
  static constexpr int OFF_O = NW * NP * PIECE, OFF_Q = OFF_O + MW * 8 * OS * 4, OFF_ML = OFF_Q + 16 * D;
  static constexpr int OFF_SEG = OFF_ML + NW * 16 * 4;
  static constexpr int SMEM = OFF_SEG + MAXSEG * 64;
  static constexpr int VPT = 8 * D / NT;  // joined values of a thread
};

// One item's part that lies in this CTA.
struct Seg {
  int seq, h, row0, rows;      // table row, kv head, first row of the step, its rows
  int p0, i0, i1, first_slot;  // position of the first row; this part's granules; where the item's first part goes
  int low, hi, ns, low_tile;   // its Span
  int item, cf, cl, slot;      // counter, CTAs that hold it, where this part goes
};
static_assert(sizeof(Seg) == 64, "segment list");

struct FewWs {
  unsigned* arrived;  // [n * Hkv], zero between calls
  float* o;           // [2 * grid][8][D]
  float2* ml;         // [2 * grid][8]
};

__device__ __forceinline__ void cp16z(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
  return y;
}

// 16-byte chunk c of row r of a 4-bit piece lies at chunk c ^ swz(r): the reads
// of K (8 lanes: 2 rows x 4 octets) and of V (4 rows x 2 octets) then touch all
// banks once.
template <int D, bool V>
__device__ __forceinline__ int swz4(int r) {
  if (D == 256) return V ? (r & 6) : (r & 1) << 2;
  return V ? ((r >> 1) & 1) | (r & 4) : r & 1;
}

// Copies granule `tile` (positions 16 * tile ..) of K or V into a ring piece;
// rows that no row of the item sees arrive as zeros (a weight of zero times what
// an unwritten row holds could be NaN).
template <class C, bool V>
__device__ __forceinline__ void copy_piece(const PagedDev& c, const AttnArgs& a, uint8_t* dst, const Seg& s, int tile,
                                           int page, int lane) {
  const uint8_t* blk = page_block(c, a.layer, max(page, 0), s.h, V);
  const int j0 = 16 * tile, slot = j0 & (c.ps - 1);
  auto size = [&](int r) {
    const int j = j0 + r;
    return page >= 0 && j < s.hi && (j >= s.low || j < a.sinks) ? 16 : 0;
  };
  if constexpr (C::BITS == 16) {
    const uint8_t* src = blk + (int64_t)slot * (2 * C::D);
    constexpr int CH = C::D / 8;
#pragma unroll
    for (int k = 0; k < 16 * CH / 32; ++k) {
      const int r = (k * 32) / CH, ch = (k * 32) % CH + lane;
      cp16z(dst + r * (2 * C::D) + ((ch ^ (r & 7)) << 4), src + r * (2 * C::D) + ch * 16, size(r));
    }
  } else {
    const uint8_t* src = blk + slot * (C::D / 2);
    const uint8_t* pairs = blk + c.ps * (C::D / 2) + slot * (C::D / 16);
    constexpr int CH = C::D / 32, PC = C::D / 256;  // chunks of a row's codes, of its pairs
#pragma unroll
    for (int k = 0; k < 16 * CH / 32; ++k) {
      const int r = (k * 32 + lane) / CH, ch = (k * 32 + lane) % CH;
      cp16z(dst + r * (C::D / 2) + ((ch ^ swz4<C::D, V>(r)) << 4), src + r * (C::D / 2) + ch * 16, size(r));
    }
    if (lane < 16 * PC) cp16z(dst + C::CODES + lane * 16, pairs + lane * 16, size(lane / PC));
  }
}

// Lane's view of the item's 8 columns: it holds columns 2t and 2t + 1 of S^T and O^T.
template <class C>
struct Acc {
  float o[C::D / 16][4];
  float corr[C::BITS == 4 ? C::NG : 1][2];  // 4-bit: sum of P (b + 8 s) - 136 P s of this lane's keys
  float m[2], l[2];
};

template <class C>
__device__ __forceinline__ void reset(Acc<C>& x) {
#pragma unroll
  for (int i = 0; i < C::D / 16; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) x.o[i][e] = 0.f;
#pragma unroll
  for (int g = 0; g < (C::BITS == 4 ? C::NG : 1); ++g) x.corr[g][0] = x.corr[g][1] = 0.f;
  x.m[0] = x.m[1] = -INFINITY;
  x.l[0] = x.l[1] = 0.f;
}

// S^T of one granule, times nothing yet.
template <class C>
__device__ __forceinline__ void scores(const uint8_t* kp, const uint32_t* qs, const float (&xs)[C::NG][2], int lane,
                                       float (&s)[4]) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (C::BITS == 16) {
    float acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
    const int r = lane & 15;
    const uint32_t row = smem_u32(kp) + r * (2 * C::D);
#pragma unroll
    for (int kk = 0; kk < C::D / 32; ++kk) {
      const uint4 b = lds_u4(qs + (kk * 32 + lane) * 4);
      uint32_t a0[4], a1[4];
      ldsm4(row + (((4 * kk + (lane >> 4)) ^ (r & 7)) << 4), a0);
      ldsm4(row + (((4 * kk + 2 + (lane >> 4)) ^ (r & 7)) << 4), a1);
      mma16816(acc[(2 * kk) & 3], a0[0], a0[1], a0[2], a0[3], b.x, b.y);
      mma16816(acc[(2 * kk + 1) & 3], a1[0], a1[1], a1[2], a1[3], b.z, b.w);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = (acc[0][e] + acc[1][e]) + (acc[2][e] + acc[3][e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = 0.f;
#pragma unroll
    for (int q4 = 0; q4 < C::NG / 4; ++q4) {  // four groups at a time: one 16-byte read each
      uint32_t w[2][2][4];                    // [key g, g + 8][octet t, t + 4][group]
      uint32_t pr[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = g + 8 * i;
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const int ch = (t + 4 * o) * (C::NG / 4) + q4;
          const uint4 v = lds_u4(kp + r * (C::D / 2) + ((ch ^ swz4<C::D, false>(r)) << 4));
          w[i][o][0] = v.x, w[i][o][1] = v.y, w[i][o][2] = v.z, w[i][o][3] = v.w;
        }
        const uint4 p = lds_u4(kp + C::CODES + r * (C::D / 16) + q4 * 16);
        pr[i][0] = p.x, pr[i][1] = p.y, pr[i][2] = p.z, pr[i][3] = p.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int gr = 4 * q4 + e;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
          const uint4 b = lds_u4(qs + ((gr * 2 + k2) * 32 + lane) * 4);
          mma16816(acc, nib_pair(w[0][0][e], 8 * k2), nib_pair(w[1][0][e], 8 * k2), nib_pair(w[0][1][e], 8 * k2),
                   nib_pair(w[1][1][e], 8 * k2), b.x, b.y);
          mma16816(acc, nib_pair(w[0][0][e], 8 * k2 + 4), nib_pair(w[1][0][e], 8 * k2 + 4),
                   nib_pair(w[0][1][e], 8 * k2 + 4), nib_pair(w[1][1][e], 8 * k2 + 4), b.z, b.w);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float sc = bf16lo(pr[i][e]), bi = fmaf(-128.f, sc, bf16hi(pr[i][e]));
          s[2 * i] = fmaf(sc, acc[2 * i], fmaf(bi, xs[gr][0], s[2 * i]));
          s[2 * i + 1] = fmaf(sc, acc[2 * i + 1], fmaf(bi, xs[gr][1], s[2 * i + 1]));
        }
      }
    }
  }
}

// O^T += V^T P^T; p: the weights of keys g, g + 8 (rows) and columns 2t, 2t + 1.
template <class C>
__device__ __forceinline__ void add_values(const uint8_t* vp, const float (&p)[4], int lane, Acc<C>& x) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (C::BITS == 16) {
    const uint32_t b0 = transpose8x8(pack_bf16x2(p[0], p[1])), b1 = transpose8x8(pack_bf16x2(p[2], p[3]));
    const int r = (lane & 7) + ((lane >> 4) << 3);
    const uint32_t row = smem_u32(vp) + r * (2 * C::D);
#pragma unroll
    for (int mt = 0; mt < C::D / 16; ++mt) {
      uint32_t a[4];
      ldsm4t(row + (((2 * mt + ((lane >> 3) & 1)) ^ (r & 7)) << 4), a);
      mma16816(x.o[mt], a[0], a[1], a[2], a[3], b0, b1);
    }
  } else {
#pragma unroll
    for (int q4 = 0; q4 < C::NG / 4; ++q4) {
      uint32_t w[4][4], pr[2][4];  // [key 2t, 2t + 1, 2t + 8, 2t + 9][group], octet g
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = 2 * t + (i & 1) + 8 * (i >> 1);
        const uint4 v = lds_u4(vp + r * (C::D / 2) + (((g * (C::NG / 4) + q4) ^ swz4<C::D, true>(r)) << 4));
        w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 v = lds_u4(vp + C::CODES + (g + 8 * i) * (C::D / 16) + q4 * 16);
        pr[i][0] = v.x, pr[i][1] = v.y, pr[i][2] = v.z, pr[i][3] = v.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int gr = 4 * q4 + e;
        const float s0 = bf16lo(pr[0][e]), s1 = bf16lo(pr[1][e]);
        const uint32_t ps0 = pack_bf16x2(p[0] * s0, p[1] * s0), ps1 = pack_bf16x2(p[2] * s1, p[3] * s1);
        // v = s (c - 8) + (b + 8 s): only the first part carries the rounding of P s
        const float z0 = fmaf(8.f, s0, bf16hi(pr[0][e])), z1 = fmaf(8.f, s1, bf16hi(pr[1][e]));
        x.corr[gr][0] = fmaf(-136.f, bf16lo(ps0) + bf16lo(ps1), fmaf(p[0], z0, fmaf(p[2], z1, x.corr[gr][0])));
        x.corr[gr][1] = fmaf(-136.f, bf16hi(ps0) + bf16hi(ps1), fmaf(p[1], z0, fmaf(p[3], z1, x.corr[gr][1])));
        const uint32_t b0 = transpose8x8(ps0), b1 = transpose8x8(ps1);
        // the pair (key 2t, key 2t + 1) of one dim in one register: even dims of
        // the octet are the low halves' nibbles, odd dims the high halves'
        const uint32_t x0 = prmt(w[0][e], w[1][e], 0x5410u), y0 = prmt(w[0][e], w[1][e], 0x7632u);
        const uint32_t x1 = prmt(w[2][e], w[3][e], 0x5410u), y1 = prmt(w[2][e], w[3][e], 0x7632u);
#pragma unroll
        for (int n = 0; n < 4; ++n)
          mma16816(x.o[4 * gr + n], nib_pair(x0, 4 * n), nib_pair(y0, 4 * n), nib_pair(x1, 4 * n), nib_pair(y1, 4 * n),
                   b0, b1);
      }
    }
  }
}

// Dim of element e of output tile mt in lane group g.
template <class C>
__device__ __forceinline__ int dim_of(int mt, int e, int g) {
  return C::BITS == 16 ? 16 * mt + g + 8 * (e >> 1) : 64 * (mt >> 2) + 8 * g + 2 * (mt & 3) + (e >> 1);
}

template <class C>
__global__ void __launch_bounds__(C::NT, 1) paged_attn_split_kernel(const PagedDev c, const BatchDev b, const AttnArgs a,
                                                                    const FewWs ws) {
  constexpr int D = C::D, NW = C::NW, NT = C::NT;
  extern __shared__ __align__(128) uint8_t sm[];
  __shared__ int2 scan_sh[NW];
  __shared__ int seg_n, last;
  __shared__ int64_t item_sh;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* ring = sm + warp * (C::NP * C::PIECE);
  float* obuf = reinterpret_cast<float*>(sm + C::OFF_O);
  uint32_t* qs = reinterpret_cast<uint32_t*>(sm + C::OFF_Q);
  float2* ml = reinterpret_cast<float2*>(sm + C::OFF_ML);  // [NW][8]
  Seg* segs = reinterpret_cast<Seg*>(sm + C::OFF_SEG);
  const int capacity = c.max_blocks << c.log_ps;

  // What sequence k0 + tid has on the line, and the sums over the chunk's sequences.
  struct Mine {
    int first, count, p0, ng;        // first row, rows, position of the first; granules of each of its items
    int at_u, at_i, sum_u, sum_i;    // granules and sequences before it in the chunk, of the chunk
    Span sp;
  };
  auto survey = [&](int k0) {
    Mine m = {};
    const int k = k0 + tid;
    if (k < b.n) {
      m.first = __ldg(b.q_start + k);
      m.count = (int)min((int64_t)__ldg(b.q_start + k + 1), b.tokens) - m.first;
      if (m.first >= 0 && m.count > 0 && m.count * (int64_t)a.share <= kFewRows) {
        const int len = __ldg(b.kv_len + k);
        m.p0 = len - m.count;
        m.sp = span_of<16>(m.p0, len - 1, a.window, a.sinks, capacity);
        m.ng = max(1, m.sp.tiles);  // an item that sees nothing still has zeros to write
      }
    }
    int x = m.ng, y = m.ng > 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int p = __shfl_up_sync(0xffffffffu, x, o), q = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) {
        x += p;
        y += q;
      }
    }
    __syncthreads();
    if (lane == 31) scan_sh[warp] = make_int2(x, y);
    __syncthreads();
    m.at_u = x - m.ng;
    m.at_i = y - (m.ng > 0);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const int2 s = scan_sh[w];
      if (w < warp) {
        m.at_u += s.x;
        m.at_i += s.y;
      }
      m.sum_u += s.x;
      m.sum_i += s.y;
    }
    return m;
  };
  const Mine mine0 = survey(0);
  auto chunk = [&](int k0) { return k0 == 0 ? mine0 : survey(k0); };

  // the line of all granules (every kv head has the same), and this CTA's part of it
  int64_t line = 0;
  for (int k0 = 0; k0 < b.n; k0 += NT) line += chunk(k0).sum_u;
  line *= c.Hkv;
  const int64_t part = max((int64_t)NW, (line + gridDim.x - 1) / gridDim.x);
  const int64_t u0 = min(line, blockIdx.x * part), u1 = min(line, u0 + part);
  if (u0 >= u1) return;

  for (int done = 0;;) {  // the segments of this part, MAXSEG at a time
    __syncthreads();
    if (tid == 0) seg_n = 0;
    if (done == 0) {  // the item that this part begins in, as its number on the line
      int64_t base = 0, items = 0;
      for (int k0 = 0; k0 < b.n; k0 += NT) {
        const Mine m = chunk(k0);
        const int64_t U = base + (int64_t)m.at_u * c.Hkv;
        if (m.ng > 0 && U <= u0 && u0 < U + (int64_t)m.ng * c.Hkv)
          item_sh = (items + m.at_i) * c.Hkv + (u0 - U) / m.ng;
        base += (int64_t)m.sum_u * c.Hkv;
        items += m.sum_i;
      }
    }
    __syncthreads();
    const int64_t item0 = item_sh + done;
    int64_t base = 0, items = 0;
    for (int k0 = 0; k0 < b.n; k0 += NT) {  // each thread lists the segments of its sequence
      const Mine m = chunk(k0);
      const int64_t U = base + (int64_t)m.at_u * c.Hkv, rel = (items + m.at_i) * c.Hkv - item0;
      if (m.ng > 0 && U < u1 && U + (int64_t)m.ng * c.Hkv > u0) {
        const int k = k0 + tid;
        for (int h = (int)max((int64_t)0, -rel); h < c.Hkv; ++h) {
          const int64_t s0 = U + (int64_t)h * m.ng, at = rel + h;
          if (s0 >= u1 || at >= C::MAXSEG) break;
          Seg s;
          s.seq = __ldg(b.seqs + k);
          s.h = h;
          s.row0 = m.first;
          s.rows = m.count * a.share;
          s.p0 = m.p0;
          s.i0 = (int)(max(u0, s0) - s0);
          s.i1 = (int)(min(u1, s0 + m.ng) - s0);
          s.low = m.sp.low;
          s.hi = m.sp.hi;
          s.ns = m.sp.ns;
          s.low_tile = m.sp.low_tile;
          s.item = k * c.Hkv + h;
          s.cf = (int)(s0 / part);
          s.cl = (int)((s0 + m.ng - 1) / part);
          s.slot = 2 * blockIdx.x + (s0 > u0);
          s.first_slot = 2 * s.cf + (s0 > s.cf * part);
          segs[at] = s;
          atomicMax(&seg_n, (int)at + 1);
        }
      }
      base += (int64_t)m.sum_u * c.Hkv;
      items += m.sum_i;
    }
    __syncthreads();
    const int n_seg = seg_n;
    if (n_seg == 0) break;

    // -- this warp's copies: granules i0 + warp, + NW, ... of each segment, K then V
    int ls = 0, li = segs[0].i0 + warp, entry = -1, entry0 = 0, entry_s = -1;
    auto page_at = [&](const Seg& s, int i, int si) {  // lanes hold the pages of the warp's next 32 granules
      const int k = (i - s.i0) / NW;
      if (entry_s != si || k >= entry0 + 32) {
        entry_s = si;
        entry0 = k;
        const int j = i + lane * NW;
        const int tile = j < s.ns ? j : s.low_tile + j - s.ns;
        entry = j < s.i1 ? page_of(c, s.seq, (16 * (int64_t)tile) >> c.log_ps) : -1;
      }
      return __shfl_sync(0xffffffffu, entry, k - entry0);
    };
    auto settle = [&]() {  // on to the warp's next granule that exists
      while (ls < n_seg && li >= segs[ls].i1)
        if (++ls < n_seg) li = segs[ls].i0 + warp;
    };
    int issued = 0;  // pieces
    auto issue = [&]() {
      if (ls < n_seg) {
        const Seg& s = segs[ls];
        const int tile = li < s.ns ? li : s.low_tile + li - s.ns;
        const int page = page_at(s, li, ls);
        uint8_t* dst = ring + (issued % C::NP) * C::PIECE;
        if (issued & 1) {
          copy_piece<C, true>(c, a, dst, s, tile, page, lane);
          li += NW;
          settle();
        } else {
          copy_piece<C, false>(c, a, dst, s, tile, page, lane);
        }
      }
      ++issued;
      cp_async_commit();
    };
    settle();
#pragma unroll 1
    for (int i = 0; i < C::NP - 1; ++i) issue();

    int used = 0;
#pragma unroll 1
    for (int si = 0; si < n_seg; ++si) {
      const Seg s = segs[si];
      // the item's 8 columns of q as B fragments, two k steps to a 16-byte read
      for (int i = tid; i < D; i += NT) {
        const int col = i / (D / 8), ch = i % (D / 8);
        uint4 v = make_uint4(0, 0, 0, 0);
        if (col < s.rows)
          v = ldg_u4(a.q + (int64_t)(s.row0 + col / a.share) * a.qs + (int64_t)(s.h * a.share + col % a.share) * D + 8 * ch);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if constexpr (C::BITS == 16)  // dims 16 ks + 8 half + 2t: lane t of chunk 2 ks + half
            qs[(((ch >> 2) * 32) + 4 * col + e) * 4 + (ch & 3)] = w[e];
          else  // octet o of a group: lane o % 4, half o / 4; pair e is k step e
            qs[(((ch >> 3) * 2 + (e >> 1)) * 32 + 4 * col + (ch & 3)) * 4 + (e & 1) * 2 + ((ch >> 2) & 1)] = w[e];
        }
      }
      __syncthreads();
      float xs[C::NG][2];
      if constexpr (C::BITS == 4) {
#pragma unroll
        for (int gr = 0; gr < C::NG; ++gr) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          const uint32_t one = 0x3f803f80u;
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            const uint4 q = lds_u4(qs + ((gr * 2 + k2) * 32 + lane) * 4);
            mma16816(acc, one, one, one, one, q.x, q.y);
            mma16816(acc, one, one, one, one, q.z, q.w);
          }
          xs[gr][0] = acc[0];
          xs[gr][1] = acc[1];
        }
      }
      Acc<C> x;
      reset<C>(x);
      const int pc0 = s.p0 + (2 * t) / a.share, pc1 = s.p0 + (2 * t + 1) / a.share;  // positions of the lane's columns
      const int p1 = s.p0 + (s.rows - 1) / a.share;
#pragma unroll 1
      for (int i = s.i0 + warp; i < s.i1; i += NW, used += 2) {
        const int j0 = 16 * (i < s.ns ? i : s.low_tile + i - s.ns);
        const int page = page_of(c, s.seq, j0 >> c.log_ps);
        float sc[4];
        issue();
        cp_async_wait_group<C::NP - 1>();
        __syncwarp();
        scores<C>(ring + (used % C::NP) * C::PIECE, qs, xs, lane, sc);
        // a missing page left zeros in the ring; its positions are masked
        const bool whole = page >= 0 && j0 + 15 <= s.p0 &&
                           (!a.window || j0 > p1 - a.window || j0 + 15 < a.sinks);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[e] *= a.sl;
          if (!whole) {
            const int j = j0 + g + 8 * (e >> 1), p = e & 1 ? pc1 : pc0;
            if (page < 0 || j > p || !(!a.window || j > p - a.window || j < a.sinks)) sc[e] = -INFINITY;
          }
        }
        float mx[2] = {fmaxf(sc[0], sc[2]), fmaxf(sc[1], sc[3])};
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
          mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], o));
          mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], o));
        }
        if (__any_sync(0xffffffffu, mx[0] > x.m[0] + 8.f || mx[1] > x.m[1] + 8.f)) {
          float f[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float mn = fmaxf(x.m[e], mx[e]);
            f[e] = x.m[e] == mn ? 1.f : ex2(x.m[e] - mn);
            x.m[e] = mn;
            x.l[e] *= f[e];
          }
#pragma unroll
          for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) x.o[mt][e] *= f[e & 1];
          if constexpr (C::BITS == 4)
#pragma unroll
            for (int gr = 0; gr < C::NG; ++gr) {
              x.corr[gr][0] *= f[0];
              x.corr[gr][1] *= f[1];
            }
        }
        const float r0 = x.m[0] == -INFINITY ? 0.f : x.m[0], r1 = x.m[1] == -INFINITY ? 0.f : x.m[1];
        float p[4] = {ex2(sc[0] - r0), ex2(sc[1] - r1), ex2(sc[2] - r0), ex2(sc[3] - r1)};
        x.l[0] += p[0] + p[2];
        x.l[1] += p[1] + p[3];
        __syncwarp();  // every lane is done with the K piece
        issue();
        cp_async_wait_group<C::NP - 1>();
        __syncwarp();
        add_values<C>(ring + ((used + 1) % C::NP) * C::PIECE, p, lane, x);
        __syncwarp();
      }

      // -- join the warps.  Sums over keys: the lanes of a column (equal t)
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        x.l[0] += __shfl_xor_sync(0xffffffffu, x.l[0], o);
        x.l[1] += __shfl_xor_sync(0xffffffffu, x.l[1], o);
        if constexpr (C::BITS == 4)
#pragma unroll
          for (int gr = 0; gr < C::NG; ++gr) {
            x.corr[gr][0] += __shfl_xor_sync(0xffffffffu, x.corr[gr][0], o);
            x.corr[gr][1] += __shfl_xor_sync(0xffffffffu, x.corr[gr][1], o);
          }
      }
      if (g == 0) {
        ml[warp * 8 + 2 * t] = make_float2(x.m[0], x.l[0]);
        ml[warp * 8 + 2 * t + 1] = make_float2(x.m[1], x.l[1]);
      }
      __syncthreads();  // the maxima are there; every warp is done with q
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, ml[w * 8 + 2 * t + e].x);
        f[e] = x.m[e] == -INFINITY ? 0.f : ex2(x.m[e] - M);
      }
      float v[C::VPT];
#pragma unroll
      for (int k = 0; k < C::VPT; ++k) v[k] = 0.f;
#pragma unroll 1
      for (int w0 = 0; w0 < NW; w0 += C::MW) {
        if (warp >= w0 && warp < w0 + C::MW) {
          float* ob = obuf + (warp - w0) * 8 * C::OS;
#pragma unroll
          for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float add = C::BITS == 4 ? x.corr[C::BITS == 4 ? mt >> 2 : 0][e & 1] : 0.f;
              // a warp without a key of this column has no say (its sums are 0, or NaN times 0)
              ob[(2 * t + (e & 1)) * C::OS + dim_of<C>(mt, e, g)] = f[e & 1] == 0.f ? 0.f : (x.o[mt][e] + add) * f[e & 1];
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < C::VPT / 4; ++k) {
          const int i = (k * NT + tid) * 4, row = i / D, d = i % D;
#pragma unroll
          for (int w = 0; w < C::MW; ++w) {
            const float4 y = *reinterpret_cast<const float4*>(obuf + (w * 8 + row) * C::OS + d);
            v[4 * k] += y.x;
            v[4 * k + 1] += y.y;
            v[4 * k + 2] += y.z;
            v[4 * k + 3] += y.w;
          }
        }
        __syncthreads();
      }
      float M[C::VPT / 4], L[C::VPT / 4];
#pragma unroll
      for (int k = 0; k < C::VPT / 4; ++k) {
        const int row = (k * NT + tid) * 4 / D;
        M[k] = -INFINITY;
        L[k] = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) M[k] = fmaxf(M[k], ml[w * 8 + row].x);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float2 y = ml[w * 8 + row];
          if (y.x > -INFINITY) L[k] += y.y * ex2(y.x - M[k]);
        }
      }
      bool write = s.cf == s.cl;
      if (!write) {
        float* po = ws.o + (int64_t)s.slot * 8 * D;
#pragma unroll
        for (int k = 0; k < C::VPT / 4; ++k) {
          const int i = (k * NT + tid) * 4;
          __stcg(reinterpret_cast<float4*>(po + i), make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]));
          if (i % D == 0) __stcg(ws.ml + s.slot * 8 + i / D, make_float2(M[k], L[k]));
        }
        __threadfence();
        __syncthreads();
        if (tid == 0) {
          last = atomicAdd(ws.arrived + s.item, 1u) == (unsigned)(s.cl - s.cf);
          if (last) ws.arrived[s.item] = 0;
        }
        __syncthreads();
        if (last) {
          __threadfence();
          write = true;
#pragma unroll
          for (int k = 0; k < C::VPT / 4; ++k) {
            const int i = (k * NT + tid) * 4, row = i / D;
            float am = -INFINITY, al = 0.f;
            float4 ao = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int q = s.cf; q <= s.cl; ++q) {
              const int slot = q == s.cf ? s.first_slot : 2 * q;
              const float2 y = __ldcg(ws.ml + slot * 8 + row);
              const float4 o = __ldcg(reinterpret_cast<const float4*>(ws.o + (int64_t)slot * 8 * D + i));
              const float mn = fmaxf(am, y.x);
              const float fa = am == mn ? 1.f : ex2(am - mn), fy = y.x == -INFINITY ? 0.f : ex2(y.x - mn);
              al = al * fa + (fy == 0.f ? 0.f : y.y * fy);
              ao.x = ao.x * fa + (fy == 0.f ? 0.f : o.x * fy);
              ao.y = ao.y * fa + (fy == 0.f ? 0.f : o.y * fy);
              ao.z = ao.z * fa + (fy == 0.f ? 0.f : o.z * fy);
              ao.w = ao.w * fa + (fy == 0.f ? 0.f : o.w * fy);
              am = mn;
            }
            v[4 * k] = ao.x;
            v[4 * k + 1] = ao.y;
            v[4 * k + 2] = ao.z;
            v[4 * k + 3] = ao.w;
            L[k] = al;
          }
        }
      }
      if (write) {
#pragma unroll
        for (int k = 0; k < C::VPT / 4; ++k) {
          const int i = (k * NT + tid) * 4, row = i / D, d = i % D;
          if (row >= s.rows) continue;
          const float inv = L[k] == 0.f ? 0.f : 1.f / L[k];
          bf16* o = a.out + ((int64_t)(s.row0 + row / a.share) * a.Hq + s.h * a.share + row % a.share) * D + d;
          *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v[4 * k] * inv, v[4 * k + 1] * inv),
                                                    pack_bf16x2(v[4 * k + 2] * inv, v[4 * k + 3] * inv));
        }
      }
    }
    cp_async_wait_all();
    if (n_seg < C::MAXSEG) break;
    done += n_seg;
  }
}

// Lane l's values l * P .. of row `slot` of a block.
template <int P>
__device__ __forceinline__ void load_page_row(const PagedDev& c, const uint8_t* blk, int slot, int lane, float (&v)[P]) {
  constexpr int D = 32 * P, LG = 64 / P, NG = P / 2;
  if (c.bits == 16) {
    const bf16* r = reinterpret_cast<const bf16*>(blk) + (int64_t)slot * D + lane * P;
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = bf2f(r[i]);
    return;
  }
  const uint32_t* words = reinterpret_cast<const uint32_t*>(blk + slot * (D / 2));
  const uint32_t pair = reinterpret_cast<const uint32_t*>(blk + c.ps * (D / 2) + slot * (D / 16))[lane / LG];
  const float s = bf16lo(pair), b = bf16hi(pair);
#pragma unroll
  for (int o = 0; o < P / 8; ++o) {
    const uint32_t w = words[((lane % LG) * (P / 8) + o) * NG + lane / LG];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[8 * o + i] = fmaf(s, (float)((w >> (4 * ((i >> 1) + 4 * (i & 1)))) & 15u), b);
  }
}

// One CTA per (row, query head); a warp takes every 8th visible position.
template <int P>
__global__ void __launch_bounds__(256) paged_attn_rows_kernel(PagedDev c, BatchDev b, AttnArgs a) {
  constexpr int D = 32 * P;
  __shared__ float sm[8], sl[8], so[8][D];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t t = blockIdx.x;
  const int h = blockIdx.y, g = h / a.share;
  int i = 0;
  for (int k = 0; k < b.n; k += blockDim.x)
    i += __syncthreads_count(k + (int)threadIdx.x < b.n && b.q_start[k + threadIdx.x + 1] <= t);
  if (i >= b.n || (b.q_start[i + 1] - b.q_start[i]) * (int64_t)a.share <= kFewRows) return;
  const int pos = b.kv_len[i] - b.q_start[i + 1] + (int)t;
  const int low = a.window ? max(0, pos - a.window + 1) : 0;
  const int first = a.window ? min(a.sinks, low) : 0;  // positions [0, first) and [low, pos]
  float q[P], o[P], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int e = 0; e < P; ++e) {
    q[e] = bf2f(a.q[t * a.qs + (int64_t)h * D + lane * P + e]) * a.sl;
    o[e] = 0.f;
  }
  const int end = min(pos + 1, c.max_blocks << c.log_ps);  // table rows hold no more
  for (int n = warp; n < first + end - low; n += 8) {
    const int j = n < first ? n : low + n - first;
    const int page = page_of(c, b.seqs[i], j >> c.log_ps);
    if (page < 0) continue;
    float x[P], s = 0.f;
    load_page_row<P>(c, page_block(c, a.layer, page, g, 0), j & (c.ps - 1), lane, x);
#pragma unroll
    for (int e = 0; e < P; ++e) s = fmaf(q[e], x[e], s);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    const float mn = fmaxf(m, s), f = ex2(m - mn), w = ex2(s - mn);
    load_page_row<P>(c, page_block(c, a.layer, page, g, 1), j & (c.ps - 1), lane, x);
    l = l * f + w;
#pragma unroll
    for (int e = 0; e < P; ++e) o[e] = o[e] * f + w * x[e];
    m = mn;
  }
  if (lane == 0) {
    sm[warp] = m;
    sl[warp] = l;
  }
#pragma unroll
  for (int e = 0; e < P; ++e) so[warp][lane * P + e] = o[e];
  __syncthreads();
  float M = -INFINITY, L = 0.f;
  for (int w = 0; w < 8; ++w) M = fmaxf(M, sm[w]);
  for (int w = 0; w < 8; ++w) L += sm[w] > -INFINITY ? sl[w] * ex2(sm[w] - M) : 0.f;
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float x = 0.f;
    for (int w = 0; w < 8; ++w) x += sm[w] > -INFINITY ? so[w][d] * ex2(sm[w] - M) : 0.f;
    a.out[(t * a.Hq + h) * D + d] = __float2bfloat16_rn(L > 0.f ? x / L : 0.f);
  }
}

// The scratch of a call: counters first (zero between calls), then the parts.
size_t carve(void* base, const PagedDev& c, int32_t n, FewWs* w) {
  Carver k(base);
  w->arrived = k.take<unsigned>((size_t)std::max(n, 1) * c.Hkv);
  w->o = k.take<float>((size_t)2 * kNumSMs * 8 * c.D);
  w->ml = k.take<float2>((size_t)2 * kNumSMs * 8);
  return align_up(k.off, 256);
}

template <class C>
int launch_split(const PagedDev& c, const BatchDev& b, const AttnArgs& a, const FewWs& w, cudaStream_t st) {
  static std::once_flag once;
  static cudaError_t err = cudaSuccess;
  std::call_once(once, [] {
    err = cudaFuncSetAttribute(paged_attn_split_kernel<C>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  });
  if (err != cudaSuccess)
    return set_error(FMOE_ERR_CUDA, "paged_attend: shared memory attribute: %s", cudaGetErrorString(err));
  ProfScope prof_(C::BITS == 16 ? "paged_attn_split_kernel<bf16>" : "paged_attn_split_kernel<4-bit>", st);
  paged_attn_split_kernel<C><<<kNumSMs, C::NT, C::SMEM, st>>>(c, b, a, w);
  return check_launch("paged_attn_split_kernel");
}

}  // namespace pa
}  // namespace fmoe

using namespace fmoe;

extern "C" {

size_t fmoe_paged_attend_workspace_bytes(const fmoe_paged_kv_t* cache, int q_heads, int32_t n, int64_t tokens,
                                         int32_t max_new) {
  PagedDev c;
  if (paged_to_dev(cache, &c, false) || q_heads < 1 || q_heads % c.Hkv || q_heads / c.Hkv > 8 || n < 0 || tokens < 0)
    return 0;
  pa::FewWs w;
  return pa::carve(nullptr, c, n, &w);
}

int fmoe_paged_attend(const fmoe_paged_kv_t* cache, int layer, const void* q, int64_t q_stride, int q_heads,
                      const fmoe_paged_batch_t* batch, int window, int sinks, float scale, void* out,
                      void* workspace, size_t workspace_bytes, void* stream) {
  PagedDev c;
  BatchDev b;
  int rc;
  if ((rc = paged_to_dev(cache, &c, true)) || (rc = batch_to_dev(batch, &b))) return rc;
  if (layer < 0 || layer >= c.layers) return set_error(FMOE_ERR_INVALID, "paged_attend: layer %d of %d", layer, c.layers);
  if (q_heads < 1 || q_heads % c.Hkv || q_heads / c.Hkv > 8)
    return set_error(FMOE_ERR_UNSUPPORTED, "paged_attend: %d query heads over %d kv heads (1..8 per kv head)", q_heads,
                     c.Hkv);
  if (window < 0 || sinks < 0) return set_error(FMOE_ERR_INVALID, "paged_attend: window %d sinks %d", window, sinks);
  if (!std::isfinite(scale)) return set_error(FMOE_ERR_INVALID, "paged_attend: scale %g", (double)scale);
  if (b.tokens == 0 || b.n == 0) return FMOE_OK;
  if (!q || !out || !aligned(q, 16) || !aligned(out, 16))
    return set_error(FMOE_ERR_ALIGN, "paged_attend: q/out null or not 16-byte aligned");
  if (q_stride % 8 || q_stride < (int64_t)q_heads * c.D)
    return set_error(FMOE_ERR_ALIGN, "paged_attend: q rows %lld values apart (a multiple of 8, at least %lld)",
                     (long long)q_stride, (long long)q_heads * c.D);
  const size_t need = fmoe_paged_attend_workspace_bytes(cache, q_heads, b.n, b.tokens, b.max_new);
  if (!workspace || workspace_bytes < need || !aligned(workspace, 16))
    return set_error(FMOE_ERR_WORKSPACE, "paged_attend: workspace of %zu bytes, %zu needed (16-byte aligned)",
                     workspace_bytes, need);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  pa::FewWs w;
  pa::carve(workspace, c, b.n, &w);
  const int share = q_heads / c.Hkv;
  const pa::AttnArgs a = {static_cast<const bf16*>(q), static_cast<bf16*>(out), q_stride, q_heads, share, layer,
                          std::min(window, 1 << 30), std::min(sinks, 1 << 30), scale * 1.4426950408889634f};
  if (c.D == 256)
    rc = c.bits == 16 ? pa::launch_split<pa::Few<256, 16>>(c, b, a, w, st) : pa::launch_split<pa::Few<256, 4>>(c, b, a, w, st);
  else
    rc = c.bits == 16 ? pa::launch_split<pa::Few<512, 16>>(c, b, a, w, st) : pa::launch_split<pa::Few<512, 4>>(c, b, a, w, st);
  if (rc || (int64_t)b.max_new * share <= pa::kFewRows) return rc;
  ProfScope prof_("paged_attn_rows_kernel", st);
  const dim3 grid((unsigned)b.tokens, (unsigned)q_heads);
  if (c.D == 256)
    pa::paged_attn_rows_kernel<8><<<grid, 256, 0, st>>>(c, b, a);
  else
    pa::paged_attn_rows_kernel<16><<<grid, 256, 0, st>>>(c, b, a);
  return check_launch("paged_attn_rows_kernel");
}

}  // extern "C"
