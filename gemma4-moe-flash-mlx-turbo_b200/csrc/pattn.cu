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
#include "tc.cuh"

namespace fmoe {
namespace pa {

// ---------------------------------------------------------------------------
// few rows: split over the keys
//
// The pages' bytes are what a decode costs, so the work is cut by them: all
// (sequence, kv head) items' keys form one line of granules of 16 positions (a
// granule never leaves its page), and every CTA takes the same length of it,
// whatever the sequences' lengths are.  A warp owns every 8th granule of its
// CTA's part and has its own ring of TMA copies, running maximum, sum and
// output, so that nothing in the loop waits for another warp and the copies run
// on across the ends of items.  At the end of an item its warps' results are
// joined in shared memory; an item that lies in several CTAs goes to scratch
// and paged_attn_join_kernel joins its parts in the order of the keys: no
// result depends on who arrives first.
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
  static constexpr int NW = 8, NT = 32 * NW;
  // A ring piece: 16 keys of K or V, bf16 in steps of 256 dims (8 KB), 4-bit
  // whole rows and their (scale, bias) pairs.  Its boxes are 16 rows of 128
  // bytes, swizzled.
  static constexpr int H = BITS == 16 ? D / 256 : 1;  // pieces of a granule's K
  static constexpr int BOXES = BITS == 16 ? 4 : D / 256, CODES = 2048 * BOXES;
  static constexpr int PAIRS = BITS == 4 ? D : 0;
  static constexpr int PIECE = BITS == 16 ? CODES : (CODES + PAIRS + 1023) / 1024 * 1024;
  static constexpr int NP = BITS == 16 ? 3 : D == 256 ? 7 : 4;  // pieces in a warp's ring
  static constexpr int OS = D + 4;                              // row stride of a joined output, floats
  static constexpr int MW = D == 256 ? 2 : 1;                   // warps that hand over their output at a time
  static constexpr int MAXSEG = 32;
  static constexpr int OFF_O = NW * NP * PIECE, OFF_Q = OFF_O + MW * 8 * OS * 4, OFF_ML = OFF_Q + 16 * D;
  static constexpr int OFF_SEG = OFF_ML + NW * 16 * 4, OFF_BAR = OFF_SEG + MAXSEG * 64;
  static constexpr int SMEM = OFF_BAR + NW * NP * 8 + 1024;  // the swizzle wants 1024-byte boxes
  static constexpr int VPT = 8 * D / NT;                     // joined values of a thread
  static_assert(SMEM <= 227 * 1024 - 256, "shared memory");
};

// One item's part that lies in this CTA.
struct Seg {
  int seq, h, row0, rows;      // table row, kv head, first row of the step, its (row, head) pairs
  int p0, i0, i1, first_slot;  // position of the first row; this part's granules; where the item's first part goes
  int low, hi, ns, low_tile;   // its Span
  int whole, cf, cl, slot;     // 1: no other part; CTAs that hold it; where this part goes
};
static_assert(sizeof(Seg) == 64, "segment list");

// An item that ends in a CTA and began in an earlier one, for the join.
struct Split {
  int row0, rows, h, cf, first_slot, pad[3];
};
struct FewWs {
  int* status;
  Split* split;  // [grid]; rows 0: none
  float* o;      // [2 * grid][8][D]
  float2* ml;    // [2 * grid][8]
};

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
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 r;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(addr) : "memory");
  return r;
}

// Which of the granule's keys row g of the score product is (row g + 8: 8
// further).  4-bit reads go straight to registers: 8 lanes together read 2 keys
// x 4 octets of K, or 4 keys x 2 octets of V, 16 bytes each, of rows 128 bytes
// apart whose chunks the copy xor-ed with the row; in these orders each such
// read touches every bank once.
template <class C>
__device__ __forceinline__ int key_of(int g) {
  if (C::BITS == 16) return g;
  return ((C::D == 256 ? 0x36147250u : 0x65742130u) >> (4 * g)) & 7;
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

// Adds piece hf of K to the scores of one granule.
template <class C>
__device__ __forceinline__ void scores(uint32_t kp, uint32_t qs, int hf, const float (&xs)[C::NG][2], int lane,
                                       float (&s)[4]) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (C::BITS == 16) {
    float acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = 0.f;
    const int r = lane & 15;
    const uint32_t q = qs + (hf * 256 + lane) * 16, sw = (r & 7) << 4;
    kp += r * 128;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {  // 32 dims
      const uint4 b = lds128(q + kk * 512);
      uint32_t a0[4], a1[4];
      ldsm4(kp + (kk >> 1) * 2048 + ((((4 * kk) & 7) * 16 + (lane & 16)) ^ sw), a0);
      ldsm4(kp + (kk >> 1) * 2048 + ((((4 * kk + 2) & 7) * 16 + (lane & 16)) ^ sw), a1);
      mma16816(acc[(2 * kk) & 3], a0[0], a0[1], a0[2], a0[3], b.x, b.y);
      mma16816(acc[(2 * kk + 1) & 3], a1[0], a1[1], a1[2], a1[3], b.z, b.w);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] += (acc[0][e] + acc[1][e]) + (acc[2][e] + acc[3][e]);
  } else {
    const int k0 = key_of<C>(g);
#pragma unroll
    for (int q4 = 0; q4 < C::NG / 4; ++q4) {  // four groups at a time: one 16-byte read each
      uint32_t w[2][2][4], pr[2][4];          // [key of row g, g + 8][octet t, t + 4][group]
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = k0 + 8 * i;
#pragma unroll
        for (int o = 0; o < 2; ++o) {
          const int ch = (t + 4 * o) * (C::NG / 4) + q4;
          const uint4 v = lds128(kp + (ch >> 3) * 2048 + r * 128 + (((ch ^ r) & 7) << 4));
          w[i][o][0] = v.x, w[i][o][1] = v.y, w[i][o][2] = v.z, w[i][o][3] = v.w;
        }
        const uint4 p = lds128(kp + C::CODES + r * (C::D / 16) + q4 * 16);
        pr[i][0] = p.x, pr[i][1] = p.y, pr[i][2] = p.z, pr[i][3] = p.w;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int gr = 4 * q4 + e;
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
          const uint4 b = lds128(qs + ((gr * 2 + k2) * 32 + lane) * 16);
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

// Piece hf of O^T += V^T P^T; p: the weights of rows g, g + 8 of the score
// product and columns 2t, 2t + 1 (bf16: their transposed fragments in b0, b1).
template <class C>
__device__ __forceinline__ void add_values(uint32_t vp, int hf, const float (&p)[4], uint32_t b0, uint32_t b1, int lane,
                                           Acc<C>& x) {
  const int g = lane >> 2, t = lane & 3;
  if constexpr (C::BITS == 16) {
    const int r = (lane & 7) + ((lane >> 4) << 3);
    vp += r * 128;
    const uint32_t sw = (r & 7) << 4, odd = (lane & 8) << 1;
#pragma unroll
    for (int mt = 0; mt < 16; ++mt) {
      uint32_t a[4];
      ldsm4t(vp + (mt >> 2) * 2048 + ((((2 * mt) & 7) * 16 + odd) ^ sw), a);
      mma16816(x.o[16 * hf + mt], a[0], a[1], a[2], a[3], b0, b1);
    }
  } else {
    const int k0 = key_of<C>(g), r0 = key_of<C>(2 * t), r1 = key_of<C>(2 * t + 1);
#pragma unroll
    for (int q4 = 0; q4 < C::NG / 4; ++q4) {
      uint32_t w[4][4], pr[2][4];  // [key of slot 2t, 2t + 1, 2t + 8, 2t + 9][group], octet g
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (i & 1 ? r1 : r0) + 8 * (i >> 1), ch = g * (C::NG / 4) + q4;
        const uint4 v = lds128(vp + (ch >> 3) * 2048 + r * 128 + (((ch ^ r) & 7) << 4));
        w[i][0] = v.x, w[i][1] = v.y, w[i][2] = v.z, w[i][3] = v.w;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 v = lds128(vp + C::CODES + (k0 + 8 * i) * (C::D / 16) + q4 * 16);
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
        const uint32_t c0 = transpose8x8(ps0), c1 = transpose8x8(ps1);
        // the pair (key of slot 2t, of 2t + 1) of one dim in one register: even dims
        // of the octet are the low halves' nibbles, odd dims the high halves'
        const uint32_t x0 = prmt(w[0][e], w[1][e], 0x5410u), y0 = prmt(w[0][e], w[1][e], 0x7632u);
        const uint32_t x1 = prmt(w[2][e], w[3][e], 0x5410u), y1 = prmt(w[2][e], w[3][e], 0x7632u);
#pragma unroll
        for (int n = 0; n < 4; ++n)
          mma16816(x.o[4 * gr + n], nib_pair(x0, 4 * n), nib_pair(y0, 4 * n), nib_pair(x1, 4 * n), nib_pair(y1, 4 * n),
                   c0, c1);
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
__global__ void __launch_bounds__(C::NT, 1)
    paged_attn_split_kernel(const __grid_constant__ CUtensorMap map, const PagedDev c, const BatchDev b, const AttnArgs a,
                            const FewWs ws) {
  constexpr int D = C::D, NW = C::NW, NT = C::NT, H = C::H, NP = C::NP;
  extern __shared__ uint8_t sm_raw[];
  __shared__ int2 scan_sh[NW];
  __shared__ int seg_n, failed_sh;
  __shared__ int64_t item_sh;
  uint8_t* sm = sm_raw + ((1024 - (smem_u32(sm_raw) & 1023)) & 1023);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  uint8_t* ring = sm + warp * (NP * C::PIECE);
  float* obuf = reinterpret_cast<float*>(sm + C::OFF_O);
  uint32_t* qs = reinterpret_cast<uint32_t*>(sm + C::OFF_Q);
  float2* ml = reinterpret_cast<float2*>(sm + C::OFF_ML);  // [NW][8]
  Seg* segs = reinterpret_cast<Seg*>(sm + C::OFF_SEG);
  uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::OFF_BAR) + warp * NP;
  volatile int* failed = &failed_sh;
  const int capacity = c.max_blocks << c.log_ps;

  griddep_launch_dependents();
  if (lane < NP) mbar_init(&full[lane], 1);
  mbar_fence_init();
  if (tid == 0) failed_sh = 0;

  // What sequence k0 + tid has on the line, and the sums over the chunk's sequences.
  struct Mine {
    int seq, first, count, p0, ng;   // table row, first row, rows, position of the first; granules of each of its items
    int at_u, at_i, sum_u, sum_i;    // granules and sequences before it in the chunk, of the chunk
    Span sp;
  };
  auto survey = [&](int k0) {
    Mine m = {};
    const int k = k0 + tid;
    if (k < b.n) {
      const int len = __ldg(b.kv_len + k);
      m.seq = __ldg(b.seqs + k);
      m.first = __ldg(b.q_start + k);
      m.count = (int)min((int64_t)__ldg(b.q_start + k + 1), b.tokens) - m.first;
      if (m.first >= 0 && m.count > 0 && m.count * (int64_t)a.share <= kFewRows) {
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
  Mine m0 = survey(0);
  auto chunk = [&](int k0) { return k0 == 0 ? m0 : survey(k0); };

  // the line of all granules (every kv head has the same), and this CTA's part of it
  int64_t line = m0.sum_u;
  for (int k0 = NT; k0 < b.n; k0 += NT) line += survey(k0).sum_u;
  line *= c.Hkv;
  const int64_t part = max((int64_t)NW, (line + gridDim.x - 1) / gridDim.x);
  const int64_t u0 = min(line, blockIdx.x * part), u1 = min(line, u0 + part);
  if (u0 >= u1) {
    if (tid == 0) ws.split[blockIdx.x].rows = 0;
    return;
  }

  int issued = 0, used = 0;  // pieces of this warp, over all rounds
  for (int done = 0;;) {     // the segments of this part, MAXSEG at a time
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
        for (int h = (int)max((int64_t)0, -rel); h < c.Hkv; ++h) {
          const int64_t s0 = U + (int64_t)h * m.ng, at = rel + h;
          if (s0 >= u1 || at >= C::MAXSEG) break;
          Seg s;
          s.seq = m.seq;
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
          s.cf = (int)(s0 / part);
          s.cl = (int)((s0 + m.ng - 1) / part);
          s.whole = s.cf == s.cl;
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
    if (done == 0 && tid == 0) {  // only the part's first item can have begun before it
      const Seg& s = segs[0];
      const bool ends = !s.whole && s.cf < (int)blockIdx.x && s.cl == (int)blockIdx.x;
      Split* r = ws.split + blockIdx.x;
      r->row0 = s.row0;
      r->rows = ends ? s.rows : 0;
      r->h = s.h;
      r->cf = s.cf;
      r->first_slot = s.first_slot;
    }
    if (n_seg == 0) break;

    // -- this warp's copies: granules i0 + warp, + NW, ... of each segment, pieces of K then of V
    int ls = 0, li = segs[0].i0 + warp, lp = 0, entry = -1, entry0 = 0, entry_s = -1;
    auto settle = [&]() {  // on to the warp's next granule that exists
      while (ls < n_seg && li >= segs[ls].i1)
        if (++ls < n_seg) li = segs[ls].i0 + warp;
    };
    auto issue = [&]() {
      if (ls >= n_seg || __any_sync(0xffffffffu, *failed)) return;
      const Seg& s = segs[ls];
      const int k = (li - s.i0) / NW;
      if (entry_s != ls || k >= entry0 + 32) {  // lanes hold the pages of the warp's next 32 granules
        entry_s = ls;
        entry0 = k;
        const int j = li + lane * NW, tile = j < s.ns ? j : s.low_tile + j - s.ns;
        entry = j < s.i1 ? page_of(c, s.seq, (16 * (int64_t)tile) >> c.log_ps) : -1;
      }
      const int page = __shfl_sync(0xffffffffu, entry, k - entry0);
      const int tile = li < s.ns ? li : s.low_tile + li - s.ns, slot = (16 * tile) & (c.ps - 1);
      const int stage = issued % NP, which = lp >= H;
      uint8_t* dst = ring + stage * C::PIECE;
      if (lane == 0) mbar_arrive_expect_tx(&full[stage], page >= 0 ? C::CODES + C::PAIRS : 0);
      __syncwarp();
      if (page >= 0) {
        const int blk = (page * c.Hkv + s.h) * 2 + which;
        if constexpr (C::BITS == 16) {
          if (lane < 4) tc::tma2d(dst + lane * 2048, &map, (lp - which * H) * 256 + lane * 64, blk * c.ps + slot, &full[stage]);
        } else {
          if (lane < C::BOXES) tc::tma3d(dst + lane * 2048, &map, lane * 128, slot, blk, &full[stage]);
          if (lane == C::BOXES)
            bulk_g2s(dst + C::CODES, page_block(c, a.layer, page, s.h, which) + c.ps * (D / 2) + slot * (D / 16), C::PAIRS,
                     &full[stage]);
        }
      }
      ++issued;
      if (++lp == 2 * H) {
        lp = 0;
        li += NW;
        settle();
      }
    };
    settle();
#pragma unroll 1
    for (int i = 0; i < NP; ++i) issue();

#pragma unroll 1
    for (int si = 0; si < n_seg; ++si) {
      const Seg s = segs[si];
      // the item's 8 columns of q as B fragments, two k steps to a 16-byte read
#pragma unroll
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
      const uint32_t qa = smem_u32(qs);
      float xs[C::NG][2];
      if constexpr (C::BITS == 4) {  // sums of q over the groups
#pragma unroll
        for (int gr = 0; gr < C::NG; ++gr) {
          float acc[4] = {0.f, 0.f, 0.f, 0.f};
          const uint32_t one = 0x3f803f80u;
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            const uint4 q = lds128(qa + ((gr * 2 + k2) * 32 + lane) * 16);
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
      for (int i = s.i0 + warp; i < s.i1; i += NW) {
        const int j0 = 16 * (i < s.ns ? i : s.low_tile + i - s.ns);
        const int page = page_of(c, s.seq, j0 >> c.log_ps);
        float sc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int hf = 0; hf < H; ++hf, ++used) {
          tc::pwait(&full[used % NP], (used / NP) & 1, failed, ws.status, 501);
          scores<C>(smem_u32(ring + (used % NP) * C::PIECE), qa, hf, xs, lane, sc);
          __syncwarp();  // every lane has read the piece
          issue();
        }
        const bool whole = page >= 0 && j0 + 15 <= s.p0 && (!a.window || j0 > p1 - a.window || j0 + 15 < a.sinks);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          sc[e] *= a.sl;
          if (!whole) {
            const int j = j0 + key_of<C>(g) + 8 * (e >> 1), p = e & 1 ? pc1 : pc0;
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
        const float p[4] = {ex2(sc[0] - r0), ex2(sc[1] - r1), ex2(sc[2] - r0), ex2(sc[3] - r1)};
        x.l[0] += p[0] + p[2];
        x.l[1] += p[1] + p[3];
        uint32_t b0 = 0, b1 = 0;
        if constexpr (C::BITS == 16) {
          b0 = transpose8x8(pack_bf16x2(p[0], p[1]));
          b1 = transpose8x8(pack_bf16x2(p[2], p[3]));
        }
        // Rows that no row of the item sees can hold anything: zeros instead, since
        // a weight of zero times an infinity is no zero.
        const bool seen = page >= 0 && j0 + 15 < s.hi && (j0 >= s.low || j0 + 15 < a.sinks);
#pragma unroll
        for (int hf = 0; hf < H; ++hf, ++used) {
          tc::pwait(&full[used % NP], (used / NP) & 1, failed, ws.status, 502);
          uint8_t* vp = ring + (used % NP) * C::PIECE;
          if (!seen) {
#pragma unroll 1
            for (int r = 0; r < 16; ++r) {
              const int j = j0 + r;
              if (page >= 0 && j < s.hi && (j >= s.low || j < a.sinks)) continue;
              if constexpr (C::BITS == 16)
                *reinterpret_cast<uint4*>(vp + (lane >> 3) * 2048 + r * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
              else if (lane < C::NG)
                *reinterpret_cast<uint32_t*>(vp + C::CODES + r * (D / 16) + lane * 4) = 0;
            }
            asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");  // before the copy that reuses the piece
            __syncwarp();
          }
          add_values<C>(smem_u32(vp), hf, p, b0, b1, lane, x);
          __syncwarp();
          issue();
        }
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
              // a warp without a key of this column has no say
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
#pragma unroll
      for (int k = 0; k < C::VPT / 4; ++k) {
        const int i = (k * NT + tid) * 4, row = i / D, d = i % D;
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, ml[w * 8 + row].x);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const float2 y = ml[w * 8 + row];
          if (y.x > -INFINITY) L += y.y * ex2(y.x - M);
        }
        if (!s.whole) {
          *reinterpret_cast<float4*>(ws.o + ((int64_t)s.slot * 8 + row) * D + d) =
              make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
          if (d == 0) ws.ml[s.slot * 8 + row] = make_float2(M, L);
        } else if (row < s.rows) {
          const float inv = L == 0.f ? 0.f : 1.f / L;
          bf16* o = a.out + ((int64_t)(s.row0 + row / a.share) * a.Hq + s.h * a.share + row % a.share) * D + d;
          *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(v[4 * k] * inv, v[4 * k + 1] * inv),
                                                    pack_bf16x2(v[4 * k + 2] * inv, v[4 * k + 3] * inv));
        }
      }
    }
    if (n_seg < C::MAXSEG) break;
    done += n_seg;
  }
  // after a wait that gave up, no copy may land in the memory of a CTA that is gone
  if (*failed)
    for (int k = max(0, issued - NP); k < issued; ++k) tc::drain_wait(&full[k % NP], (k / NP) & 1);
}

// Joins the parts of the items that lie in several CTAs: block (q, row) the
// item that ends in CTA q, a thread four dims.
template <int D>
__global__ void __launch_bounds__(D / 4) paged_attn_join_kernel(const AttnArgs a, const FewWs ws) {
  __shared__ float w[kNumSMs], red[D / 128];
  griddep_wait();
  const int q = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const Split s = ws.split[q];
  if (row >= s.rows) return;
  const int n = q - s.cf + 1;
  auto slot = [&](int i) { return i == 0 ? s.first_slot : 2 * (s.cf + i); };
  auto all = [&](float v, bool maxi) {  // over the block, the same in every thread
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float y = __shfl_xor_sync(0xffffffffu, v, o);
      v = maxi ? fmaxf(v, y) : v + y;
    }
    __syncthreads();
    if (lane == 0) red[tid >> 5] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int k = 1; k < D / 128; ++k) v = maxi ? fmaxf(v, red[k]) : v + red[k];
    return v;
  };
  float M = -INFINITY, L = 0.f;
  for (int i = tid; i < n; i += D / 4) M = fmaxf(M, w[i] = ws.ml[slot(i) * 8 + row].x);
  M = all(M, true);
  for (int i = tid; i < n; i += D / 4) {
    const float f = w[i] == -INFINITY ? 0.f : ex2(w[i] - M);
    w[i] = f;
    if (f != 0.f) L += f * ws.ml[slot(i) * 8 + row].y;
  }
  L = all(L, false);  // its barriers also publish w
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
  for (int i = 0; i < n; ++i) {
    const float f = w[i];
    const float4 o = *reinterpret_cast<const float4*>(ws.o + ((int64_t)slot(i) * 8 + row) * D + 4 * tid);
    acc.x = fmaf(f, o.x, acc.x);
    acc.y = fmaf(f, o.y, acc.y);
    acc.z = fmaf(f, o.z, acc.z);
    acc.w = fmaf(f, o.w, acc.w);
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
  bf16* o = a.out + ((int64_t)(s.row0 + row / a.share) * a.Hq + s.h * a.share + row % a.share) * D + 4 * tid;
  *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
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

// The scratch of a call: the status word, then what the parts of split items leave.
size_t carve(void* base, const PagedDev& c, FewWs* w) {
  Carver k(base);
  w->status = k.take<int>(64);
  w->split = k.take<Split>(kNumSMs);
  w->o = k.take<float>((size_t)2 * kNumSMs * 8 * c.D);
  w->ml = k.take<float2>((size_t)2 * kNumSMs * 8);
  return align_up(k.off, 256);
}

// The pages of one layer as the split kernel copies them: bf16 rows, or the
// rows of codes of every block.
int encode_pages(CUtensorMap* m, const PagedDev& c, int layer) {
  const int64_t blocks = 2ll * c.num_pages * c.Hkv;
  if (blocks * c.ps > INT32_MAX)
    return set_error(FMOE_ERR_UNSUPPORTED, "paged_attend: %lld rows in a layer's pages", (long long)(blocks * c.ps));
  const void* base = c.pages + layer * c.layer;
  if (c.bits == 16) {
    const cuuint64_t dims[2] = {(cuuint64_t)c.D, (cuuint64_t)(blocks * c.ps)}, strides[1] = {(cuuint64_t)c.D * 2};
    const cuuint32_t box[2] = {64, 16};
    return encode(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, "pages");
  }
  const cuuint64_t dims[3] = {(cuuint64_t)c.D / 2, (cuuint64_t)c.ps, (cuuint64_t)blocks};
  const cuuint64_t strides[2] = {(cuuint64_t)c.D / 2, (cuuint64_t)c.block};
  const cuuint32_t box[3] = {128, 16, 1};
  return encode(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, "pages");
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
  CUtensorMap map;
  if (int rc = encode_pages(&map, c, a.layer)) return rc;
  {
    ProfScope prof_(C::BITS == 16 ? "paged_attn_split_kernel<bf16>" : "paged_attn_split_kernel<4-bit>", st);
    paged_attn_split_kernel<C><<<kNumSMs, C::NT, C::SMEM, st>>>(map, c, b, a, w);
  }
  if (int rc = check_launch("paged_attn_split_kernel")) return rc;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(kNumSMs, kFewRows);
  cfg.blockDim = dim3(C::D / 4);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  ProfScope prof_("paged_attn_join_kernel", st);
  cudaLaunchKernelEx(&cfg, paged_attn_join_kernel<C::D>, a, w);
  return check_launch("paged_attn_join_kernel");
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
  return pa::carve(nullptr, c, &w);
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
  pa::carve(workspace, c, &w);
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
