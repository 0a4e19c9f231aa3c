// Attention over [shared prefix | own pages] for 16-bit types on the 5th-generation tensor cores.
//
// One persistent CTA per SM walks its stretch of the line (hc_prefix.cuh) in row tiles of up to 256 rows
// and key tiles of 128. Per key tile: S = Q K^T (M = 128 rows, N = 128 keys, fp32 in TMEM), P = 2^(S scale
// log2 e - m) rounded to the operand type (off by half a step of each probability, as large as the
// rounding of the result itself) and written over S in TMEM, O += P V with P as the TMEM operand and V read
// in place as an MN-major operand; O stays in TMEM for the whole piece. The softmax is online, and O is
// only rescaled when a row's maximum has grown by more than 2^8 since the last time: until then P exceeds 1
// by at most that, which neither type minds, and the 32-bit sums carry the same factor.
//
// Roles: warp 0 brings K and V tiles by TMA into a ring (pages as boxes of their own, absent pages as
// boxes out of range, which read as zeros); warps 1 and 2 each issue the MMAs of one stream; warps 4-7 and
// 8-11 are the softmax of the two streams, a thread per row. Of a row tile above 128 rows the streams take
// a half each and share the K/V tiles; of a smaller one (a decode step of one sequence's pages, a small
// batch) they take every second key tile of the same rows, with results of their own that the merge joins,
// so that one stream's softmax runs under the other's MMAs in both cases.
//
// Bound: HBM while 2 (rows) D flops a key cost less than its 2 D elements, i.e. up to about 256 rows a row
// tile; beyond that the MMAs (1024 cycles per 128 x 128 x 128 pair) and the 128 x 128 exponentials (1024
// cycles at 16 a cycle) of each tile.

#include <cuda.h>
#include <cudaTypedefs.h>

#include "hc_prefix.cuh"

namespace hc {

constexpr int kMmaThreads = 384, kMmaR = 256, kMmaK = 128;
constexpr float kLazy = 8.f;  // log2 of how far P may exceed 1 before O is rescaled

template <int D>
struct MmaSmem {
  static constexpr int PL = D / 64;                 // planes of 64 elements (128 bytes, the swizzle width)
  static constexpr uint32_t tile = 128u * 128u * PL;  // 128 rows
  static constexpr int NB = D == 128 ? 5 : 8;       // K/V tiles in the ring
  static constexpr uint32_t q = 0;
  static constexpr uint32_t ring = 2 * tile;
  static constexpr uint32_t bars = ring + NB * tile;  // full[NB] empty[NB] s_full[2] p_ready[2] pv_done[2] q_ready[2] fin
  static constexpr uint32_t misc = bars + 8 * (2 * NB + 9);  // tmem address, dead flag, poison[2], armed
  static constexpr uint32_t scan = (misc + 32 + 15) & ~15u;
  static constexpr uint32_t bytes = scan + 8 * (kMmaThreads / 32 + 4);
};

struct PrefixMaps {
  CUtensorMap pk, pv, kp, vp;
  int pk_tok, pv_tok;  // which coordinate (1 or 2) of the prefix maps is the token
};

__device__ __forceinline__ void tma_load_3d(void* dst_smem, const void* tmap, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst_smem)),
      "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// D[tmem] (+)= A[tmem] . B[smem] (A: 128 lanes, two 16-bit K elements a column).
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem, uint32_t atmem, uint64_t bdesc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}\n" ::"r"(tmem),
      "r"(atmem), "l"(bdesc), "r"(idesc), "r"(acc), "r"(0u), "r"(0u), "r"(0u), "r"(0u)
      : "memory");
}
// 32 lanes x 32 columns, this warp's lane quarter; the caller waits with tmem_wait_ld.
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_x32(uint32_t taddr, const float* v) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  tmem_st_x16(taddr, r);
  tmem_st_x16(taddr + 16, r + 16);
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void named_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (DT == HC_F16) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// A wait that gives up after kMaxPolls polls and marks the CTA dead; from then on no wait of the CTA
// lasts, every role runs through its remaining pieces, and the results are marked invalid by the status.
__device__ __forceinline__ void wait_bar(uint64_t* bar, uint32_t parity, volatile int* dead, int32_t* status) {
  for (int i = 0; i < kMaxPolls; ++i) {
    if (mbar_try_wait(bar, parity)) return;
    if (*dead) return;
  }
  *dead = 1;
  if (status) atomicOr(status, HC_DEV_TIMEOUT);
}

// Waits until ring position n is filled. A stream that takes only every second tile, or none of several
// pieces, does not see every fill of a buffer, so its parity alone could name an older fill: it first waits
// until the producer has armed position n, which it does once every earlier fill of that buffer is used up.
template <int NB>
__device__ __forceinline__ void wait_full(uint64_t* full, uint32_t n, volatile uint32_t* armed, volatile int* dead,
                                          int32_t* status) {
  for (int i = 0; *armed <= n; ++i) {
    if (*dead) return;
    if (i == kMaxPolls) {
      *dead = 1;
      if (status) atomicOr(status, HC_DEV_TIMEOUT);
      return;
    }
    __nanosleep(64);
  }
  wait_bar(&full[n % NB], (n / NB) & 1, dead, status);
}

template <int DT, int D>
__global__ void __launch_bounds__(kMmaThreads, 1)
    prefix_mma_kernel(PrefixArgs a, LineShape ls, int64_t* hdr, float2* ml, float* part, const __grid_constant__ PrefixMaps maps) {
  using T = typename Elem<DT>::T;
  using SM = MmaSmem<D>;
  constexpr int PL = SM::PL, NB = SM::NB;
  constexpr uint32_t kFmt = DT == HC_BF16 ? 1u : 0u;
  constexpr uint32_t kIdS = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((uint32_t)(kMmaK >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
  // P V: N = D, B (V) MN-major
  constexpr uint32_t kIdO = (1u << 4) | (kFmt << 7) | (kFmt << 10) | (1u << 16) | ((uint32_t)(D >> 3) << 17) |
                            ((uint32_t)(128 >> 4) << 24);
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + SM::bars);
  uint64_t *empty = full + NB, *s_full = empty + NB, *p_ready = s_full + 2, *pv_done = p_ready + 2, *q_ready = pv_done + 2;
  uint64_t* fin = q_ready + 2;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + SM::misc);
  volatile int* dead = reinterpret_cast<volatile int*>(smem + SM::misc + 4);
  int* poison = reinterpret_cast<int*>(smem + SM::misc + 8);  // per stream: a hidden value was not finite
  volatile uint32_t* armed = reinterpret_cast<volatile uint32_t*>(smem + SM::misc + 16);  // ring positions armed
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = ls.G;

  if (tid == 0) {
    for (int i = 0; i < NB; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 2);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&s_full[x], 1);
      mbar_init(&p_ready[x], 4);
      mbar_init(&pv_done[x], 1);
      mbar_init(&q_ready[x], 4);
    }
    mbar_init(fin, 2);
    fence_mbar_init();
    *dead = 0;
    *armed = 0;
    poison[0] = poison[1] = 0;
    prefetch_tensormap(&maps.kp);
    prefetch_tensormap(&maps.vp);
    if (ls.P > 0) {
      prefetch_tensormap(&maps.pk);
      prefetch_tensormap(&maps.pv);
    }
  }
  if (warp == 3) tmem_alloc(s_tmem, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = *s_tmem;
  pdl_wait();
  const LineGeom g(ls, min(a.T, max(a.cu_new[ls.n_seq], 0)));
  LineWalk walk;
  walk.c = blockIdx.x;
  walk.st = line_setup<kMmaThreads>(a, ls, g, blockIdx.x, hdr, reinterpret_cast<int64_t*>(smem + SM::scan));
  Piece p;

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      // ---- producer --------------------------------------------------------------------
      const int sh = __ffs(a.page_size) - 1;
      const int bx = min(a.page_size, kMmaK), nbx = kMmaK / bx;
      const int y_out = a.n_pages * ls.Hk * a.page_size;  // out of range: reads as zeros
      uint32_t n = 0;
      bool stop = false;
      while (!stop && walk.next(a, ls, g, p)) {
        for (int kt = p.kt0; kt < p.kt1; ++kt) {
          stop = __any_sync(0xffffffffu, *dead);
          if (stop) break;
          int y = y_out;
          if (p.own && lane < nbx) {
            const int key = kt * kMmaK + lane * bx;
            if (key < p.kend) {
              const int page = a.block_table[(size_t)p.b * a.max_blocks + (key >> sh)];
              if (page >= 0 && page < a.n_pages) y = (page * ls.Hk + p.h) * a.page_size + (key & (a.page_size - 1));
              else if (a.status) atomicOr(a.status, HC_DEV_INDEX);
            }
          }
#pragma unroll
          for (int kv = 0; kv < 2; ++kv, ++n) {
            const uint32_t b = n % NB;
            wait_bar(&empty[b], ((n / NB) & 1) ^ 1, dead, a.status);
            unsigned char* dst = smem + SM::ring + b * SM::tile;
            if (lane == 0) {
              mbar_arrive_expect_tx(&full[b], SM::tile);
              *armed = n + 1;
            }
            __syncwarp();
            if (p.own) {
              if (lane < nbx)
#pragma unroll
                for (int pl = 0; pl < PL; ++pl)
                  tma_load_2d(dst + pl * 16384 + lane * bx * 128, kv ? &maps.vp : &maps.kp, pl * 64, y, &full[b]);
            } else if (lane < PL) {
              const bool tok1 = (kv ? maps.pv_tok : maps.pk_tok) == 1;
              tma_load_3d(dst + lane * 16384, kv ? &maps.pv : &maps.pk, lane * 64, tok1 ? kt * kMmaK : p.h,
                          tok1 ? p.h : kt * kMmaK, &full[b]);
            }
          }
        }
      }
      // copies still in flight write this CTA's shared memory: they land before it ends
      for (uint32_t i = n > NB ? n - NB : 0; i < n; ++i) mbar_wait(&full[i % NB], (i / NB) & 1);
    } else if (warp < 3) {
      // ---- MMA issue of stream x ---------------------------------------------------------
      if (lane == 0) {
        const int x = warp - 1;
        const uint32_t tS = tbase + x * 128, tO = tbase + 256 + x * 128;
        const uint32_t sq = smem_u32(smem + SM::q + x * SM::tile), sr = smem_u32(smem + SM::ring);
        uint32_t base = 0, np = 0, nt = 0;  // ring position, pieces and tiles of this stream
        while (walk.next(a, ls, g, p)) {
          const bool both = p.ntok * G > 128;
          const int tiles = p.kt1 - p.kt0, step = both ? 1 : 2;
          bool begun = false;
          for (int i = both ? 0 : x; i < tiles; i += step, ++nt) {
            const uint32_t nk = base + 2 * i, nv = nk + 1, bk = nk % NB, bv = nv % NB;
            if (!begun) wait_bar(&q_ready[x], np & 1, dead, a.status);
            wait_full<NB>(full, nk, armed, dead, a.status);
            if (nt > 0) wait_bar(&pv_done[x], (nt - 1) & 1, dead, a.status);  // P of the last tile has been read
            tc_fence_after();
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
              umma_f16(tS, umma_desc_k_sw128(sq + (ks >> 2) * 16384u + (ks & 3) * 32u),
                       umma_desc_k_sw128(sr + bk * SM::tile + (ks >> 2) * 16384u + (ks & 3) * 32u), kIdS, ks > 0);
            umma_commit(&s_full[x]);
            umma_commit(&empty[bk]);
            if (!both) umma_commit(&empty[bk]);
            wait_bar(&p_ready[x], nt & 1, dead, a.status);
            wait_full<NB>(full, nv, armed, dead, a.status);
            tc_fence_after();
#pragma unroll
            for (int ks = 0; ks < kMmaK / 16; ++ks)
              umma_f16_ts(tO, tS + ks * 8, umma_desc_mn_sw128(sr + bv * SM::tile + ks * 2048u, 16384u), kIdO,
                          (begun || ks > 0) ? 1u : 0u);
            umma_commit(&pv_done[x]);
            umma_commit(&empty[bv]);
            if (!both) umma_commit(&empty[bv]);
            begun = true;
          }
          if (begun) ++np;
          base += 2 * tiles;
        }
        umma_commit(fin);
      }
      __syncwarp();
    }
  } else {
    // ---- softmax of stream x: thread = row -------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int x = (warp >> 2) - 1, r = tid & 127;
    const uint32_t quarter = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tS = tbase + x * 128 + quarter, tO = tbase + 256 + x * 128 + quarter;
    unsigned char* sQ = smem + SM::q + x * SM::tile;
    const float sc = a.scale * 1.4426950408889634f;
    uint32_t base = 0, nt = 0;
    while (walk.next(a, ls, g, p)) {
      const int rows = p.ntok * G, tiles = p.kt1 - p.kt0;
      const bool both = rows > 128;
      const int row_at = both ? x * 128 : 0;                 // this stream's first row of the row tile
      const int nr = min(max(rows - row_at, 0), 128);
      const int64_t out_row = p.row0 + (both ? x * 128 : x * rows) + r;
      const int first = both ? 0 : x, step = both ? 1 : 2;
      float m = kNegInf, l = 0.f;
      if (first < tiles) {
        // Q rows, 16 bytes a thread at a time, in the swizzled K-major layout
        constexpr int CPR = D / 8;
#pragma unroll 4
        for (int k = r; k < 128 * CPR; k += 128) {
          const int rr = k / CPR, c = k % CPR;
          if (rr < nr) {
            const int row = row_at + rr;
            const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(p.tok0 + row / G) * a.q_st +
                           (int64_t)(p.h * G + row % G) * a.q_sh;
            *reinterpret_cast<uint4*>(sQ + (c >> 3) * 16384 + rr * 128 + (((c & 7) ^ (rr & 7)) << 4)) =
                reinterpret_cast<const uint4*>(src)[c];
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_ready[x]);
      }
      const bool live = (warp & 3) * 32 < nr;  // of a warp without rows nothing is read
      // own keys of this row: j < lim
      const int lim = p.own ? min(p.c0 + (row_at + r) / G + 1, p.kend) : p.kend;
      const bool hides = p.own && p.c0 + 1 < p.kend;  // some key here is hidden from some row
      bool any_poison = false;
      for (int i = first; i < tiles; i += step, ++nt) {
        const int k0 = (p.kt0 + i) * kMmaK;
        uint32_t w[4] = {~0u, ~0u, ~0u, ~0u};
        uint32_t wr = ~0u;  // the word of this thread's V row
        bool masked = false;
        if (a.mask && !p.own) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = k0 + j * 32 + lane;
            w[j] = __ballot_sync(0xffffffffu, key < p.kend && a.mask[key] != 0);
            masked |= w[j] != ~0u;
            if (j == (warp & 3)) wr = w[j];
          }
        }
        wait_bar(&s_full[x], nt & 1, dead, a.status);
        tc_fence_after();
        if (live) {
          float s[128];
#pragma unroll
          for (int j = 0; j < 4; ++j) tmem_ld_x32(tS + j * 32, s + j * 32);
          tmem_wait_ld();
          const int n = lim - k0;  // columns seen
          if (masked || __any_sync(0xffffffffu, n < kMmaK)) {
#pragma unroll
            for (int j = 0; j < 128; ++j) s[j] = j < n && (w[j >> 5] >> (j & 31) & 1u) ? s[j] : kNegInf;
          }
          float mx0 = s[0], mx1 = s[1], mx2 = s[2], mx3 = s[3];
#pragma unroll
          for (int j = 4; j < 128; j += 4) {
            mx0 = fmaxf(mx0, s[j]);
            mx1 = fmaxf(mx1, s[j + 1]);
            mx2 = fmaxf(mx2, s[j + 2]);
            mx3 = fmaxf(mx3, s[j + 3]);
          }
          const float mt = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * sc;
          if (__any_sync(0xffffffffu, r < nr && mt > m + kLazy)) {  // rows of no token hold anything: no vote
            const float mn = fmaxf(m, mt), al = ex2_approx(m - (mn == kNegInf ? 0.f : mn));
            m = mn;
            l *= al;
            if (i > first) {
#pragma unroll
              for (int j = 0; j < D; j += 32) {
                float o[32];
                tmem_ld_x32(tO + j, o);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] *= al;
                tmem_st_x32(tO + j, o);
              }
            }
          }
          const float ref = m == kNegInf ? 0.f : m;
          float l0 = 0.f, l1 = 0.f;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t pk[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const float p0 = ex2_approx(fmaf(s[j * 32 + 2 * e], sc, -ref));
              const float p1 = ex2_approx(fmaf(s[j * 32 + 2 * e + 1], sc, -ref));
              l0 += p0;
              l1 += p1;
              pk[e] = pack2<DT>(p0, p1);
            }
            tmem_st_x16(tS + j * 16, pk);
          }
          l += l0 + l1;
          tmem_wait_st();
        }
        // V rows that no row here attends (masked, behind the end, absent) may hold anything: they become
        // zeros, since the MMA multiplies them by 0
        const uint32_t nv = base + 2 * i + 1, bv = nv % NB;
        const bool scan = hides && k0 + kMmaK > p.c0 + 1;
        if (masked || (p.own && k0 + kMmaK > p.kend) || scan) {
          wait_full<NB>(full, nv, armed, dead, a.status);
          unsigned char* sV = smem + SM::ring + bv * SM::tile + r * 128;
          const int key = k0 + r;
          if (key >= p.kend || !(wr >> lane & 1u)) {
#pragma unroll
            for (int c = 0; c < PL * 8; ++c) *reinterpret_cast<uint4*>(sV + (c >> 3) * 16384 + (c & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          } else if (scan && key > p.c0 && (!both || x == 0)) {
            // hidden from the first rows and attended by the last: values that are not finite are taken
            // out here and added to the rows that attend them at the end
            bool odd = false;
            for (int c = 0; c < PL * 8; ++c) {
              uint4* at = reinterpret_cast<uint4*>(sV + (c >> 3) * 16384 + (c & 7) * 16);
              uint4 u = *at;
              float f[8];
              unpack16<DT>(u, f);
              bool bad = false;
              for (int e = 0; e < 8; ++e) bad |= !isfinite(f[e]);
              if (bad) {
                odd = true;
                alignas(16) T t[8];
                for (int e = 0; e < 8; ++e) t[e] = Elem<DT>::from_f(isfinite(f[e]) ? f[e] : 0.f);
                *at = *reinterpret_cast<uint4*>(t);
              }
            }
            if (odd) atomicOr(&poison[x], 1);
          }
          fence_proxy_async_smem();
          if (scan) {
            named_sync(both ? 3 : 1 + x, both ? 256 : 128);
            any_poison |= *reinterpret_cast<volatile int*>(&poison[both ? 0 : x]) != 0;
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_ready[x]);
      }
      if (first < tiles) {
        wait_bar(&pv_done[x], (nt - 1) & 1, dead, a.status);
        tc_fence_after();
        if (live) {
          const T* vp = reinterpret_cast<const T*>(a.v_pages);
          const int sh = __ffs(a.page_size) - 1;
#pragma unroll
          for (int j = 0; j < D; j += 32) {
            float o[32];
            tmem_ld_x32(tO + j, o);
            tmem_wait_ld();
            if (any_poison && r < nr) {
              for (int i = first; i < tiles; i += step) {
                const int k0 = (p.kt0 + i) * kMmaK;
                for (int key = max(k0, p.c0 + 1); key < min(k0 + kMmaK, lim); ++key) {
                  const int page = a.block_table[(size_t)p.b * a.max_blocks + (key >> sh)];
                  if (page < 0 || page >= a.n_pages) continue;
                  const T* v = vp + (((size_t)page * ls.Hk + p.h) * a.page_size + (key & (a.page_size - 1))) * D + j;
#pragma unroll
                  for (int e = 0; e < 32; ++e) {
                    const float f = Elem<DT>::to_f(v[e]);
                    if (!isfinite(f)) o[e] += f;
                  }
                }
              }
            }
            if (r < nr) {
              float4* dst = reinterpret_cast<float4*>(part + (size_t)out_row * D + j);
#pragma unroll
              for (int e = 0; e < 8; ++e) dst[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
            }
          }
        }
        tc_fence_before();
      }
      if (r < nr) ml[out_row] = make_float2(m, l);
      base += 2 * tiles;
      if (any_poison) {  // cleared for the next piece once every thread that reads it has
        named_sync(both ? 3 : 1 + x, both ? 256 : 128);
        if (r == 0) poison[both ? 0 : x] = 0;
        named_sync(both ? 3 : 1 + x, both ? 256 : 128);
      }
    }
  }
  __syncthreads();
  if (warp == 3) {
    mbar_wait(fin, 0);  // every MMA has ended
    tc_fence_after();
    tmem_dealloc(tbase, 512);
  }
}

// ----------------------------------------------------------------------------------------
// host
// ----------------------------------------------------------------------------------------
static PFN_cuTensorMapEncodeTiled_v12000 tensor_map_encoder() {
  static std::mutex mu;
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  std::lock_guard<std::mutex> lock(mu);
  if (!fn) {
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    void* p = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      (void)cudaGetLastError();
    else
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  }
  return fn;
}

static bool encode_rows(CUtensorMap* m, PFN_cuTensorMapEncodeTiled_v12000 enc, int dtype, const void* base, int rank,
                        const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  const cuuint32_t estr[3] = {1u, 1u, 1u};
  return enc(m, dtype == HC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank,
             const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
             CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// (heads, tokens, D) with any strides: the dimension of the smaller stride comes first.
static bool encode_prefix(CUtensorMap* m, int* tok, PFN_cuTensorMapEncodeTiled_v12000 enc, int dtype, const void* base,
                          int Hk, int P, int D, int64_t sh, int64_t st) {
  *tok = st <= sh ? 1 : 2;
  const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)(*tok == 1 ? P : Hk), (cuuint64_t)(*tok == 1 ? Hk : P)};
  const cuuint64_t strides[2] = {(cuuint64_t)(*tok == 1 ? st : sh) * 2, (cuuint64_t)(*tok == 1 ? sh : st) * 2};
  const cuuint32_t box[3] = {64u, *tok == 1 ? (cuuint32_t)kMmaK : 1u, *tok == 1 ? 1u : (cuuint32_t)kMmaK};
  return encode_rows(m, enc, dtype, base, 3, dims, strides, box);
}

template <int DT, int D>
static cudaError_t mma_t(const PrefixArgs& a, const LineShape& s, int64_t* hdr, float2* ml, float* part, cudaStream_t stream) {
  PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
  if (!enc) return cudaErrorNotSupported;
  PrefixMaps maps{};
  bool ok = true;
  if (a.P > 0)
    ok = encode_prefix(&maps.pk, &maps.pk_tok, enc, DT, a.pk, a.Hk, a.P, D, a.pk_sh, a.pk_st) &&
         encode_prefix(&maps.pv, &maps.pv_tok, enc, DT, a.pv, a.Hk, a.P, D, a.pv_sh, a.pv_st);
  const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)a.n_pages * a.Hk * a.page_size};
  const cuuint64_t strides[1] = {(cuuint64_t)D * 2};
  const cuuint32_t box[2] = {64u, (cuuint32_t)(a.page_size < kMmaK ? a.page_size : kMmaK)};
  ok = ok && encode_rows(&maps.kp, enc, DT, a.k_pages, 2, dims, strides, box) &&
       encode_rows(&maps.vp, enc, DT, a.v_pages, 2, dims, strides, box);
  if (!ok) return cudaErrorInvalidValue;
  auto kern = prefix_mma_kernel<DT, D>;
  cudaError_t e = ensure_smem(kern, MmaSmem<D>::bytes);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3((unsigned)s.nc), dim3(kMmaThreads), (size_t)MmaSmem<D>::bytes, stream, a, s, hdr, ml, part, maps);
}

LineShape prefix_mma_shape(int T, int n_seq, int Hk, int G, int P, int sms) {
  return line_shape(T, n_seq, Hk, G, P, kMmaR, kMmaK, sms, 2);
}

cudaError_t launch_prefix_mma(const PrefixArgs& a, const LineShape& s, int dtype, int D, int64_t* hdr, float2* ml, float* part,
                              cudaStream_t stream) {
  if (dtype == HC_F16 && D == 128) return mma_t<HC_F16, 128>(a, s, hdr, ml, part, stream);
  if (dtype == HC_BF16 && D == 128) return mma_t<HC_BF16, 128>(a, s, hdr, ml, part, stream);
  if (dtype == HC_F16 && D == 64) return mma_t<HC_F16, 64>(a, s, hdr, ml, part, stream);
  if (dtype == HC_BF16 && D == 64) return mma_t<HC_BF16, 64>(a, s, hdr, ml, part, stream);
  return cudaErrorInvalidValue;
}

}  // namespace hc
