// Attention over [shared prefix | own pages] for 16-bit types on the 5th-generation tensor cores.
//
// One persistent CTA per SM walks its stretch of the line (hc_prefix.cuh) in row tiles of up to 256 rows
// and key tiles of 128. Softmax is online over the key tiles: P = 2^(S scale log2 e - m), rounded to the
// operand type (off by half a step of each probability, as large as the rounding of the result itself); O
// stays in TMEM for the whole piece and is only rescaled when a row's maximum has grown by more than 2^8
// since the last time: until then P exceeds 1 by at most that, which neither type minds, and the 32-bit sums
// carry the same factor.
//
// Roles: warp 0 brings K and V tiles by TMA into a ring (pages as boxes of their own, absent pages as
// boxes out of range, which read as zeros); warps 1 and 2 each issue the MMAs of one stream; warps 4-7 and
// 8-11 are the softmax of the two streams. What a stream is depends on the piece's rows:
//   above 128  a half of the rows each, both over all key tiles. S = Q K^T (M = 128 rows, N = 128 keys), a
//              thread per row; P goes back to TMEM over S as the A operand of O += P V, V read in place as
//              an MN-major operand.
//   65 to 128  the same rows, every second key tile each, each with a result of its own for the merge.
//   up to 64   whole pieces in turn, transposed: S^T = K Q^T (M = 128 keys, N = the rows), a thread per key,
//              so that all 128 threads have work where a thread per row would leave one warp 128 columns;
//              P^T through shared memory as the B operand of O^T += V^T P^T.
// Either way one stream's softmax runs under the other's MMAs and copies.
//
// Bound: by its bytes up to about 256 rows a row tile, beyond that by the MMAs (1024 cycles per 128 x 128 x 128
// pair) and the 128 x 128 exponentials (1024 cycles at 16 a cycle) of each tile. Measured on one B200, D = 128
// in 16 bits: a key tile of 256 rows 2.6 to 2.8 us (its bytes at a 148th of HBM 1.5, MMAs 1.1, exponentials 1.1), of
// 65 to 128 rows 1.2 us, of up to 64 rows 1.15 us where pieces alternate and 1.8 to 3.2 us where a stretch is one
// piece and so one stream's; 64 sequences over 128k prefix keys 244 us (2.5 TB/s, 564 TFLOP/s), a chunk of 8 x 257
// over 16k 434 us (690 TFLOP/s). What the tall tile loses is in its chain: softmax 1.4 us, then [O += P V, next S]
// 1.4 us, in turns, since P lies over S and the next S has to wait for P V.

#include <cuda.h>
#include <cudaTypedefs.h>

#include "hc_prefix.cuh"

namespace hc {

constexpr int kMmaThreads = 384, kMmaR = 256, kMmaK = 128;
constexpr int kPieces = 8;    // pieces listed ahead

template <int DT>
struct PRange {
  static constexpr float kLift = DT == HC_F16 ? 11.f : 0.f;  // log2 of what P of a row's maximum is
  static constexpr float kLazy = DT == HC_F16 ? 4.f : 8.f;   // log2 of how far P may exceed that before O is rescaled
};

template <int D>
struct MmaSmem {
  static constexpr int PL = D / 64;                   // planes of 64 elements (128 bytes, the swizzle width)
  static constexpr uint32_t tile = 128u * 128u * PL;  // 128 rows
  static constexpr int NB = D == 128 ? 5 : 8;         // K/V tiles in the ring
  static constexpr uint32_t qbuf = 32768;             // per stream: Q (transposed pieces: Q, then P^T from ptr on)
  static constexpr uint32_t pt = 16384;
  static constexpr uint32_t ring = 2 * qbuf;
  static constexpr uint32_t bars = ring + NB * tile;  // full[NB] empty[NB] s_full[2] p_ready[2] pv_done[2] q_ready[2] fin both
  static constexpr uint32_t misc = (bars + 8 * (2 * NB + 10) + 15) & ~15u;  // tmem address, dead, armed, q_here, poison[3], turns[2]
  static constexpr uint32_t red = misc + 48;  // per stream [4 warps][64 rows]; the setup's scan before that
  static constexpr uint32_t pieces = red + 2 * 4 * 64 * 4;           // the next pieces, and their barriers
  static constexpr uint32_t pbars = pieces + kPieces * sizeof(Piece);  // full[kPieces] empty[kPieces]
  static constexpr uint32_t bytes = pbars + 16 * kPieces;
  static_assert(bytes <= 227 * 1024, "shared memory of a CTA");
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
    if (i == 16 * kMaxPolls) {
      *dead = 1;
      if (status) atomicOr(status, HC_DEV_TIMEOUT);
      return;
    }
  }
  wait_bar(&full[n % NB], (n / NB) & 1, dead, status);
}

// 32 lanes x N columns (N = 8, 16, 32 or 64) and back.
template <int N>
__device__ __forceinline__ void tmem_ld_n(uint32_t taddr, float* v) {
  if constexpr (N == 8) {
    tmem_ld_x8(taddr, v);
  } else if constexpr (N == 16) {
    tmem_ld_x8(taddr, v);
    tmem_ld_x8(taddr + 8, v + 8);
  } else {
#pragma unroll
    for (int j = 0; j < N; j += 32) tmem_ld_x32(taddr + j, v + j);
    tmem_wait_ld();
  }
}
__device__ __forceinline__ void tmem_st_x8(uint32_t taddr, const float* v) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]),
               "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ float redux_max(float x) {
  float y;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}

// Stream x's turn for its tall tile number n: the first stream goes when the other has issued all S tiles
// before n, the second when the first has issued S tile n.
__device__ __forceinline__ void wait_turn(volatile uint32_t* turns, int x, uint32_t n, volatile int* dead) {
  for (int i = 0; turns[x ^ 1] < n + x && !*dead && i < 16 * kMaxPolls; ++i) {
  }
}
// Shared-memory descriptors from their low word's address (see umma_desc_k_sw128, umma_desc_mn_sw128).
__device__ __forceinline__ uint64_t desc_k(uint32_t addr16) {
  return ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32) | (addr16 | (1u << 16));
}
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr16, uint32_t lbo16) {
  return ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32) | (addr16 | (lbo16 << 16));
}
__device__ __forceinline__ bool elect_one() {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
  return ok != 0;
}

// The CTA's pieces, listed ahead in shared memory by one thread (a role that walked the line itself would
// carry its state in registers and wait for the tables at every piece). Every role reads every piece, and an
// entry is written anew once all have copied it. These waits outlast the others and do not give up with them
// when the CTA is dead: no role waits for anything else then, so all arrive here, and every warp sees the
// same pieces (the barriers among a stream's four warps depend on nothing but the piece).
__device__ __forceinline__ void mbar_wait_long(uint64_t* bar, uint32_t parity) {
  for (int i = 0; i < 8; ++i)
    if (mbar_wait(bar, parity)) return;
}
struct PieceRing {
  const Piece* e;
  uint64_t *full, *empty;
  uint32_t k;
  // Whether the next piece is listed, for the whole warp.
  __device__ __forceinline__ bool listed() const {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(&full[k % kPieces])), "r"((k / kPieces) & 1)
        : "memory");
    return __all_sync(0xffffffffu, ok);
  }
  // Copies the next piece; false after the last. `lanes`: the threads of the warp that read it.
  __device__ __forceinline__ bool next(Piece& p, uint32_t lanes, bool first) {
    mbar_wait_long(&full[k % kPieces], (k / kPieces) & 1);
    p = e[k % kPieces];
    __syncwarp(lanes);
    if (first) mbar_arrive(&empty[k % kPieces]);
    ++k;
    return p.kt1 > p.kt0;
  }
};

// What a stream does with a piece.
enum { kSkip = 0, kHalf, kEvery2nd, kTransposed };
struct Part {
  int mode, rows, row_at, nr;  // rows of the piece, this stream's first row and its rows
  int first, step, tiles;      // its key tiles: first, first + step, ... < tiles
};
__device__ __forceinline__ Part piece_part(const Piece& p, int G, int x, uint32_t turn) {
  Part t;
  t.rows = p.ntok * G;
  t.tiles = p.kt1 - p.kt0;
  t.row_at = 0;
  t.nr = t.rows;
  t.first = 0;
  t.step = 1;
  if (t.rows > 128) {
    t.mode = kHalf;
    t.row_at = x * 128;
    t.nr = min(t.rows - t.row_at, 128);
  } else if (prefix_two_streams(t.rows)) {
    t.mode = x < t.tiles ? kEvery2nd : kSkip;
    t.first = x;
    t.step = 2;
  } else {
    t.mode = (turn & 1) == (uint32_t)x ? kTransposed : kSkip;
  }
  return t;
}
// Rows of the transposed MMAs' N for nr rows, and the values a softmax thread holds.
__device__ __forceinline__ int t_cols(int nr) { return nr <= 16 ? 16 : nr <= 32 ? 32 : 64; }

// State of one softmax stream while it works on a piece.
struct Soft {
  const PrefixArgs& a;
  const LineShape& ls;
  const Piece& p;
  const Part& t;
  unsigned char* smem;
  uint64_t *full, *s_full, *p_ready, *pv_done, *both;
  volatile uint32_t* armed;
  volatile int* dead;
  int* poison;  // this piece's flag
  float sc;
  uint32_t base;  // ring position of the piece
  int x, r, lane, warp4;
  uint32_t tS, tO;
  uint32_t& meets;  // meetings of the two streams so far
  // The two streams of a tall row tile meet.
  __device__ __forceinline__ void meet() const {
    __syncwarp();
    if (lane == 0) mbar_arrive(both);
    wait_bar(both, meets & 1, dead, a.status);
    ++meets;
  }
};

// The prefix mask of a key tile: bits of this warp's 32 V rows and, for the row-wise softmax, of all 128.
__device__ __forceinline__ bool tile_mask(const Soft& f, int k0, uint32_t* w, uint32_t& wr) {
  wr = ~0u;
#pragma unroll
  for (int j = 0; j < 4; ++j) w[j] = ~0u;
  if (!f.a.mask || f.p.own) return false;
  bool masked = false;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int key = k0 + j * 32 + f.lane;
    w[j] = __ballot_sync(0xffffffffu, key < f.p.kend && f.a.mask[key] != 0);
    masked |= w[j] != ~0u;
    if (j == f.warp4) wr = w[j];
  }
  return masked;
}

// V rows that no row here attends (masked, behind the end, absent) may hold anything: they become zeros,
// since the MMA multiplies them by 0. Values hidden from the first rows and attended by the last that are
// not finite are taken out here and added to the rows that attend them at the end of the piece. Returns
// whether the piece has any of those.
template <int DT, int D>
__device__ __forceinline__ bool clean_v(const Soft& f, int i, int k0, bool masked, uint32_t wr, bool any) {
  using T = typename Elem<DT>::T;
  using SM = MmaSmem<D>;
  const bool scan = f.p.own && f.p.c0 + 1 < f.p.kend && k0 + kMmaK > f.p.c0 + 1;
  if (!(masked || (f.p.own && k0 + kMmaK > f.p.kend) || scan)) return any;
  const uint32_t nv = f.base + 2 * i + 1;
  wait_full<SM::NB>(f.full, nv, f.armed, f.dead, f.a.status);
  unsigned char* sV = f.smem + SM::ring + (nv % SM::NB) * SM::tile + f.r * 128;
  const int key = k0 + f.r, rot = f.r & 7;  // chunks in an order that spreads a warp over the banks
  const bool half = f.t.mode == kHalf;
  if (key >= f.p.kend || !(wr >> f.lane & 1u)) {
#pragma unroll
    for (int c = 0; c < SM::PL * 8; ++c)
      *reinterpret_cast<uint4*>(sV + (c >> 3) * 16384 + (((c & 7) ^ rot) << 4)) = make_uint4(0u, 0u, 0u, 0u);
  } else if (scan && key > f.p.c0 && (!half || f.x == 0)) {
    // a 16-bit value is not finite when its exponent bits are all ones, i.e. carry into the top bit
    constexpr uint32_t kExp = DT == HC_F16 ? 0x7c007c00u : 0x7f807f80u, kOne = DT == HC_F16 ? 0x04000400u : 0x00800080u;
    bool odd = false;
#pragma unroll 4
    for (int c = 0; c < SM::PL * 8; ++c) {
      uint4* at = reinterpret_cast<uint4*>(sV + (c >> 3) * 16384 + (((c & 7) ^ rot) << 4));
      const uint4 u = *at;
      if ((((u.x & kExp) + kOne) | ((u.y & kExp) + kOne) | ((u.z & kExp) + kOne) | ((u.w & kExp) + kOne)) & 0x80008000u) {
        odd = true;
        const uint32_t y[4] = {u.x, u.y, u.z, u.w};
        uint32_t z[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t bad = (((y[e] & kExp) + kOne) & 0x80008000u) >> 15;  // 1 in each half that is not finite
          z[e] = y[e] & ~(bad * 0xffffu);
        }
        *at = make_uint4(z[0], z[1], z[2], z[3]);
      }
    }
    if (odd) atomicOr(f.poison, 1);
  }
  fence_proxy_async_smem();
  if (scan) {
    if (half) f.meet();
    else named_sync(1 + f.x, 128);
    any |= *reinterpret_cast<volatile int*>(f.poison) != 0;
  }
  return any;
}

// Calls fn(key, row of V) for the own keys of this stream's tiles in [c0 + 1, lim).
template <int DT, int D, typename F>
__device__ __forceinline__ void hidden_rows(const Soft& f, int lim, F fn) {
  using T = typename Elem<DT>::T;
  const int sh = __ffs(f.a.page_size) - 1;
  for (int i = f.t.first; i < f.t.tiles; i += f.t.step) {
    const int k0 = (f.p.kt0 + i) * kMmaK;
    for (int key = max(k0, f.p.c0 + 1); key < min(k0 + kMmaK, lim); ++key) {
      const int page = f.a.block_table[(size_t)f.p.b * f.a.max_blocks + (key >> sh)];
      if (page >= 0 && page < f.a.n_pages)
        fn(key, reinterpret_cast<const T*>(f.a.v_pages) +
                    (((size_t)page * f.ls.Hk + f.p.h) * f.a.page_size + (key & (f.a.page_size - 1))) * D);
    }
  }
}

// A thread per row: the key tiles of the piece. nt counts the stream's tiles.
template <int DT, int D>
__device__ __forceinline__ void rows_tiles(const Soft& f, uint32_t& nt, float& m, float& l, bool& any) {
  const Piece& p = f.p;
  const bool live = f.warp4 * 32 < f.t.nr;  // of a warp without rows nothing is read
  const int lg = __ffs(f.ls.G) - 1;
  const int lim = p.own ? min(p.c0 + ((f.t.row_at + f.r) >> lg) + 1, p.kend) : p.kend;  // keys this row sees
  for (int i = f.t.first; i < f.t.tiles; i += f.t.step, ++nt) {
    const int k0 = (p.kt0 + i) * kMmaK;
    uint32_t w[4], wr;
    const bool masked = tile_mask(f, k0, w, wr);
    wait_bar(f.s_full, nt & 1, f.dead, f.a.status);
    tc_fence_after();
    if (live) {
      const int n = lim - k0;  // columns seen
      const bool edge = masked || __any_sync(0xffffffffu, n < kMmaK);
      // 32 columns at a time, in loops that stay loops: S is read from TMEM twice, and the code of a tile is
      // a few kilobytes (unrolled over 128 columns it ran from instruction cache misses: measured 3.9 us for
      // a tile of 256 rows)
      auto load = [&](int j, float* s) {
        tmem_ld_x32(f.tS + j * 32, s);
        tmem_wait_ld();
        if (edge) {
          const int c = n - j * 32;
          uint32_t seen = j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3];
          seen &= c >= 32 ? ~0u : c <= 0 ? 0u : (1u << c) - 1u;
#pragma unroll
          for (int e = 0; e < 32; ++e) s[e] = seen >> e & 1u ? s[e] : kNegInf;
        }
      };
      float mx0 = kNegInf, mx1 = kNegInf;
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        float s[32];
        load(j, s);
#pragma unroll
        for (int e = 0; e < 32; e += 4) {
          mx0 = fmaxf(mx0, fmaxf(s[e], s[e + 1]));
          mx1 = fmaxf(mx1, fmaxf(s[e + 2], s[e + 3]));
        }
      }
      const float mt = fmaxf(mx0, mx1) * f.sc;
      if (__any_sync(0xffffffffu, f.r < f.t.nr && mt > m + PRange<DT>::kLazy)) {  // rows of no token hold anything: no vote
        const float mn = fmaxf(m, mt), al = ex2_approx(m - (mn == kNegInf ? 0.f : mn));
        m = mn;
        l *= al;
        if (i > f.t.first) {
#pragma unroll 1
          for (int j = 0; j < D; j += 32) {
            float o[32];
            tmem_ld_x32(f.tO + j, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] *= al;
            tmem_st_x32(f.tO + j, o);
          }
        }
      }
      const float ref = m == kNegInf ? 0.f : m - PRange<DT>::kLift;
      float l0 = 0.f, l1 = 0.f;
#pragma unroll 1
      for (int j = 0; j < 4; ++j) {
        float s[32];
        load(j, s);
        uint32_t pk[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float p0 = ex2_approx(fmaf(s[2 * e], f.sc, -ref));
          const float p1 = ex2_approx(fmaf(s[2 * e + 1], f.sc, -ref));
          l0 += p0;
          l1 += p1;
          pk[e] = pack2<DT>(p0, p1);
        }
        tmem_st_x16(f.tS + j * 16, pk);
      }
      l += l0 + l1;
      tmem_wait_st();
    }
    any = clean_v<DT, D>(f, i, k0, masked, wr, any);
    tc_fence_before();
    __syncwarp();
    if (f.lane == 0) mbar_arrive(f.p_ready);
  }
}

template <int DT, int D>
__device__ __forceinline__ void rows_out(const Soft& f, float m, float l, bool any, float2* ml, float* part) {
  const Piece& p = f.p;
  const int nr = f.t.nr, lg = __ffs(f.ls.G) - 1;
  const int64_t blk = p.row0 + (f.t.mode == kHalf ? f.x * 128 : f.x * f.t.rows);
  if (f.warp4 * 32 < nr) {
    const int lim = p.own ? min(p.c0 + ((f.t.row_at + f.r) >> lg) + 1, p.kend) : p.kend;
#pragma unroll 1
    for (int j = 0; j < D; j += 32) {
      float o[32];
      tmem_ld_x32(f.tO + j, o);
      tmem_wait_ld();
      if (any && f.r < nr)
        hidden_rows<DT, D>(f, lim, [&](int, const typename Elem<DT>::T* v) {
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const float y = Elem<DT>::to_f(v[j + e]);
            if (!isfinite(y)) o[e] += y;
          }
        });
      if (f.r < nr) {
        float4* dst = reinterpret_cast<float4*>(part + (size_t)blk * D) + (size_t)(j / 4) * nr + f.r;
#pragma unroll
        for (int e = 0; e < 8; ++e) dst[(size_t)e * nr] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
      }
    }
  }
  if (f.r < nr) ml[blk + f.r] = make_float2(m - PRange<DT>::kLift, l);
}

// A thread per key: the key tiles of a piece of up to N rows, and its maxima and sums.
template <int DT, int D, int N>
__device__ __forceinline__ bool cols_tiles(const Soft& f, uint32_t& nt, float2* ml) {
  using T = typename Elem<DT>::T;
  using SM = MmaSmem<D>;
  constexpr int NQ = N < 16 ? 16 : N;  // rows of the operands
  const Piece& p = f.p;
  const int nr = f.t.nr, lane = f.lane;
  float* red = reinterpret_cast<float*>(f.smem + SM::red) + f.x * 256;  // [4 warps][64]
  unsigned char* sP = f.smem + f.x * SM::qbuf + SM::pt + (f.r >> 6) * (NQ * 128) + (f.r & 7) * 2;
  const int chunk = (f.r & 63) >> 3;
  // reference maxima: of row `lane`, and of row 32 + lane
  float m0 = kNegInf, m1 = kNegInf, l[N];
#pragma unroll
  for (int n = 0; n < N; ++n) l[n] = 0.f;
  bool any = false;
  for (int i = 0; i < f.t.tiles; ++i, ++nt) {
    const int k0 = (p.kt0 + i) * kMmaK, key = k0 + f.r;
    uint32_t w[4], wr;
    const bool masked = tile_mask(f, k0, w, wr);
    const bool ok = key < p.kend && (wr >> lane & 1u);
    // own key `key` is seen by the rows from (key - c0) G on
    const int from = !ok ? N : p.own ? max(key - p.c0, 0) * f.ls.G : 0;
    wait_bar(f.s_full, nt & 1, f.dead, f.a.status);
    tc_fence_after();
    float s[N];
    tmem_ld_n<N>(f.tS, s);
    float w0 = kNegInf, w1 = kNegInf;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      s[n] = n >= from ? s[n] : kNegInf;
      const float y = redux_max(s[n]);
      if (lane == (n & 31)) (n < 32 ? w0 : w1) = y;
    }
    if (lane < N) red[f.warp4 * 64 + lane] = w0;
    if (N > 32) red[f.warp4 * 64 + 32 + lane] = w1;
    named_sync(1 + f.x, 128);
    // every warp finds the same maxima; the buffer is free again once all have arrived at p_ready
    float t0 = kNegInf, t1 = kNegInf;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (lane < N) t0 = fmaxf(t0, red[j * 64 + lane]);
      if (N > 32) t1 = fmaxf(t1, red[j * 64 + 32 + lane]);
    }
    t0 *= f.sc;
    t1 *= f.sc;
    if (i > 0) {  // the last tile's O += P V: its P^T is written over now, and O may be rescaled
      wait_bar(f.pv_done, (nt - 1) & 1, f.dead, f.a.status);
      tc_fence_after();
    }
    const bool up = (lane < nr && t0 > m0 + PRange<DT>::kLazy) || (N > 32 && 32 + lane < nr && t1 > m1 + PRange<DT>::kLazy);
    if (__any_sync(0xffffffffu, up)) {
      const float n0 = fmaxf(m0, t0), n1 = fmaxf(m1, t1);
      const float a0 = ex2_approx(m0 - (n0 == kNegInf ? 0.f : n0)), a1 = ex2_approx(m1 - (n1 == kNegInf ? 0.f : n1));
      m0 = n0;
      m1 = n1;
#pragma unroll
      for (int n = 0; n < N; ++n) l[n] *= __shfl_sync(0xffffffffu, n < 32 ? a0 : a1, n & 31);
      if (i > 0) {
#pragma unroll
        for (int j = 0; j < N; j += 8) {
          float o[8];
          tmem_ld_x8(f.tO + j, o);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] *= __shfl_sync(0xffffffffu, j < 32 ? a0 : a1, (j + e) & 31);
          tmem_st_x8(f.tO + j, o);
        }
        tmem_wait_st();
      }
    }
    const float r0 = m0 == kNegInf ? 0.f : m0 - PRange<DT>::kLift, r1 = m1 == kNegInf ? 0.f : m1 - PRange<DT>::kLift;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const float pr = ex2_approx(fmaf(s[n], f.sc, -__shfl_sync(0xffffffffu, n < 32 ? r0 : r1, n & 31)));
      l[n] += pr;
      *reinterpret_cast<T*>(sP + n * 128 + ((chunk ^ (n & 7)) << 4)) = Elem<DT>::from_f(pr);
    }
    fence_proxy_async_smem();
    any = clean_v<DT, D>(f, i, k0, masked, wr, any);
    tc_fence_before();
    __syncwarp();
    if (lane == 0) mbar_arrive(f.p_ready);
  }
  // sums over the keys: a warp's, then the four warps' (every warp has read the last tile's maxima)
  float w0 = 0.f, w1 = 0.f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const float y = warp_sum(l[n]);
    if (lane == (n & 31)) (n < 32 ? w0 : w1) = y;
  }
  named_sync(1 + f.x, 128);
  if (lane < N) red[f.warp4 * 64 + lane] = w0;
  if (N > 32) red[f.warp4 * 64 + 32 + lane] = w1;
  named_sync(1 + f.x, 128);
  if (f.r < nr)
    ml[p.row0 + f.r] = make_float2((f.r < 32 ? m0 : m1) - PRange<DT>::kLift, red[f.r] + red[64 + f.r] + red[128 + f.r] + red[192 + f.r]);
  return any;
}

template <int DT, int D, int N>
__device__ __forceinline__ void cols_out(const Soft& f, bool any, float* part) {
  using T = typename Elem<DT>::T;
  const Piece& p = f.p;
  const int nr = f.t.nr;
  if (f.r < D) {  // thread = output column; whole warps
    float o[N];
    tmem_ld_n<N>(f.tO, o);
    if (any)
      hidden_rows<DT, D>(f, p.kend, [&](int key, const T* v) {
        const float y = Elem<DT>::to_f(v[f.r]);
        if (!isfinite(y))
#pragma unroll
          for (int n = 0; n < N; ++n)
            if (n >= (key - p.c0) * f.ls.G) o[n] += y;
      });
    float* dst = part + (size_t)p.row0 * D + (size_t)(f.r >> 2) * nr * 4 + (f.r & 3);
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (n < nr) dst[n * 4] = o[n];
  }
}

template <int DT, int D>
__global__ void __launch_bounds__(kMmaThreads, 1)
    prefix_mma_kernel(PrefixArgs a, LineShape ls, int64_t* hdr, float2* ml, float* part, const __grid_constant__ PrefixMaps maps) {
  using T = typename Elem<DT>::T;
  using SM = MmaSmem<D>;
  constexpr int PL = SM::PL, NB = SM::NB;
  constexpr uint32_t kFmt = DT == HC_BF16 ? 1u : 0u;
  constexpr uint32_t kId = (1u << 4) | (kFmt << 7) | (kFmt << 10) | ((uint32_t)(128 >> 4) << 24);  // fp32 sums, M = 128
  constexpr uint32_t kIdS = kId | ((uint32_t)(kMmaK >> 3) << 17);
  constexpr uint32_t kIdO = kId | (1u << 16) | ((uint32_t)(D >> 3) << 17);  // N = D, B (V) MN-major
  extern __shared__ __align__(1024) unsigned char smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + SM::bars);
  uint64_t *empty = full + NB, *s_full = empty + NB, *p_ready = s_full + 2, *pv_done = p_ready + 2, *q_ready = pv_done + 2;
  uint64_t* fin = q_ready + 2;
  uint32_t* s_tmem = reinterpret_cast<uint32_t*>(smem + SM::misc);
  volatile int* dead = reinterpret_cast<volatile int*>(smem + SM::misc + 4);
  volatile uint32_t* armed = reinterpret_cast<volatile uint32_t*>(smem + SM::misc + 8);  // ring positions armed
  uint64_t* both = fin + 1;
  volatile uint32_t* q_here = armed + 1;  // the first Q rows have arrived
  volatile uint32_t* turns = armed + 5;   // per stream: S tiles of tall row tiles issued
  int* poison = reinterpret_cast<int*>(smem + SM::misc + 16);  // a hidden value was not finite: per stream, and both halves'
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, G = ls.G;
  PieceRing ring{reinterpret_cast<const Piece*>(smem + SM::pieces), reinterpret_cast<uint64_t*>(smem + SM::pbars),
                 reinterpret_cast<uint64_t*>(smem + SM::pbars) + kPieces, 0};

  if (tid == 0) {
    for (int i = 0; i < kPieces; ++i) {
      mbar_init(&ring.full[i], 1);
      mbar_init(&ring.empty[i], 11);  // producer, two issuers, eight softmax warps
    }
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
    mbar_init(both, 8);
    fence_mbar_init();
    *dead = 0;
    *armed = *q_here = 0;
    poison[0] = poison[1] = poison[2] = 0;
    turns[0] = turns[1] = 0;
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
  const Stretch st = line_setup<kMmaThreads>(a, ls, g, blockIdx.x, hdr, reinterpret_cast<int64_t*>(smem + SM::red));
  __syncthreads();  // the setup's buffer is used anew

  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0) {
      // ---- producer --------------------------------------------------------------------
      const int sh = __ffs(a.page_size) - 1;
      const int bx = min(a.page_size, kMmaK), nbx = kMmaK / bx;
      const int y_out = a.n_pages * ls.Hk * a.page_size;  // out of range: reads as zeros
      uint32_t n = 0;
      Piece p;
      while (ring.next(p, 0xffffffffu, lane == 0)) {
        for (int kt = p.kt0; kt < p.kt1; ++kt) {
          if (__any_sync(0xffffffffu, *dead)) break;
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
            // the first Q rows do not queue behind a ring full of tiles
            if (n == 2)
              for (int i = 0; !*q_here && !*dead && i < kMaxPolls; ++i) __nanosleep(20);
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
      // ---- MMA issue of stream x: the warp walks together, one thread issues ----------------
      const int x = warp - 1;
      const bool leader = elect_one();
      const uint32_t tS = tbase + x * 128, tO = tbase + 256 + x * 128;
      // low words of the operands' descriptors (address / 16), stepped by adding
      const uint32_t dq = smem_u32(smem + x * SM::qbuf) >> 4, dr = smem_u32(smem + SM::ring) >> 4;
      uint32_t base = 0, np = 0, nt = 0, turn = 0, tall = 0;  // ring position; pieces, tiles, tall tiles of this stream
      Piece p;
      while (ring.next(p, 0xffffffffu, lane == 0)) {
        const Part t = piece_part(p, G, x, turn);
        if (t.rows <= 64) ++turn;
        if (t.mode != kSkip) {
          const bool tr = t.mode == kTransposed, half = t.mode == kHalf;
          const uint32_t nq = t_cols(t.nr), idt = kId | ((nq >> 3) << 17);
          wait_bar(&q_ready[x], np & 1, dead, a.status);
          ++np;
          for (int i = t.first; i < t.tiles; i += t.step, ++nt) {
            const uint32_t nk = base + 2 * i, nv = nk + 1, bk = nk % NB, bv = nv % NB;
            const uint32_t dk = dr + bk * (SM::tile >> 4), dv = dr + bv * (SM::tile >> 4);
            wait_full<NB>(full, nk, armed, dead, a.status);
            // P of the last tile, in the columns of S, has been read; transposed, the scores of the last tile were
            // in registers once P^T was ready
            if (!tr && i > t.first) wait_bar(&pv_done[x], (nt - 1) & 1, dead, a.status);
            if (half && i == 0) wait_turn(turns, x, tall, dead);
            tc_fence_after();
            if (leader) {
              if (tr) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                  umma_f16(tS, desc_k(dk + (ks >> 2) * 1024 + (ks & 3) * 2), desc_k(dq + (ks >> 2) * nq * 8 + (ks & 3) * 2), idt,
                           ks > 0);
              } else {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks)
                  umma_f16(tS, desc_k(dq + (ks >> 2) * 1024 + (ks & 3) * 2), desc_k(dk + (ks >> 2) * 1024 + (ks & 3) * 2), kIdS,
                           ks > 0);
              }
              umma_commit(&s_full[x]);
              if (half) turns[x] = tall + 1;
              umma_commit(&empty[bk]);
              if (!half) umma_commit(&empty[bk]);  // the tile is this stream's alone
            }
            if (half) ++tall;
            wait_full<NB>(full, nv, armed, dead, a.status);
            wait_bar(&p_ready[x], nt & 1, dead, a.status);
            // The two halves of a tall row tile take turns, [O += P V, next S] each: mixed with one another
            // they would finish together, and then both softmaxes run while the tensor cores wait.
            if (half && i + 1 < t.tiles) wait_turn(turns, x, tall, dead);
            tc_fence_after();
            if (leader) {
              const uint32_t more = i > t.first;
              if (tr) {
                // A = V^T from its MN-major rows. M is 128: for D = 64 the same plane serves as both halves
                // (a plane stride of 0) and the lower half of the result is not read
                const uint32_t dp = dq + (SM::pt >> 4);
#pragma unroll
                for (int ks = 0; ks < kMmaK / 16; ++ks)
                  umma_f16(tO, desc_mn(dv + ks * 128, D == 128 ? 1024 : 0), desc_k(dp + (ks >> 2) * nq * 8 + (ks & 3) * 2),
                           idt | (1u << 15), more | (ks > 0));
              } else {
#pragma unroll
                for (int ks = 0; ks < kMmaK / 16; ++ks)
                  umma_f16_ts(tO, tS + ks * 8, desc_mn(dv + ks * 128, 1024), kIdO, more | (ks > 0));
              }
              umma_commit(&pv_done[x]);
              umma_commit(&empty[bv]);
              if (!half) umma_commit(&empty[bv]);
            }
            __syncwarp();
          }
        }
        base += 2 * t.tiles;
      }
      if (leader) umma_commit(fin);
    } else if (lane == 0) {
      // ---- lists the pieces --------------------------------------------------------------
      LineWalk walk(a, ls, g, st, blockIdx.x);
      Piece* out = reinterpret_cast<Piece*>(smem + SM::pieces);
      Piece p{};
      bool more = true;
      for (uint32_t k = 0; more; ++k) {
        more = walk.next(a, ls, g, p);
        if (!more) p.kt0 = p.kt1 = 0;  // the end
        mbar_wait_long(&ring.empty[k % kPieces], ((k / kPieces) & 1) ^ 1);
        out[k % kPieces] = p;
        mbar_arrive(&ring.full[k % kPieces]);
      }
    }
    __syncwarp();
  } else {
    // ---- softmax of stream x ---------------------------------------------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int x = (warp >> 2) - 1, r = tid & 127, warp4 = warp & 3, lg = __ffs(G) - 1;
    const uint32_t quarter = (uint32_t)(warp4 * 32) << 16;
    unsigned char* sQ = smem + x * SM::qbuf;
    uint32_t base = 0, next_base = 0, nt = 0, turn = 0, meets = 0;
    Piece p, q;
    Part tq;
    // The next piece of this stream; `base` goes along. A stream that still has work on its piece may not
    // wait here: it can have many pieces to pass by, which are listed only as the others get on, and those may
    // need this stream's work (its share of the ring, the meetings). So it looks ahead as far as pieces are
    // listed, and waits only once it is done.
    enum { kNone = 0, kHave, kEnd };  // not listed yet; found; no more
    auto advance = [&](bool wait) -> int {
      while (wait || ring.listed()) {
        if (!ring.next(q, 0xffffffffu, lane == 0)) return kEnd;
        tq = piece_part(q, G, x, turn);
        base = next_base;
        next_base += 2 * tq.tiles;
        if (tq.rows <= 64) ++turn;
        if (tq.mode != kSkip) return kHave;
        // too few key tiles for this stream: its block of partial rows holds nothing
        if (prefix_two_streams(tq.rows) && r < tq.rows) ml[q.row0 + tq.rows + r] = make_float2(kNegInf, 0.f);
      }
      return kNone;
    };
    // its Q rows: a thread takes one 16-byte column of every RS-th row (a whole number of tokens apart, since
    // the group divides RS), all loads in flight, then into the swizzled K-major layout
    constexpr int CPR = D / 8, RS = 128 / CPR, QB = 128 / RS;
    const int qc = r % CPR, qr = r / CPR;
    auto load_q = [&](uint4* u) {
      const int row = tq.row_at + qr;
      const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(q.tok0 + (row >> lg)) * a.q_st +
                     (int64_t)(q.h * G + (row & (G - 1))) * a.q_sh + qc * 8;
      const int64_t step = (int64_t)(RS >> lg) * a.q_st;
#pragma unroll
      for (int j = 0; j < QB; ++j) {
        u[j] = qr + j * RS < tq.nr ? *reinterpret_cast<const uint4*>(src) : make_uint4(0u, 0u, 0u, 0u);
        src += step;
      }
    };
    auto store_q = [&](const uint4* u) {
      const uint32_t plane = tq.mode == kTransposed ? t_cols(tq.nr) * 128u : 16384u;
      unsigned char* dst = sQ + (qc >> 3) * plane + qr * 128 + (((qc & 7) ^ (qr & 7)) << 4);
#pragma unroll
      for (int j = 0; j < QB; ++j)
        if (qr + j * RS < tq.nr) *reinterpret_cast<uint4*>(dst + j * RS * 128) = u[j];
      fence_proxy_async_smem();
    };
    auto q_arrive = [&]() {
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_ready[x]);
    };
    int got = advance(true);
    if (got == kHave) {
      uint4 u[QB];
      load_q(u);
      store_q(u);
      if (r == 0) *q_here = 1;
      q_arrive();
    }
    while (got == kHave) {
      p = q;
      const Part t = tq;
      const Soft f{a, ls, p, t, smem, full, &s_full[x], &p_ready[x], &pv_done[x], both, armed, dead,
                   &poison[t.mode == kHalf ? 2 : x], a.scale * 1.4426950408889634f, base, x, r, lane, warp4,
                   tbase + x * 128 + quarter, tbase + 256 + x * 128 + quarter, meets};
      // The next piece's Q is loaded and its first MMAs begin while this one's result is written: all MMAs
      // that read Q, P or S have ended, and O is only overwritten after the next p_ready.
      float m = kNegInf, l = 0.f;
      bool any = false;
      const bool tr = t.mode == kTransposed;
      // its Q rows are under way during this one's tiles, where a thread has registers for them
      uint4 u[QB];
      auto fetch = [&](bool wait) {
        got = advance(wait);
        if (got == kHave) load_q(u);
      };
      if (!tr) {
        rows_tiles<DT, D>(f, nt, m, l, any);
        fetch(false);
      } else if (t.nr <= 8) {
        fetch(false);
        any = cols_tiles<DT, D, 8>(f, nt, ml);
      } else if (t.nr <= 16) {
        fetch(false);
        any = cols_tiles<DT, D, 16>(f, nt, ml);
      } else if (t.nr <= 32) {
        fetch(false);
        any = cols_tiles<DT, D, 32>(f, nt, ml);
      } else {
        any = cols_tiles<DT, D, 64>(f, nt, ml);
        fetch(false);
      }
      wait_bar(&pv_done[x], (nt - 1) & 1, dead, a.status);
      tc_fence_after();
      if (got == kHave) {
        store_q(u);
        q_arrive();
      }
      if (!tr) rows_out<DT, D>(f, m, l, any, ml, part);
      else if (t.nr <= 8) cols_out<DT, D, 8>(f, any, part);
      else if (t.nr <= 16) cols_out<DT, D, 16>(f, any, part);
      else if (t.nr <= 32) cols_out<DT, D, 32>(f, any, part);
      else cols_out<DT, D, 64>(f, any, part);
      tc_fence_before();
      if (p.own && p.c0 + 1 < p.kend) {  // the flag is cleared once every thread has read it
        if (t.mode == kHalf) f.meet();
        else named_sync(1 + x, 128);
        if (r == 0) *f.poison = 0;
        if (t.mode == kHalf) f.meet();
        else named_sync(1 + x, 128);
      }
      if (got == kNone) {
        fetch(true);
        if (got == kHave) {
          store_q(u);
          q_arrive();
        }
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
