// Attention of a batch over [shared prefix | the sequence's own pages]:
//   o_t = sum_j softmax_j(scale q_t . k_j) v_j,  j over the unmasked prefix keys and own keys j <= len_b - n_b + i
// (t the i-th of sequence b's n_b new tokens). The division of the work is in hc_prefix.cuh.
//
// 16-bit types run on the tensor cores (hc_prefix_mma.cu). prefix_simt_kernel serves fp32 layers: 64 rows x
// 64 keys with fp32 FMAs; scores and probabilities pass through shared memory, the output stays in
// registers. A call is divided among two CTAs an SM: at D = 64 two fit, at D = 128 (114 KB of shared memory and 1 KB
// of the system's each, of 228) one does, and the stretches run as two waves. One B200, 8 sequences over 4k keys, 8/2
// heads of 128, replayed from a graph: one new token each 39 us, 8 each 79 us, 64 each 349 us. prefix_merge_kernel
// joins the partial results of both.

#include "hc_prefix.cuh"

namespace hc {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

constexpr int kSimtThreads = 256, kSimtR = 64, kSimtK = 64;

template <int D>
struct SimtSmem {
  static constexpr int KS = D + 4;  // padded key row: 16 rows' float4 reads hit distinct banks
  static constexpr size_t q = 0;
  static constexpr size_t k = q + sizeof(float) * kSimtR * D;
  static constexpr size_t v = k + sizeof(float) * kSimtK * KS;
  static constexpr size_t s = v + sizeof(float) * kSimtK * D;
  static constexpr size_t al = s + sizeof(float) * kSimtR * (kSimtK + 4);
  static constexpr size_t hd = al + sizeof(float) * kSimtR;
  static constexpr size_t bytes = hd + sizeof(int64_t) * (kSimtThreads / 32 + 4);
};

template <int D>
__global__ void __launch_bounds__(kSimtThreads, 2) prefix_simt_kernel(PrefixArgs a, LineShape ls, int64_t* hdr, float2* ml,
                                                                      float* part) {
  constexpr int DT = HC_F32;
  using E = Elem<DT>;
  using T = typename E::T;
  using SM = SimtSmem<D>;
  constexpr int VEC = 16 / sizeof(T), CPR = D / VEC, KS = SM::KS, PS = kSimtK + 4, NC = D / 64;
  extern __shared__ __align__(16) unsigned char smem[];
  float* sQ = reinterpret_cast<float*>(smem + SM::q);
  float* sK = reinterpret_cast<float*>(smem + SM::k);
  float* sV = reinterpret_cast<float*>(smem + SM::v);
  float* sS = reinterpret_cast<float*>(smem + SM::s);
  float* sAl = reinterpret_cast<float*>(smem + SM::al);
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4, G = ls.G;
  pdl_wait();
  const LineGeom g(ls, min(a.T, max(a.cu_new[ls.n_seq], 0)));
  LineWalk walk(a, ls, g, line_setup<kSimtThreads>(a, ls, g, blockIdx.x, hdr, reinterpret_cast<int64_t*>(smem + SM::hd)),
                blockIdx.x);
  const int sh = __ffs(a.page_size) - 1;
  const float sc = a.scale * kLog2e;
  Piece p;
  while (walk.next(a, ls, g, p)) {
    const int rows = p.ntok * G;
    __syncthreads();
    for (int x = tid; x < kSimtR * CPR; x += kSimtThreads) {
      const int r = x / CPR, c = x % CPR;
      float f[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) f[e] = 0.f;
      if (r < rows) {
        const T* src = reinterpret_cast<const T*>(a.q) + (int64_t)(p.tok0 + r / G) * a.q_st + (int64_t)(p.h * G + r % G) * a.q_sh;
        unpack16<DT>(reinterpret_cast<const uint4*>(src)[c], f);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) sQ[r * D + c * VEC + e] = f[e];
    }
    float o[4][4 * NC];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4 * NC; ++j) o[i][j] = 0.f;
    float m = kNegInf, l = 0.f;  // of row tid / 4, in units of log2
    for (int kt = p.kt0; kt < p.kt1; ++kt) {
      const int k0 = kt * kSimtK;
      bool odd = false;  // a value that is not finite
      __syncthreads();
      // a thread takes one 16-byte column of every 8th (16th) row; four rows' loads in flight at a time
      constexpr int RS = kSimtThreads / CPR, LB = 4;
#pragma unroll
      for (int r0 = 0; r0 < kSimtK; r0 += RS * LB) {
        uint4 uk[LB], uv[LB];
#pragma unroll
        for (int u = 0; u < LB; ++u) {
          const int key = k0 + r0 + u * RS + tid / CPR, c = tid % CPR;
          const T *kr = nullptr, *vr = nullptr;
          if (key < p.kend) {
            if (p.own) {
              const int page = a.block_table[(size_t)p.b * a.max_blocks + (key >> sh)];
              if (page >= 0 && page < a.n_pages) {
                const size_t off = (((size_t)page * ls.Hk + p.h) * a.page_size + (key & (a.page_size - 1))) * D;
                kr = reinterpret_cast<const T*>(a.k_pages) + off;
                vr = reinterpret_cast<const T*>(a.v_pages) + off;
              } else if (a.status) {
                atomicOr(a.status, HC_DEV_INDEX);
              }
            } else if (!a.mask || a.mask[key]) {
              kr = reinterpret_cast<const T*>(a.pk) + p.h * a.pk_sh + (int64_t)key * a.pk_st;
              vr = reinterpret_cast<const T*>(a.pv) + p.h * a.pv_sh + (int64_t)key * a.pv_st;
            }
          }
          uk[u] = kr ? reinterpret_cast<const uint4*>(kr)[c] : make_uint4(0u, 0u, 0u, 0u);
          uv[u] = vr ? reinterpret_cast<const uint4*>(vr)[c] : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int u = 0; u < LB; ++u) {
          const int r = r0 + u * RS + tid / CPR, c = tid % CPR;
          *reinterpret_cast<uint4*>(sK + r * KS + c * VEC) = uk[u];
          *reinterpret_cast<uint4*>(sV + r * D + c * VEC) = uv[u];
          float f[VEC];
          unpack16<DT>(uv[u], f);
#pragma unroll
          for (int e = 0; e < VEC; ++e) odd |= !isfinite(f[e]);
        }
      }
      // a causal tile whose hidden keys hold values that are not finite takes the careful product
      const bool causal = p.own && k0 + kSimtK > p.c0 + 1;
      const bool careful = __syncthreads_or(odd && causal);
      float acc[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        float4 x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(sQ + (ty * 4 + i) * D + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = *reinterpret_cast<const float4*>(sK + (tx + 16 * j) * KS + d);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            acc[i][j] = fmaf(x[i].x, y[j].x, fmaf(x[i].y, y[j].y, fmaf(x[i].z, y[j].z, fmaf(x[i].w, y[j].w, acc[i][j]))));
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = k0 + tx + 16 * j;
        const bool seen = key < p.kend && (p.own || !a.mask || a.mask[key]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = ty * 4 + i;
          const bool hid = p.own && key > p.c0 + r / G;
          sS[r * PS + tx + 16 * j] = seen && !hid ? acc[i][j] * sc : kNegInf;
        }
      }
      __syncthreads();
      {  // four threads a row, 16 keys each
        const int r = tid >> 2, part4 = tid & 3;
        float* row = sS + r * PS + part4 * 4;
        float x[16], mx = kNegInf;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            x[j * 4 + e] = row[j * 16 + e];
            mx = fmaxf(mx, x[j * 4 + e]);
          }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m, mx), ref = mn == kNegInf ? 0.f : mn;
        const float al = ex2(m - ref);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float pr = ex2(x[j * 4 + e] - ref);
            row[j * 16 + e] = pr;
            sum += pr;
          }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        l = l * al + sum;
        m = mn;
        if (part4 == 0) sAl[r] = al;
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float al = sAl[ty * 4 + i];
#pragma unroll
        for (int j = 0; j < 4 * NC; ++j) o[i][j] *= al;
      }
      if (!careful) {
#pragma unroll 2
        for (int k = 0; k < kSimtK; k += 4) {
          float4 x[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4*>(sS + (ty * 4 + i) * PS + k);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
#pragma unroll
            for (int n = 0; n < NC; ++n) {
              const float4 y = *reinterpret_cast<const float4*>(sV + (k + kk) * D + n * 64 + tx * 4);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float pr = kk == 0 ? x[i].x : kk == 1 ? x[i].y : kk == 2 ? x[i].z : x[i].w;
                o[i][n * 4] = fmaf(pr, y.x, o[i][n * 4]);
                o[i][n * 4 + 1] = fmaf(pr, y.y, o[i][n * 4 + 1]);
                o[i][n * 4 + 2] = fmaf(pr, y.z, o[i][n * 4 + 2]);
                o[i][n * 4 + 3] = fmaf(pr, y.w, o[i][n * 4 + 3]);
              }
            }
        }
      } else {
        for (int k = 0; k < kSimtK; ++k)
          for (int i = 0; i < 4; ++i) {
            const int r = ty * 4 + i;
            if (k0 + k > p.c0 + r / G) continue;  // hidden from this row: its value is not read
            const float pr = sS[r * PS + k];
            for (int n = 0; n < NC; ++n)
              for (int e = 0; e < 4; ++e) o[i][n * 4 + e] = fmaf(pr, sV[k * D + n * 64 + tx * 4 + e], o[i][n * 4 + e]);
          }
      }
    }
    if ((tid & 3) == 0 && (tid >> 2) < rows) ml[p.row0 + (tid >> 2)] = make_float2(m, l);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = ty * 4 + i;
      if (r < rows)
#pragma unroll
        for (int n = 0; n < NC; ++n)
          *reinterpret_cast<float4*>(part + (size_t)p.row0 * D + ((size_t)(n * 16 + tx) * rows + r) * 4) =
              make_float4(o[i][n * 4], o[i][n * 4 + 1], o[i][n * 4 + 2], o[i][n * 4 + 3]);
    }
  }
}

// ----------------------------------------------------------------------------------------
// Joins the partial results of the G rows of (token, KV head): out = sum_p w_p O_p / sum_p w_p l_p with
// w_p = 2^(m_p - max m). A CTA lists the pieces that cover the rows, a warp per row works out the weights,
// then a thread takes 16-byte columns of a row, neighbours the group's rows (they lie next to each other).
// A row with no attended key at all is 0 with a log-sum of -inf. Bound by the partial results it reads
// (from L2) and, for a decode step, by its launch and three dependent reads.
// ----------------------------------------------------------------------------------------
constexpr int kMaxCtas = 448;     // CTAs a call's work is divided among
constexpr int kMergeList = 512;   // >= partial results of a row: one per CTA and one more per group of the row (17)

template <int DT, int D, int kMergeThreads>
__global__ void __launch_bounds__(kMergeThreads) prefix_merge_kernel(PrefixArgs a, LineShape s, const int64_t* hdr,
                                                                     const float2* ml, const float* part) {
  using E = Elem<DT>;
  using T = typename E::T;
  __shared__ int64_t list[kMergeList];
  __shared__ float wts[kMergeList * 8];
  __shared__ float4 sum[kMergeThreads];
  __shared__ float s_ml[8];
  __shared__ int s_b, s_geo[4], s_lo[17], s_at[18], s_sec[17];
  __shared__ int64_t s_row[17];
  const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) s_b = -1;
  pdl_wait();
  const int64_t W = hdr[0];
  const int R = min(a.T, max(a.cu_new[s.n_seq], 0));
  __syncthreads();
  for (int b = tid; b < s.n_seq; b += kMergeThreads)
    if (a.cu_new[b] <= t && t < a.cu_new[b + 1]) s_b = b;
  if (t >= R) return;  // rows behind the last sequence are left as they were ...
  const LineGeom g(s, R);
  __syncthreads();
  if (s_b < 0) return;  // ... and so are rows before the first
  // the blocks of partial rows over these rows, in a fixed order: segment j < nch the prefix chunk j, segment
  // nch the own pages; where a CTA ran two streams over the keys, both of its blocks
  if (warp == 0) {
    int64_t row = 0;
    int lo = 0, hi = -1, rows = 0, q0 = 0;
    if (lane < s.nch && g.ktp > 0) {
      const int i = t / g.tt, tok0 = i * g.tt;
      const int tiles = min(g.ct, g.ktp - lane * g.ct);
      const int64_t v0 = h * g.head + (int64_t)lane * g.nrt * (g.ct * g.pre.a + g.pre.b) +
                         (int64_t)i * (tiles * g.pre.a + g.pre.b) + g.pre.b;
      rows = min(g.tt, R - tok0) * s.G, q0 = (t - tok0) * s.G;
      lo = line_div(v0, W), hi = line_div(v0 + (int64_t)(tiles - 1) * g.pre.a, W);
      row = s.dup * (((int64_t)h * s.nch + lane) * s.T + tok0) * s.G;
    } else if (lane == s.nch) {
      const SeqLens q = seq_lens(a, s_b);
      const int r = (t - q.cu) / g.tt, nr = ceil_div(q.n, g.tt), tok1 = min(q.n, (r + 1) * g.tt);
      const int tiles = ceil_div(seq_keys(q, tok1), s.kt);
      rows = (tok1 - r * g.tt) * s.G, q0 = (t - q.cu - r * g.tt) * s.G;
      if (tiles > 0) {
        const LineCost k = line_cost(s, min(q.n * s.G, s.rt), true);
        const int64_t v0 = hdr[1 + s_b] + ((int64_t)h * nr + r) * g.seq_group(s, q) + k.b;
        lo = line_div(v0, W), hi = line_div(v0 + (int64_t)(tiles - 1) * k.a, W);
        row = s.dup * ((int64_t)s.Hk * s.T * (s.P > 0 ? s.nch : 0) + (int64_t)q.cu * s.Hk + (int64_t)h * q.n + r * g.tt) * s.G;
      }
    }
    // a row tile above 128 rows is two blocks; of a smaller one's two streams each has a block of its own
    const bool halves = s.dup == 2 && rows > 128, second = s.dup == 2 && prefix_two_streams(rows);
    const int blk = halves && q0 >= 128 ? 128 : 0, n_blk = halves ? min(128, rows - blk) : rows;
    const int mine = (hi - lo + 1) * (second ? 2 : 1);
    int at = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += y;
    }
    if (lane <= s.nch) {
      s_lo[lane] = lo;
      s_row[lane] = row + blk;
      s_sec[lane] = second ? rows : 0;
      s_at[lane + 1] = min(at, kMergeList);
    }
    if (lane == 0 || lane == s.nch) {  // rows of a block, and the first of these rows in it: prefix, own pages
      s_geo[lane ? 2 : 0] = n_blk;
      s_geo[lane ? 3 : 1] = q0 - blk;
    }
    if (lane == 0) s_at[0] = 0;
  }
  __syncthreads();
  const int np = s_at[s.nch], n = s_at[s.nch + 1];
  for (int gq = warp; gq < s.G; gq += kMergeThreads / 32) {
    // a lane's first block stays in registers; the maximum needs the others once more
    float M = kNegInf, L = 0.f;
    float2 z0 = make_float2(kNegInf, 0.f);
    auto load = [&](int x) {
      int j = 0;
      while (x >= s_at[j + 1]) ++j;
      const int i = x - s_at[j], sec = s_sec[j];
      const int64_t base = s_row[j] + (int64_t)(s_lo[j] + (sec ? i >> 1 : i)) * s.rt + (sec && (i & 1) ? sec : 0);
      if (gq == 0) list[x] = base;
      return __ldcg(&ml[base + (j < s.nch ? s_geo[1] : s_geo[3]) + gq]);
    };
    if (lane < n) z0 = load(lane);
    M = z0.x;
    for (int x = lane + 32; x < n; x += 32) M = fmaxf(M, load(x).x);
    M = warp_max(M);
    const float ref = M == kNegInf ? 0.f : M;
    for (int x = lane; x < n; x += 32) {
      const float2 z = x < 32 ? z0 : load(x);
      const float w = ex2(z.x - ref);
      wts[x * s.G + gq] = w;
      L = fmaf(w, z.y, L);
    }
    L = warp_sum(L);
    if (lane == 0) {
      s_ml[gq] = L;
      if (a.lse) a.lse[(size_t)t * a.Hq + (size_t)h * s.G + gq] = L == 0.f ? kNegInf : (M + log2f(L)) * kLn2;
    }
  }
  __syncthreads();
  // columns of 16 bytes x rows, and where there are fewer of them than threads the blocks in as many shares
  const int items = s.G * (D / 4), shares = items < kMergeThreads ? kMergeThreads / items : 1;
  for (int k0 = 0; k0 < items; k0 += kMergeThreads) {
    const int k = k0 + tid % items, share = tid / items;
    const int gq = k & (s.G - 1), c4 = k / s.G;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const size_t off_p = ((size_t)c4 * s_geo[0] + s_geo[1] + gq) * 4, off_s = ((size_t)c4 * s_geo[2] + s_geo[3] + gq) * 4;
    for (int x0 = share; x0 < n; x0 += 8 * shares) {
      float4 y[8];
      float w[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int x = x0 + u * shares;
        w[u] = x < n ? wts[x * s.G + gq] : 0.f;
        // a block without a key may not have been written
        y[u] = w[u] != 0.f ? __ldcg(reinterpret_cast<const float4*>(part + (size_t)list[x] * D + (x < np ? off_p : off_s)))
                           : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        o.x = fmaf(w[u], y[u].x, o.x);
        o.y = fmaf(w[u], y[u].y, o.y);
        o.z = fmaf(w[u], y[u].z, o.z);
        o.w = fmaf(w[u], y[u].w, o.w);
      }
    }
    if (shares > 1) {
      sum[tid] = o;
      __syncthreads();
      if (share > 0) break;
      for (int z = 1; z < shares; ++z) {
        const float4 y = sum[z * items + k];
        o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
      }
    }
    const float L = s_ml[gq], inv = L == 0.f ? 0.f : 1.f / L;
    alignas(16) T r[4];
    r[0] = E::from_f(L == 0.f ? 0.f : o.x * inv);
    r[1] = E::from_f(L == 0.f ? 0.f : o.y * inv);
    r[2] = E::from_f(L == 0.f ? 0.f : o.z * inv);
    r[3] = E::from_f(L == 0.f ? 0.f : o.w * inv);
    T* dst = reinterpret_cast<T*>(a.out) + ((size_t)t * a.Hq + (size_t)h * s.G + gq) * D + c4 * 4;
    if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<uint4*>(r);
    else *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<uint2*>(r);
  }
}

// ----------------------------------------------------------------------------------------
// host
// ----------------------------------------------------------------------------------------
static int sm_count() {
  static int n[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  int& x = n[dev & 63];
  if (!x && (cudaDeviceGetAttribute(&x, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || x <= 0)) {
    (void)cudaGetLastError();
    return 148;
  }
  return x;
}

static LineShape prefix_shape(int dtype, int T, int n_seq, int Hq, int Hk, int P) {
  const int sms = sm_count() < kMaxCtas / 2 ? sm_count() : kMaxCtas / 2;
  if (dtype != HC_F32) return prefix_mma_shape(T, n_seq, Hk, Hq / Hk, P, sms);
  return line_shape(T, n_seq, Hk, Hq / Hk, P, kSimtR, kSimtK, 2 * sms, 1);
}

static size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

size_t prefix_scratch_bytes(int dtype, int T, int n_seq, int Hq, int Hk, int D, int P) {
  const LineShape s = prefix_shape(dtype, T, n_seq, Hq, Hk, P);
  const size_t rows = line_rows(s);
  return up256(sizeof(int64_t) * (n_seq + 1)) + up256(rows * sizeof(float2)) + rows * D * sizeof(float);
}

template <int DT, int D>
static cudaError_t prefix_t(const PrefixArgs& a, void* scratch, cudaStream_t stream) {
  const LineShape s = prefix_shape(DT, a.T, a.n_seq, a.Hq, a.Hk, a.P);
  char* p = static_cast<char*>(scratch);
  int64_t* hdr = reinterpret_cast<int64_t*>(p);
  p += up256(sizeof(int64_t) * (a.n_seq + 1));
  float2* ml = reinterpret_cast<float2*>(p);
  p += up256(line_rows(s) * sizeof(float2));
  float* part = reinterpret_cast<float*>(p);
  cudaError_t e;
  if constexpr (DT == HC_F32) {
    auto kern = prefix_simt_kernel<D>;
    const size_t smem = SimtSmem<D>::bytes;
    e = ensure_smem(kern, smem);
    if (e == cudaSuccess) e = launch_pdl(kern, dim3((unsigned)s.nc), dim3(kSimtThreads), smem, stream, a, s, hdr, ml, part);
  } else {
    e = launch_prefix_mma(a, s, DT, D, hdr, ml, part, stream);
  }
  if (e != cudaSuccess) return e;
  // few rows have many blocks each: wide CTAs take shares of them (8 rows of 68 blocks: 21 us with 256 threads);
  // many rows have few, and fill the GPU by themselves
  const bool wide = (int64_t)a.T * a.Hk < 2048;
  return launch_pdl(wide ? prefix_merge_kernel<DT, D, 512> : prefix_merge_kernel<DT, D, 128>,
                    dim3((unsigned)a.T, (unsigned)a.Hk), dim3(wide ? 512 : 128), 0, stream, a, s, (const int64_t*)hdr,
                    (const float2*)ml, (const float*)part);
}

cudaError_t launch_prefix_attention(const PrefixArgs& a, int dtype, int D, void* scratch, cudaStream_t stream) {
  HC_DISPATCH_DT_D(dtype, D, prefix_t, a, scratch, stream);
}

}  // namespace hc
