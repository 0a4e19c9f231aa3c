// Paged storage of a batch's own tokens (the part of each sequence behind a shared prefix): block
// tables and slot maps built from request lengths, their release, and the rotary append into pages.
//
// Tables. Sequence b holds len_b tokens in ceil(len_b / ps) pages of ps tokens, block_table[b][j] the
// page of its tokens [j ps, (j + 1) ps). The free pages are a stack; the step's fresh pages come off
// its top in the order of (sequence, block):
//   need_b = ceil((len_b + new_b) / ps) - ceil(len_b / ps),   first_b = sum of need_a over a < b
//   block_table[b][have_b + i] = free[n_free - 1 - first_b - i],  i < need_b
//   token t of sequence b (cu_b <= t < cu_{b+1}) sits at p = len_b + t - cu_b, slot = page * ps + p % ps
// It is bound by latency (a launch, two dependent loads, one block scan): 12 bytes a sequence and 20 a
// token. Every CTA scans the lengths of all sequences for itself (at most 4096, 8 a thread), so the tokens
// spread over CTAs without a second launch. lens and n_free may be updated in place, which has to come
// after every CTA has read them: up to 8 CTAs are a cluster and meet before the first one does it; the
// slot maps of whole prompts take as many CTAs as they fill, and a second launch of one CTA commits.

#include "hc_internal.cuh"

namespace hc {

constexpr int kPlanThreads = 512;
constexpr int kPlanMaxSeq = 4096;
constexpr int kPlanPer = kPlanMaxSeq / kPlanThreads;  // sequences per thread

// The largest b with s[b] <= x in s[0..n), s[0] = 0 <= x, s ascending.
__device__ __forceinline__ int last_not_above(const int* s, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (s[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// Exclusive sums over the block of two counts per thread, and their totals. 64 bits: the totals of refused
// lengths are looked at too. `sh` takes 2 * kPlanThreads / 32 values. (64-bit atomics on one shared word
// took 15 us for 256 threads.)
__device__ __forceinline__ void scan_pair(int64_t x, int64_t y, int64_t* sh, int64_t& bx, int64_t& by, int64_t& tx, int64_t& ty) {
  constexpr int NW = kPlanThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  bx = x;
  by = y;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t p = __shfl_up_sync(0xffffffffu, bx, o), q = __shfl_up_sync(0xffffffffu, by, o);
    if (lane >= o) bx += p, by += q;
  }
  if (lane == 31) sh[warp] = bx, sh[NW + warp] = by;
  __syncthreads();
  bx -= x;
  by -= y;
  tx = ty = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if (w == warp) bx += tx, by += ty;
    tx += sh[w];
    ty += sh[NW + w];
  }
}

__device__ __forceinline__ void cluster_sync_all() {
  __syncthreads();
  cluster_arrive();
  cluster_wait();
}

__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(PagePlanArgs a) {
  __shared__ int s_cu[kPlanMaxSeq], s_first[kPlanMaxSeq];
  __shared__ int64_t s_scan[2 * kPlanThreads / 32];
  pdl_wait();
  const int tid = threadIdx.x, rank = blockIdx.x, nct = gridDim.x;
  const int sh = __ffs(a.page_size) - 1, pm = a.page_size - 1;
  const long long cap = (long long)a.max_blocks << sh;
  const int n_free = *a.n_free;
  const int per = (a.n_seq + kPlanThreads - 1) / kPlanThreads;
  int len[kPlanPer], add[kPlanPer];
  int bits = (n_free < 0 || n_free > a.n_pages) ? HC_DEV_INDEX : 0;
  long long nn = 0, np = 0;
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) {
    const int b = tid * per + i;
    if (i >= per || b >= a.n_seq) continue;
    len[i] = a.lens[b];
    add[i] = a.new_lens[b];
    if (len[i] < 0 || add[i] < 0 || len[i] > cap) bits |= HC_DEV_INDEX;
    else if (len[i] + (long long)add[i] > cap) bits |= HC_DEV_CAPACITY;
    else {
      nn += add[i];
      np += (int)(((long long)len[i] + add[i] + pm) >> sh) - (int)(((long long)len[i] + pm) >> sh);
    }
  }
  int64_t cu0, first0, all_new, all_fresh;
  scan_pair(nn, np, s_scan, cu0, first0, all_new, all_fresh);
  const int bad_index = __syncthreads_or(bits & HC_DEV_INDEX), bad_cap = __syncthreads_or(bits & HC_DEV_CAPACITY);
  bits = (bad_index ? HC_DEV_INDEX : 0) | (bad_cap || all_new > a.n_tokens || all_fresh > n_free ? HC_DEV_CAPACITY : 0);
  const bool ok = bits == 0;
  const int total = ok ? (int)all_new : 0, fresh = ok ? (int)all_fresh : 0;
  int cu = ok ? (int)cu0 : 0, first = ok ? (int)first0 : 0;
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) {
    const int b = tid * per + i;
    if (i >= per || b >= a.n_seq) continue;
    s_cu[b] = cu;
    s_first[b] = first;
    if (rank == 0 && !a.only_commit) a.cu_new[b] = cu;
    if (ok) {
      cu += add[i];
      first += (int)(((long long)len[i] + add[i] + pm) >> sh) - (int)(((long long)len[i] + pm) >> sh);
    }
  }
  if (tid == 0) {
    if (rank == 0 && !a.only_commit) a.cu_new[a.n_seq] = total;
    if (rank == 0 && bits && a.status) atomicOr(a.status, bits);
  }
  __syncthreads();
  const int step = nct * kPlanThreads;
  if (!a.only_commit) {
    for (int f = rank * kPlanThreads + tid; f < fresh; f += step) {
      const int b = last_not_above(s_first, a.n_seq, f);
      a.block_table[(size_t)b * a.max_blocks + ((a.lens[b] + pm) >> sh) + (f - s_first[b])] = a.free_pages[n_free - 1 - f];
    }
#pragma unroll 2
    for (int t = rank * kPlanThreads + tid; t < a.n_tokens; t += step) {
      int64_t slot = -1, pos = -1;
      int b = -1;
      if (t < total) {
        b = last_not_above(s_cu, a.n_seq, t);
        const int len0 = a.lens[b], p = len0 + (t - s_cu[b]), j = p >> sh, have = (len0 + pm) >> sh;
        const int page = j < have ? a.block_table[(size_t)b * a.max_blocks + j] : a.free_pages[n_free - 1 - s_first[b] - (j - have)];
        if (page >= 0 && page < a.n_pages) slot = ((int64_t)page << sh) + (p & pm);
        else if (a.status) atomicOr(a.status, HC_DEV_INDEX);
        pos = (int64_t)a.base_pos + p;
      }
      a.slots[t] = slot;
      a.seq_ids[t] = b;
      a.positions[t] = pos;
    }
  }
  if (!a.lens_out) return;  // committed by another launch
  if (a.in_place && nct > 1) cluster_sync_all();  // every CTA has read lens and n_free
  else __syncthreads();
  if (rank == 0) {
#pragma unroll
    for (int i = 0; i < kPlanPer; ++i) {
      const int b = tid * per + i;
      if (i < per && b < a.n_seq) a.lens_out[b] = ok ? len[i] + add[i] : len[i];
    }
    if (tid == 0) *a.n_free_out = n_free - fresh;
  }
}

// Sequence b keeps its first keep_b tokens; the pages behind them go back on the stack in the reverse of
// the order plan_pages_kernel takes them, so that taking a step back restores the stack as it was. One CTA: the
// bytes are 12 a sequence and 8 a page, the time launch, scan and for each page a search and two dependent accesses. One
// B200: 64 sequences of 2 pages 2.4 us, 256 of 64 pages each all at once 20 us, 4096 of 4 pages 28 us.
__global__ void __launch_bounds__(kPlanThreads) release_pages_kernel(PagePlanArgs a) {
  __shared__ int s_first[kPlanMaxSeq], s_have[kPlanMaxSeq];
  __shared__ int64_t s_scan[2 * kPlanThreads / 32];
  pdl_wait();
  const int tid = threadIdx.x;
  const int sh = __ffs(a.page_size) - 1, pm = a.page_size - 1;
  const long long cap = (long long)a.max_blocks << sh;
  const int n_free = *a.n_free;
  const int per = (a.n_seq + kPlanThreads - 1) / kPlanThreads;
  int n = 0, bits = (n_free < 0 || n_free > a.n_pages) ? HC_DEV_INDEX : 0;
  int keep[kPlanPer], give[kPlanPer];
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) {
    const int b = tid * per + i;
    if (i >= per || b >= a.n_seq) continue;
    const int len = a.lens[b];
    keep[i] = a.new_lens[b];
    give[i] = 0;
    if (len < 0 || len > cap || keep[i] < 0 || keep[i] > len) bits |= HC_DEV_INDEX;
    else give[i] = ((len + pm) >> sh) - ((keep[i] + pm) >> sh);
    n += give[i];
  }
  int64_t first0, total0, none0, none1;
  scan_pair(n, 0, s_scan, first0, none0, total0, none1);
  const int bad = __syncthreads_or(bits);
  bits = bad ? HC_DEV_INDEX : (total0 > a.n_pages - n_free ? HC_DEV_CAPACITY : 0);
  if (bits) {  // nothing is given back
    if (tid == 0 && a.status) atomicOr(a.status, bits);
    return;
  }
  const int total = (int)total0;
  int first = (int)first0;
#pragma unroll
  for (int i = 0; i < kPlanPer; ++i) {
    const int b = tid * per + i;
    if (i >= per || b >= a.n_seq) continue;
    s_first[b] = first;
    s_have[b] = (keep[i] + pm) >> sh;
    first += give[i];
    a.lens[b] = keep[i];
  }
  __syncthreads();
  for (int f = tid; f < total; f += kPlanThreads) {
    const int b = last_not_above(s_first, a.n_seq, f);
    a.free_out[n_free + total - 1 - f] = a.block_table[(size_t)b * a.max_blocks + s_have[b] + (f - s_first[b])];
  }
  if (tid == 0) *a.n_free_out = n_free + total;
}

// One B200: a step of 64 tokens takes 5.2 us, 131 thousand tokens of 256 prompts 6.0 us on as many CTAs as a
// thousand tokens each fill (2.7 MB written; 51 us on a cluster of 8). Both are launch, scan and two dependent
// loads; the bytes are 0.4 us.
cudaError_t launch_plan_pages(const PagePlanArgs& args, cudaStream_t stream) {
  PagePlanArgs a = args;
  a.in_place = a.lens == a.lens_out || a.new_lens == a.lens_out || a.n_free == a.n_free_out;
  const int want = (int)(((int64_t)a.n_tokens + kPlanThreads - 1) / kPlanThreads);
  if (want > 16) {
    const int ctas = want / 2 < 296 ? want / 2 : 296;
    if (a.in_place) a.lens_out = nullptr;
    cudaError_t e = launch_pdl(plan_pages_kernel, dim3((unsigned)ctas), dim3(kPlanThreads), 0, stream, a);
    if (e != cudaSuccess || !a.in_place) return e;
    a.lens_out = args.lens_out;
    a.only_commit = 1;
    return launch_pdl(plan_pages_kernel, dim3(1), dim3(kPlanThreads), 0, stream, a);
  }
  int ctas = 1;
  while (ctas < 8 && ctas < want) ctas *= 2;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)ctas;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kPlanThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, plan_pages_kernel, a);
}

cudaError_t launch_release_pages(const PagePlanArgs& a, cudaStream_t stream) {
  return launch_pdl(release_pages_kernel, dim3(1), dim3(kPlanThreads), 0, stream, a);
}

// ----------------------------------------------------------------------------------------
// Rotary append: x'[i] = x[i] cos - x[i + D/2] sin, x'[i + D/2] = x[i + D/2] cos + x[i] sin with the
// angle position * inv_freq[i], for queries and keys; keys and values go to the row their slot names.
// Bound by HBM: every element is read once and written once. A CTA takes one token with a thread for each
// pair of 16-byte chunks (i, i + D/2) of its rows, so that a token's loads are all in flight while D/2
// threads work out its angles. The angle is reduced in 64 bits (a 32-bit product is off by 0.008 rad at
// position 131072); the rotation is done in 32 bits and rounded once.
// One B200, 32/8 heads of 128 in bf16: 8.5 thousand tokens (209 MB) 42 us, 5.0 TB/s, 76 % of the measured copy
// rate; 64 tokens 3.8 us.
// ----------------------------------------------------------------------------------------
constexpr int kAppThreads = 512;

template <int DT, int D>
__global__ void __launch_bounds__(kAppThreads) append_pages_kernel(PageAppendArgs a) {
  using E = Elem<DT>;
  using T = typename E::T;
  constexpr int VEC = 16 / sizeof(T), H = D / 2, CH = H / VEC;  // chunks per half row
  __shared__ float s_cos[H], s_sin[H];
  pdl_wait();
  const int t = blockIdx.x, tid = threadIdx.x;
  const int nq = a.q_out ? a.Hq : 0, items = (nq + 2 * a.Hk) * CH;
  // a pair of chunks: of a query head, of a key head, of a value head
  auto source = [&](int x) {
    const int hh = x / CH;
    if (hh < nq) return reinterpret_cast<const T*>(a.q) + t * a.q_st + hh * a.q_sh;
    if (hh < nq + a.Hk) return reinterpret_cast<const T*>(a.k) + t * a.k_st + (hh - nq) * a.k_sh;
    return reinterpret_cast<const T*>(a.v) + t * a.v_st + (hh - nq - a.Hk) * a.v_sh;
  };
  // the rows, the slot and the position are read side by side
  uint4 lo = make_uint4(0u, 0u, 0u, 0u), hi = lo;
  if (tid < items) {
    const uint4* src = reinterpret_cast<const uint4*>(source(tid)) + tid % CH;
    lo = src[0];
    hi = src[CH];
  }
  const int64_t slot = a.slots[t];
  if (a.inv_freq && tid < H) {
    const double ang = (double)a.inv_freq[tid] * (double)a.positions[t];
    const double n = rint(ang * 0.15915494309189535);  // 1 / (2 pi)
    // 2 pi as the nearest double and what that leaves
    const double r = fma(-n, 2.4492935982947064e-16, fma(-n, 6.283185307179586, ang));
    float cs, sn;
    sincosf((float)r, &sn, &cs);
    s_cos[tid] = cs * a.rope_scaling;
    s_sin[tid] = sn * a.rope_scaling;
  }
  __syncthreads();
  if (slot < 0 || slot >= (int64_t)a.n_pages * a.page_size) {
    if (slot != -1 && tid == 0 && a.status) atomicOr(a.status, HC_DEV_INDEX);
    return;
  }
  const int64_t page = slot >> (__ffs(a.page_size) - 1);
  const int row = (int)slot & (a.page_size - 1);
  for (int x = tid; x < items; x += blockDim.x) {
    const int hh = x / CH, c = x % CH;
    if (x != tid) {
      const uint4* src = reinterpret_cast<const uint4*>(source(x)) + c;
      lo = src[0];
      hi = src[CH];
    }
    T* dst;
    if (hh < nq) {
      dst = reinterpret_cast<T*>(a.q_out) + ((size_t)t * a.Hq + hh) * D;
    } else {
      const bool key = hh < nq + a.Hk;
      const size_t off = (((size_t)page * a.Hk + hh - nq - (key ? 0 : a.Hk)) * a.page_size + row) * D;
      dst = reinterpret_cast<T*>(key ? a.k_pages : a.v_pages) + off;
    }
    if (a.inv_freq && hh < nq + a.Hk) {
      float fl[VEC], fh[VEC];
      unpack16<DT>(lo, fl);
      unpack16<DT>(hi, fh);
      alignas(16) T ol[VEC], oh[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float cs = s_cos[c * VEC + e], sn = s_sin[c * VEC + e];
        ol[e] = E::from_f(fl[e] * cs - fh[e] * sn);
        oh[e] = E::from_f(fh[e] * cs + fl[e] * sn);
      }
      lo = *reinterpret_cast<uint4*>(ol);
      hi = *reinterpret_cast<uint4*>(oh);
    }
    reinterpret_cast<uint4*>(dst)[c] = lo;
    reinterpret_cast<uint4*>(dst + H)[c] = hi;
  }
}

template <int DT, int D>
static cudaError_t append_pages_t(const PageAppendArgs& a, cudaStream_t stream) {
  const int items = ((a.q_out ? a.Hq : 0) + 2 * a.Hk) * (D / 2) / (DT == HC_F32 ? 4 : 8);
  int threads = (items + 31) / 32 * 32;
  if (threads < D / 2) threads = D / 2;
  if (threads > kAppThreads) threads = kAppThreads;
  return launch_pdl(append_pages_kernel<DT, D>, dim3((unsigned)a.n_tokens), dim3((unsigned)threads), 0, stream, a);
}

cudaError_t launch_append_pages(const PageAppendArgs& a, int dtype, int D, cudaStream_t stream) {
  HC_DISPATCH_DT_D(dtype, D, append_pages_t, a, stream);
}

}  // namespace hc
