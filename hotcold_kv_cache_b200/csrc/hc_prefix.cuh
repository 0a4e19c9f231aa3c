// How the attention of a batch over [shared prefix | own pages] is divided among CTAs.
//
// A query token t of sequence b sees every (unmasked) prefix key and its own sequence's keys up to
// itself. The prefix part is the same for all sequences, so the rows (t, query head of a KV head's
// group) of the whole batch are stacked into row tiles and each prefix key tile is read once per row
// tile, not once per sequence. The own-pages part has row tiles per sequence. A group is
//   prefix: (KV head, chunk of key tiles, row tile)      suffix: (sequence, KV head, row tile)
// and all groups lie one behind the other on a line, each as long as it takes (line_cost: so much to start
// it and so much a key tile). CTA c works on the key tiles that begin in the stretch [c W, (c + 1) W) of the
// line, so that CTAs get about the same work: the busiest of 148 has 1.01 times the mean with 64 decode steps over
// 128k keys and 1.04 with a chunk of 8 x 257 over 16k. Not so where causal own tokens outweigh the rest: every
// row tile of a sequence is as long on the line as if it saw all of the sequence's keys, and a short last row tile as a
// whole one (1.29 with 4 x 4096 new tokens over 4k, 1.69 with 8192 over 1k, 1.89 with 16384 and no prefix). Where a
// stretch ends inside a group its rows are left as several partial results (running maximum, sum, unnormalised output), joined by the merge
// kernel. A piece (c, group) has its partial rows at  2 * (rows of the groups before it) + c * ROWS:
// pieces follow one another in c or in the group, and each takes at most min(2 rows, ROWS).
// The prefix is cut into chunks (nch > 1) when there are several row tiles, so that row tiles reading
// the same keys sit next to each other on the line and share them through L2.
#pragma once
#include "hc_internal.cuh"

namespace hc {

// Host constants of one call.
struct LineShape {
  int T, n_seq, Hk, G, P;
  int rt, kt;  // rows per row tile, keys per key tile
  int nc;      // CTAs
  int nch;     // prefix chunks
  int dup;     // 2 where one piece may leave two partial results per row (two streams over the keys)
};

// What a group costs on the line: b to start it, a for each key tile.
struct LineCost {
  int a, b;
};

__host__ __device__ inline int ceil_div(int a, int b) { return (a + b - 1) / b; }

inline LineShape line_shape(int T, int n_seq, int Hk, int G, int P, int rt, int kt, int nc, int dup) {
  LineShape s{T, n_seq, Hk, G, P, rt, kt, nc, 1, dup};
  const int nrt = ceil_div(T, rt / G), ktp = ceil_div(P, kt);
  if (nrt > 1 && ktp > 0) {
    const int want = nc / (nrt * Hk);
    s.nch = want < 1 ? 1 : want > 16 ? 16 : want;
    if (s.nch > ktp) s.nch = ktp;
    s.nch = ceil_div(ktp, ceil_div(ktp, s.nch));  // no empty chunk
  }
  return s;
}

// Rows of partial results the call may leave.
inline size_t line_rows(const LineShape& s) {
  const size_t rows = (size_t)s.T * s.G * s.Hk;
  return s.dup * (rows * (s.P > 0 ? s.nch : 0) + rows) + (size_t)s.nc * s.rt;
}

// The 16-bit kernel (hc_prefix_mma.cu) and its division of a call on `sms` SMs.
LineShape prefix_mma_shape(int T, int n_seq, int Hk, int G, int P, int sms);
cudaError_t launch_prefix_mma(const PrefixArgs& a, const LineShape& s, int dtype, int D, int64_t* hdr, float2* ml, float* part,
                              cudaStream_t stream);

// Whether a row tile of `rows` rows is taken by two streams over its key tiles, each with a result of its own
// (hc_prefix_mma.cu): above that its halves, below it whole pieces go to one stream each.
__host__ __device__ inline bool prefix_two_streams(int rows) { return rows > 64 && rows <= 128; }

// fp32: alike. 16 bits, in units of about 0.55 us as measured on whole lines of one kind at D = 128: tall row
// tiles 2.8 us a key tile and 4.5 us to load Q and write the result (9.5 us behind causal tiles, where the streams
// meet and V is looked through), up to 64 rows 1.15 and 1.6 us. 65 to 128 rows lie between by choice; a key tile of
// theirs was measured later at 1.2 us. D = 64 is divided by the same costs: there a key tile takes 2.5 us (tall) and 1.4.
__device__ __forceinline__ LineCost line_cost(const LineShape& s, int rows, bool own) {
  if (s.dup == 1) return {1, 1};
  if (rows > 128) return {5, own ? 17 : 8};
  if (prefix_two_streams(rows)) return {3, own ? 12 : 6};
  return {2, 3};
}

// The shortest stretch is >= every a: no CTA between a group's first and last is without a tile.
__device__ __forceinline__ int min_stretch(const LineShape& s) { return s.dup == 1 ? 2 : 7; }

struct Piece {
  bool own;         // suffix (own pages) or prefix
  int b, h;         // sequence (suffix) and KV head
  int tok0, ntok;   // query tokens
  int kt0, kt1;     // key tiles
  int kend;         // keys that exist for these tokens
  int c0;           // suffix: token tok0 + i sees keys j < c0 + i + 1
  int64_t row0;     // first partial row
};

// The lengths of sequence b as every kernel reads them: bounded, whatever the tables hold.
struct SeqLens {
  int cu, n, len;
};
__device__ __forceinline__ SeqLens seq_lens(const PrefixArgs& a, int b) {
  SeqLens s;
  const int c0 = min(max(a.cu_new[b], 0), a.T), c1 = min(max(a.cu_new[b + 1], 0), a.T);
  s.cu = c0;
  s.n = max(c1 - c0, 0);
  const int64_t cap = (int64_t)a.max_blocks * a.page_size;
  const int len = a.lens[b];
  s.len = (int)min((int64_t)max(len, 0), cap);
  if (len != s.len && a.status) atomicOr(a.status, HC_DEV_INDEX);
  return s;
}
__device__ __forceinline__ int seq_keys(const SeqLens& s, int tok1) {  // keys seen by tokens below tok1 (of n)
  return min(max(s.len - s.n + tok1, 0), s.len);
}

// Quotient of line positions: 64-bit division, out of the way, only where 32 bits do not hold them (a kernel
// starts with cold instruction caches, and its first microseconds are fetches of what it runs through).
static __device__ __noinline__ int64_t line_div64(int64_t x, int64_t y) { return x / y; }
__device__ __forceinline__ int line_div(int64_t x, int64_t y) {  // numbers of CTAs, groups or tiles: 32 bits hold them
  return (x | y) >> 32 ? (int)line_div64(x, y) : (int)((uint32_t)x / (uint32_t)y);
}

struct LineGeom {
  int R;              // query tokens of the call's sequences
  int tt;             // query tokens per row tile
  int nrt, ktp, ct;   // prefix row tiles, key tiles, key tiles per chunk
  LineCost pre;       // of a prefix group
  int64_t head;       // length of one KV head's prefix groups
  int64_t vpre;       // length of all prefix groups
  __device__ LineGeom(const LineShape& s, int R_) {
    R = R_;
    tt = s.rt / s.G;
    nrt = ceil_div(R, tt);
    ktp = ceil_div(s.P, s.kt);
    ct = ktp > 0 ? ceil_div(ktp, s.nch) : 0;
    pre = line_cost(s, min(R * s.G, s.rt), false);
    head = ktp > 0 ? (int64_t)nrt * (ktp * pre.a + s.nch * pre.b) : 0;
    vpre = head * s.Hk;
  }
  __device__ int64_t seq_group(const LineShape& s, const SeqLens& q) const {  // one group of a sequence
    if (q.n <= 0 || q.len <= 0) return 0;
    const LineCost c = line_cost(s, min(q.n * s.G, s.rt), true);
    return (int64_t)ceil_div(q.len, s.kt) * c.a + c.b;
  }
  __device__ int64_t seq_total(const LineShape& s, const SeqLens& q) const {
    return seq_group(s, q) * s.Hk * ceil_div(q.n, tt);
  }
};

// Header of the scratch: hdr[0] = W, hdr[1 + b] = where sequence b's groups start on the line.
// Every CTA of NT threads calls it; CTA 0 writes the header. Returns the stretch of this CTA and the
// sequence in which it starts (b0, at vb0) where that is behind the prefix.
struct Stretch {
  int64_t W, v, v_end, vb;
  int b;
};
template <int NT>
__device__ __forceinline__ Stretch line_setup(const PrefixArgs& a, const LineShape& s, const LineGeom& g, int c,
                                              int64_t* hdr, int64_t* sh /* NT / 32 + 4 */) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  constexpr int NW = NT / 32;
  const int per = ceil_div(s.n_seq, NT);
  const int b0 = tid * per, b1 = min(b0 + per, s.n_seq);
  int64_t mine = 0, last = 0;
  for (int b = b0; b < b1; ++b) mine += last = g.seq_total(s, seq_lens(a, b));
  int64_t x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sh[warp] = x;
  __syncthreads();
  int64_t before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const int64_t t = sh[w];
    if (w < warp) before += t;
    total += t;
  }
  before += x - mine + g.vpre;
  total += g.vpre;
  Stretch r;
  // a stretch may pass 32 bits: 65536 tokens of one sequence over 2^30 keys are 4.6e9 long
  const int64_t up = total + s.nc - 1;
  r.W = max(up >> 32 ? line_div64(up, s.nc) : (int64_t)((uint32_t)up / (uint32_t)s.nc), (int64_t)min_stretch(s));
  r.v = min(c * r.W, total);
  r.v_end = min((c + 1) * r.W, total);
  if (c == 0 && tid == 0) hdr[0] = r.W;
  // the sequence in which the stretch starts (or the first one, when it starts in the prefix)
  const int64_t at = max(r.v, g.vpre);
  if (tid == 0) {
    sh[NW] = 0;
    sh[NW + 1] = g.vpre;
  }
  __syncthreads();
  int64_t vb = before;
  for (int b = b0; b < b1; ++b) {
    const int64_t n = per == 1 ? last : g.seq_total(s, seq_lens(a, b));
    if (c == 0) hdr[1 + b] = vb;
    if (n > 0 && vb <= at && at < vb + n) {
      sh[NW] = b;
      sh[NW + 1] = vb;
    }
    vb += n;
  }
  __syncthreads();
  r.b = (int)sh[NW];
  r.vb = sh[NW + 1];
  return r;
}

// The pieces of a CTA's stretch, one after the other. Uniform over the threads that walk it. The position
// is found once by division; from there groups follow one another by counting, and a sequence's lengths are
// read once.
struct LineWalk {
  int64_t v, v_end, cw;  // start of the current group, end and start of the stretch
  int c, b, h, r, j;     // prefix: head h, chunk j, row tile r; own pages: sequence b, head h, row tile r
  bool own;
  SeqLens q;
  int len, nr;           // own pages: length of a group, row tiles of the sequence
  LineCost cost;         // of the sequence's groups
  // the key tiles of the group at v that begin in the stretch
  __device__ __forceinline__ void clip(LineCost k, int tiles, int& lo, int& hi) const {
    const int64_t s = cw - v - k.b, e = v_end - v - k.b;
    const int64_t all = (int64_t)tiles * k.a;  // beyond it every tile counts
    lo = s <= 0 ? 0 : s >= all ? tiles : line_div(s + k.a - 1, k.a);
    hi = e <= 0 ? 0 : e >= all ? tiles : line_div(e + k.a - 1, k.a);
  }
  __device__ __forceinline__ void seq(const PrefixArgs& a, const LineShape& s, const LineGeom& g) {
    q = seq_lens(a, b);
    len = (int)g.seq_group(s, q);
    cost = line_cost(s, min(q.n * s.G, s.rt), true);
    nr = len > 0 ? ceil_div(q.n, g.tt) : 0;
  }
  __device__ __forceinline__ LineWalk(const PrefixArgs& a, const LineShape& s, const LineGeom& g, const Stretch& st, int cta) {
    c = cta;
    cw = st.v;
    v_end = st.v_end;
    b = st.b;
    own = st.v >= g.vpre;
    len = nr = h = r = j = 0;
    v = st.v;
    if (v >= v_end) return;
    if (!own) {
      h = line_div(v, g.head);
      const int64_t rem = v - h * g.head, full = (int64_t)g.nrt * (g.ct * g.pre.a + g.pre.b);
      j = min(line_div(rem, full), s.nch - 1);
      const int64_t n = (int64_t)min(g.ct, g.ktp - j * g.ct) * g.pre.a + g.pre.b;
      r = line_div(rem - j * full, n);
      v = h * g.head + j * full + r * n;
    } else {
      seq(a, s, g);
      if (len > 0) {
        const int x = line_div(v - st.vb, len);
        h = x / nr;
        r = x % nr;
        v = st.vb + (int64_t)x * len;
      }
    }
  }
  __device__ __forceinline__ bool next(const PrefixArgs& a, const LineShape& s, const LineGeom& g, Piece& p) {
    while (v < v_end) {
      if (!own) {
        const int tiles = min(g.ct, g.ktp - j * g.ct);
        int lo, hi;
        clip(g.pre, tiles, lo, hi);
        p.own = false;
        p.b = 0;
        p.h = h;
        p.tok0 = r * g.tt;
        p.ntok = min(g.tt, g.R - p.tok0);
        p.kt0 = j * g.ct + lo;
        p.kt1 = j * g.ct + hi;
        p.kend = s.P;
        p.c0 = 0;
        p.row0 = s.dup * (((int64_t)h * s.nch + j) * s.T + p.tok0) * s.G + (int64_t)c * s.rt;
        v += (int64_t)tiles * g.pre.a + g.pre.b;
        if (++r == g.nrt) {
          r = 0;
          if (++j == s.nch) {
            j = 0;
            if (++h == s.Hk) {
              own = true;
              b = h = 0;
              if (v < v_end) seq(a, s, g);
            }
          }
        }
        if (lo < hi) return true;
        continue;
      }
      if (nr == 0) {  // a sequence without groups
        if (++b >= s.n_seq) return false;
        seq(a, s, g);
        continue;
      }
      const int tok1 = min(q.n, (r + 1) * g.tt), keys = seq_keys(q, tok1), tiles = ceil_div(keys, s.kt);
      int lo, hi;
      clip(cost, tiles, lo, hi);
      p.own = true;
      p.b = b;
      p.h = h;
      p.tok0 = q.cu + r * g.tt;
      p.ntok = tok1 - r * g.tt;
      p.kt0 = lo;
      p.kt1 = hi;
      p.kend = keys;
      p.c0 = q.len - q.n + r * g.tt;
      p.row0 = s.dup * ((int64_t)s.Hk * s.T * (s.P > 0 ? s.nch : 0) + (int64_t)q.cu * s.Hk + (int64_t)h * q.n + r * g.tt) * s.G +
               (int64_t)c * s.rt;
      v += len;
      if (++r == nr) {
        r = 0;
        if (++h == s.Hk) {
          h = 0;
          if (++b >= s.n_seq) nr = 0, b = s.n_seq;
          else if (v < v_end) seq(a, s, g);
        }
      }
      if (lo < hi) return true;
    }
    return false;
  }
};

}  // namespace hc
