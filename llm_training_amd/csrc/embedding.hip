// Embedding lookup with scaling and its weight gradient by sorted tokens, for gfx950.
//
//   forward   y[t] = scale * w[ids[t] - v0]                       (zeros for an id outside [v0, v0 + V))
//   backward  dw[v] (+)= scale * sum over t with ids[t] - v0 == v of g[t]
//
// The sums are taken in fp32 in ascending order of t and rounded once, so a gradient is the same bits in every
// run: no floating-point atomics. Up to kSmallMax tokens one kernel does it all: every workgroup looks through the
// ids for its few vocabulary rows (embed_small_kernel; 333 tokens, 32064 x 768 fp32: the four dependent launches of
// the general way are most of its time). Beyond, the tokens are put in order of (id, t) first:
//   * up to kRankMax tokens: every token counts the tokens in front of it, all pairs, over the whole chip
//     (8192 tokens: 67 M compares of one packed word, a few us in one launch, where a radix sort needs five
//     launches of that length);
//   * more: least-significant-digit radix passes of 9 bits, two kernels each: a histogram per tile of tokens, and
//     a stable scatter whose workgroups add up the histograms in front of them by themselves (up to kScanSelf tiles;
//     a scan kernel for more). Counting the next histogram inside the scatter would save a launch, but its global
//     atomics meet on a few words when a few ids make up most of a text: 85 us against 6 for the kernel.
// Then the sorted list is cut into equal chunks, whatever ids it holds (a padding id can own half of it): a run of
// one id inside a chunk is summed and stored at once; a run over several chunks leaves fp32 partial rows that the
// finishing kernel adds in chunk order, beside writing the zeros of rows without a token. Bound by HBM: g is read
// once and dw written once.
#include "elem_types.h"

namespace llmt {

constexpr int kSmallMax = 512;
constexpr int kSmallRows = 16;   // vocabulary rows of a workgroup of the small kernel
constexpr int kRankMax = 8192;   // 13 bits of position beside 19 bits of id in one word
constexpr int kRadixBits = 9, kRadix = 1 << kRadixBits;
constexpr int kTile = 1024;      // keys per workgroup of a radix pass: 4 waves x 256, 4 rounds of 64
constexpr int kScanSelf = 64;    // tiles up to which a scatter workgroup sums the histograms itself
constexpr int kRankTile = 256;   // tokens compared against by one workgroup of the rank kernel

template <typename I>
__device__ __forceinline__ uint32_t local_key(const I* ids, int64_t i, int64_t v0, int valid, int V, int* err) {
  const int64_t l = (int64_t)ids[i] - v0;
  if (l >= 0 && l < valid) return (uint32_t)l;
  if (err) err[2] = 1;  // (an unsharded table: every id has to be in it)
  return (uint32_t)V;   // sorts behind every row; dropped
}

// ---------------------------------------------------------------------------------------------- forward
template <typename T, typename I, bool VEC, bool NT>
__global__ __launch_bounds__(256) void embed_fwd_kernel(const I* __restrict__ ids, const T* __restrict__ w,
                                                        T* __restrict__ y, int64_t N, int V, int H, int64_t v0,
                                                        float scale, int rows, int* __restrict__ err) {
  const int64_t r0 = (int64_t)blockIdx.x * rows;
  const int nr = (int)(N - r0 < rows ? N - r0 : rows);
  const int per = VEC ? H >> 3 : H;
  const unsigned items = (unsigned)nr * (unsigned)per;
  if constexpr (VEC) {
    constexpr int U = sizeof(T) == 4 ? 2 : 4;  // vectors in flight a thread
    for (unsigned e0 = threadIdx.x; e0 < items; e0 += 256 * U) {
      typename Elem<T>::Raw x[U];
      unsigned r[U], c[U];
      bool ok[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const unsigned e = e0 + 256 * u < items ? e0 + 256 * u : e0;
        r[u] = e / (unsigned)per;
        c[u] = e - r[u] * (unsigned)per;
        const int64_t l = (int64_t)ids[r0 + r[u]] - v0;
        ok[u] = l >= 0 && l < V;
        if (!ok[u] && err && c[u] == 0) err[2] = 1;
        if (V > 0) x[u] = load8(w + (ok[u] ? l : 0) * H + 8 * c[u]);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (e0 + 256 * u >= items) break;
        float f[8];
        Elem<T>::unpack(x[u], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = ok[u] ? f[i] * scale : 0.f;
        if constexpr (NT)
          store8_nt(y + (r0 + r[u]) * H + 8 * c[u], f);
        else
          store8(y + (r0 + r[u]) * H + 8 * c[u], f);
      }
    }
  } else {
    for (unsigned e = threadIdx.x; e < items; e += 256) {
      const unsigned r = e / (unsigned)per, c = e - r * (unsigned)per;
      const int64_t l = (int64_t)ids[r0 + r] - v0;
      const bool ok = l >= 0 && l < V;
      if (!ok && err && c == 0) err[2] = 1;
      y[(r0 + r) * H + c] = Elem<T>::from_float(ok ? Elem<T>::to_float(w[l * H + c]) * scale : 0.f);
    }
  }
}

// ---------------------------------------------------------------------------------------------- order of tokens
// part[jb][i]: how many tokens of the jb-th kRankTile come before token i. grid (>= ceil(N / 256), ceil(N / kRankTile)).
// Also clears the run table of the vocabulary rows (workgroups behind the last token do nothing else).
template <typename I>
__global__ __launch_bounds__(256) void embed_rank_kernel(const I* __restrict__ ids, int N, int64_t v0, int valid, int V,
                                                         int* __restrict__ part, int* __restrict__ run_start,
                                                         int* __restrict__ err) {
  __shared__ __attribute__((aligned(16))) uint32_t tile[kRankTile];
  const int tid = threadIdx.x, i = blockIdx.x * 256 + tid, j0 = blockIdx.y * kRankTile;
  const int nblk = gridDim.x * gridDim.y, blk = blockIdx.y * gridDim.x + blockIdx.x;
  for (int v = blk * 256 + tid; v < V; v += nblk * 256) run_start[v] = -1;
  if ((int)blockIdx.x * 256 >= N) return;
  for (int j = tid; j < kRankTile; j += 256)  // a word above every key past the end: counted for nobody
    tile[j] = j0 + j < N ? (local_key(ids, j0 + j, v0, valid, V, nullptr) << 13) | (uint32_t)(j0 + j) : 0xffffffffu;
  __syncthreads();
  const uint32_t mine = i < N ? (local_key(ids, i, v0, valid, V, blockIdx.y == 0 ? err : nullptr) << 13) | (uint32_t)i : 0u;
  int n = 0;
#pragma unroll 4
  for (int j = 0; j < kRankTile; j += 4) {
    const uint4 k = *reinterpret_cast<const uint4*>(tile + j);
    n += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
  }
  if (i < N) part[(int64_t)blockIdx.y * N + i] = n;
}
template <typename I>
__global__ __launch_bounds__(256) void embed_place_kernel(const I* __restrict__ ids, int N, int64_t v0, int valid, int V,
                                                          const int* __restrict__ part, int parts,
                                                          uint32_t* __restrict__ skey, int* __restrict__ order) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= N) return;
  int r = 0;
  for (int p = 0; p < parts; ++p) r += part[(int64_t)p * N + i];
  skey[r] = local_key(ids, i, v0, valid, V, nullptr);
  order[r] = i;
}

// radix pass, step 1: hist[block][digit]. The first pass also clears the run table.
template <typename I, bool FIRST>
__global__ __launch_bounds__(256) void embed_hist_kernel(const I* __restrict__ ids, const uint32_t* __restrict__ kin,
                                                         int64_t N, int64_t v0, int valid, int V, int shift,
                                                         int* __restrict__ hist, int nblk, int* __restrict__ run_start,
                                                         int* __restrict__ err) {
  __shared__ int h[kRadix];
  const int tid = threadIdx.x;
  for (int d = tid; d < kRadix; d += 256) h[d] = 0;
  __syncthreads();
  for (int e = tid; e < kTile; e += 256) {
    const int64_t i = (int64_t)blockIdx.x * kTile + e;
    if (i < N) {
      const uint32_t k = FIRST ? local_key(ids, i, v0, valid, V, err) : kin[i];
      atomicAdd(&h[(k >> shift) & (kRadix - 1)], 1);
    }
  }
  __syncthreads();
  for (int d = tid; d < kRadix; d += 256) hist[(int64_t)blockIdx.x * kRadix + d] = h[d];
  if constexpr (FIRST)
    for (int64_t v = (int64_t)blockIdx.x * 256 + tid; v < V; v += (int64_t)nblk * 256) run_start[v] = -1;
}

// step 2 (more than kScanSelf tiles): hist[b][d] becomes the count of digit d in the tiles before b, row nblk the
// digits' totals. One thread a digit.
__global__ __launch_bounds__(64) void embed_scan_kernel(int* __restrict__ hist, int nblk) {
  int* h = hist + blockIdx.x * 64 + threadIdx.x;
  int sum = 0, b = 0;
  for (; b + 8 <= nblk; b += 8) {
    int v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = h[(int64_t)(b + i) * kRadix];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      h[(int64_t)(b + i) * kRadix] = sum;
      sum += v[i];
    }
  }
  for (; b < nblk; ++b) {
    const int v = h[(int64_t)b * kRadix];
    h[(int64_t)b * kRadix] = sum;
    sum += v;
  }
  h[(int64_t)nblk * kRadix] = sum;
}

// step 3: stable scatter by the digit at `shift`. Each wave owns 256 consecutive keys of the tile and takes them in
// rounds of 64: the lanes with an equal digit find each other through one ballot per bit, so a lane's place is the
// wave's running count of its digit plus the equal lanes below it.
template <typename I, bool FIRST>
__global__ __launch_bounds__(256) void embed_scatter_kernel(const I* __restrict__ ids, const uint32_t* __restrict__ kin,
                                                            const int* __restrict__ vin, int64_t N, int64_t v0, int valid, int V,
                                                            int shift, const int* __restrict__ hist, int nblk,
                                                            uint32_t* __restrict__ kout, int* __restrict__ vout) {
  __shared__ int cnt[4][kRadix];
  __shared__ int base[kRadix];  // where this tile's keys of a digit begin
  __shared__ int wsum[4];
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  for (int d = tid; d < 4 * kRadix; d += 256) (&cnt[0][0])[d] = 0;
  {  // digits 2 tid, 2 tid + 1: keys of the digit in the tiles before, and in all; then the digits' prefix sums
    int before[2], total[2];
    const int* h = hist + 2 * tid;
    const int me = (int)blockIdx.x;
    if (nblk <= kScanSelf) {
      before[0] = before[1] = total[0] = total[1] = 0;
#pragma unroll 8
      for (int b = 0; b < nblk; ++b) {
        const int2 v = *reinterpret_cast<const int2*>(h + (int64_t)b * kRadix);
        if (b < me) {
          before[0] += v.x;
          before[1] += v.y;
        }
        total[0] += v.x;
        total[1] += v.y;
      }
    } else {
      const int2 v = *reinterpret_cast<const int2*>(h + (int64_t)me * kRadix);
      const int2 t = *reinterpret_cast<const int2*>(h + (int64_t)nblk * kRadix);
      before[0] = v.x;
      before[1] = v.y;
      total[0] = t.x;
      total[1] = t.y;
    }
    const int mine = total[0] + total[1];
    int inc = mine;  // inclusive sum over the wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(inc, o, 64);
      if (lane >= o) inc += t;
    }
    if (lane == 63) wsum[wid] = inc;
    __syncthreads();
    int at = inc - mine;
    for (int w = 0; w < wid; ++w) at += wsum[w];
    base[2 * tid] = at + before[0];
    base[2 * tid + 1] = at + total[0] + before[1];
  }
  __syncthreads();
  constexpr int R = kTile / 256;
  uint32_t key[R];
  int val[R], place[R];
  const int64_t t0 = (int64_t)blockIdx.x * kTile + wid * (kTile / 4);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int64_t i = t0 + r * 64 + lane;
    key[r] = 0;
    val[r] = 0;
    if (i < N) {
      key[r] = FIRST ? local_key(ids, i, v0, valid, V, nullptr) : kin[i];
      val[r] = FIRST ? (int)i : vin[i];
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool live = t0 + r * 64 + lane < N;
    const int d = (int)(key[r] >> shift) & (kRadix - 1);
    uint64_t same = __ballot(live);
#pragma unroll
    for (int b = 0; b < kRadixBits; ++b) {
      const uint64_t one = __ballot((d >> b) & 1);
      same &= ((d >> b) & 1) ? one : ~one;
    }
    const int below = __popcll(same & ((1ull << lane) - 1));
    int n0 = 0;
    if (live) n0 = cnt[wid][d];
    place[r] = n0 + below;
    // (a wave's LDS operations complete in order: every lane has read the count before its last lane adds to it)
    __builtin_amdgcn_wave_barrier();
    if (live && (same >> lane) == 1ull) cnt[wid][d] = n0 + __popcll(same);
    __builtin_amdgcn_wave_barrier();
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (t0 + r * 64 + lane >= N) continue;
    const int d = (int)(key[r] >> shift) & (kRadix - 1);
    int p = base[d] + place[r];
    for (int w = 0; w < wid; ++w) p += cnt[w][d];
    kout[p] = key[r];
    vout[p] = val[r];
  }
}

// ---------------------------------------------------------------------------------------------- sums
// One subgroup of `tpr` threads (a power of two) sums one chunk of C sorted tokens for 8 * tpr columns (tpr when not
// VEC). part: [2 * chunk + slot][H] fp32; slot 0: a run that began before this chunk, slot 1: one that begins here
// and goes on. run_start / run_end of the ids found are written by the first column block.
template <typename T, typename TO, bool VEC>
__global__ __launch_bounds__(256) void embed_sum_kernel(const T* __restrict__ g, const uint32_t* __restrict__ skey,
                                                        const int* __restrict__ order, int64_t N, int V, int H, int C,
                                                        int tpr, float scale, int accumulate, TO* __restrict__ dw,
                                                        float* __restrict__ part, int* __restrict__ run_start,
                                                        int* __restrict__ run_end) {
  constexpr int W = VEC ? 8 : 1;
  constexpr int U = sizeof(T) == 4 ? 4 : 8;  // rows in flight
  const int sub = threadIdx.x / tpr, ln = threadIdx.x & (tpr - 1);
  const int64_t chunk = (int64_t)blockIdx.x * (256 / tpr) + sub;
  const int64_t p0 = chunk * C;
  if (p0 >= N) return;
  const int64_t p1 = p0 + C < N ? p0 + C : N;
  const int col = ((int)blockIdx.y * tpr + ln) * W;
  const bool on = col < H;
  const int cc = on ? col : 0;
  const bool mark = blockIdx.y == 0 && ln == 0;

  uint32_t cur = skey[p0];
  if (cur >= (uint32_t)V) return;
  bool head = p0 > 0 && skey[p0 - 1] == cur;  // the current run began in an earlier chunk
  if (mark && !head) run_start[cur] = (int)p0;
  float acc[W];
#pragma unroll
  for (int i = 0; i < W; ++i) acc[i] = 0.f;

  auto flush = [&](uint32_t key, bool open) {  // open: the run goes on behind this chunk
    if (!on) return;
    if (head || open) {
      float* o = part + (2 * chunk + (head ? 0 : 1)) * H + cc;
#pragma unroll
      for (int i = 0; i < W; ++i) o[i] = acc[i];
      return;
    }
    TO* o = dw + (int64_t)key * H + cc;
    float f[8];
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = 0.f;
      if (accumulate) Elem<TO>::unpack(load8(o), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = fmaf(acc[i], scale, f[i]);
      store8(o, f);
    } else {
      f[0] = accumulate ? Elem<TO>::to_float(o[0]) : 0.f;
      o[0] = Elem<TO>::from_float(fmaf(acc[0], scale, f[0]));
    }
  };

  uint32_t nkey[U];
  int nrow[U];
  auto fetch = [&](int64_t p) {  // keys and rows of the U tokens from p on (the chunk's last one where it ends)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t pp = p + u < p1 ? p + u : p1 - 1;
      nkey[u] = skey[pp];
      nrow[u] = order[pp];
    }
  };
  fetch(p0);
  for (int64_t p = p0; p < p1; p += U) {
    uint32_t key[U];
    int64_t row[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      key[u] = nkey[u];
      row[u] = nrow[u];
    }
    if constexpr (VEC) {
      typename Elem<T>::Raw x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = load8_nt(g + row[u] * H + cc);
      if (p + U < p1) fetch(p + U);  // under the rows' loads
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p + u >= p1) break;
        if (key[u] != cur) {
          flush(cur, false);
          if (mark) run_end[cur] = (int)(p + u);
          cur = key[u];
          if (cur >= (uint32_t)V) return;  // only dropped ids follow
          head = false;
          if (mark) run_start[cur] = (int)(p + u);
#pragma unroll
          for (int i = 0; i < W; ++i) acc[i] = 0.f;
        }
        float f[8];
        Elem<T>::unpack(x[u], f);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += f[i];
      }
    } else {
      float x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = Elem<T>::to_float(g[row[u] * H + cc]);
      if (p + U < p1) fetch(p + U);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (p + u >= p1) break;
        if (key[u] != cur) {
          flush(cur, false);
          if (mark) run_end[cur] = (int)(p + u);
          cur = key[u];
          if (cur >= (uint32_t)V) return;
          head = false;
          if (mark) run_start[cur] = (int)(p + u);
          acc[0] = 0.f;
        }
        acc[0] += x[u];
      }
    }
  }
  const bool open = p1 < N && skey[p1] == cur;
  flush(cur, open);
  if (mark && !open) run_end[cur] = (int)p1;
}

// What the sums leave. Workgroups below `zero_blocks` write the zeros of vocabulary rows without a token, kZeroRows
// rows a wave (none when accumulating), past the caches (32768 tokens in 128256 x 4096 bf16: 313 -> 280 us in all). The others take a chunk each, 256 vectors of columns: if a run begins in it and goes
// on behind it, they add its partial rows in chunk order and store the row.
constexpr int kZeroRows = 4;
template <typename TO, bool VEC>
__global__ __launch_bounds__(256) void embed_finish_kernel(const float* __restrict__ part, const uint32_t* __restrict__ skey,
                                                           const int* __restrict__ run_start,
                                                           const int* __restrict__ run_end, int64_t N, int V, int H, int C,
                                                           float scale, int accumulate, int zero_blocks, int pieces,
                                                           TO* __restrict__ dw) {
  constexpr int W = VEC ? 8 : 1;
  const int tid = threadIdx.x, lane = tid & 63;
  if ((int)blockIdx.x < zero_blocks) {
    const int64_t v0 = ((int64_t)blockIdx.x * 4 + (tid >> 6)) * kZeroRows;
    const bool none = lane < kZeroRows && v0 + lane < V && run_start[v0 + lane] < 0;
    uint64_t rows = __ballot(none);
    const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    while (rows) {
      TO* o = dw + (v0 + __builtin_ctzll(rows)) * H;
      rows &= rows - 1;
      for (int c = lane * W; c < H; c += 64 * W) {
        if constexpr (VEC)
          store8_nt(o + c, z);
        else
          o[c] = Elem<TO>::from_float(0.f);
      }
    }
    return;
  }
  const int64_t job = (int64_t)blockIdx.x - zero_blocks;
  const int64_t c0 = pieces == 1 ? job : job / pieces;
  const int c = ((int)(job - c0 * pieces) * 256 + tid) * W;
  const int64_t next = (c0 + 1) * C;
  if (next >= N || c >= H) return;
  const uint32_t key = skey[next];
  if (key >= (uint32_t)V || skey[next - 1] != key || run_start[key] < c0 * C) return;
  const int64_t c1 = (run_end[key] - 1) / C;
  const float* p = part + (2 * c0 + 1) * H + c;
  float acc[8];
#pragma unroll
  for (int i = 0; i < W; ++i) acc[i] = p[i];
  p = part + 2 * (c0 + 1) * H + c;
  const int64_t st = 2 * (int64_t)H;
  int64_t k = c0 + 1;
  for (; k + 8 <= c1 + 1; k += 8, p += 8 * st) {
    float x[8][W];
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int i = 0; i < W; ++i) x[u][i] = p[u * st + i];
#pragma unroll
    for (int u = 0; u < 8; ++u)
#pragma unroll
      for (int i = 0; i < W; ++i) acc[i] += x[u][i];
  }
  for (; k <= c1; ++k, p += st)
#pragma unroll
    for (int i = 0; i < W; ++i) acc[i] += p[i];
  TO* o = dw + (int64_t)key * H + c;
  if constexpr (VEC) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = 0.f;
    if (accumulate) Elem<TO>::unpack(load8(o), f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = fmaf(acc[i], scale, f[i]);
    store8(o, f);
  } else {
    o[0] = Elem<TO>::from_float(fmaf(acc[0], scale, accumulate ? Elem<TO>::to_float(o[0]) : 0.f));
  }
}

// ---------------------------------------------------------------------------------------------- few tokens
// grid (ceil(V / kSmallRows), column blocks of tpr vectors). A workgroup's rows lie gridDim.x apart: the most frequent
// ids are neighbours in most vocabularies, and one workgroup with all of them would be the kernel's time. The tokens of
// its rows are listed, ordered by (row, token) by counting, and summed row by row by a subgroup of `tpr` threads (a
// power of two).
template <typename T, typename TO, typename I, bool VEC>
__global__ __launch_bounds__(256) void embed_small_kernel(const I* __restrict__ ids, const T* __restrict__ g, int N,
                                                          int64_t v0, int valid, int V, int H, int tpr, float scale,
                                                          int accumulate, TO* __restrict__ dw, int* __restrict__ err) {
  constexpr int W = VEC ? 8 : 1, U = 8;
  __shared__ int found[kSmallMax], sorted[kSmallMax];  // row in the workgroup << 16 | token
  __shared__ int start[kSmallRows + 1];
  __shared__ int count;
  const int tid = threadIdx.x;
  const unsigned me0 = blockIdx.x, stride = gridDim.x;
  if (tid == 0) count = 0;
  if (tid <= kSmallRows) start[tid] = 0;
  __syncthreads();
  for (int i = tid; i < N; i += 256) {
    const uint32_t k = local_key(ids, i, v0, valid, V, me0 == 0 && blockIdx.y == 0 ? err : nullptr);
    const unsigned l = k / stride;
    if (k < (uint32_t)V && k - l * stride == me0) found[atomicAdd(&count, 1)] = (int)(l << 16) | i;
  }
  __syncthreads();
  const int n = count;
  if (n == 0 && accumulate) return;
  for (int e = tid; e < n; e += 256) {  // distinct words: the order in which they were found does not matter
    const int me = found[e];
    int at = 0;
    for (int j = 0; j < n; ++j) at += found[j] < me;
    sorted[at] = me;
  }
  if (tid <= kSmallRows) {
    int at = 0;
    for (int j = 0; j < n; ++j) at += found[j] < tid << 16;
    start[tid] = at;
  }
  __syncthreads();
  const int sub = tid / tpr, ln = tid & (tpr - 1), subs = 256 / tpr;
  const int col = ((int)blockIdx.y * tpr + ln) * W;
  if (col >= H) return;
  for (int l = sub; l < kSmallRows && me0 + (int64_t)l * stride < V; l += subs) {
    const int e0 = start[l], e1 = start[l + 1];
    if (e0 == e1 && accumulate) continue;
    float acc[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    for (int e = e0; e < e1; e += U) {
      if constexpr (VEC) {
        typename Elem<T>::Raw x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) x[u] = load8(g + (int64_t)(sorted[e + u < e1 ? e + u : e1 - 1] & 0xffff) * H + col);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float f[8];
          Elem<T>::unpack(x[u], f);
          if (e + u < e1)
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] += f[i];
        }
      } else {
        float x[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
          x[u] = Elem<T>::to_float(g[(int64_t)(sorted[e + u < e1 ? e + u : e1 - 1] & 0xffff) * H + col]);
#pragma unroll
        for (int u = 0; u < U; ++u) acc[0] += e + u < e1 ? x[u] : 0.f;
      }
    }
    TO* o = dw + (me0 + (int64_t)l * stride) * H + col;
    if constexpr (VEC) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = 0.f;
      if (accumulate) Elem<TO>::unpack(load8(o), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = fmaf(acc[i], scale, f[i]);
      store8_nt(o, f);
    } else {
      o[0] = Elem<TO>::from_float(fmaf(acc[0], scale, accumulate ? Elem<TO>::to_float(o[0]) : 0.f));
    }
  }
}

// ---------------------------------------------------------------------------------------------- launches
template <typename T, typename I>
static void launch_fwd(const void* ids, const void* w, void* y, int64_t N, int V, int H, int64_t v0, float scale,
                       bool vec, int* err, hipStream_t stream) {
  // about 2048 items a workgroup, but short batches spread over the chip
  const int per = vec ? H / 8 : H;
  int rows = per >= 2048 ? 1 : 2048 / per;
  if ((N + rows - 1) / rows < 512) rows = (int)((N + 511) / 512);
  if (rows < 1) rows = 1;
  const unsigned grid = (unsigned)((N + rows - 1) / rows);
  // outputs that exceed the caches go past them, which leaves those to the table's frequent rows (32768 x 4096 bf16,
  // 268 MB: 82 -> 62 us); smaller ones stay for the layer that reads them next
  const bool nt = vec && N * (int64_t)H * (int64_t)sizeof(T) > (128LL << 20);
#define LLMT_EMB_FWD(VEC, NT) \
  embed_fwd_kernel<T, I, VEC, NT><<<grid, 256, 0, stream>>>((const I*)ids, (const T*)w, (T*)y, N, V, H, v0, scale, rows, err)
  if (nt)
    LLMT_EMB_FWD(true, true);
  else if (vec)
    LLMT_EMB_FWD(true, false);
  else
    LLMT_EMB_FWD(false, false);
#undef LLMT_EMB_FWD
}

template <typename T, typename TO>
static void launch_small(const void* ids, int ids64, const void* g, int N, int64_t v0, int valid, int V, int H, bool vec,
                         float scale, int accumulate, void* dw, int* err, hipStream_t stream) {
  const int per = vec ? H / 8 : H;
  int tpr = 1;
  while (tpr < 256 && tpr < per) tpr <<= 1;
  const dim3 grid((unsigned)((V + kSmallRows - 1) / kSmallRows), (unsigned)((per + tpr - 1) / tpr));
#define LLMT_EMB_SMALL(I, VEC)                                                                                      \
  embed_small_kernel<T, TO, I, VEC><<<grid, 256, 0, stream>>>((const I*)ids, (const T*)g, N, v0, valid, V, H, tpr, scale, \
                                                              accumulate, (TO*)dw, err)
  if (ids64 && vec)
    LLMT_EMB_SMALL(int64_t, true);
  else if (ids64)
    LLMT_EMB_SMALL(int64_t, false);
  else if (vec)
    LLMT_EMB_SMALL(int, true);
  else
    LLMT_EMB_SMALL(int, false);
#undef LLMT_EMB_SMALL
}

template <typename T, typename TO>
static void launch_sum(const void* g, const uint32_t* skey, const int* order, int64_t N, int V, int H, int C, bool vec,
                       float scale, int accumulate, void* dw, float* part, int* rs, int* re, hipStream_t stream) {
  const int per = vec ? H / 8 : H;
  int tpr = 1;
  while (tpr < 256 && tpr < per) tpr <<= 1;
  const int64_t chunks = (N + C - 1) / C;
  const dim3 grid((unsigned)((chunks + 256 / tpr - 1) / (256 / tpr)), (unsigned)((per + tpr - 1) / tpr));
  const int pieces = (per + 255) / 256;
  const int zero_blocks = accumulate ? 0 : (V + 4 * kZeroRows - 1) / (4 * kZeroRows);
  const unsigned gf = (unsigned)(zero_blocks + chunks * pieces);
  if (vec) {
    embed_sum_kernel<T, TO, true><<<grid, 256, 0, stream>>>((const T*)g, skey, order, N, V, H, C, tpr, scale, accumulate,
                                                           (TO*)dw, part, rs, re);
    embed_finish_kernel<TO, true><<<gf, 256, 0, stream>>>(part, skey, rs, re, N, V, H, C, scale, accumulate, zero_blocks,
                                                              pieces, (TO*)dw);
  } else {
    embed_sum_kernel<T, TO, false><<<grid, 256, 0, stream>>>((const T*)g, skey, order, N, V, H, C, tpr, scale,
                                                            accumulate, (TO*)dw, part, rs, re);
    embed_finish_kernel<TO, false><<<gf, 256, 0, stream>>>(part, skey, rs, re, N, V, H, C, scale, accumulate, zero_blocks,
                                                              pieces, (TO*)dw);
  }
}

// tokens per chunk: 64 keeps the partial rows few; short batches are cut finer, so that their chunks still reach
// every CU
static int chunk_of(int64_t N) { return N > 16384 ? 64 : N > 2048 ? 32 : 16; }

struct EmbedWs {
  int64_t keys, vals, hist, start, end, part, total;  // offsets in 4-byte words
  int nblk, passes;
  bool rank;
};
static EmbedWs embed_ws(int64_t N, int V, int H) {
  EmbedWs w{};
  if (N <= kSmallMax) return w;  // (none)
  int bits = 1;
  while (bits < 31 && ((int64_t)V >> bits) > 0) ++bits;  // keys 0 .. V
  w.rank = N <= kRankMax && bits <= 19;
  w.passes = (bits + kRadixBits - 1) / kRadixBits;
  w.nblk = (int)((N + kTile - 1) / kTile);
  auto up = [](int64_t n) { return (n + 63) / 64 * 64; };
  w.keys = 0;                                  // two buffers each
  w.vals = w.keys + 2 * up(N);
  w.hist = w.vals + 2 * up(N);
  const int64_t hist = w.rank ? (int64_t)((N + kRankTile - 1) / kRankTile) * N : kRadix * ((int64_t)w.nblk + 1);
  w.start = w.hist + up(hist);
  w.end = w.start + up(V);
  w.part = w.end + up(V);
  const int C = chunk_of(N);
  w.total = w.part + 2 * ((N + C - 1) / C) * (int64_t)H;
  return w;
}

template <typename I>
static void sort_tokens(const I* ids, int64_t N, int64_t v0, int valid, int V, const EmbedWs& w, int* ws, int* err, uint32_t*& skey,
                        int*& order, hipStream_t stream) {
  const int64_t Np = (N + 63) / 64 * 64;
  uint32_t* k[2] = {(uint32_t*)(ws + w.keys), (uint32_t*)(ws + w.keys + Np)};
  int* v[2] = {ws + w.vals, ws + w.vals + Np};
  int *hist = ws + w.hist, *rs = ws + w.start;
  if (w.rank) {
    const int parts = (int)((N + kRankTile - 1) / kRankTile);
    const int64_t gx = (N + 255) / 256, gc = ((int64_t)V + 2047) / 2048 / parts;  // (clearing: 8 words a thread)
    embed_rank_kernel<I><<<dim3((unsigned)(gx > gc ? gx : gc), (unsigned)parts), 256, 0, stream>>>(ids, (int)N, v0, valid, V, hist,
                                                                                                rs, err);
    embed_place_kernel<I><<<(unsigned)((N + 255) / 256), 256, 0, stream>>>(ids, (int)N, v0, valid, V, hist, parts, k[0], v[0]);
    skey = k[0];
    order = v[0];
    return;
  }
  for (int p = 0; p < w.passes; ++p) {
    const int shift = p * kRadixBits;
    const uint32_t* kin = k[(p + 1) & 1];
    const int* vin = v[(p + 1) & 1];
    if (p == 0)
      embed_hist_kernel<I, true><<<(unsigned)w.nblk, 256, 0, stream>>>(ids, nullptr, N, v0, valid, V, 0, hist, w.nblk, rs, err);
    else
      embed_hist_kernel<I, false><<<(unsigned)w.nblk, 256, 0, stream>>>(ids, kin, N, v0, valid, V, shift, hist, w.nblk,
                                                                        nullptr, nullptr);
    if (w.nblk > kScanSelf) embed_scan_kernel<<<kRadix / 64, 64, 0, stream>>>(hist, w.nblk);
    if (p == 0)
      embed_scatter_kernel<I, true><<<(unsigned)w.nblk, 256, 0, stream>>>(ids, nullptr, nullptr, N, v0, valid, V, 0, hist,
                                                                          w.nblk, k[0], v[0]);
    else
      embed_scatter_kernel<I, false><<<(unsigned)w.nblk, 256, 0, stream>>>(ids, kin, vin, N, v0, valid, V, shift, hist,
                                                                           w.nblk, k[p & 1], v[p & 1]);
  }
  skey = k[(w.passes + 1) & 1];
  order = v[(w.passes + 1) & 1];
}

}  // namespace llmt

using namespace llmt;

extern "C" hipError_t llmt_embedding_fwd(const void* ids, int ids64, const void* w, void* y, int type, int64_t N, int V,
                                         int H, int64_t v0, float scale, int* err, hipStream_t stream) {
  if (N <= 0 || H <= 0) return hipSuccess;
  const bool vec = H % 8 == 0 && ((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(y)) & 15) == 0;
#define LLMT_EMB(T)                                                                              \
  if (ids64)                                                                                     \
    launch_fwd<T, int64_t>(ids, w, y, N, V, H, v0, scale, vec, err, stream);                     \
  else                                                                                           \
    launch_fwd<T, int>(ids, w, y, N, V, H, v0, scale, vec, err, stream);
  switch (type) {
    case kElemBf16: { LLMT_EMB(bf16) } break;
    case kElemF16: { LLMT_EMB(__half) } break;
    case kElemF32: { LLMT_EMB(float) } break;
    default: return hipErrorInvalidValue;
  }
#undef LLMT_EMB
  return hipGetLastError();
}

// 4-byte words of workspace llmt_embedding_bwd needs
extern "C" int64_t llmt_embedding_bwd_ws(int64_t N, int V, int H) { return embed_ws(N, V, H).total; }

extern "C" hipError_t llmt_embedding_bwd(const void* ids, int ids64, const void* g, int gtype, void* dw, int wtype,
                                         int64_t N, int valid, int V, int H, int64_t v0, float scale, int accumulate, int* ws,
                                         int* err, hipStream_t stream) {
  if (V <= 0 || H <= 0 || N <= 0 || N >= (1LL << 31) - kTile) return hipErrorInvalidValue;
  const EmbedWs w = embed_ws(N, V, H);
  const bool vec = H % 8 == 0 && ((reinterpret_cast<uintptr_t>(g) | reinterpret_cast<uintptr_t>(dw)) & 15) == 0;
  uint32_t* skey = nullptr;
  int* order = nullptr;
  const bool small = N <= kSmallMax;
  if (!small && ids64)
    sort_tokens((const int64_t*)ids, N, v0, valid, V, w, ws, err, skey, order, stream);
  else if (!small)
    sort_tokens((const int*)ids, N, v0, valid, V, w, ws, err, skey, order, stream);
  const int C = chunk_of(N);
  float* part = reinterpret_cast<float*>(ws + w.part);
  int *rs = ws + w.start, *re = ws + w.end;
#define LLMT_EMB(T, TO)                                                                                                \
  small ? launch_small<T, TO>(ids, ids64, g, (int)N, v0, valid, V, H, vec, scale, accumulate, dw, err, stream)        \
        : launch_sum<T, TO>(g, skey, order, N, V, H, C, vec, scale, accumulate, dw, part, rs, re, stream)
  // the gradient's type, into a buffer of the same type or of fp32
  if (gtype == kElemBf16 && wtype == kElemBf16) LLMT_EMB(bf16, bf16);
  else if (gtype == kElemBf16 && wtype == kElemF32) LLMT_EMB(bf16, float);
  else if (gtype == kElemF16 && wtype == kElemF16) LLMT_EMB(__half, __half);
  else if (gtype == kElemF16 && wtype == kElemF32) LLMT_EMB(__half, float);
  else if (gtype == kElemF32 && wtype == kElemF32) LLMT_EMB(float, float);
  else if (gtype == kElemF32 && wtype == kElemBf16) LLMT_EMB(float, bf16);
  else if (gtype == kElemF32 && wtype == kElemF16) LLMT_EMB(float, __half);
  else return hipErrorInvalidValue;
#undef LLMT_EMB
  return hipGetLastError();
}
