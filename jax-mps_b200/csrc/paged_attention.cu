// Attention of one new token per sequence over a cache of pages (custom call b200.paged_attention).
//
//   out[b, h] = sum_j w_j v_j,  w = softmax_j(scale * q[b, h] . k_j)  over the visible positions j of sequence b
//
// The token stands at position p: the last cached one, or, where its own key and value are given beside the cache, the one
// behind them. Position j is visible when j <= p and (no window, p - j < window, or j < sinks). A row that sees nothing is zero.
// Sums, maxima and the weights' normaliser are held in 32 bits; the running maximum m, sum l and output o of a part of the
// positions are joined with those of the others by o = sum o_i 2^(m_i - m) / sum l_i 2^(m_i - m).
//
// Bound by memory: the visible keys and values are read once, 4 bytes of 16-bit data for each feature, position and key-value
// head, and take part in 4 * group operations each.
#include <algorithm>
#include <type_traits>

#include "operators.cuh"

namespace b200 {
namespace {

constexpr int kPartHeads = 8;         // query heads that a block takes along
constexpr int kMinPart = 128;         // positions: a shorter part is not worth a place in the second pass
constexpr int kParts = kSMs * 4;      // parts that fill the chip

struct Paged {
  const void *q, *cache, *fresh;
  const int *table, *lengths;
  void* out;
  float* parts;                       // per part and query head: dim outputs, the maximum and the sum
  int* first;                         // per sequence: its first part and how many it has
  int batch, heads, kv_heads, dim, group, chunks, pages, page, width, window, sinks, has_new;
  long long plane;                    // elements between the keys and the values of a layer
  float scale;                        // of the scores, times log2(e)
};

// Positions of a sequence as a row: the sinks that lie in front of the window, then the window, then the token itself.
struct Span {
  int seen;                           // how many cached ones are visible
  int sinks, start;                   // place i < sinks is position i, another position start + i - sinks
};
__device__ __forceinline__ Span span_of(const Paged& a, int b) {
  long long most = (long long)a.width * a.page;
  int n = a.lengths[b];
  n = n < 0 ? 0 : n > most ? (int)most : n;
  Span s;
  s.start = 0;
  if (a.window > 0) {
    const int p = a.has_new ? n : n - 1;
    s.start = max(0, p - a.window + 1);
    s.start = min(s.start, n);        // a window of one sees the token itself alone
  }
  s.sinks = min(a.sinks, s.start);
  s.seen = n - s.start + s.sinks;
  return s;
}

struct Part {
  int b, index, count;                // the sequence, which of its parts, how many it has
  int from, to;                       // places of the row, the token itself included
  int place;                          // where the part's result goes
  Span span;
};

// Which part a block works on. All parts have the same number of positions, so that a long sequence among short ones is spread
// over the chip: every block adds up the sequences' lengths for itself (they are on the device only). False: no such part.
template <int THREADS>
__device__ __forceinline__ bool part_of(const Paged& a, int want, Part& r) {
  __shared__ long long sums[THREADS / 32 + 1];
  __shared__ int found[4];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.batch + THREADS - 1) / THREADS, lo = min(a.batch, tid * per), hi = min(a.batch, lo + per);
  long long mine = 0;
  for (int b = lo; b < hi; ++b) mine += span_of(a, b).seen + a.has_new;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xFFFFFFFFu, mine, o);
  if (lane == 0) sums[warp] = mine;
  if (tid < 4) found[tid] = -1;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) total += sums[w];
  const int room = max(1, kParts / a.chunks);
  const long long even = (total + room - 1) / room;
  const int len = (int)((min(max((long long)kMinPart, even), 1LL << 30) + 63) / 64 * 64);
  // the part's sequence: an inclusive sum over the threads' stretches of the batch
  int parts = 0;
  for (int b = lo; b < hi; ++b) parts += max(1, (span_of(a, b).seen + a.has_new + len - 1) / len);
  int upto = parts;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
    if (lane >= o) upto += v;
  }
  __syncthreads();
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  for (int w = 0; w < warp; ++w) upto += (int)sums[w];
  int at = upto - parts;
  if (want >= at && want < upto)
    for (int b = lo; b < hi; ++b) {
      const int n = max(1, (span_of(a, b).seen + a.has_new + len - 1) / len);
      if (want < at + n) { found[0] = b; found[1] = want - at; found[2] = n; break; }
      at += n;
    }
  __syncthreads();
  if (found[0] < 0) return false;
  r.b = found[0];
  r.index = found[1];
  r.count = found[2];
  r.span = span_of(a, r.b);
  r.from = r.index * len;
  r.to = min(r.from + len, r.span.seen + a.has_new);
  r.place = want;
  return true;
}

// The first element of the keys at a place of the row, and how far behind it the values are. Null where the table names no page of
// the cache: such a position is left out.
template <typename T>
__device__ __forceinline__ const T* key_at(const Paged& a, const Part& r, int place, int kvh, long long& to_value) {
  if (place >= r.span.seen) {
    to_value = (long long)a.batch * a.kv_heads * a.dim;
    return (const T*)a.fresh + ((long long)r.b * a.kv_heads + kvh) * a.dim;
  }
  to_value = a.plane;
  const int pos = place < r.span.sinks ? place : r.span.start + place - r.span.sinks;
  const int page = a.table[(long long)r.b * a.width + pos / a.page];
  if (page < 0 || page >= a.pages) return nullptr;
  return (const T*)a.cache + (((long long)page * a.page + pos % a.page) * a.kv_heads + kvh) * a.dim;
}

// A block takes up to eight query heads of one key-value head over one part: tiles of 32 positions go to shared memory as floats,
// a warp forms the scores of two heads with a position per lane, a thread adds up one feature (or two) of the outputs.
template <typename T>
__global__ void __launch_bounds__(128) paged_simple_kernel(const __grid_constant__ Paged a) {
  pdl_prologue();
  extern __shared__ __align__(16) float smem[];
  const int D = a.dim, KP = D + 4, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float *ks = smem, *vs = ks + 32 * KP, *qs = vs + 32 * D, *ps = qs + kPartHeads * D, *ms = ps + 32 * kPartHeads, *ls = ms + kPartHeads, *fs = ls + kPartHeads;
  const int chunk = blockIdx.x % a.chunks, per = (a.group + kPartHeads - 1) / kPartHeads;
  const int kvh = chunk / per, h0 = kvh * a.group + chunk % per * kPartHeads, nh = min(kPartHeads, kvh * a.group + a.group - h0);
  Part r;
  if (!part_of<128>(a, blockIdx.x / a.chunks, r)) return;
  for (int i = tid; i < kPartHeads * D; i += 128) qs[i] = i < nh * D ? to_float(((const T*)a.q)[((long long)r.b * a.heads + h0) * D + i]) * a.scale : 0.f;
  if (tid < kPartHeads) { ms[tid] = neg_inf(); ls[tid] = 0.f; }
  float acc[2][kPartHeads];
#pragma unroll
  for (int h = 0; h < kPartHeads; ++h) acc[0][h] = acc[1][h] = 0.f;
  constexpr int N = Pack<T>::N;
  const int pieces = D / N;
  for (int t0 = r.from; t0 < r.to; t0 += 32) {
    __syncthreads();
    for (int i = tid; i < 32 * pieces; i += 128) {
      const int row = i / pieces, c = i % pieces * N;
      long long to_value = 0;
      const T* k = t0 + row < r.to ? key_at<T>(a, r, t0 + row, kvh, to_value) : nullptr;
      uint4 kv = {0, 0, 0, 0}, vv = kv;
      if (k) { kv = *(const uint4*)(k + c); vv = *(const uint4*)(k + to_value + c); }
      float f[N];
      unpack<T>(kv, f);
#pragma unroll
      for (int e = 0; e < N; ++e) ks[row * KP + c + e] = f[e];
      unpack<T>(vv, f);
#pragma unroll
      for (int e = 0; e < N; ++e) vs[row * D + c + e] = f[e];
    }
    long long unused;
    const bool there = t0 + lane < r.to && key_at<T>(a, r, t0 + lane, kvh, unused) != nullptr;
    __syncthreads();
    for (int h = warp; h < nh; h += 4) {
      float s = 0.f;
      for (int d = 0; d < D; d += 4) {
        const float4 k = *(const float4*)(ks + lane * KP + d), q = *(const float4*)(qs + h * D + d);
        s = fmaf(k.x, q.x, fmaf(k.y, q.y, fmaf(k.z, q.z, fmaf(k.w, q.w, s))));
      }
      if (!there) s = neg_inf();
      const float was = ms[h], m = fmaxf(was, warp_max(s)), ref = m == neg_inf() ? 0.f : m;
      const float p = there ? exp2f(s - ref) : 0.f, sum = warp_sum(p), keep = exp2f(was - ref);
      ps[lane * kPartHeads + h] = p;
      __syncwarp();
      if (lane == 0) { ms[h] = m; ls[h] = ls[h] * keep + sum; fs[h] = keep; }
    }
    __syncthreads();
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int d = tid + 128 * part;
      if (d < D) {
        for (int h = 0; h < nh; ++h) acc[part][h] *= fs[h];
        const int n = min(32, r.to - t0);
        for (int t = 0; t < n; ++t) {
          const float v = vs[t * D + d];
#pragma unroll
          for (int h = 0; h < kPartHeads; ++h) if (h < nh) acc[part][h] = fmaf(ps[t * kPartHeads + h], v, acc[part][h]);
        }
      }
    }
  }
  __syncthreads();
  if (r.index == 0 && chunk == 0 && tid == 0) { a.first[2 * r.b] = r.place; a.first[2 * r.b + 1] = r.count; }
  for (int part = 0; part < 2; ++part) {
    const int d = tid + 128 * part;
    if (d >= D) continue;
#pragma unroll
    for (int h = 0; h < kPartHeads; ++h) {
      if (h >= nh) continue;
      if (r.count == 1) ((T*)a.out)[((long long)r.b * a.heads + h0 + h) * D + d] = from_float<T>(ls[h] > 0.f || ls[h] != ls[h] ? acc[part][h] / ls[h] : 0.f);
      else a.parts[((long long)r.place * a.heads + h0 + h) * (D + 2) + d] = acc[part][h];
    }
  }
  if (r.count > 1 && tid < nh) {
    float* ml = a.parts + ((long long)r.place * a.heads + h0 + tid) * (D + 2) + D;
    ml[0] = ms[tid];
    ml[1] = ls[tid];
  }
}

// ---- 16-bit data on the tensor cores -------------------------------------------------------------------
// A warp streams 16 positions at a time through a ring of its own in shared memory (cp.async, no block barrier in the loop), and
// takes 8 * NT query heads along: scores^T [16 positions, 8 heads] = K Q^T and outputs^T [features, 8 heads] += V^T P^T by
// mma.sync.m16n8k16, whose eight columns fit the heads that share a key-value head (with heads as rows half of every product and of
// the accumulators would be padding). The scores' fragments become the weights' by an 8 x 8 transpose within the warp. The weights go
// into the second product as two 16-bit pieces, their rounding and what it leaves, so that they lose nothing beside the result's own
// rounding: the products are not what bounds this kernel. The warps of a block and then the parts of a sequence are joined at the end.
constexpr int kWarps = 4;

template <int DP, int NT>
struct Ring {
  static constexpr int CHUNKS = DP / 8;                              // pieces of 16 bytes in a row
  static constexpr int TILE = 16 * DP * 2, STAGE = 2 * TILE;         // bytes of the keys, of keys and values
  static constexpr int STAGES = DP <= 128 ? 3 : 3;
  static constexpr int BYTES = kWarps * STAGES * STAGE;
  static constexpr int JOIN = kWarps * 8 * NT * (DP + 2) * 4;
  static constexpr int SMEM = BYTES > JOIN ? BYTES : JOIN;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Two floats as a pair of 16-bit values, rounded to nearest even; `low` what that leaves of them, rounded again.
template <typename T>
__device__ __forceinline__ uint32_t pair16(float x, float y, uint32_t& low) {
  if (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y), l = __floats2bfloat162_rn(x - __low2float(h), y - __high2float(h));
    low = *reinterpret_cast<const uint32_t*>(&l);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(x, y), l = __floats2half2_rn(x - __low2float(h), y - __high2float(h));
  low = *reinterpret_cast<const uint32_t*>(&l);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float power(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float column_max(float v) {             // over the lanes of the same quarter: the positions of a head
  v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 16));
}

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(kWarps * 32) paged_mma_kernel(const __grid_constant__ Paged a) {
  pdl_prologue();
  using R = Ring<DP, NT>;
  extern __shared__ __align__(128) uint8_t ring[];
  constexpr int HEADS = 8 * NT, S = R::STAGES;
  const int D = a.dim, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int chunk = blockIdx.x % a.chunks, per = (a.group + HEADS - 1) / HEADS;
  const int kvh = chunk / per, h0 = kvh * a.group + chunk % per * HEADS, nh = min(HEADS, kvh * a.group + a.group - h0);
  Part r;
  if (!part_of<kWarps * 32>(a, blockIdx.x / a.chunks, r)) return;

  // Q^T as the second operand: lane holds head lane / 4, features 2 (lane % 4) + {0, 1} and eight further of each 16
  uint32_t q[DP / 16][NT][2];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int h = t * 8 + lane / 4;
    const T* src = (const T*)a.q + ((long long)r.b * a.heads + h0 + h) * D;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int d = k * 16 + i * 8 + lane % 4 * 2;
        q[k][t][i] = h < nh && d < D ? *(const uint32_t*)(src + d) : 0u;
      }
  }
  const int ntiles = (r.to - r.from + 15) / 16;
  const uint32_t base = smem_u32(ring) + warp * S * R::STAGE;
  // where a position's keys are: lanes 0-15 look up one each, in front of the tile that asks for them
  struct Where { const T* key; long long to_value; };
  auto locate = [&](int tile) {
    Where w = {nullptr, 0};
    const int place = r.from + tile * 16 + (lane & 15);
    if (tile < ntiles && place < r.to) w.key = key_at<T>(a, r, place, kvh, w.to_value);
    return w;
  };
  auto fetch = [&](const Where& w, int slot) -> uint32_t {          // gives which of the tile's positions are there
    const uint32_t to = base + slot * R::STAGE;
#pragma unroll
    for (int i = 0; i < R::CHUNKS / 2; ++i) {
      const int piece = lane + 32 * i, row = piece / R::CHUNKS, c = piece % R::CHUNKS;
      const T* key = (const T*)__shfl_sync(0xFFFFFFFFu, (unsigned long long)w.key, row);
      const long long to_value = __shfl_sync(0xFFFFFFFFu, w.to_value, row);
      const bool real = key != nullptr && c * 8 < D;
      const T *ksrc = real ? key + c * 8 : (const T*)a.q, *vsrc = real ? ksrc + to_value : (const T*)a.q;
      const uint32_t dst = to + row * (DP * 2) + ((c ^ (row & 7)) << 4), bytes = real ? 16 : 0;
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(ksrc), "r"(bytes) : "memory");
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + R::TILE), "l"(vsrc), "r"(bytes) : "memory");
    }
    return __ballot_sync(0xFFFFFFFFu, w.key != nullptr) & 0xFFFFu;
  };
  float m[NT][2], l[NT][2], o[DP / 16][NT][4];                      // heads 2 (lane % 4) + {0, 1} of each eight
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t][0] = m[t][1] = neg_inf();
    l[t][0] = l[t][1] = 0.f;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) o[k][t][0] = o[k][t][1] = o[k][t][2] = o[k][t][3] = 0.f;
  }
  uint32_t there[S];
  Where next = locate(warp);
#pragma unroll
  for (int s = 0; s < S - 1; ++s) {
    there[s] = fetch(next, s);
    asm volatile("cp.async.commit_group;" ::: "memory");
    next = locate(warp + (s + 1) * kWarps);
  }
  for (int tile0 = warp; tile0 < ntiles; tile0 += S * kWarps) {
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const int tile = tile0 + s * kWarps;
      if (tile < ntiles) {
        constexpr int AHEAD = S - 1;
        there[(s + AHEAD) % S] = fetch(next, (s + AHEAD) % S);
        asm volatile("cp.async.commit_group;" ::: "memory");
        next = locate(tile + S * kWarps);
        asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
        __syncwarp();
        const uint32_t kt = base + s * R::STAGE, vt = kt + R::TILE;
        // scores: rows are positions lane / 4 and eight further, columns heads
        float sc[NT][4];
#pragma unroll
        for (int t = 0; t < NT; ++t) sc[t][0] = sc[t][1] = sc[t][2] = sc[t][3] = 0.f;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          uint32_t f[4];
          const int row = lane & 15, c = 2 * k + (lane >> 4);
          ldmatrix4(f, kt + row * (DP * 2) + ((c ^ (row & 7)) << 4));
#pragma unroll
          for (int t = 0; t < NT; ++t) mma16<T>(sc[t], f, q[k][t][0], q[k][t][1]);
        }
        const uint32_t seen = there[s] >> (lane / 4);
        uint32_t hi[NT][2], lo[NT][2];
        bool grown = false;
        float keep[NT][2];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            sc[t][i] = seen & 1u ? sc[t][i] * a.scale : neg_inf();
            sc[t][2 + i] = seen & 0x100u ? sc[t][2 + i] * a.scale : neg_inf();
            const float top = fmaxf(m[t][i], column_max(fmaxf(sc[t][i], sc[t][2 + i])));
            grown |= top > m[t][i];
            const float ref = top == neg_inf() ? 0.f : top;
            keep[t][i] = power(m[t][i] - ref);
            m[t][i] = top;
            sc[t][i] = power(sc[t][i] - ref);
            sc[t][2 + i] = power(sc[t][2 + i] - ref);
            l[t][i] = l[t][i] * keep[t][i] + sc[t][i] + sc[t][2 + i];
          }
          hi[t][0] = transpose8(pair16<T>(sc[t][0], sc[t][1], lo[t][0]));
          hi[t][1] = transpose8(pair16<T>(sc[t][2], sc[t][3], lo[t][1]));
          lo[t][0] = transpose8(lo[t][0]);
          lo[t][1] = transpose8(lo[t][1]);
        }
        if (__any_sync(0xFFFFFFFFu, grown)) {
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              o[k][t][0] *= keep[t][0];
              o[k][t][1] *= keep[t][1];
              o[k][t][2] *= keep[t][0];
              o[k][t][3] *= keep[t][1];
            }
        }
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          uint32_t f[4];
          const int row = (lane & 7) + (lane >> 4) * 8, c = 2 * k + ((lane >> 3) & 1);
          ldmatrix4_trans(f, vt + row * (DP * 2) + ((c ^ (row & 7)) << 4));
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma16<T>(o[k][t], f, hi[t][0], hi[t][1]);
            mma16<T>(o[k][t], f, lo[t][0], lo[t][1]);
          }
        }
        __syncwarp();                                               // the tile's place may be filled again
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncthreads();
  // the block's warps are joined through the ring's memory: [warp][head][feature], then maxima and sums
  float* os = reinterpret_cast<float*>(ring);
  float* ms = os + kWarps * HEADS * DP;
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[t][i] += __shfl_xor_sync(0xFFFFFFFFu, l[t][i], 4);
      l[t][i] += __shfl_xor_sync(0xFFFFFFFFu, l[t][i], 8);
      l[t][i] += __shfl_xor_sync(0xFFFFFFFFu, l[t][i], 16);
      const int h = t * 8 + lane % 4 * 2 + i;
      if (lane < 4) { ms[(warp * HEADS + h) * 2] = m[t][i]; ms[(warp * HEADS + h) * 2 + 1] = l[t][i]; }
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        os[(warp * HEADS + h) * DP + k * 16 + lane / 4] = o[k][t][i];
        os[(warp * HEADS + h) * DP + k * 16 + lane / 4 + 8] = o[k][t][2 + i];
      }
    }
  __syncthreads();
  if (r.index == 0 && chunk == 0 && tid == 0) { a.first[2 * r.b] = r.place; a.first[2 * r.b + 1] = r.count; }
  for (int i = tid; i < nh * DP; i += kWarps * 32) {
    const int h = i / DP, d = i % DP;
    if (d >= D) continue;
    float top = neg_inf();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ms[(w * HEADS + h) * 2]);
    const float ref = top == neg_inf() ? 0.f : top;
    float sum = 0.f, out = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = power(ms[(w * HEADS + h) * 2] - ref);
      sum = fmaf(f, ms[(w * HEADS + h) * 2 + 1], sum);
      out = fmaf(f, os[(w * HEADS + h) * DP + d], out);
    }
    if (r.count == 1) {
      ((T*)a.out)[((long long)r.b * a.heads + h0 + h) * D + d] = from_float<T>(sum > 0.f || sum != sum ? out / sum : 0.f);
    } else {
      float* to = a.parts + ((long long)r.place * a.heads + h0 + h) * (D + 2);
      to[d] = out;
      if (d == 0) { to[D] = top; to[D + 1] = sum; }
    }
  }
}

// Joins the parts of the sequences that have several, in their order: a block per sequence, query head and 32 features.
template <typename T>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ Paged a) {
  pdl_prologue();
  const int b = blockIdx.x / a.heads, h = blockIdx.x % a.heads, tid = threadIdx.x, lane = tid & 31, row = tid >> 5;
  const int n = a.first[2 * b + 1];
  if (n == 1) return;
  __shared__ float most[8], sums[8], acc[8][32];
  const long long step = (long long)a.heads * (a.dim + 2);
  const float* base = a.parts + (long long)a.first[2 * b] * step + (long long)h * (a.dim + 2);
  float m = neg_inf();
  for (int i = tid; i < n; i += 256) m = fmaxf(m, base[i * step + a.dim]);
  m = warp_max(m);
  if (lane == 0) most[row] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, most[w]);
  const float ref = m == neg_inf() ? 0.f : m;
  const int d = blockIdx.y * 32 + lane;
  float o = 0.f, l = 0.f;
  for (int i = row; i < n; i += 8) {
    const float w = exp2f(base[i * step + a.dim] - ref);
    l = fmaf(w, base[i * step + a.dim + 1], l);
    if (d < a.dim) o = fmaf(w, base[i * step + d], o);
  }
  acc[row][lane] = o;
  if (lane == 0) sums[row] = l;
  __syncthreads();
  if (row || d >= a.dim) return;
  o = l = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) { o += acc[w][lane]; l += sums[w]; }
  ((T*)a.out)[((long long)b * a.heads + h) * a.dim + d] = from_float<T>(l > 0.f || l != l ? o / l : 0.f);
}

// Parts that there can be at most: those that fill the chip and one more for each sequence, or what the tables have room for.
long long most_parts(const OperatorLaunch& op, int chunks, bool* several) {
  long long cap = (long long)op.width * op.page;
  if (op.window > 0) cap = std::min<long long>(cap, (long long)op.window + op.sinks);
  cap += op.has_new;
  const long long each = std::max<long long>(1, (cap + kMinPart - 1) / kMinPart);
  *several = each > 1;
  return std::min<long long>(std::max(1, kParts / chunks) + (long long)op.batch, each * op.batch);
}

// Query heads that a block takes along: sixteen where more than eight share a key-value head and the data is 16-bit.
int heads_of(const OperatorLaunch& op) { return op.type != 0 && op.heads / op.kv_heads > 8 ? 16 : 8; }
int chunks_of(const OperatorLaunch& op) {
  const int group = op.heads / op.kv_heads, each = heads_of(op);
  return op.kv_heads * ((group + each - 1) / each);
}

template <typename T>
cudaError_t launch_join(const Paged& a, bool several, cudaStream_t stream, int* launches) {
  if (!several) return cudaSuccess;
  return launch_op(paged_join_kernel<T>, dim3((unsigned)(a.batch * a.heads), (unsigned)((a.dim + 31) / 32)), 256, 0, stream, launches, a);
}

cudaError_t launch_fma(const Paged& a, long long parts, bool several, cudaStream_t stream, int* launches) {
  static bool done[64] = {};
  const size_t most = (size_t)(32 * 260 + 32 * 256 + kPartHeads * 256 + 32 * kPartHeads + 3 * kPartHeads) * 4;
  if (cudaError_t e = allow_smem(paged_simple_kernel<float>, most, done)) return e;
  const size_t smem = (size_t)(32 * (a.dim + 4) + 32 * a.dim + kPartHeads * a.dim + 32 * kPartHeads + 3 * kPartHeads) * 4;
  if (cudaError_t e = launch_op(paged_simple_kernel<float>, dim3((unsigned)(parts * a.chunks)), 128, smem, stream, launches, a)) return e;
  return launch_join<float>(a, several, stream, launches);
}

template <typename T, int DP, int NT>
cudaError_t launch_mma(const Paged& a, long long parts, bool several, cudaStream_t stream, int* launches) {
  static bool done[64] = {};
  constexpr size_t smem = Ring<DP, NT>::SMEM;
  if (cudaError_t e = allow_smem(paged_mma_kernel<T, DP, NT>, smem, done)) return e;
  if (cudaError_t e = launch_op(paged_mma_kernel<T, DP, NT>, dim3((unsigned)(parts * a.chunks)), kWarps * 32, smem, stream, launches, a)) return e;
  return launch_join<T>(a, several, stream, launches);
}
template <typename T>
cudaError_t launch_16bit(const Paged& a, int heads, long long parts, bool several, cudaStream_t stream, int* launches) {
  if (heads == 8) {
    if (a.dim <= 64) return launch_mma<T, 64, 1>(a, parts, several, stream, launches);
    if (a.dim <= 128) return launch_mma<T, 128, 1>(a, parts, several, stream, launches);
    if (a.dim <= 192) return launch_mma<T, 192, 1>(a, parts, several, stream, launches);
    return launch_mma<T, 256, 1>(a, parts, several, stream, launches);
  }
  if (a.dim <= 64) return launch_mma<T, 64, 2>(a, parts, several, stream, launches);
  if (a.dim <= 128) return launch_mma<T, 128, 2>(a, parts, several, stream, launches);
  if (a.dim <= 192) return launch_mma<T, 192, 2>(a, parts, several, stream, launches);
  return launch_mma<T, 256, 2>(a, parts, several, stream, launches);
}

}  // namespace

const char* paged_attention_plan(OperatorLaunch& op) {
  if ((long long)op.width * op.page >= (1LL << 30)) return "tables of 2^30 positions and more";
  bool several;
  const int chunks = chunks_of(op);
  const long long parts = most_parts(op, chunks, &several);
  if (parts * chunks >= (1LL << 31) || (long long)op.batch * op.heads >= (1LL << 31)) return "too many sequences and heads";
  op.scratch_bytes = ((long long)op.batch * 8 + 255) / 256 * 256 + (several ? parts * op.heads * (op.dim + 2) * 4 : 0);
  op.launches = several ? 2 : 1;
  return nullptr;
}

cudaError_t launch_paged_attention(const OperatorLaunch& op, void* const* args, void* scratch, cudaStream_t stream, int* launches) {
  Paged a = {};
  const size_t size = op.type == 0 ? 4 : 2;
  a.out = args[0];
  a.q = args[1];
  a.plane = (long long)op.pages * op.page * op.kv_heads * op.dim;
  a.cache = (const char*)args[2] + (size_t)op.layer * 2 * a.plane * size;
  a.table = (const int*)args[3];
  a.lengths = (const int*)args[4];
  a.fresh = op.has_new ? args[5] : nullptr;
  a.first = (int*)scratch;
  a.parts = (float*)((char*)scratch + ((long long)op.batch * 8 + 255) / 256 * 256);
  a.batch = op.batch; a.heads = op.heads; a.kv_heads = op.kv_heads; a.dim = op.dim; a.group = op.heads / op.kv_heads;
  a.pages = op.pages; a.page = op.page; a.width = op.width; a.window = op.window; a.sinks = op.sinks; a.has_new = op.has_new;
  a.scale = op.scale * kLog2e;
  a.chunks = chunks_of(op);
  bool several;
  const long long parts = most_parts(op, a.chunks, &several);
  if (op.type == 0) return launch_fma(a, parts, several, stream, launches);
  if (op.type == 1) return launch_16bit<__nv_bfloat16>(a, heads_of(op), parts, several, stream, launches);
  return launch_16bit<__half>(a, heads_of(op), parts, several, stream, launches);
}

}  // namespace b200
