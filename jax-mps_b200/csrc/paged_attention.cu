// Attention of one new token per sequence over a cache of pages (custom call b200.paged_attention).
//
//   out[b, h] = sum_j w_j v_j,  w = softmax_j(scale * q[b, h] . k_j)  over the visible positions j of sequence b
//
// The token stands at position p: the last cached one, or, where its own key and value are given beside the cache, the one
// behind them. Position j is visible when j <= p and (no window, p - j < window, or j < sinks). A row that sees nothing is zero.
// Sums, maxima and the weights' normaliser are held in 32 bits; the running maximum m, sum l and output o of some of the
// positions are joined with those of the others by o = sum o_i 2^(m_i - m) / sum l_i 2^(m_i - m).
//
// Bound by memory: the visible keys and values are read once, 4 bytes of 16-bit data for each feature, position and key-value
// head, and take part in 4 * group operations each.
#include <algorithm>
#include <type_traits>

#include "operators.cuh"

namespace b200 {
namespace {

// Positions: a shorter part is not worth a place in the second pass, and a shorter sequence is counted as so many, for what it costs a block
// is mostly its own chain of loads (46 sequences of up to 10 positions in one block's row took 89 us, 5.5 in blocks of their own).
constexpr int kMinPart = 128;

struct Paged {
  const void *q, *cache, *fresh;
  const int *table, *lengths;
  void* out;
  float* parts;                       // two places per block: for each query head dim outputs, the maximum and the sum
  int2* spans;                        // per sequence: its first part and how many it has
  int batch, heads, kv_heads, dim, group, chunks, blocks, step, pages, page, width, window, sinks, has_new;
  unsigned page_inverse;              // 2^32 / page, cut
  long long plane;                    // elements between the keys and the values of a layer
  float scale;                        // of the scores, times log2(e)
};

// Positions of a sequence as a row: the sinks that lie in front of the window, then the window, then the token itself.
struct Span {
  int seen;                           // how many cached ones are visible
  int sinks, start;                   // place i < sinks is position i, another position start + i - sinks
};
__device__ __forceinline__ Span span_of(const Paged& a, int b) {
  const long long most = (long long)a.width * a.page;
  int n = a.lengths[b];
  n = n < 0 ? 0 : n > most ? (int)most : n;
  Span s;
  s.start = 0;
  if (a.window > 0) {
    const int p = a.has_new ? n : n - 1;
    s.start = min(max(0, p - a.window + 1), n);        // a window of one sees the token itself alone
  }
  s.sinks = min(a.sinks, s.start);
  s.seen = n - s.start + s.sinks;
  return s;
}
// Places that a row counts as; every sequence has a block that writes its result.
__device__ __forceinline__ int places(const Paged& a, const Span& s) { return max(kMinPart, s.seen + a.has_new); }

// The rows of all sequences, one behind another, are cut into as many equal parts as there are blocks for a group of heads, whatever
// the sequences' lengths: a block starts in the middle of one sequence and ends in the middle of another, and no block has more to
// read than the others. (With parts that end with their sequence, 32 sequences of 0 to 4096 positions took 2.4 waves of blocks:
// 66 us instead of 55.) Lengths are on the device only, so each block adds them up for itself.
template <int THREADS>
struct Cut {
  int len;                            // places of a part
  int b;                              // the sequence in which the block's part begins
  long long at;                       // places in front of that sequence
  long long total;
};
template <int THREADS>
__device__ __forceinline__ bool cut_of(const Paged& a, int block, Cut<THREADS>& r) {
  __shared__ long long sums[THREADS / 32];
  __shared__ int found;
  __shared__ long long found_at;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.batch + THREADS - 1) / THREADS, lo = min(a.batch, tid * per), hi = min(a.batch, lo + per);
  long long mine = 0;
  for (int b = lo; b < hi; ++b) mine += places(a, span_of(a, b));
  long long upto = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long v = __shfl_up_sync(0xFFFFFFFFu, upto, o);
    if (lane >= o) upto += v;
  }
  if (lane == 31) sums[warp] = upto;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) upto += sums[w];
    total += sums[w];
  }
  r.total = total;
  r.len = (int)min(max((long long)kMinPart, ((total + a.blocks - 1) / a.blocks + a.step - 1) / a.step * a.step), 1LL << 30);
  const long long want = (long long)block * r.len;
  if (want >= total) return false;
  long long at = upto - mine;
  if (want >= at && want < upto)
    for (int b = lo; b < hi; ++b) {
      const int n = places(a, span_of(a, b));
      if (want < at + n) { found = b; found_at = at; break; }
      at += n;
    }
  __syncthreads();
  r.b = found;
  r.at = found_at;
  return true;
}

constexpr unsigned kNowhere = 0xFFFFFFFFu, kFresh = 0xFFFFFFFEu;

// Where the keys at a place of a row begin, in pieces of 16 bytes behind the layer's first; kFresh: the token's own, kNowhere: not at
// all (behind the part, or the table names no page of the cache: such a position is left out). In two steps: a warp that made use of the
// table's entry at once would stand still until it is there (a quarter of the time), so the second comes a tile later.
struct Place {
  int page;
  unsigned in;                        // position in the page, or one of the two above
};
__device__ __forceinline__ Place look_up(const Paged& a, const Span& s, int b, int place, int end) {
  Place p = {0, kNowhere};
  if (place >= end) return p;
  if (place >= s.seen) {
    if (a.has_new) p.in = kFresh;
    return p;
  }
  const unsigned pos = place < s.sinks ? place : s.start + place - s.sinks;
  unsigned which = __umulhi(pos, a.page_inverse);                   // one below the quotient at most
  p.in = pos - which * (unsigned)a.page;
  if (p.in >= (unsigned)a.page) { ++which; p.in -= a.page; }
  p.page = a.table[(long long)b * a.width + which];
  return p;
}
__device__ __forceinline__ unsigned key_at(const Paged& a, const Place& p, int kvh, int row_pieces) {
  if (p.in >= kFresh) return p.in;
  if (p.page < 0 || p.page >= a.pages) return kNowhere;
  return (((unsigned)p.page * (unsigned)a.page + p.in) * (unsigned)a.kv_heads + (unsigned)kvh) * (unsigned)row_pieces;
}

// ---- the products ------------------------------------------------------------------------------------
// A warp streams 16 positions at a time through a ring of its own in shared memory (cp.async, no block barrier in the loop), and
// takes 8 * NT query heads along: scores^T [16 positions, 8 heads] = K Q^T and outputs^T [features, 8 heads] += V^T P^T by
// mma.sync, whose eight columns fit the heads that share a key-value head (with heads as rows half of every product and of the
// accumulators would be padding). The scores' fragments become the weights' by 8 x 8 transposes within the warp.
//   16-bit data (m16n8k16): the weights go into the second product as two 16-bit pieces, their rounding and what it leaves, so that
//   they lose nothing beside the result's own rounding: the products are not what bounds this kernel.
//   32-bit data (tf32 m16n8k8): every product is hi hi + hi lo + lo hi, hi a word rounded to the 19 bits that the tensor core reads and
//   lo what that leaves; a tile's outputs are added up apart and then to the others in 32 bits, since the tensor core cuts its sums.
template <typename T, int DP, int NT>
struct Ring {
  static constexpr int ROW = DP * (int)sizeof(T), PIECES = ROW / 16;
  // Warps and the tiles that each has on its way or in use, by the bytes of a row: as many warps as registers let be, for a tile's products
  // are a chain (heads of 128, 32 sequences of up to 4096 positions, 16-bit: 8 warps an SM with three tiles 55.3 us, 12 with two 54.2; 32-bit
  // heads of 64 58 and 46, which are 42 since).
  static constexpr int WARPS = ROW >= 768 ? 2 : ROW > 256 ? 6 : 4, STAGES = ROW >= 768 ? 3 : ROW > 128 ? 2 : 3;
  static constexpr int TILE = 16 * ROW, STAGE = 2 * TILE;            // bytes of the keys, of keys and values
  static constexpr int BYTES = WARPS * STAGES * STAGE;
  static constexpr int JOIN = WARPS * 8 * NT * (DP + 2) * 4;
  static constexpr int SMEM = BYTES > JOIN ? BYTES : JOIN;
  static constexpr int FIT = 232448 / (SMEM + 2048), MOST = ROW > 256 ? 1 : NT == 2 ? 2 : ROW > 128 ? 3 : 4;
  static_assert(SMEM + 2048 <= 232448, "more than an SM has");
  static constexpr int PER_SM = FIT > MOST ? MOST : FIT;             // blocks that an SM has room for (memory, registers)
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t load_word(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else if (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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
// A word rounded to the 19 bits that a tf32 product reads, and what that leaves, rounded to as many; nothing of an infinity.
// (With hi cut instead of rounded, both errors lean to one side: three times the error of the result.)
__device__ __forceinline__ uint32_t high_part(uint32_t v) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(__uint_as_float(v)));
  return r;
}
__device__ __forceinline__ uint32_t low_part(uint32_t v, uint32_t high) {
  const float rest = __uint_as_float(v) - __uint_as_float(high);
  return rest == rest ? high_part(__float_as_uint(rest)) : 0u;
}
// Whether a word has an infinity: one of two 16-bit values, or one 32-bit value that is one or whose high part is.
template <typename T>
__device__ __forceinline__ bool infinite_word(uint32_t v) {
  if (sizeof(T) == 4) return (v & 0x7FFFFFFFu) >= 0x7F7FF000u && (v & 0x7FFFFFFFu) <= 0x7F800000u;
  constexpr uint32_t inf = std::is_same<T, __nv_bfloat16>::value ? 0x7F80u : 0x7C00u;
  return (v & 0x7FFFu) == inf || (v & 0x7FFF0000u) == inf << 16;
}
__device__ __forceinline__ float column_max(float v) {             // over the lanes that hold the positions of a head
  v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 4));
  v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 8));
  return fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, 16));
}

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(Ring<T, DP, NT>::WARPS * 32, Ring<T, DP, NT>::PER_SM) paged_kernel(const __grid_constant__ Paged a) {
  pdl_prologue();
  using R = Ring<T, DP, NT>;
  constexpr bool WIDE = sizeof(T) == 4;
  constexpr int HEADS = 8 * NT, S = R::STAGES, W = R::WARPS, STEP = WIDE ? 8 : 16, KSTEPS = DP / STEP;
  // f16: weights, sums and outputs in units of 2^-14, so that weights keep their bits down to 2^-28 of the largest and no long row of
  // small ones is lost (they end at 2^-24 otherwise, which 60000 positions make 2^-8 of the result)
  constexpr float LIFT = std::is_same<T, __half>::value ? 14.f : 0.f;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ float stats[W][HEADS][2];
  const int D = a.dim, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row_pieces = D * (int)sizeof(T) / 16;
  const int chunk = blockIdx.x % a.chunks, block = blockIdx.x / a.chunks, per = (a.group + HEADS - 1) / HEADS;
  const int kvh = chunk / per, h0 = kvh * a.group + chunk % per * HEADS, nh = min(HEADS, kvh * a.group + a.group - h0);
  Cut<W * 32> cut;
  if (!cut_of<W * 32>(a, block, cut)) return;
  const uint32_t base = smem_u32(ring) + warp * S * R::STAGE;
  // where a lane's parts of a tile are, for the k-steps of 128 bytes of a row; 16-byte pieces are permuted by their row
  uint32_t key_piece[4], value_piece[4], value_word[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int row = lane & 15, vrow = (lane & 7) + (lane >> 4) * 8;
    key_piece[k] = row * R::ROW + (((2 * k + (lane >> 4)) ^ (row & 7)) << 4);
    value_piece[k] = vrow * R::ROW + (((2 * k + ((lane >> 3) & 1)) ^ (vrow & 7)) << 4);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int row = lane % 4 * 2 + (i >> 2), d = (i & 1) * 16 + (i >> 1 & 1) * 8 + lane / 4;
    value_word[i] = row * R::ROW + (((d >> 2) ^ (row & 7)) << 4) + (d & 3) * 4;
  }
  const long long from0 = (long long)block * cut.len, to0 = min(from0 + cut.len, cut.total);
  for (long long at = cut.at; cut.b < a.batch && at < to0; ++cut.b) {
    const int b = cut.b;
    const Span span = span_of(a, b);
    const int n = places(a, span), from = (int)(max(from0, at) - at), end = (int)min((long long)(span.seen + a.has_new), to0 - at);
    const int first = (int)(at / cut.len), count = (int)((at + n - 1) / cut.len) - first + 1;      // the blocks that share the sequence
    at += n;

    // Q^T as the second operand: lane holds head lane / 4 and, of each k-step, features 2 (lane % 4) + {0, 1} and those eight further
    // (16-bit), or lane % 4 and that four further (32-bit)
    uint32_t q[KSTEPS][NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const int h = t * 8 + lane / 4;
      const T* src = (const T*)a.q + ((long long)b * a.heads + h0 + h) * D;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int d = k * STEP + i * (STEP / 2) + (WIDE ? lane % 4 : lane % 4 * 2);
          q[k][t][i] = h < nh && d < D ? *(const uint32_t*)(src + d) : 0u;
        }
    }
    const int ntiles = end > from ? (end - from + 15) / 16 : 0;
    const uint8_t *keys = (const uint8_t*)a.cache, *fresh_key = (const uint8_t*)a.fresh + ((long long)b * a.kv_heads + kvh) * D * (long long)sizeof(T);
    const long long plane = a.plane * (long long)sizeof(T), fresh_plane = (long long)a.batch * a.kv_heads * D * (long long)sizeof(T);
    // lanes look up a position each (the upper half those of the lower once more), in front of the tile that asks for them
    auto locate = [&](int tile) { return look_up(a, span, b, from + tile * 16 + (lane & 15), tile < ntiles ? end : 0); };
    auto fetch = [&](const Place& place, uint32_t to) -> uint32_t { // gives which of the tile's positions are there
      constexpr int P = R::PIECES;
      const unsigned where = key_at(a, place, kvh, row_pieces);
      if (__all_sync(0xFFFFFFFFu, where < kFresh) && D == DP) {
        // a tile of cached positions, as most are: a lane's piece of a row is the same in all of its rows, or every other one
#pragma unroll
        for (int i = 0; i < P / 2; ++i) {
          const int row = (lane + 32 * i) / P, c = (lane + 32 * i) % P;
          const uint8_t* src = keys + ((unsigned long long)(__shfl_sync(0xFFFFFFFFu, where, row) + c) << 4);
          const uint32_t dst = to + row * R::ROW + ((c ^ (row & 7)) << 4);
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + R::TILE), "l"(src + plane) : "memory");
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < P / 2; ++i) {
          const int row = (lane + 32 * i) / P, c = (lane + 32 * i) % P;
          const unsigned w = __shfl_sync(0xFFFFFFFFu, where, row);
          const bool real = w != kNowhere && c < row_pieces, own = w == kFresh;
          const uint8_t* src = !real ? (const uint8_t*)a.q : own ? fresh_key + c * 16 : keys + ((unsigned long long)w + c) * 16;
          const uint32_t dst = to + row * R::ROW + ((c ^ (row & 7)) << 4), bytes = real ? 16 : 0;
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + R::TILE), "l"(!real ? src : src + (own ? fresh_plane : plane)), "r"(bytes) : "memory");
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      return __ballot_sync(0xFFFFFFFFu, where != kNowhere) & 0xFFFFu;
    };
    float m[NT][2], l[NT][2], o[DP / 16][NT][4];                    // heads 2 (lane % 4) + {0, 1} of each eight
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      m[t][0] = m[t][1] = neg_inf();
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) o[k][t][0] = o[k][t][1] = o[k][t][2] = o[k][t][3] = 0.f;
    }
    // Tiles go round the ring, whose places are offsets and not copies of the loop's body: unrolled, it did not fit the instruction
    // cache (32-bit data: 1.8 of 4.7 cycles an instruction were waits for the next).
    uint32_t there[S], into = base, out = base;
    auto past = [&](uint32_t& at) { at = at + R::STAGE == base + S * R::STAGE ? base : at + R::STAGE; };
    Place next = locate(warp);
#pragma unroll
    for (int s = 0; s < S - 1; ++s) {
      there[s] = fetch(next, into);
      past(into);
      next = locate(warp + (s + 1) * W);
    }
#pragma unroll 1
    for (int tile = warp; tile < ntiles; tile += W) {
      constexpr int AHEAD = S - 1;
      there[AHEAD] = fetch(next, into);
      past(into);
      next = locate(tile + S * W);
      asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD) : "memory");
      __syncwarp();
      const uint32_t kt = out, vt = kt + R::TILE;
      // scores: rows are positions lane / 4 and eight further, columns heads; two chains, so that a product need not wait for the last
      float sc[2][NT][4];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[0][t][i] = sc[1][t][i] = 0.f;
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k) {
        uint32_t f[4];
        ldmatrix4(f, kt + key_piece[k % 4] + k / 4 * 128);
        if (WIDE) {
          uint32_t g[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t v = f[e];
            f[e] = high_part(v);
            g[e] = low_part(v, f[e]);
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            const uint32_t q0 = high_part(q[k][t][0]), q1 = high_part(q[k][t][1]);
            mma<T>(sc[k % 2][t], g, q0, q1);
            mma<T>(sc[k % 2][t], f, low_part(q[k][t][0], q0), low_part(q[k][t][1], q1));
            mma<T>(sc[k % 2][t], f, q0, q1);
          }
        } else {
#pragma unroll
          for (int t = 0; t < NT; ++t) mma<T>(sc[k % 2][t], f, q[k][t][0], q[k][t][1]);
        }
      }
      const uint32_t seen = there[0] >> (lane / 4);
      // the weights as second operand, in two pieces: [eight positions][of the pieces' words]
      uint32_t hi[NT][WIDE ? 4 : 2], lo[NT][WIDE ? 4 : 2];
      bool grown = false;
      float keep[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float x = seen & 1u ? (sc[0][t][i] + sc[1][t][i]) * a.scale : neg_inf(), y = seen & 0x100u ? (sc[0][t][2 + i] + sc[1][t][2 + i]) * a.scale : neg_inf();
          const float top = fmaxf(m[t][i], column_max(fmaxf(x, y)));
          grown |= top > m[t][i];
          const float ref = top == neg_inf() ? 0.f : top;
          keep[t][i] = power(m[t][i] - ref);
          m[t][i] = top;
          p[i] = power(LIFT > 0.f ? x - ref + LIFT : x - ref);
          p[2 + i] = power(LIFT > 0.f ? y - ref + LIFT : y - ref);
          l[t][i] = l[t][i] * keep[t][i] + p[i] + p[2 + i];
        }
        if (WIDE) {
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const uint32_t x = __float_as_uint(p[2 * u]), y = __float_as_uint(p[2 * u + 1]);
            const uint32_t upper = transpose8(__byte_perm(x, y, 0x7632)), lower = transpose8(__byte_perm(x, y, 0x5410));
            constexpr int M = WIDE ? 4 : 2;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t v = __byte_perm(lower, upper, e ? 0x7632 : 0x5410);
              hi[t][(2 * u + e) % M] = high_part(v);
              lo[t][(2 * u + e) % M] = low_part(v, hi[t][(2 * u + e) % M]);
            }
          }
        } else {
          hi[t][0] = transpose8(pair16<T>(p[0], p[1], lo[t][0]));
          hi[t][1] = transpose8(pair16<T>(p[2], p[3], lo[t][1]));
          lo[t][0] = transpose8(lo[t][0]);
          lo[t][1] = transpose8(lo[t][1]);
        }
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
        if (WIDE) {
          float add[NT][4];
#pragma unroll
          for (int t = 0; t < NT; ++t) add[t][0] = add[t][1] = add[t][2] = add[t][3] = 0.f;
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            // features lane / 4 and eight further as rows; positions 2 (lane % 4) and the next, which the weights' words hold
            // (a product does not mind the order of what it adds up, and so no two lanes meet in a bank)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              f[e] = load_word(vt + value_word[(e >> 1) * 4 + (e & 1) * 2 + k % 2] + u * 8 * R::ROW + k / 2 * 128);
            }
            uint32_t g[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t v = f[e];
              f[e] = high_part(v);
              g[e] = low_part(v, f[e]);
            }
            constexpr int M = WIDE ? 4 : 2;
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              mma<T>(add[t], g, hi[t][2 * u % M], hi[t][(2 * u + 1) % M]);
              mma<T>(add[t], f, lo[t][2 * u % M], lo[t][(2 * u + 1) % M]);
              mma<T>(add[t], f, hi[t][2 * u % M], hi[t][(2 * u + 1) % M]);
            }
          }
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) o[k][t][i] += add[t][i];
        } else {
          ldmatrix4_trans(f, vt + value_piece[k % 4] + k / 4 * 128);
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            mma<T>(o[k][t], f, hi[t][0], hi[t][1]);
            mma<T>(o[k][t], f, lo[t][0], lo[t][1]);
          }
        }
      }
      __syncwarp();                                             // the tile's place may be filled again
      past(out);
#pragma unroll
      for (int s = 0; s < AHEAD; ++s) there[s] = there[s + 1];
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    bool odd[NT][2], any_odd = false;
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        l[t][i] += __shfl_xor_sync(0xFFFFFFFFu, l[t][i], 4);
        l[t][i] += __shfl_xor_sync(0xFFFFFFFFu, l[t][i], 8);
        l[t][i] += __shfl_xor_sync(0xFFFFFFFFu, l[t][i], 16);
        // Products in parts make no numbers of infinities: a part of a weight may be zero or below it, and one of an infinite word is no
        // number. (16-bit scores are products in one part, so that weights without a number are what the definition gives.)
        bool nan = false;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) nan |= o[k][t][i] != o[k][t][i] || o[k][t][2 + i] != o[k][t][2 + i];
        nan = (nan && (WIDE || l[t][i] == l[t][i])) || (WIDE && l[t][i] != l[t][i]);
        odd[t][i] = (__ballot_sync(0xFFFFFFFFu, nan) & 0x11111111u << (lane & 3)) && t * 8 + lane % 4 * 2 + i < nh;
        any_odd |= odd[t][i];
      }
    bool again = __any_sync(0xFFFFFFFFu, any_odd);
    if (again) {
      // NaN that come of NaN are right as they are: only where the warp's values (32 bits: or keys or queries) have an infinity, or a word that rounds to one,
      // is there more to do.
      bool found = false;
#pragma unroll 1
      for (int tile = warp; tile < ntiles; tile += W) {
        const unsigned where = key_at(a, locate(tile), kvh, row_pieces);
#pragma unroll 1
        for (int i = 0; i < R::PIECES / 2; ++i) {
          const unsigned w = __shfl_sync(0xFFFFFFFFu, where, (lane + 32 * i) / R::PIECES), c = (lane + 32 * i) % R::PIECES;
          if (w == kNowhere || c >= (unsigned)row_pieces) continue;
          const uint8_t* src = w == kFresh ? fresh_key + c * 16 : keys + ((unsigned long long)w + c) * 16;
          const uint4 v = *(const uint4*)(src + (w == kFresh ? fresh_plane : plane)), k = WIDE ? *(const uint4*)src : v;
          found |= infinite_word<T>(v.x) | infinite_word<T>(v.y) | infinite_word<T>(v.z) | infinite_word<T>(v.w) | infinite_word<T>(k.x) | infinite_word<T>(k.y) |
                   infinite_word<T>(k.z) | infinite_word<T>(k.w);
        }
      }
      if (WIDE)
        for (int i = lane; i < nh * D; i += 32) found |= infinite_word<T>(((const uint32_t*)a.q)[((long long)b * a.heads + h0) * D + i]);
      again = __any_sync(0xFFFFFFFFu, found);
    }
    if (again) {
      // Such heads are made again from the warp's positions, one after another with whole words and weights, in the places of the products'
      // fragments. (32 sequences of 2048, 32 heads of 128 on 8, in bf16: 55 us, with a NaN in every page 136, with an infinity 1270.)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (odd[t][i]) {
            m[t][i] = neg_inf();
            l[t][i] = 0.f;
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) o[k][t][i] = o[k][t][2 + i] = 0.f;
          }
#pragma unroll 1
      for (int tile = warp; tile < ntiles; tile += W)
#pragma unroll 1
        for (int place = from + tile * 16; place < min(end, from + tile * 16 + 16); ++place) {
          const unsigned where = key_at(a, look_up(a, span, b, place, end), kvh, row_pieces);
          if (where == kNowhere) continue;
          const uint8_t* row = where == kFresh ? fresh_key : keys + ((unsigned long long)where << 4);
          const T *key = (const T*)row, *value = (const T*)(row + (where == kFresh ? fresh_plane : plane));
          float x[NT][2] = {};
#pragma unroll 1
          for (int d = lane / 4; d < D; d += 8) {
            const float kd = to_float(key[d]);
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const int h = min(t * 8 + lane % 4 * 2 + i, nh - 1);
                x[t][i] = fmaf(to_float(((const T*)a.q)[((long long)b * a.heads + h0 + h) * D + d]), kd, x[t][i]);
              }
          }
          float keep[NT][2], p[NT][2];
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
              for (int by = 4; by < 32; by *= 2) x[t][i] += __shfl_xor_sync(0xFFFFFFFFu, x[t][i], by);
              x[t][i] *= a.scale;
              const float top = fmaxf(m[t][i], x[t][i]), ref = top == neg_inf() ? 0.f : top;
              keep[t][i] = power(m[t][i] - ref);
              p[t][i] = power(LIFT > 0.f ? x[t][i] - ref + LIFT : x[t][i] - ref);
              if (odd[t][i]) {
                m[t][i] = top;
                l[t][i] = l[t][i] * keep[t][i] + p[t][i];
              }
            }
#pragma unroll
          for (int k = 0; k < DP / 16; ++k)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int d = k * 16 + e * 8 + lane / 4;
              const float v = d < D ? to_float(value[d]) : 0.f;
#pragma unroll
              for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                  if (odd[t][i]) o[k][t][2 * e + i] = fmaf(p[t][i], v, o[k][t][2 * e + i] * keep[t][i]);
            }
        }
    }
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (lane < 4) { stats[warp][t * 8 + lane * 2 + i][0] = m[t][i]; stats[warp][t * 8 + lane * 2 + i][1] = l[t][i]; }
    __syncthreads();                                                // nobody reads the ring any more, all maxima are known
    // the warps' outputs go through the ring's memory in units of the block's maximum: [warp][head][feature]
    float* os = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int h = t * 8 + lane % 4 * 2 + i;
        float top = neg_inf();
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, stats[w][h][0]);
        const float f = power(m[t][i] - (top == neg_inf() ? 0.f : top));
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          os[(warp * HEADS + h) * DP + k * 16 + lane / 4] = o[k][t][i] * f;
          os[(warp * HEADS + h) * DP + k * 16 + lane / 4 + 8] = o[k][t][2 + i] * f;
        }
      }
    __syncthreads();
    // a part of a sequence is its block's last when the sequence goes on behind it, and else its first
    const int place = block * 2 + (block == first ? 1 : 0);
    if (block == first && chunk == 0 && tid == 0) a.spans[b] = make_int2(first, count);
    constexpr int LANES = DP / 4;                                   // four features a thread
    for (int i = tid; i < nh * LANES; i += W * 32) {
      const int h = i / LANES, d = i % LANES * 4;
      if (d >= D) continue;
      float top = neg_inf(), sum = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) top = fmaxf(top, stats[w][h][0]);
      const float ref = top == neg_inf() ? 0.f : top;
      float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) {
        sum = fmaf(power(stats[w][h][0] - ref), stats[w][h][1], sum);
        const float4 x = *reinterpret_cast<const float4*>(os + (w * HEADS + h) * DP + d);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
      }
      if (count == 1) {
        const float inv = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
        if (inv == 0.f) v = {0.f, 0.f, 0.f, 0.f};                   // no weight at all, whatever the values are
        T* to = (T*)a.out + ((long long)b * a.heads + h0 + h) * D + d;
        to[0] = from_float<T>(v.x * inv);
        to[1] = from_float<T>(v.y * inv);
        to[2] = from_float<T>(v.z * inv);
        to[3] = from_float<T>(v.w * inv);
      } else {
        float* to = a.parts + ((long long)place * a.heads + h0 + h) * (D + 4);
        *reinterpret_cast<float4*>(to + d) = v;
        if (d == 0) { to[D] = top; to[D + 1] = sum; }
      }
    }
    __syncthreads();                                                // the ring and the maxima may be filled again
  }
}

// Joins the parts of the sequences that have several, in their order. A warp takes a sequence and head with up to eight parts, one block
// of eight those of its seven neighbours; with more parts a block does, whose warps take every eighth part. 128 features at a time.
constexpr int kFewParts = 8;
template <typename T>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ Paged a) {
  pdl_prologue();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, D = a.dim;
  auto part = [&](int first, int i, int h) { return a.parts + ((long long)(2 * (first + i) + (i == 0 ? 1 : 0)) * a.heads + h) * (D + 4); };
  auto finish = [&](int pair, int d, float4 v, float l) {
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    if (inv == 0.f) v = {0.f, 0.f, 0.f, 0.f};
    T* to = (T*)a.out + (long long)pair * D + d;
    to[0] = from_float<T>(v.x * inv);
    to[1] = from_float<T>(v.y * inv);
    to[2] = from_float<T>(v.z * inv);
    to[3] = from_float<T>(v.w * inv);
  };
  auto add = [](float4& v, float f, const float4& x) { v.x = fmaf(f, x.x, v.x); v.y = fmaf(f, x.y, v.y); v.z = fmaf(f, x.z, v.z); v.w = fmaf(f, x.w, v.w); };
  if (blockIdx.x % 8 == 0 && blockIdx.y == 0) {
    const int pair = blockIdx.x + warp;
    if (pair < a.batch * a.heads) {
      const int h = pair % a.heads;
      const int2 span = a.spans[pair / a.heads];
      if (span.y > 1 && span.y <= kFewParts) {
        const float mine = lane < span.y ? part(span.x, lane, h)[D] : neg_inf(), sum = lane < span.y ? part(span.x, lane, h)[D + 1] : 0.f;
        float m = mine;
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
        m = __shfl_sync(0xFFFFFFFFu, m, 0);
        const float f = power(mine - (m == neg_inf() ? 0.f : m));
        float l = 0.f;
        for (int i = 0; i < span.y; ++i) l += __shfl_sync(0xFFFFFFFFu, f * sum, i);
        for (int d = lane * 4; d < (D + 127) / 128 * 128; d += 128) {
          float4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
          for (int i = 0; i < span.y; ++i) {
            const float g = __shfl_sync(0xFFFFFFFFu, f, i);
            if (d < D) add(v, g, *reinterpret_cast<const float4*>(part(span.x, i, h) + d));
          }
          if (d < D) finish(pair, d, v, l);
        }
      }
    }
  }
  const int pair = blockIdx.x, h = pair % a.heads;
  const int2 span = a.spans[pair / a.heads];
  if (span.y <= kFewParts) return;
  __shared__ float most[8], sums[8];
  __shared__ float4 acc[8][32];
  float m = neg_inf();
  for (int i = tid; i < span.y; i += 256) m = fmaxf(m, part(span.x, i, h)[D]);
  m = warp_max(m);
  if (lane == 0) most[warp] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) m = fmaxf(m, most[w]);
  const float ref = m == neg_inf() ? 0.f : m;
  const int d = blockIdx.y * 128 + lane * 4;
  float4 v = {0.f, 0.f, 0.f, 0.f};
  float l = 0.f;
#pragma unroll 4
  for (int i = warp; i < span.y; i += 8) {
    const float* p = part(span.x, i, h);
    const float f = power(p[D] - ref);
    l = fmaf(f, p[D + 1], l);
    if (d < D) add(v, f, *reinterpret_cast<const float4*>(p + d));
  }
  acc[warp][lane] = v;
  if (lane == 0) sums[warp] = l;
  __syncthreads();
  if (warp || d >= D) return;
#pragma unroll
  for (int w = 1; w < 8; ++w) {
    add(v, 1.f, acc[w][lane]);
    l += sums[w];
  }
  finish(pair, d, v, l);
}

// The one place that turns an operator into a kernel's type: f gets a Ring.
template <typename F>
auto with_ring(const OperatorLaunch& op, F&& f) {
  const int d = op.dim;
  const bool many = op.heads / op.kv_heads > 8;                     // sixteen heads a block where more than eight share keys
#define B200_BY_DIM(T, NT) \
  return d <= 64 ? f(T(), std::integral_constant<int, 64>(), std::integral_constant<int, NT>()) \
       : d <= 128 ? f(T(), std::integral_constant<int, 128>(), std::integral_constant<int, NT>()) \
       : d <= 192 ? f(T(), std::integral_constant<int, 192>(), std::integral_constant<int, NT>()) \
                  : f(T(), std::integral_constant<int, 256>(), std::integral_constant<int, NT>())
  if (op.type == 0) { B200_BY_DIM(float, 1); }                      // (32-bit queries of sixteen heads would not stay in registers)
  if (op.type == 1) { if (many) { B200_BY_DIM(__nv_bfloat16, 2); } else { B200_BY_DIM(__nv_bfloat16, 1); } }
  if (many) { B200_BY_DIM(__half, 2); } else { B200_BY_DIM(__half, 1); }
#undef B200_BY_DIM
}

struct Shape {
  int chunks, blocks;                 // groups of heads; blocks for each
  int step;                           // of a part's length
  bool several;                       // whether a sequence can have several parts
};
Shape shape_of(const OperatorLaunch& op) {
  return with_ring(op, [&](auto t, auto dp, auto nt) {
    using R = Ring<decltype(t), decltype(dp)::value, decltype(nt)::value>;
    Shape s;
    const int group = op.heads / op.kv_heads, heads = 8 * decltype(nt)::value;
    s.chunks = op.kv_heads * ((group + heads - 1) / heads);
    // places that the tables have room for
    long long cap = (long long)op.width * op.page;
    if (op.window > 0) cap = std::min<long long>(cap, (long long)op.window + op.sinks);
    cap = std::max<long long>(kMinPart, cap + op.has_new);
    s.blocks = (int)std::min<long long>(std::max(1, kSMs * R::PER_SM / s.chunks), (cap * op.batch + kMinPart - 1) / kMinPart);
    s.several = cap > kMinPart;
    s.step = s.several ? 16 : kMinPart;                             // sequences of one part each stay whole
    return s;
  });
}

long long spans_bytes(const OperatorLaunch& op) { return ((long long)op.batch * 8 + 255) / 256 * 256; }

}  // namespace

const char* paged_attention_plan(OperatorLaunch& op) {
  if ((long long)op.width * op.page >= (1LL << 30)) return "tables of 2^30 positions and more";
  if ((long long)op.pages * op.page * op.kv_heads * op.dim * (op.type == 0 ? 4 : 2) >= 16 * 0xFFFFFFFELL) return "64 GB and more of a layer's keys";
  const Shape s = shape_of(op);
  if (((long long)op.width * op.page + kMinPart) * op.batch / s.blocks >= (1LL << 30) - kMinPart) return "more positions than the blocks can share";
  if ((long long)s.blocks * s.chunks >= (1LL << 31) || (long long)op.batch * op.heads >= (1LL << 31)) return "too many sequences and heads";
  op.scratch_bytes = spans_bytes(op) + (s.several ? 2LL * s.blocks * op.heads * (op.dim + 4) * 4 : 0);
  op.launches = s.several ? 2 : 1;
  return nullptr;
}

cudaError_t launch_paged_attention(const OperatorLaunch& op, void* const* args, void* scratch, cudaStream_t stream, int* launches) {
  Paged a = {};
  a.out = args[0];
  a.q = args[1];
  a.plane = (long long)op.pages * op.page * op.kv_heads * op.dim;
  a.cache = (const char*)args[2] + (size_t)op.layer * 2 * a.plane * (op.type == 0 ? 4 : 2);
  a.table = (const int*)args[3];
  a.lengths = (const int*)args[4];
  a.fresh = op.has_new ? args[5] : nullptr;
  a.spans = (int2*)scratch;
  a.parts = (float*)((char*)scratch + spans_bytes(op));
  a.batch = op.batch; a.heads = op.heads; a.kv_heads = op.kv_heads; a.dim = op.dim; a.group = op.heads / op.kv_heads;
  a.pages = op.pages; a.page = op.page; a.width = op.width; a.window = op.window; a.sinks = op.sinks; a.has_new = op.has_new;
  a.scale = op.scale * kLog2e;
  a.page_inverse = op.page == 1 ? 0xFFFFFFFFu : (unsigned)((1ULL << 32) / op.page);
  const Shape s = shape_of(op);
  a.chunks = s.chunks;
  a.blocks = s.blocks;
  a.step = s.step;
  return with_ring(op, [&](auto t, auto dp, auto nt) -> cudaError_t {
    using T = decltype(t);
    constexpr int DP = decltype(dp)::value, NT = decltype(nt)::value;
    using R = Ring<T, DP, NT>;
    static bool done[64] = {};
    if (cudaError_t e = allow_smem(paged_kernel<T, DP, NT>, R::SMEM, done)) return e;
    if (cudaError_t e = launch_op(paged_kernel<T, DP, NT>, dim3((unsigned)(s.blocks * s.chunks)), R::WARPS * 32, R::SMEM, stream, launches, a)) return e;
    if (!s.several) return cudaSuccess;
    return launch_op(paged_join_kernel<T>, dim3((unsigned)(a.batch * a.heads), (unsigned)((a.dim + 127) / 128)), 256, 0, stream, launches, a);
  });
}

}  // namespace b200
