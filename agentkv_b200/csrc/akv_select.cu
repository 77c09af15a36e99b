// akv_select.cu — the blocks of each row that matter most to its new token.
//
// With a block's key bounds kmin <= k <= kmax by dimension, no key of it
// scores above sum_d max(q_d kmin_d, q_d kmax_d).  max(q a, q b) is q b for
// q > 0 and q a for q < 0, so the sum over a group of query heads is
//   sum_d P_d kmax_d + N_d kmin_d,  P_d = sum_heads max(q_d, 0), N_d = sum_heads min(q_d, 0):
// two products per dimension whatever the group.
//
// A score is a number in 64 bits: which of two blocks is taken hangs on the
// last places of their scores, and products of 16-bit numbers and their sums are
// exact there, so the choice does not depend on the order of a sum.  But 64-bit
// arithmetic on every block took 8 times the time that reading them does (212 us
// for 171 MB of bounds), so k_score works in 32 bits and brings, beside the
// scores, a bound on the sum of their terms' magnitudes: a score is off by at most
// (group + 32) * 2^-23 of that (each of a lane's at most 16 products and 5 sums,
// and of the group's sums in the coefficients, is off by 2^-24 of its own).  Only the
// blocks that this leaves on both sides of the border (a few, unless
// blocks are alike) are scored again in 64 bits, by k_select.
//
// What bounds it: 2 head_dim elements read per block and key head.  Measured: bounds
// of 32 rows' 41,700 blocks (171 MB, 8 key heads of 128) scored in 62 us, 2.8 TB/s
// (what issues is each score's sum over the lanes; about 100 bytes a thread are
// spilled at 128 registers), chosen from in 22 us.
#include <climits>

#include "akv_paged.cuh"

namespace {

constexpr int kThreads = 256;
constexpr int kWindow = 32;        // blocks whose ids a warp holds
constexpr int kSharedKeys = 8192;  // keys that k_select holds in shared memory
constexpr double kLargest = 1.7976931348623157e308;

struct SelectParams {
  AkvLayer kv;  // geometry only
  AkvTables tab;
  const char* bounds;
  int64_t bounds_page;  // bytes
  const void* q;
  int64_t q_row, q_head;
  int32_t group, keep, first, last;
  int32_t q_words;  // the queries allow loads of whole words
  int32_t task;    // blocks that a warp takes for one row and head, a multiple of kWindow
  float* near;     // [rows][heads][width]: scores in 32 bits
  float* most;     // [rows][heads][tasks of a row]: what their terms' magnitudes add up to at most
  uint64_t* keys;  // [rows][heads][width]: of blocks that were scored in 64 bits
  int32_t* selected;
  AkvStatus* st;
};

AKV_DEV float warp_max(float x) {
#pragma unroll
  for (int off = 16; off; off >>= 1) x = max_nan(x, __shfl_xor_sync(kFullWarp, x, off));
  return x;
}

AKV_DEV int32_t blocks_of(const SelectParams& p, int32_t s) {
  return static_cast<int32_t>((static_cast<int64_t>(akv_held(p.tab, p.kv.bs_log2, s)) + (1 << p.kv.bs_log2) - 1) >>
                              p.kv.bs_log2);
}

// The score as a whole number of the same order, above 0 and below the
// largest; NaN counts as the highest score.
AKV_DEV uint64_t key_of(double x) {
  x = x != x ? kLargest : fmin(fmax(x, -kLargest), kLargest);
  const uint64_t u = static_cast<uint64_t>(__double_as_longlong(x + 0.0));  // -0 and 0 are equal
  return u >> 63 ? ~u : u | (1ull << 63);
}

template <typename T, int kE, int kJ>
__global__ void __launch_bounds__(kThreads, 2) k_score(SelectParams p) {
  using Word = AkvPack<T, kE>;
  constexpr int kBytes = kE * kJ * static_cast<int>(sizeof(T)), kB = kBytes <= 16 ? 8 : kBytes <= 32 ? 4 : 2;
  const int lane = threadIdx.x & 31, dim = p.kv.dim;
  const int64_t groups = (p.tab.width + p.task - 1) / p.task;
  const int64_t tasks = p.tab.rows * groups * p.kv.heads;
  const int64_t layer_bytes = 2ll * p.kv.row_bytes;
  for (int64_t t = blockIdx.x * (kThreads / 32ll) + threadIdx.x / 32; t < tasks; t += gridDim.x * (kThreads / 32ll)) {
    const int32_t h = static_cast<int32_t>(t % p.kv.heads);
    const int32_t s = static_cast<int32_t>(t / p.kv.heads / groups);
    const int32_t j0 = static_cast<int32_t>(t / p.kv.heads % groups) * p.task;
    const int32_t n = blocks_of(p, s);
    if (n <= p.keep || j0 >= n) continue;
    float coef[kJ * kE], most = 0.f;  // (the sum of the lanes' greatest is no less than any block's sum)
#pragma unroll
    for (int j = 0; j < kJ; ++j)
#pragma unroll
      for (int i = 0; i < kE; ++i) coef[j * kE + i] = 0.f;
    for (int32_t g = 0; g < p.group; ++g) {
      const T* row = static_cast<const T*>(p.q) + s * p.q_row + (static_cast<int64_t>(h) * p.group + g) * p.q_head;
#pragma unroll
      for (int j = 0; j < kJ; ++j) {
        const int at = (j * 32 + lane) * kE;
        if (at < 2 * dim) {
          const bool high = at >= dim;
          const T* from = row + (high ? at - dim : at);
          float q[kE];
          if (p.q_words) {
            akv_unpack<T, kE>(q, akv_load<T, kE>(from));
          } else {
#pragma unroll
            for (int i = 0; i < kE; ++i) q[i] = to_f32<T>(from[i]);
          }
#pragma unroll
          for (int i = 0; i < kE; ++i) coef[j * kE + i] += high ? max_nan(q[i], 0.f) : min_nan(q[i], 0.f);
        }
      }
    }
    const char* base = p.bounds + h * layer_bytes;
    const int32_t stop = n - j0 < p.task ? n - j0 : p.task;
    auto id_of = [&](int32_t c) -> int32_t {
      if (c >= stop) return 0;
      const int32_t id = p.tab.ids[s * p.tab.stride + j0 + c];
      if (static_cast<uint32_t>(id) < static_cast<uint32_t>(p.kv.total)) return id;
      if (h == 0) akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, id, p.kv.total);
      return 0;
    };
    int32_t id = id_of(lane), later = id_of(lane + kWindow);  // of this window and the next
    // kB blocks at a time, the next kB's bounds on their way (behind the row's
    // last block: block 0's, whose scores go nowhere)
    Word w[kB][kJ];
    auto ask = [&](int32_t c, Word(&to)[kB][kJ]) {
#pragma unroll
      for (int u = 0; u < kB; ++u) {
        const char* box = base + __shfl_sync(kFullWarp, id, c % kWindow + u) * p.bounds_page;
#pragma unroll
        for (int j = 0; j < kJ; ++j) {
          const int at = (j * 32 + lane) * kE;
          if (at < 2 * dim) to[u][j] = akv_load<T, kE>(box + at * sizeof(T));
        }
      }
    };
    ask(0, w);
    for (int32_t c = 0; c < stop; c += kB) {
      Word ahead[kB][kJ];
      if ((c + kB) % kWindow == 0) {
        id = later;
        later = id_of(c + kB + kWindow + lane);
      }
      if (c + kB < stop) ask(c + kB, ahead);
      float sum[kB];
#pragma unroll
      for (int u = 0; u < kB; ++u) {
        float all = 0.f;
        sum[u] = 0.f;
#pragma unroll
        for (int j = 0; j < kJ; ++j)
          if ((j * 32 + lane) * kE < 2 * dim) {
            float x[kE];
            akv_unpack<T, kE>(x, w[u][j]);
#pragma unroll
            for (int i = 0; i < kE; ++i) {
              sum[u] = fmaf(coef[j * kE + i], x[i], sum[u]);
              all = fmaf(fabsf(coef[j * kE + i]), fabsf(x[i]), all);
            }
          }
        if (c + u < stop) most = max_nan(most, all);
      }
      // sum u ends, whole, in lanes u * 32 / kB ..
      int off = 16;
#pragma unroll
      for (int x = kB / 2; x >= 1; x >>= 1, off >>= 1) {
        const bool up = lane & off;
#pragma unroll
        for (int i = 0; i < x; ++i) {
          const float a = up ? sum[i] : sum[i + x];
          sum[i] = (up ? sum[i + x] : sum[i]) + __shfl_xor_sync(kFullWarp, a, off);
        }
      }
#pragma unroll
      for (int x = 16 / kB; x >= 1; x >>= 1) sum[0] += __shfl_xor_sync(kFullWarp, sum[0], x);
      const int32_t mine = c + lane / (32 / kB);
      if (lane % (32 / kB) == 0 && mine < stop)
        p.near[(static_cast<int64_t>(s) * p.kv.heads + h) * p.tab.width + j0 + mine] = sum[0];
#pragma unroll
      for (int u = 0; u < kB; ++u)
#pragma unroll
        for (int j = 0; j < kJ; ++j) w[u][j] = ahead[u][j];
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) most += __shfl_xor_sync(kFullWarp, most, off);
    if (lane == 0) p.most[(static_cast<int64_t>(s) * p.kv.heads + h) * groups + j0 / p.task] = most;
  }
}

// A finite score in 32 bits as a whole number of the same order, and back.
AKV_DEV uint32_t order_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}
AKV_DEV float value_of(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k); }

// The score of one block in 64 bits (a warp together; in the same order for every block).
template <typename T>
AKV_DEV double exact_score(const SelectParams& p, int32_t s, int32_t h, int32_t j, int lane) {
  int32_t id = p.tab.ids[s * p.tab.stride + j];
  if (static_cast<uint32_t>(id) >= static_cast<uint32_t>(p.kv.total)) id = 0;
  const T* box = reinterpret_cast<const T*>(p.bounds + id * p.bounds_page + h * 2ll * p.kv.row_bytes);
  const T* q = static_cast<const T*>(p.q) + s * p.q_row + static_cast<int64_t>(h) * p.group * p.q_head;
  double sum = 0.0;
  for (int d = lane; d < p.kv.dim; d += 32) {
    double up = 0.0, down = 0.0;
    for (int32_t g = 0; g < p.group; ++g) {
      const float x = to_f32<T>(q[g * p.q_head + d]);
      up += x != x ? x : fmaxf(x, 0.f);
      down += x != x ? x : fminf(x, 0.f);
    }
    sum = fma(up, static_cast<double>(to_f32<T>(box[p.kv.dim + d])), sum);
    sum = fma(down, static_cast<double>(to_f32<T>(box[d])), sum);
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(kFullWarp, sum, off);
  return sum;
}

template <typename K, int kSelectWarps>
struct RadixShared {
  K ends[2][kSelectWarps];
  int32_t bins[256];
  int32_t found[2];  // digit, keys above it
};

// Narrows [prefix, prefix | ~mask] down to the `need`-th highest of the keys that
// each(f) calls f(key) for, digit by digit from the highest bit in which they
// differ, until a digit's keys are all taken (kWhole: down to one key's
// value, so that few lie too near to it).  `need` becomes how many of the
// range are; at least one is.
template <bool kWhole, typename K, int kSelectWarps, class Each>
AKV_DEV void radix(RadixShared<K, kSelectWarps>& sh, Each each, int32_t& need, K& mask, K& prefix) {
  constexpr int kBits = 8 * sizeof(K);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  K lo = ~static_cast<K>(0), hi = 0;
  each([&](K k) {
    lo = k < lo ? k : lo;
    hi = k > hi ? k : hi;
  });
  auto spread = [&](int width) {
    for (int off = width; off; off >>= 1) {
      const K a = __shfl_xor_sync(kFullWarp, lo, off), b = __shfl_xor_sync(kFullWarp, hi, off);
      lo = a < lo ? a : lo;
      hi = b > hi ? b : hi;
    }
  };
  spread(16);
  __syncthreads();
  if (lane == 0) {
    sh.ends[0][warp] = lo;
    sh.ends[1][warp] = hi;
  }
  __syncthreads();
  lo = sh.ends[0][lane % kSelectWarps];
  hi = sh.ends[1][lane % kSelectWarps];
  spread(16);
  int bit = lo == hi ? 0 : sizeof(K) == 8 ? 64 - __clzll(static_cast<long long>(lo ^ hi)) : 32 - __clz(static_cast<int>(lo ^ hi));
  mask = bit == kBits ? 0 : ~static_cast<K>(0) << bit;
  prefix = hi & mask;
  while (bit > 0) {
    const int width = bit < 8 ? bit : 8;
    bit -= width;
    if (tid < 256) sh.bins[tid] = 0;
    __syncthreads();
    each([&](K k) {
      if ((k & mask) == prefix) atomicAdd(&sh.bins[static_cast<int>(k >> bit) & ((1 << width) - 1)], 1);
    });
    __syncthreads();
    if (warp == 0) {
      // lane i: digits 255 - 8 i .. 248 - 8 i, highest first
      int32_t sum = 0, at[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        at[i] = sh.bins[255 - 8 * lane - i];
        sum += at[i];
      }
      int32_t incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t up = __shfl_up_sync(kFullWarp, incl, o);
        if (lane >= o) incl += up;
      }
      int32_t above = incl - sum;
      if (above < need && incl >= need) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          if (above < need && above + at[i] >= need) {
            sh.found[0] = 255 - 8 * lane - i;
            sh.found[1] = above;
          }
          above += at[i];
        }
      }
    }
    __syncthreads();
    const int32_t digit = sh.found[0], count = sh.bins[digit];
    need -= sh.found[1];
    mask |= static_cast<K>((1 << width) - 1) << bit;
    prefix |= static_cast<K>(digit) << bit;
    __syncthreads();
    if (!kWhole && count == need) break;  // all of them
  }
}

// One CTA per (row, key head): the border in 32 bits by a radix selection, the
// blocks that lie too near to it again in 64 bits and among them a second one;
// then the places, in order.
template <typename T, int kSelectThreads>
__global__ void __launch_bounds__(kSelectThreads) k_select(SelectParams p) {
  constexpr int kSelectWarps = kSelectThreads / 32;
  extern __shared__ __align__(16) float held[];
  __shared__ union {
    RadixShared<uint32_t, kSelectWarps> near;
    RadixShared<uint64_t, kSelectWarps> exact;
  } radix_sh;
  __shared__ int32_t counts[2][kSelectWarps];
  __shared__ float top[kSelectWarps];
  akv_grid_wait();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int32_t s = blockIdx.x / p.kv.heads, h = blockIdx.x % p.kv.heads;
  const int32_t n = blocks_of(p, s);
  int32_t* out = p.selected + static_cast<int64_t>(blockIdx.x) * p.keep;
  if (tid == 0 && h == 0 && p.tab.lengths[s] != akv_held(p.tab, p.kv.bs_log2, s))
    akv_fail(p.st, AKV_ERR_OUT_OF_RANGE, s, p.tab.lengths[s], p.tab.width);
  if (n <= p.keep) {
    for (int32_t i = tid; i < p.keep; i += kSelectThreads) out[i] = i < n ? i : -1;
    return;
  }
  const float* near = p.near + static_cast<int64_t>(blockIdx.x) * p.tab.width;
  uint64_t* keys = p.keys + static_cast<int64_t>(blockIdx.x) * p.tab.width;
  const bool local = n <= kSharedKeys;
  const int32_t from = p.first, to = n - p.last;  // [from, to) are ranked
  int32_t need = p.keep - p.first - p.last;
  if (local)
#pragma unroll 8
    for (int32_t j = from + tid; j < to; j += kSelectThreads) held[j] = __ldcg(near + j);
  // (with infinities and NaN among the terms this is none that is finite: every
  // block is scored again)
  float most = 0.f;
  const int32_t tasks = (p.tab.width + p.task - 1) / p.task, used = (n + p.task - 1) / p.task;
  for (int32_t i = tid; i < used; i += kSelectThreads)
    most = max_nan(most, __ldcg(p.most + static_cast<int64_t>(blockIdx.x) * tasks + i));
  most = warp_max(most);
  if (lane == 0) top[warp] = most;
  __syncthreads();
  most = warp_max(top[lane % kSelectWarps]);
  const float off = (p.group + 32) * 1.1920929e-7f * most + 1e-35f;  // no score is further off than that
  auto score = [&](int32_t j) { return local ? held[j] : __ldcg(near + j); };
  // scores above `high` are taken, below `low` not
  float low = -INFINITY, high = INFINITY;
  if (isfinite(off) && need > 0) {
    uint32_t mask, prefix;
    int32_t left = need;
    radix<true>(
        radix_sh.near,
        [&](auto f) {
#pragma unroll 4
          for (int32_t j = from + tid; j < to; j += kSelectThreads) f(order_of(score(j)));
        },
        left, mask, prefix);
    low = value_of(prefix) - 2.f * off;
    high = value_of(prefix | ~mask) + 2.f * off;
    low -= fabsf(low) * 2.4e-7f;  // these two sums' own rounding
    high += fabsf(high) * 2.4e-7f;
    if (!(low > -INFINITY)) low = -INFINITY;
    if (!(high < INFINITY)) high = INFINITY;
  }
  // Each warp counts its stretch.
  const int32_t per = ((n + kSelectWarps - 1) / kSelectWarps + 31) / 32 * 32;
  const int32_t w0 = warp * per, w1 = min(n, w0 + per);
  // 2: taken, 1: in question, 0: not taken
  auto class_of = [&](int32_t j) {
    if (j < from || j >= to) return 2;
    if (need == 0) return 0;
    const float x = score(j);
    return x > high ? 2 : x < low ? 0 : 1;
  };
  auto total = [&](int32_t* of) {  // of the warps' counts
    int32_t x = lane < kSelectWarps ? of[lane] : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(kFullWarp, x, o);
    return x;
  };
  int32_t sure = 0, open = 0;
  for (int32_t j = w0 + lane; j < w1; j += 32) {
    const int c = class_of(j);
    sure += c == 2;
    open += c == 1;
  }
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    sure += __shfl_xor_sync(kFullWarp, sure, o);
    open += __shfl_xor_sync(kFullWarp, open, o);
  }
  if (lane == 0) {
    counts[0][warp] = sure;
    counts[1][warp] = open;
  }
  __syncthreads();
  int32_t left = p.keep - total(counts[0]);  // to take of those in question
  const int32_t in_question = total(counts[1]);
  uint64_t mask = 0, prefix = 0;  // (all of them equal)
  if (left > 0 && left < in_question) {
    for (int32_t j0 = w0; j0 < w1; j0 += 32) {
      uint32_t open_here = __ballot_sync(kFullWarp, j0 + lane < w1 && class_of(j0 + lane) == 1);
      for (; open_here; open_here &= open_here - 1) {
        const int32_t j = j0 + __ffs(open_here) - 1;
        const uint64_t k = key_of(exact_score<T>(p, s, h, j, lane));
        if (lane == 0) keys[j] = k;
      }
    }
    __syncthreads();  // (the keys are this CTA's own)
    radix<false>(
        radix_sh.exact,
        [&](auto f) {
          for (int32_t j = from + tid; j < to; j += kSelectThreads)
            if (class_of(j) == 1) f(keys[j]);
        },
        left, mask, prefix);
  }
  // Taken: the sure ones, those in question above the prefix's range, and the
  // first `left` of those in it.
  auto classes = [&](int32_t j, uint32_t& gt, uint32_t& eq) {
    const int c = j < w1 ? class_of(j) : 0;
    const uint64_t k = c == 1 && mask != 0 ? keys[j] & mask : 0;
    gt = __ballot_sync(kFullWarp, c == 2 || (c == 1 && k > prefix));
    eq = __ballot_sync(kFullWarp, c == 1 && k == prefix);
  };
  int32_t above = 0, equal = 0;
  for (int32_t j0 = w0; j0 < w1; j0 += 32) {
    uint32_t gt, eq;
    classes(j0 + lane, gt, eq);
    above += __popc(gt);
    equal += __popc(eq);
  }
  __syncthreads();
  if (lane == 0) {
    counts[0][warp] = above;
    counts[1][warp] = equal;
  }
  __syncthreads();
  above = lane < warp ? counts[0][lane % kSelectWarps] : 0;
  equal = lane < warp ? counts[1][lane % kSelectWarps] : 0;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    above += __shfl_xor_sync(kFullWarp, above, o);
    equal += __shfl_xor_sync(kFullWarp, equal, o);
  }
  for (int32_t j0 = w0; j0 < w1; j0 += 32) {
    uint32_t gt, eq;
    classes(j0 + lane, gt, eq);
    const uint32_t below = (1u << lane) - 1;
    const int32_t g = above + __popc(gt & below), e = equal + __popc(eq & below);
    if ((gt >> lane & 1) || ((eq >> lane & 1) && e < left)) out[g + min(e, left)] = j0 + lane;
    above += __popc(gt);
    equal += __popc(eq);
  }
}

using ScoreKernel = void (*)(SelectParams);

// The widest word that the addresses and the head dim allow; a lane holds
// every 32nd word of a block's bounds.
template <typename T>
ScoreKernel score_kernel(int dim, int elements) {
  constexpr int kWide = 16 / sizeof(T);
  if (elements >= kWide) {
    if (2 * dim <= 32 * kWide) return k_score<T, kWide, 1>;
    if (2 * dim <= 64 * kWide) return k_score<T, kWide, 2>;
    return k_score<T, kWide, sizeof(T) == 4 ? 4 : 2>;
  }
  if (elements >= 2) return k_score<T, 2, 8>;
  return k_score<T, 1, 16>;
}

ScoreKernel score_kernel(int32_t dtype, int dim, int elements) {
  return dtype == AKV_F32 ? score_kernel<float>(dim, elements)
                          : dtype == AKV_F16 ? score_kernel<__half>(dim, elements)
                                             : score_kernel<__nv_bfloat16>(dim, elements);
}

int64_t key_bytes(int64_t rows, int64_t heads, int64_t width, int64_t keep) {
  return width <= keep ? 0 : rows * heads * width * 16;  // a key, a score and (at most one a block) a bound each
}

template <int kN>
ScoreKernel select_kernel(int32_t dtype) {
  return dtype == AKV_F32 ? k_select<float, kN> : dtype == AKV_F16 ? k_select<__half, kN> : k_select<__nv_bfloat16, kN>;
}

}  // namespace

int akv_select_prepare() {
  for (int32_t dtype : {AKV_F32, AKV_F16, AKV_BF16})
    for (int dim : {32, 64, 128, 256})
      for (int elements : {1, 2, 8})
        if (int rc = akv_load_kernel(reinterpret_cast<const void*>(score_kernel(dtype, dim, elements)),
                                     "akv_prepare: k_score"))
          return rc;
  for (int32_t dtype : {AKV_F32, AKV_F16, AKV_BF16})
    for (ScoreKernel k : {select_kernel<512>(dtype), select_kernel<1024>(dtype)})
      if (int rc = akv_load_kernel(reinterpret_cast<const void*>(k), "akv_prepare: k_select")) return rc;
  return AKV_OK;
}

extern "C" int64_t akv_select_blocks_scratch_bytes(int32_t rows, int32_t num_kv_heads, int32_t table_width,
                                                   int32_t keep) {
  if (rows < 0 || num_kv_heads <= 0 || table_width < 0 || keep <= 0) {
    akv_set_error("akv_select_blocks_scratch_bytes: bad arguments");
    return -1;
  }
  return key_bytes(rows, num_kv_heads, table_width, keep);
}

extern "C" int akv_select_blocks(const AkvPagedPool* pool, const void* bounds, const AkvPageBatch* batch,
                                 const AkvHeads* query, int32_t group, int32_t keep, int32_t first, int32_t last,
                                 int32_t* selected, void* scratch, int64_t scratch_bytes, AkvStatus* status,
                                 void* stream) {
  const char* what = "akv_select_blocks";
  SelectParams p = {};
  if (int rc = akv_layer_view(what, pool, &p.kv)) return rc;
  if (int rc = akv_tables_view(what, batch, pool->block_size, &p.tab)) return rc;
  AKV_ARG_CHECK(group > 0 && keep > 0 && first >= 0 && last >= 0 && static_cast<int64_t>(first) + last <= keep,
                "%s: group=%d keep=%d first=%d last=%d", what, group, keep, first, last);
  if (p.tab.rows == 0) return AKV_OK;
  AKV_ARG_CHECK(bounds && query && query->data && selected, "%s: NULL pointer", what);
  AKV_ARG_CHECK(query->stride_token >= 0 && query->stride_head >= 0, "%s: negative stride", what);
  const int es = akv_dtype_bytes(pool->dtype);
  AKV_ARG_CHECK(akv_aligned(bounds, es) && akv_aligned(query->data, es) && akv_aligned(selected, 4) &&
                    akv_aligned(scratch, 16),
                "%s: misaligned pointer", what);
  const int64_t need = key_bytes(p.tab.rows, p.kv.heads, p.tab.width, keep);
  AKV_ARG_CHECK(scratch_bytes >= need && (scratch || need == 0), "%s: scratch has %lld bytes, %lld are needed", what,
                static_cast<long long>(scratch_bytes), static_cast<long long>(need));
  const int64_t pairs = static_cast<int64_t>(p.tab.rows) * p.kv.heads;
  AKV_ARG_CHECK(pairs <= INT_MAX, "%s: too many rows", what);
  const int64_t head_bytes = 2ll * p.kv.row_bytes, layer_bytes = head_bytes * p.kv.heads;
  p.bounds = static_cast<const char*>(bounds) + layer_bytes * pool->layer;
  p.bounds_page = layer_bytes * pool->num_layers;
  p.q = query->data;
  p.q_row = query->stride_token;
  p.q_head = query->stride_head;
  p.group = group;
  p.keep = keep;
  p.first = first;
  p.last = last;
  p.keys = static_cast<uint64_t*>(scratch);
  p.near = reinterpret_cast<float*>(p.keys + need / 16);
  p.most = p.near + need / 16;
  p.selected = selected;
  p.st = status;
  cudaStream_t st = akv_stream(stream);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(pairs));
  // 1,024 threads fill an SM: while there is one for each pair they finish
  // sooner (19.5 against 24.8 us for 8 pairs of 8,126 blocks); beyond it two
  // CTAs of 512 an SM do (21 against 25 us for 256 pairs of 560 to 2,048).
  const bool few = pairs <= kAkvSMs;
  cfg.blockDim = dim3(few ? 1024 : 512);
  cfg.stream = st;
  // Its launch is prepared while k_score runs (which releases nothing early: the
  // blocks start when it has ended).  Without it the scoring and choosing of one
  // row took 2 to 4 us longer, those of 32 rows 2 to 3.
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  if (need) {
    const uint64_t bits = reinterpret_cast<uintptr_t>(bounds) | static_cast<uint64_t>(p.kv.row_bytes);
    const int low = static_cast<int>(bits & (~bits + 1) & 31);
    p.q_words = ((reinterpret_cast<uintptr_t>(query->data) | static_cast<uint64_t>(query->stride_token * es) |
                  static_cast<uint64_t>(query->stride_head * es)) % 16) == 0;
    // A task reads its row's queries and its first ids before it can start (3
    // latencies): as many blocks each as leave every resident warp four, to even them out.
    const int64_t per = kThreads / 32, most = 2ll * kAkvSMs;
    const int64_t share = pairs * p.tab.width / (most * per * kWindow);
    p.task = kWindow * static_cast<int32_t>(share < 8 ? 1 : share > 64 ? 16 : share / 4);
    const int64_t warps = pairs * ((p.tab.width + p.task - 1) / p.task);
    const int64_t ctas = (warps + per - 1) / per;
    score_kernel(pool->dtype, p.kv.dim, (low == 0 || low > 16 ? 16 : low) / es)<<<
        static_cast<unsigned>(ctas < most ? ctas : most), kThreads, 0, st>>>(p);
    AKV_LAUNCH_CHECK(what);
    cfg.dynamicSmemBytes = static_cast<size_t>(p.tab.width < kSharedKeys ? p.tab.width : kSharedKeys) * 4;
    cfg.numAttrs = 1;
  }
  const cudaError_t err = cudaLaunchKernelEx(&cfg, few ? select_kernel<1024>(pool->dtype) : select_kernel<512>(pool->dtype), p);
  if (err != cudaSuccess) return akv_cuda_fail(err, what);
  return AKV_OK;
}
