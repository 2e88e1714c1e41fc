// Kernels of the verification of drafted tokens (include/et_speculative.h).
//
// A sequence has K + 1 target rows and, with a draft model, K draft rows.  Three launches:
//   verify_stats   every row is cut into chunks; a workgroup reduces one chunk to (max, sum of
//                  exp((l - max) / T)), or, for a greedy sequence, to its best (key, ~index)
//   verify_rest    (draft model only) per sequence: which position decides, then the mass of
//                  max(p - q, 0) of every chunk of that position's rows
//   verify_finish  one workgroup per sequence: the decision again, the chunk in which the drawn token
//                  lies, and a scan of that chunk
// The kernel boundaries order the three; nothing is handed over inside a launch, so a launch needs no
// waits and leaves no state behind.
//
// Weights are computed in 64 bits: a token is the place where a running sum over up to 2^18 weights
// crosses a threshold, and an error e of that sum moves about e x (entries that matter) draws over a
// border; at 1e-13 that is one draw in 1e8.  The 64-bit rate of the vector unit is its 32-bit rate, so
// what this costs is registers and about twice the instructions of a 32-bit exponential.
#pragma once

#include "ets_kernels.h"

namespace ets {

constexpr int kVerifyBlock = 256;    // lanes of verify_stats and verify_rest
constexpr int kFinishBlock = 1024;   // lanes of verify_finish
constexpr int kMaxDrafts = 64;       // drafts per sequence: one lane of a wave each
constexpr int kExp2Steps = 256;      // entries of the table of 2^(j / 256)
constexpr int kSmallChunk = 2048, kLargeChunk = 8192;  // entries per chunk

struct ChunkStat {
  double sum;   // of exp((l - max) / T); NaN where the chunk holds a NaN or +inf (greedy: the bits of the best key)
  float max;
  float pad;
};

struct VerifyParams {
  const void* target;
  const void* draft;  // or null
  int64_t target_seq, target_pos, draft_seq, draft_pos;  // strides in elements
  const int32_t* draft_tokens;
  int64_t draft_tokens_stride;
  const int32_t* lengths;
  const float* temperatures;
  float temperature;
  const float* coins;
  int64_t coins_stride;
  int32_t* tokens;
  int64_t tokens_stride;
  int32_t* accepted;
  int32_t vocab, drafts, sequences;
  int32_t chunks;          // per row
  int32_t rows_per_seq;    // K + 1, or 2K + 1 with a draft model
  ChunkStat* stats;        // [sequences, rows_per_seq, chunks]
  double* rest;            // [sequences, chunks]
  const double* exp2_table;
};

// A 16-byte load from an address aligned to an element only (global loads need no more than that).
template <int DT>
struct __attribute__((packed, aligned(DT == kDtypeFloat ? 4 : 2))) LooseVec {
  uint32_t w[4];
};

// Entries [first, first + VecElems) of a row as raw bits; those at n and behind read as -inf and are
// not touched in memory.
template <int DT>
__device__ __forceinline__ uint4 load_raw(const char* row, int first, int n) {
  constexpr int VE = VecElems<DT>::value, ES = ElemSize<DT>::value;
  if (first + VE <= n) {
    const LooseVec<DT> v = *reinterpret_cast<const LooseVec<DT>*>(row + static_cast<int64_t>(first) * ES);
    return make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
  }
  constexpr uint32_t kFill = DT == kDtypeFloat ? 0xff800000u : (DT == kDtypeBFloat16 ? 0xff80ff80u : 0xfc00fc00u);
  uint32_t w[4] = {kFill, kFill, kFill, kFill};
#pragma unroll
  for (int e = 0; e < VE; ++e) {
    if (first + e < n) {
      if (DT == kDtypeFloat) {
        w[e] = reinterpret_cast<const uint32_t*>(row)[first + e];
      } else {
        const uint32_t h = reinterpret_cast<const uint16_t*>(row)[first + e];
        w[e >> 1] = (e & 1) ? ((w[e >> 1] & 0xffffu) | (h << 16)) : ((w[e >> 1] & 0xffff0000u) | h);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// exp((l - m) / T) for l <= m, c = 256 log2(e) / T: 2^(k/256) 2^(r/256) with k = round((l - m) c), the
// first factor from the table (a copy in LDS) and k's high bits, the second, |r| <= 1/2, by its series to
// the third power: the first term left out is (ln 2 / 512)^4 / 24 = 1.4e-13.  l = -inf gives 0, whatever T:
// the argument is cut off where the result is 0 (fmax also drops the NaN of -inf * 0 at T = inf).
__device__ __forceinline__ double exp_weight(float l, double m, double c, const double* table) {
  constexpr double kStep = 0.69314718055994530942 / kExp2Steps;
  const double t = fmax((static_cast<double>(l) - m) * c, -600000.0);
  const double kd = __builtin_rint(t);
  const double r = t - kd;
  const int k = static_cast<int>(kd);
  const double poly = fma(r, fma(r, fma(r, kStep * kStep * kStep / 6.0, kStep * kStep / 2.0), kStep), 1.0);
  return ldexp(poly * table[k & (kExp2Steps - 1)], k >> 8);
}

// The same for one entry, without the table.
__device__ __forceinline__ double exact_weight(float l, float m, float temperature) {
  return l == -INFINITY ? 0.0 : exp((static_cast<double>(l) - m) / temperature);
}

__device__ __forceinline__ double temperature_factor(float temperature) {
  return (kExp2Steps * 1.44269504088896340736) / static_cast<double>(temperature);
}

__device__ __forceinline__ float sequence_temperature(const VerifyParams& p, int b) {
  const float t = p.temperatures ? p.temperatures[b] : p.temperature;
  return t < 0.0f ? 0.0f : t;
}

__device__ __forceinline__ int sequence_length(const VerifyParams& p, int b) {
  return p.lengths ? min(max(p.lengths[b], 0), p.drafts) : p.drafts;
}

template <int DT>
__device__ __forceinline__ const char* target_row(const VerifyParams& p, int b, int i) {
  return static_cast<const char*>(p.target) + (b * p.target_seq + i * p.target_pos) * ElemSize<DT>::value;
}
template <int DT>
__device__ __forceinline__ const char* draft_row(const VerifyParams& p, int b, int i) {
  return static_cast<const char*>(p.draft) + (b * p.draft_seq + i * p.draft_pos) * ElemSize<DT>::value;
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
__device__ __forceinline__ float wave_max_f32(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}

// Sum over the workgroup, in a fixed order; every lane gets it.  `red`: one double per wave.
template <int WAVES>
__device__ __forceinline__ double block_sum_f64(double v, double* red) {
  v = wave_sum_f64(v);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = red[0];
#pragma unroll
  for (int w = 1; w < WAVES; ++w) s += red[w];
  __syncthreads();
  return s;
}

// ---- statistics of every chunk ------------------------------------------------------------------
// U vectors per lane, all of them in registers: the chunk is read once, its maximum found, then its sum.
template <int DT, int U>
__global__ void __launch_bounds__(kVerifyBlock)
verify_stats_kernel(const VerifyParams p) {
  constexpr int VE = VecElems<DT>::value;
  constexpr int kWavesHere = kVerifyBlock / 64;
  __shared__ double table[kExp2Steps];
  __shared__ float red_max[kWavesHere];
  __shared__ int red_bad[kWavesHere];
  __shared__ double red_sum[kWavesHere];
  __shared__ uint64_t red_best[kWavesHere];
  const int tid = threadIdx.x, wave = tid >> 6;
  const int row = blockIdx.x / p.chunks, chunk = blockIdx.x - row * p.chunks;
  const int b = row / p.rows_per_seq, j = row - b * p.rows_per_seq;
  const bool is_draft = j > p.drafts;
  const int pos = is_draft ? j - p.drafts - 1 : j;
  const int len = sequence_length(p, b);
  if (is_draft ? pos >= len : pos > len) return;  // (the row is not the sequence's)
  const float temperature = sequence_temperature(p, b);
  const bool greedy = temperature == 0.0f;
  if (is_draft && greedy) return;
  const char* src = is_draft ? draft_row<DT>(p, b, pos) : target_row<DT>(p, b, pos);
  const int first = chunk * (kVerifyBlock * VE * U);
  ChunkStat* out = p.stats + static_cast<int64_t>(row) * p.chunks + chunk;

  uint4 raw[U];
#pragma unroll
  for (int u = 0; u < U; ++u) raw[u] = load_raw<DT>(src, first + (u * kVerifyBlock + tid) * VE, p.vocab);
  for (int i = tid; i < kExp2Steps; i += kVerifyBlock) table[i] = p.exp2_table[i];

  if (greedy) {
    uint64_t best = 0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[VE];
      decode_vec<DT>(raw[u], v);
      const int at = first + (u * kVerifyBlock + tid) * VE;
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        const uint64_t key = pack_best(order_key(v[e]), at + e);
        if (at + e < p.vocab && key > best) best = key;
      }
    }
    best = wave_max_u64(best);
    if ((tid & 63) == 0) red_best[wave] = best;
    __syncthreads();
    if (tid == 0) {
      for (int w = 1; w < kWavesHere; ++w) best = red_best[w] > best ? red_best[w] : best;
      out->sum = __longlong_as_double(static_cast<long long>(best));
    }
    return;
  }

  float m = -INFINITY;
  int bad = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[VE];
    decode_vec<DT>(raw[u], v);
#pragma unroll
    for (int e = 0; e < VE; ++e) {
      m = fmaxf(m, v[e]);
      bad |= v[e] != v[e];
    }
  }
  m = wave_max_f32(m);
  bad = __any(bad);
  if ((tid & 63) == 0) red_max[wave] = m, red_bad[wave] = bad;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWavesHere; ++w) m = fmaxf(m, red_max[w]), bad |= red_bad[w];
  if (bad || m == INFINITY || m == -INFINITY || temperature != temperature) {  // (the same in every lane)
    if (tid == 0) {
      out->max = m;
      out->sum = (m == -INFINITY && !bad && temperature == temperature) ? 0.0 : static_cast<double>(NAN);
    }
    return;
  }
  const double c = temperature_factor(temperature), md = m;
  double sum = 0.0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[VE];
    decode_vec<DT>(raw[u], v);
#pragma unroll
    for (int e = 0; e < VE; ++e) sum += exp_weight(v[e], md, c, table);
  }
  sum = block_sum_f64<kWavesHere>(sum, red_sum);
  if (tid == 0) {
    out->max = m;
    out->sum = sum;
  }
}

// ---- the decision -------------------------------------------------------------------------------
struct RowNorm {
  double sum;  // of exp((l - max) / T) over the row; not above 0 where the row has no distribution
  float max;
  int32_t best;  // greedy sequences: the row's arg-max
};

// One wave: the row's statistics from its chunks', in a fixed order.
__device__ __forceinline__ RowNorm combine_chunks(const ChunkStat* st, int chunks, bool greedy, float temperature) {
  const int lane = threadIdx.x & 63;
  RowNorm r = {0.0, -INFINITY, 0};
  if (greedy) {
    uint64_t best = 0;
    for (int c = lane; c < chunks; c += 64) {
      const uint64_t k = static_cast<uint64_t>(__double_as_longlong(st[c].sum));
      best = k > best ? k : best;
    }
    best = wave_max_u64(best);
    r.best = static_cast<int32_t>(0xffffffffu - static_cast<uint32_t>(best));
    return r;
  }
  float m = -INFINITY;
  for (int c = lane; c < chunks; c += 64) m = fmaxf(m, st[c].max);
  m = wave_max_f32(m);
  double s = 0.0;
  for (int c = lane; c < chunks; c += 64) {
    const double sc = st[c].sum;  // (a chunk without a finite entry: 0; exp(-inf) stays out of the sum)
    s += st[c].max == -INFINITY ? sc : sc * exact_weight(st[c].max, m, temperature);
  }
  r.max = m;
  r.sum = wave_sum_f64(s);
  return r;
}

struct Decision {
  int kept;        // drafts accepted
  int len;         // the sequence's drafts
  int valid;       // 0: a row at `kept` has no distribution
  int best;        // greedy: the arg-max of the target row at `kept`
  float temperature;
  RowNorm t, d;    // rows at `kept` (d: with draft logits and kept < len only)
};

// Which position decides, worked out by the whole workgroup of WAVES waves from the statistics (every
// workgroup that needs it does so for itself: it is a few hundred bytes and one exponential per draft).
template <int DT, int WAVES>
__device__ __forceinline__ Decision decide(const VerifyParams& p, int b, RowNorm* rows /* [2 kMaxDrafts + 1], LDS */, int* shared /* LDS */) {
  const int tid = threadIdx.x, wave = tid >> 6;
  Decision out;
  out.len = sequence_length(p, b);
  out.temperature = sequence_temperature(p, b);
  const bool greedy = out.temperature == 0.0f;
  const ChunkStat* st = p.stats + static_cast<int64_t>(b) * p.rows_per_seq * p.chunks;
  for (int j = wave; j < p.rows_per_seq; j += WAVES) {
    const bool is_draft = j > p.drafts;
    const int pos = is_draft ? j - p.drafts - 1 : j;
    if ((is_draft && greedy) || (is_draft ? pos >= out.len : pos > out.len)) continue;
    const RowNorm r = combine_chunks(st + static_cast<int64_t>(j) * p.chunks, p.chunks, greedy, out.temperature);
    if ((tid & 63) == 0) rows[j] = r;
  }
  __syncthreads();
  if (wave == 0) {
    bool accept = false, valid = true;
    if (tid <= out.len) {
      const RowNorm t = rows[tid];
      valid = greedy || t.sum > 0.0;
      if (tid < out.len) {
        const int x = p.draft_tokens[b * p.draft_tokens_stride + tid];
        if (greedy) {
          accept = x == t.best;
        } else {
          double q = 1.0;
          if (p.draft) {
            const RowNorm d = rows[p.drafts + 1 + tid];
            valid = valid && d.sum > 0.0;
            if (x >= 0 && x < p.vocab)
              q = exact_weight(load_elem<DT>(draft_row<DT>(p, b, tid), x), d.max, out.temperature) / d.sum;
          }
          if (valid && x >= 0 && x < p.vocab) {
            const double pt = exact_weight(load_elem<DT>(target_row<DT>(p, b, tid), x), t.max, out.temperature) / t.sum;
            accept = static_cast<double>(p.coins[b * p.coins_stride + tid]) * q < pt;
          }
        }
      }
    }
    // (lane 64 does not exist: with 64 drafts the row behind the last one is looked at below)
    const uint64_t stop = __ballot(tid < out.len && !accept);
    const int kept = stop ? __ffsll(static_cast<unsigned long long>(stop)) - 1 : out.len;
    const uint64_t good = __ballot(valid);
    if (tid == 0) {
      shared[0] = kept;
      shared[1] = kept < 64 ? static_cast<int>((good >> kept) & 1) : (greedy || rows[kept].sum > 0.0);
    }
  }
  __syncthreads();
  out.kept = shared[0];
  out.valid = shared[1];
  out.t = rows[out.kept];
  out.best = out.t.best;
  if (p.draft && out.kept < out.len && !greedy) {
    out.d = rows[p.drafts + 1 + out.kept];
  } else {
    out.d = RowNorm{1.0, 0.0f, 0};
  }
  return out;
}

// max(p - q, 0) of one entry.
__device__ __forceinline__ double rest_weight(float t, float d, const Decision& dec, double c, double inv_t, double inv_d,
                                              const double* table) {
  return fmax(exp_weight(t, dec.t.max, c, table) * inv_t - exp_weight(d, dec.d.max, c, table) * inv_d, 0.0);
}

// ---- mass of max(p - q, 0) per chunk ------------------------------------------------------------
template <int DT, int U>
__global__ void __launch_bounds__(kVerifyBlock)
verify_rest_kernel(const VerifyParams p) {
  constexpr int VE = VecElems<DT>::value;
  constexpr int kWavesHere = kVerifyBlock / 64;
  __shared__ double table[kExp2Steps];
  __shared__ RowNorm rows[2 * kMaxDrafts + 1];
  __shared__ int shared[2];
  __shared__ double red[kWavesHere];
  const int tid = threadIdx.x;
  const int b = blockIdx.x / p.chunks, chunk = blockIdx.x - b * p.chunks;
  for (int i = tid; i < kExp2Steps; i += kVerifyBlock) table[i] = p.exp2_table[i];
  const Decision dec = decide<DT, kWavesHere>(p, b, rows, shared);
  if (dec.kept >= dec.len || !dec.valid || dec.temperature == 0.0f) return;  // (the same in every lane)
  const char* t_row = target_row<DT>(p, b, dec.kept);
  const char* d_row = draft_row<DT>(p, b, dec.kept);
  const int first = chunk * (kVerifyBlock * VE * U);
  const double c = temperature_factor(dec.temperature), inv_t = 1.0 / dec.t.sum, inv_d = 1.0 / dec.d.sum;
  double sum = 0.0;
#pragma unroll 1
  for (int u = 0; u < U; ++u) {
    const int at = first + (u * kVerifyBlock + tid) * VE;
    float tv[VE], dv[VE];
    decode_vec<DT>(load_raw<DT>(t_row, at, p.vocab), tv);
    decode_vec<DT>(load_raw<DT>(d_row, at, p.vocab), dv);
#pragma unroll
    for (int e = 0; e < VE; ++e) sum += rest_weight(tv[e], dv[e], dec, c, inv_t, inv_d, table);
  }
  sum = block_sum_f64<kWavesHere>(sum, red);
  if (tid == 0) p.rest[static_cast<int64_t>(b) * p.chunks + chunk] = sum;
}

// ---- the draw -----------------------------------------------------------------------------------
constexpr double kEmptyRest = 1.0 / (1 << 30);  // residual masses up to this are rounding noise of p - q

template <int DT, int CHUNK>
__global__ void __launch_bounds__(kFinishBlock)
verify_finish_kernel(const VerifyParams p) {
  constexpr int VE = VecElems<DT>::value;
  constexpr int kWavesHere = kFinishBlock / 64;
  constexpr int E = CHUNK / kFinishBlock < VE ? VE : CHUNK / kFinishBlock;  // consecutive entries per lane
  static_assert(E % VE == 0 && CHUNK % E == 0 && CHUNK / E <= kFinishBlock, "lanes cover the chunk");
  __shared__ double table[kExp2Steps];
  __shared__ RowNorm rows[2 * kMaxDrafts + 1];
  __shared__ int shared[2];
  __shared__ double red[kWavesHere];
  __shared__ double pick_at;   // what is left of the threshold when the chunk begins
  __shared__ int pick_chunk;
  __shared__ int found, last;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int b = blockIdx.x;
  for (int i = tid; i < kExp2Steps; i += kFinishBlock) table[i] = p.exp2_table[i];
  if (tid == 0) found = CHUNK, last = -1;
  const Decision dec = decide<DT, kWavesHere>(p, b, rows, shared);
  int32_t* out = p.tokens + b * p.tokens_stride;
  const int32_t* drafted = p.draft_tokens + b * p.draft_tokens_stride;
  auto answer = [&](int token) {  // (by every lane, with the same token)
    for (int i = tid; i <= p.drafts; i += kFinishBlock) out[i] = i < dec.kept ? drafted[i] : (i == dec.kept ? token : -1);
    if (tid == 0) p.accepted[b] = dec.kept;
  };
  if (!dec.valid) return answer(-1);
  if (dec.temperature == 0.0f) return answer(dec.best);

  const bool rejected = dec.kept < dec.len;
  const char* t_row = target_row<DT>(p, b, dec.kept);
  const char* d_row = p.draft && rejected ? draft_row<DT>(p, b, dec.kept) : t_row;
  const double c = temperature_factor(dec.temperature), inv_t = 1.0 / dec.t.sum, inv_d = 1.0 / dec.d.sum;
  const ChunkStat* st = p.stats + (static_cast<int64_t>(b) * p.rows_per_seq + dec.kept) * p.chunks;
  const double* rest = p.rest + static_cast<int64_t>(b) * p.chunks;

  // the weights of this lane's entries of a chunk: p (unnormalised), p without the entry `skip`, or p - q
  auto weights = [&](int chunk, bool minus_q, int skip, double* w) {
    const int at = chunk * CHUNK + tid * E;
#pragma unroll
    for (int g = 0; g < E / VE; ++g) {
      float tv[VE], dv[VE];
      const bool mine = tid * E < CHUNK;
      decode_vec<DT>(load_raw<DT>(t_row, at + g * VE, mine ? p.vocab : 0), tv);
      if (minus_q) decode_vec<DT>(load_raw<DT>(d_row, at + g * VE, mine ? p.vocab : 0), dv);
#pragma unroll
      for (int e = 0; e < VE; ++e) {
        w[g * VE + e] = minus_q ? rest_weight(tv[e], dv[e], dec, c, inv_t, inv_d, table)
                                : (at + g * VE + e == skip ? 0.0 : exp_weight(tv[e], dec.t.max, c, table));
      }
    }
  };

  // the mode: p - q of the draft model; p without the drafted token; p
  bool minus_q = p.draft && rejected;
  int skip = -1;
  double skip_chunk_mass = 0.0;
  if (!p.draft && rejected) {
    const int x = drafted[dec.kept];
    if (x >= 0 && x < p.vocab) {
      // the mass of x's chunk without x, summed anew: p(x) may be all but 1, and a difference would cancel
      skip = x;
      double w[E], s = 0.0;
      weights(x / CHUNK, false, skip, w);
#pragma unroll
      for (int e = 0; e < E; ++e) s += w[e];
      skip_chunk_mass = block_sum_f64<kWavesHere>(s, red);
    }
  }
  if (wave == 0) {
    auto mass = [&](int k) {
      if (k >= p.chunks) return 0.0;
      if (minus_q) return rest[k];
      if (skip >= 0 && k == skip / CHUNK) return skip_chunk_mass;
      return st[k].sum * exact_weight(st[k].max, dec.t.max, dec.temperature);
    };
    auto total_of = [&] {
      double s = 0.0;
      for (int k = lane; k < p.chunks; k += 64) s += mass(k);
      return wave_sum_f64(s);
    };
    double total = total_of();
    if ((minus_q && !(total > kEmptyRest)) || (skip >= 0 && !(total * inv_t > kEmptyRest))) {
      minus_q = false, skip = -1;
      total = total_of();
    }
    const double threshold = static_cast<double>(p.coins[b * p.coins_stride + p.drafts]) * total;
    double before = 0.0;  // of the chunks of the groups of 64 already passed
    int chunk = -1, last_mass = 0;
    double at = INFINITY;
    for (int k0 = 0; k0 < p.chunks && chunk < 0; k0 += 64) {
      const double m = mass(k0 + lane);
      double incl = m;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(incl, d);
        if (lane >= d) incl += o;
      }
      incl += before;
      const uint64_t hit = __ballot(m > 0.0 && incl > threshold);
      const uint64_t some = __ballot(m > 0.0);
      if (some) last_mass = k0 + 63 - __clzll(static_cast<long long>(some));
      if (hit) {
        const int l = __ffsll(static_cast<unsigned long long>(hit)) - 1;
        chunk = k0 + l;
        at = threshold - (__shfl(incl, l) - __shfl(m, l));
      }
      before = __shfl(incl, 63);
    }
    if (chunk < 0) chunk = last_mass;  // (a coin of 1 or more, or a sum that rounds below the threshold: the last entry)
    if (lane == 0) pick_chunk = chunk, pick_at = at, shared[0] = minus_q, shared[1] = skip;
  }
  __syncthreads();
  const int chunk = pick_chunk;
  double w[E];
  weights(chunk, shared[0] != 0, shared[1], w);
  double mine = 0.0;
#pragma unroll
  for (int e = 0; e < E; ++e) mine += w[e];
  // inclusive scan over the lanes
  double incl = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double o = __shfl_up(incl, d);
    if (lane >= d) incl += o;
  }
  if (lane == 63) red[wave] = incl;
  __syncthreads();
  double run = incl - mine;
  for (int v = 0; v < wave; ++v) run += red[v];
  int first_hit = CHUNK, last_some = -1;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    run += w[e];
    if (w[e] > 0.0) {
      last_some = tid * E + e;
      if (run > pick_at && first_hit == CHUNK) first_hit = tid * E + e;
    }
  }
  if (first_hit < CHUNK) atomicMin(&found, first_hit);
  if (last_some >= 0) atomicMax(&last, last_some);
  __syncthreads();
  const int in_chunk = found < CHUNK ? found : last;
  answer(in_chunk < 0 ? -1 : chunk * CHUNK + in_chunk);
}

}  // namespace ets
