// The waves of a decode row's workgroup: queries, keys and values of one kv head, with their online
// softmax. Shared by the decode kernels and the windowed prefill's launch, which takes decode rows
// along.
#pragma once

#include "common.hpp"
#include "paged_attention.hpp"

namespace mvllm {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
// Tokens per row group per step (each step's K/V rows are requested together).
#ifndef MVLLM_DECODE_UNROLL
#define MVLLM_DECODE_UNROLL 4
#endif
constexpr int kUnroll = MVLLM_DECODE_UNROLL;

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ u32x4 load16_stream(const char* p) {
  return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p));
}

// One lane's E elements of a query head, and their dot product with a 16-byte chunk of a K
// row in fp32. 16-bit queries stay packed and use the two-element dot instruction (exact
// products, one rounding per pair: against 64 bits 1.27e-8 where the multiply-adds of widened
// values give 1.32e-8 for bfloat16, 3.94e-8 and 3.94e-8 for float16) over K as it is, or
// over fp8 codes widened exactly to the query's type: per key and head 4 instructions
// instead of 8, and no widening of a 16-bit K.
template <typename TQ, typename TKV> struct Query {
  static constexpr int E = Chunk<TKV>::kN;
  float f[E];
  __device__ void load(const void* q, int64_t base) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = Elem<TQ>::load(q, base + e);
  }
  __device__ static void widen(const u32x4& k, float (&kf)[E]) { Chunk<TKV>::unpack(k, kf); }
  using Key = float[E];
  __device__ float dot(const float (&kf)[E]) const {
    float d = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) d = fmaf(f[e], kf[e], d);
    return d;
  }
};

template <typename TQ> __device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
  if constexpr (__is_same(TQ, bf16_t)) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2, a), __builtin_bit_cast(v2, b), c,
                                           false);
  } else {
    typedef _Float16 v2 __attribute__((ext_vector_type(2)));
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2, a), __builtin_bit_cast(v2, b), c, false);
  }
}

template <typename TQ, typename TKV> struct PackedQuery {
  static constexpr int E = Chunk<TKV>::kN;
  uint32_t w[E / 2];
  __device__ void load(const void* q, int64_t base) {
    if (reinterpret_cast<uintptr_t>(q) % 16 == 0) {
#pragma unroll
      for (int i = 0; i < E / 8; ++i) set(i, load16(static_cast<const char*>(q) + (base + 8 * i) * 2));
    } else {  // (the rows start at any element: nothing requires more of q)
      const uint16_t* e = static_cast<const uint16_t*>(q) + base;
#pragma unroll
      for (int i = 0; i < E / 2; ++i) w[i] = e[2 * i] | (static_cast<uint32_t>(e[2 * i + 1]) << 16);
    }
  }
  __device__ void set(int i, const u32x4& v) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[4 * i + j] = v[j];
  }
  using Key = uint32_t[E / 2];
  __device__ static void widen(const u32x4& k, uint32_t (&kw)[E / 2]) {
    if constexpr (Elem<TKV>::kBytes == 2) {
#pragma unroll
      for (int j = 0; j < 4; ++j) kw[j] = k[j];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (__is_same(TQ, bf16_t)) {
          kw[2 * j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k[j], 1.0f, false));
          kw[2 * j + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(k[j], 1.0f, true));
        } else {
          kw[2 * j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(k[j], 1.0f, false));
          kw[2 * j + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(k[j], 1.0f, true));
        }
      }
    }
  }
  __device__ float dot(const uint32_t (&kw)[E / 2]) const {
    float d = 0.0f;
#pragma unroll
    for (int j = 0; j < E / 2; ++j) d = dot2<TQ>(w[j], kw[j], d);
    return d;
  }
};
template <> struct Query<bf16_t, bf16_t> : PackedQuery<bf16_t, bf16_t> {};
template <> struct Query<f16_t, f16_t> : PackedQuery<f16_t, f16_t> {};
template <> struct Query<bf16_t, fp8_t> : PackedQuery<bf16_t, fp8_t> {};
template <> struct Query<f16_t, fp8_t> : PackedQuery<f16_t, fp8_t> {};

// Where the entries of a sequence's key list lie: all positions in order, or for windowed
// attention the sinks and then, `gap` positions on, the window's keys.
struct EveryKey {
  static constexpr bool kListed = false;
  __device__ int operator()(int v) const { return v; }
};
struct WindowKeys {
  static constexpr bool kListed = true;
  int sinks, gap;
  __device__ int operator()(int v) const { return v < sinks ? v : v + gap; }
};

// Per-wave online-softmax state over a run of keys, for GC query heads.
template <int GC, int E>
struct WaveState {
  float m[GC];
  float l[GC];
  float acc[GC][E];
};

template <typename TQ, typename TKV, int D, int GC>
struct Decode {
  static constexpr int E = Chunk<TKV>::kN;   // elements per 16-byte chunk
  static constexpr int R = D / E;            // lanes per token row
  static constexpr int RG = kWave / R;       // row groups per wave
  static constexpr bool kFp8 = Elem<TKV>::kBytes == 1;
  static_assert(R >= 1 && R <= kWave && (kWave % R) == 0, "head dim / dtype mismatch");
  using State = WaveState<GC, E>;

  using Q = Query<TQ, TKV>;

  __device__ static void load_queries(const PagedParams& p, int row, int h0, int r, Q (&qf)[GC]) {
#pragma unroll
    for (int h = 0; h < GC; ++h) {
      qf[h].load(p.q, (static_cast<int64_t>(row) * p.hq + h0 + h) * D + r * E);
    }
  }

  __device__ static void init(State& st) {
#pragma unroll
    for (int h = 0; h < GC; ++h) {
      st.m[h] = -INFINITY;
      st.l[h] = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) st.acc[h][e] = 0.0f;
    }
  }

  // Stream keys [sb, se) of one sequence for kv head `kvh` into `st`. Page ids come
  // from `lds_pages` (page i of the run at lds_pages[i - first_page]) when given,
  // otherwise from the sequence's block table, or with none (a dense cache, table_shift 0)
  // are the slots of positions 16 i from dense_base on; the next step's ids are requested
  // before this step is computed. (Requesting the next step's K/V rows early as well
  // measured slower: on shuffled pages more requests in flight per CU cost DRAM
  // efficiency.)
  __device__ static void stream(const PagedParams& p, const int32_t* table, int dense_base,
                                const int* lds_pages, int first_page, int kvh, int sb, int se, int g, int r,
                                const Q (&qf)[GC], float score_scale, State& st) {
    const Fresh none{-1, {}, {}};
    stream_with<false>(p, table, dense_base, lds_pages, first_page, kvh, sb, se, g, r, qf, score_scale, st,
                       [] {}, none, EveryKey{});
  }

  // The same over entries [sb, se) of a windowed sequence's key list.
  __device__ static void stream_window(const PagedParams& p, const int32_t* table, const WindowKeys& keys,
                                       int kvh, int sb, int se, int g, int r, const Q (&qf)[GC],
                                       float score_scale, State& st) {
    const Fresh none{-1, {}, {}};
    stream_with<false>(p, table, 0, nullptr, 0, kvh, sb, se, g, r, qf, score_scale, st, [] {}, none, keys);
  }

  // The new token of a fresh-token stream: token `tok` of the run (< 0: none) takes this
  // lane's chunks `k` and `v` as its K and V rows instead of the pool's.
  struct Fresh {
    int tok;
    u32x4 k, v;
  };

  // stream() with two additions: `prep()` runs once the first step's page ids have been
  // requested (a fresh-token stream forms its queries and the new token's rows there, in
  // qf and `fresh`, so that arithmetic overlaps those loads), and with kFresh the step
  // holding fresh.tok takes that token's rows from `fresh`. (Forming them under the
  // first step's K/V requests instead measured the same, with 60% more registers.)
  // `at` gives the position of an entry of the run.
  template <bool kFresh, typename Prep, typename Keys>
  __device__ static void stream_with(const PagedParams& p, const int32_t* table,
                                     int dense_base, const int* lds_pages, int first_page, int kvh, int sb, int se,
                                     int g, int r, const Q (&qf)[GC], float score_scale,
                                     State& st, Prep&& prep, const Fresh& fresh, const Keys& at) {
    static_assert(!(kFresh && kFp8), "the fresh-token stream serves 16-bit pools");
    const char* kbase = static_cast<const char*>(p.k_pool);
    const char* vbase = static_cast<const char*>(p.v_pool);
    constexpr int kElemBytes = Elem<TKV>::kBytes;
    constexpr int kStep = RG * kUnroll;

    auto page_of = [&](int tok) -> int {
      if (table == nullptr) return dense_base + (tok & ~p.block_mask);
      const int pi = at(tok) >> p.block_shift;
      return lds_pages != nullptr ? lds_pages[pi - first_page] : table[pi];
    };

    int pg[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) pg[u] = page_of(min(sb + u * RG + g, se - 1));
    prep();

    for (int t0 = sb; t0 < se; t0 += kStep) {
      u32x4 kw[kUnroll], vw[kUnroll];
      bool valid[kUnroll];
      float ks[kUnroll], vs[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        int tok = t0 + u * RG + g;
        valid[u] = tok < se;
        tok = valid[u] ? tok : se - 1;
        // (here and not where the ids are requested, which would wait for them there)
        if constexpr (Keys::kListed) pg[u] = held_page(p, pg[u]);
        const int64_t slot = (static_cast<int64_t>(pg[u]) << p.table_shift) + (at(tok) & p.block_mask);
        const int64_t off = slot * p.kv_row_bytes + kvh * p.kv_head_bytes + r * E * kElemBytes;
        kw[u] = load16_stream(kbase + off);
        vw[u] = load16_stream(vbase + off);
        if constexpr (kFp8) {
          ks[u] = p.k_scales[static_cast<int64_t>(pg[u]) * p.hk + kvh];
          vs[u] = p.v_scales[static_cast<int64_t>(pg[u]) * p.hk + kvh];
        }
      }
      if (t0 + kStep < se) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) pg[u] = page_of(min(t0 + kStep + u * RG + g, se - 1));
      }
      if constexpr (kFresh) {
        // The step holding the new token (wave-uniform test): its pool slot, read above
        // before this launch wrote it, is replaced by the rows formed in the launch.
        if (fresh.tok >= 0 && t0 + kStep > fresh.tok) [[unlikely]] {
          // a real branch, taken once per share: without the barrier the compiler turns
          // the substitution into selects executed in every step
          asm volatile("" ::: "memory");
#pragma unroll
          for (int u = 0; u < kUnroll; ++u) {
            if (t0 + u * RG + g == fresh.tok) {
              kw[u] = fresh.k;
              vw[u] = fresh.v;
            }
          }
        }
      }

      float s[kUnroll][GC];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        typename Q::Key kf;
        Q::widen(kw[u], kf);
#pragma unroll
        for (int h = 0; h < GC; ++h) {
          const float dot = group_sum<R>(qf[h].dot(kf));
          // The reference scales after the reduction (paged_attention.cu:181-183).
          float sc = dot * score_scale;
          if constexpr (kFp8) sc *= ks[u];
          s[u][h] = valid[u] ? sc : -INFINITY;
        }
      }

      float pr[kUnroll][GC];
#pragma unroll
      for (int h = 0; h < GC; ++h) {
        float mx = st.m[h];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) mx = fmaxf(mx, s[u][h]);
        // A row group that has seen no valid key yet keeps m = -inf; exponentiate
        // against 0 then, so 2^(-inf - 0) = 0 instead of 2^(-inf + inf) = NaN
        // (the empty-split rule of paged_attention.cu:210-213).
        const float mu = mx == -INFINITY ? 0.0f : mx;
        const float alpha = fast_exp2(st.m[h] - mu);
        float sum = 0.0f;
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          pr[u][h] = fast_exp2(s[u][h] - mu);
          sum += pr[u][h];
        }
        st.l[h] = st.l[h] * alpha + sum;
        st.m[h] = mx;
#pragma unroll
        for (int e = 0; e < E; ++e) st.acc[h][e] *= alpha;
      }

#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float vf[E];
        Chunk<TKV>::unpack(vw[u], vf);
#pragma unroll
        for (int h = 0; h < GC; ++h) {
          float w = pr[u][h];
          if constexpr (kFp8) w *= vs[u];
#pragma unroll
          for (int e = 0; e < E; ++e) st.acc[h][e] = fmaf(w, vf[e], st.acc[h][e]);
        }
      }
    }
  }

  // f over the lanes of the same r (one of each row group), in all of them: rotations within 16 lanes,
  // then exchanges of 16-lane rows and of the wave's halves, none of them through LDS.
  template <typename F>
  __device__ static float over_row_groups(float v, F f) {
    if constexpr (R <= 8) v = f(v, dpp<0x128>(v));  // row_ror:8
    if constexpr (R <= 4) v = f(v, dpp<0x124>(v));
    if constexpr (R <= 2) v = f(v, dpp<0x122>(v));
    if constexpr (R <= 1) v = f(v, dpp<0x121>(v));
    if constexpr (R <= 16) {
      const auto rows = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
      v = f(__uint_as_float(rows[0]), __uint_as_float(rows[1]));
    }
    if constexpr (R <= 32) {
      const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
      v = f(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
    }
    return v;
  }

  // Combine the wave's row groups against their common maximum, as windowed calls do: what a row group
  // holds is scaled once, and the sums take no trip through LDS (merge_row_groups makes log2(RG) of
  // them a value, 288 with 4 heads over fp8 at D = 64: 89 lists of 70 keys for 4 kv heads 18.1 us a
  // call, 14.0 so; at D = 128, 64 of 70 for 8 16.9 and 14.3, with 2 heads 8.4 and 7.7, over bf16 level;
  // the stream over one list of 64, 4 heads, 17.2 and 13.9, 2 heads 11.8 and 10.7).
  __device__ static void sum_row_groups(State& st) {
#pragma unroll
    for (int h = 0; h < GC; ++h) {
      const float mx = over_row_groups(st.m[h], [](float x, float y) { return fmaxf(x, y); });
      const float a = fast_exp2(st.m[h] - (mx == -INFINITY ? 0.0f : mx));
      auto add = [](float x, float y) { return x + y; };
      st.m[h] = mx;
      st.l[h] = over_row_groups(st.l[h] * a, add);
#pragma unroll
      for (int e = 0; e < E; ++e) st.acc[h][e] = over_row_groups(st.acc[h][e] * a, add);
    }
  }

  // Combine the wave's row groups: xor partners share r and differ in g. Afterwards
  // every row group holds the totals.
  __device__ static void merge_row_groups(State& st) {
#pragma unroll
    for (int off = R; off < kWave; off <<= 1) {
#pragma unroll
      for (int h = 0; h < GC; ++h) {
        const float mo = __shfl_xor(st.m[h], off, kWave);
        const float lo = __shfl_xor(st.l[h], off, kWave);
        const float mx = fmaxf(st.m[h], mo);
        const float mu = mx == -INFINITY ? 0.0f : mx;
        const float a = fast_exp2(st.m[h] - mu);
        const float b = fast_exp2(mo - mu);
        st.l[h] = st.l[h] * a + lo * b;
        st.m[h] = mx;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float other = __shfl_xor(st.acc[h][e], off, kWave);
          st.acc[h][e] = st.acc[h][e] * a + other * b;
        }
      }
    }
  }

  __device__ static void write_output(const PagedParams& p, int row, int h0, int r, const State& st) {
#pragma unroll
    for (int h = 0; h < GC; ++h) {
      const float inv = st.l[h] > 0.0f ? 1.0f / st.l[h] : 0.0f;
      const int64_t base = (static_cast<int64_t>(row) * p.hq + h0 + h) * D + r * E;
#pragma unroll
      for (int e = 0; e < E; ++e) Elem<TQ>::store(p.out, base + e, st.acc[h][e] * inv);
    }
  }

  // Partial of head h0 + h at index (pidx0 + h * pstride).
  __device__ static void write_partial(const PagedParams& p, int64_t pidx0, int64_t pstride, int r,
                                       const State& st) {
#pragma unroll
    for (int h = 0; h < GC; ++h) {
      const int64_t pidx = pidx0 + h * pstride;
      float* po = p.part_o + pidx * D + r * E;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        *reinterpret_cast<f32x4*>(po + e) =
            f32x4{st.acc[h][e], st.acc[h][e + 1], st.acc[h][e + 2], st.acc[h][e + 3]};
      }
      if (r == 0) {
        p.part_ml[pidx * 2] = st.m[h];
        p.part_ml[pidx * 2 + 1] = st.l[h];
      }
    }
  }
};

// The (kv head, head chunk) unit of a wave; false when the wave has none.
template <int GC>
__device__ __forceinline__ bool wave_unit(const PagedParams& p, int unit, int& kvh, int& h0) {
  const int chunks = p.hq / p.hk / GC;
  if (unit >= p.hk * chunks) return false;
  kvh = unit / chunks;
  h0 = kvh * (p.hq / p.hk) + (unit % chunks) * GC;
  return true;
}

// A windowed decode row's list for one chunk of a kv head's query heads, by a workgroup of kWaves waves
// that take equal runs of it and meet in `s_o` (kWaves GC D floats) and `s_ml` (2 kWaves GC).
template <typename TQ, typename TKV, int D, int GC, int kWaves>
__device__ __forceinline__ void decode_list(const PagedParams& p, int seq, int unit, float* s_o, float* s_ml) {
  using K = Decode<TQ, TKV, D, GC>;
  float* const s_m = s_ml;  // [kWaves][GC]
  float* const s_l = s_m + kWaves * GC;
  if (sload(p.seq_lens + seq) != 1) return;  // a prefill chunk: the prefill kernel has it
  const int context = max(sload(p.context_lens + seq), 0);
  const int row = sload(p.cu_seqlens_q + seq);
  const int entries = window_keys(context, p.window, p.sinks);
  int kvh, h0;
  if (!wave_unit<GC>(p, unit, kvh, h0)) return;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), lane = threadIdx.x % kWave;
  const int g = lane / K::R, r = lane % K::R;
  constexpr int kStep = K::RG * kUnroll;
  const int per = ((entries + kWaves - 1) / kWaves + kStep - 1) / kStep * kStep;
  const int sb = min(wave * per, entries), se = min(sb + per, entries);
  typename K::State st;
  K::init(st);
  if (sb < se) {
    typename K::Q qf[GC];
    K::load_queries(p, row, h0, r, qf);
    const int32_t* table = p.block_tables + static_cast<int64_t>(seq) * p.max_blocks;
    K::stream_window(p, table, WindowKeys{p.sinks, context - entries}, kvh, sb, se, g, r, qf,
                     p.scale * kLog2e, st);
    K::sum_row_groups(st);
  }
  if (g == 0) {
#pragma unroll
    for (int h = 0; h < GC; ++h) {
#pragma unroll
      for (int e = 0; e < K::E; e += 4) {
        *reinterpret_cast<f32x4*>(&s_o[(wave * GC + h) * D + r * K::E + e]) =
            f32x4{st.acc[h][e], st.acc[h][e + 1], st.acc[h][e + 2], st.acc[h][e + 3]};
      }
      if (r == 0) {
        s_m[wave * GC + h] = st.m[h];
        s_l[wave * GC + h] = st.l[h];
      }
    }
  }
  __syncthreads();
  for (int j = threadIdx.x; j < GC * D; j += kWaves * kWave) {
    const int h = j / D, d = j % D;
    float m = s_m[h];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s_m[w * GC + h]);
    const float mu = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, o = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float a = fast_exp2(s_m[w * GC + h] - mu);
      l = fmaf(s_l[w * GC + h], a, l);
      o = fmaf(s_o[(w * GC + h) * D + d], a, o);
    }
    // (no key at all: l = 0, a row of zeros)
    Elem<TQ>::store(p.out, (static_cast<int64_t>(row) * p.hq + h0 + h) * D + d,
                    l > 0.0f ? o * (1.0f / l) : 0.0f);
  }
}

}  // namespace

}  // namespace mvllm
