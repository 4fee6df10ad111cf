// Paged decode attention for CDNA4, with split-K ("flash decoding") and a merge.
//
// Behaviour follows the reference's paged_decode_kernel / paged_decode_merge_kernel
// (csrc/paged_attention.cu:97-302): for every query row whose sequence computes one
// token (seq_lens[s] == 1), out = softmax(q K^T * scale) V over the context_lens[s]
// keys that the sequence's block table maps to physical slots
// (slot = table[p >> shift] << shift | (p & mask), paged_attention.cu:87-93).
//
// The work decomposition is this library's own.
//
// Inside a workgroup: one wave per (kv head, chunk of up to four query heads of that
// head's GQA group). The wave holds the queries of its group in registers, so each
// K/V byte is fetched from HBM exactly once however many query heads share it. A
// token's (kv head) row is D elements = D / E lanes of 16 bytes (E = 8 for bf16/fp16,
// 4 for fp32, 16 for fp8); the 64 lanes split into 64 / (D / E) row groups, each
// streaming its own tokens with its own online-softmax state, so the main loop needs
// no cross-row-group traffic and no barrier: a dot product is reduced with 16-lane DPP
// all-reduces only. Row groups are merged once at the end with the reference's
// rescale exp(m_i - M) (paged_attention.cu:284-301).
//
// Across workgroups, two schedules, and a third of windowed calls:
//
//  * stream (the decode hot path): a persistent grid of a few workgroups per CU. The
//    decode sequences' keys are laid end to end (an in-kernel prefix scan of
//    context_lens, no host read) and every workgroup streams an equal share of that
//    token axis, so every CU moves the same bytes whatever the length distribution.
//    A share that covers a whole sequence writes its output directly; a sequence cut
//    between workgroups leaves one (m, l, O) partial per piece, in slot
//    (workgroup + sequence), which is unique because shares and sequences are both
//    contiguous ranges of the same axis. A second small kernel merges the pieces.
//    (Merging in the decode kernel instead -- the last workgroup to finish a piece
//    merges, on an atomic counter -- measured slower: every merge then sits at the
//    end of the launch behind a chain of dependent memory round trips.)
//  * grid (fallback, and the by-row mode that also serves prefill rows when no MFMA
//    prefill kernel fits the shape): one workgroup per (row, split) with splits of
//    `split_tokens` keys, page ids staged in LDS, merged by a second kernel.
//  * direct (windowed: a row's keys are at most sinks + window): one workgroup per (sequence, kv
//    head), whose waves take equal runs of its list and meet in LDS: one launch, no workspace, no
//    page id fetched twice. With prefill chunks in the batch, workgroups of the pair prefill's launch
//    (paged_prefill.hip); their body is paged_decode_rows.hpp's.
//
// Fresh-token stream (a decode-only batch over a 16-bit pool): every sequence's last
// key is the step's new token, taken from the q/k/v projection's output rather than
// the pool. Each wave QK-norms and rotates its queries itself (norm_rope_chunk, the
// QK-norm + RoPE kernel's code: this file is compiled with -ffp-contract=off so it
// rounds the same), the share holding a sequence's last key forms that key's row
// likewise, writes it and v to the pool slot, and uses them from registers in its last
// step; the result is the QK-norm + RoPE + KV-write launch followed by the plain
// stream, bit for bit, with one launch fewer.
//
// K/V are read with nontemporal 16-byte loads (they are streamed once); page ids are
// fetched one step ahead of the K/V loads that need them. Scores are kept in the
// log2 domain: s = (q.k) * scale * log2(e), p = 2^(s - m), exactly
// exp((q.k)*scale - max) in real arithmetic, at one v_exp_f32 per score.

#include "common.hpp"
#include "paged_attention.hpp"
#include "paged_decode_rows.hpp"

namespace mvllm {

namespace {

// Which query row, sequence and visible context a grid-schedule workgroup serves.
// Returns false when the workgroup has nothing to do in this pass.
__device__ __forceinline__ bool resolve_row(const PagedParams& p, int index, int& seq, int& row,
                                            int& visible) {
  if (p.by_row) {
    // Every query row is a unit: find its sequence by binary search over cu_seqlens_q.
    row = index;
    int lo = 0, hi = p.num_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (p.cu_seqlens_q[mid] <= row) lo = mid; else hi = mid - 1;
    }
    seq = lo;
    const int query_len = p.seq_lens[seq];
    const int local = row - p.cu_seqlens_q[seq];
    // The L queries are the last L positions of the context (causal offset S - L,
    // reference attention.py:76-92 / paged_attention.cu:348-349).
    visible = p.context_lens[seq] - query_len + local + 1;
    return visible > 0;
  }
  seq = index;
  if (p.seq_lens[seq] != 1) return false;  // a prefill chunk: the prefill kernel has it
  row = p.cu_seqlens_q[seq];
  visible = p.context_lens[seq];
  return visible > 0;
}

// The same for windowed attention, whose rows without a key are zeros: true for every row that is
// this pass's to write, `visible` then at most 0 where it has none. (By row: not the rows of q
// behind the last sequence.)
__device__ __forceinline__ bool resolve_window_row(const PagedParams& p, int index, int& seq, int& row,
                                                   int& visible) {
  if (resolve_row(p, index, seq, row, visible)) {
    return !p.by_row || row - p.cu_seqlens_q[seq] < p.seq_lens[seq];
  }
  return p.by_row ? row - p.cu_seqlens_q[seq] < p.seq_lens[seq] : p.seq_lens[seq] == 1;
}

}  // namespace

// ------------------------------------------------------------ stream schedule

// kFresh: every sequence's last key is the step's new token, formed here from the
// projection's output (FreshParams) instead of read from the pool.
// kWindow: a sequence's keys are the entries of its windowed list (WindowKeys), at most window +
// sinks of them whatever its context: the same loop over fewer keys, no key read for nothing and
// no mask, with two instructions an entry more for its position.
template <typename TQ, typename TKV, int D, int GC, bool kFresh, bool kWindow>
__global__ __launch_bounds__(512) void paged_decode_stream_kernel(const PagedParams p,
                                                                  const FreshParams f) {
  using K = Decode<TQ, TKV, D, GC>;
  __shared__ int s_prefix[kMaxStreamSeqs + 1];  // decode keys before sequence s

  const int n = p.num_seqs;
  const int tid = threadIdx.x;
  // Prefix sums of the decode sequences' context lengths (0 for prefill chunks). Up to 64
  // sequences: every wave for itself, lane s holding the keys up to and with sequence s's,
  // no barrier and no LDS. More: through s_prefix, by all waves, loads side by side (by one
  // wave, each lane summing a contiguous run, 2000 sequences of 20 to 200 keys took 6 to 10 us
  // longer).
  // A dense cache: every sequence holds dense_keys, nothing is read.
  const bool dense = !kFresh && p.dense_keys > 0;
  const bool by_lane = n <= kWave;
  auto listed = [&](int context) __attribute__((always_inline)) -> int {
    return kWindow ? window_keys(max(context, 0), p.window, p.sinks) : max(context, 0);
  };
  int upto = 0;
  if (dense) {
  } else if (by_lane) {
    const int s = tid % kWave;
    upto = wave_inclusive_scan(s < n && p.seq_lens[s] == 1 ? listed(p.context_lens[s]) : 0);
  } else {
    // Each wave its run of sequences, 64 at a time: their sum, then their places after the
    // runs before.
    __shared__ int s_run[kMaxDecodeWaves];
    constexpr int kAhead = 4;
    const int waves = blockDim.x / kWave, lane = tid % kWave;
    const int w = __builtin_amdgcn_readfirstlane(tid / kWave);
    const int per = (n + blockDim.x - 1) / blockDim.x * kWave;
    const int first = min(w * per, n), end = min(first + per, n);
    auto keys = [&](int s) __attribute__((always_inline)) -> int {
      return s < end && p.seq_lens[s] == 1 ? listed(p.context_lens[s]) : 0;
    };
    int run = 0;
#pragma unroll 4
    for (int s = first; s < end; s += kWave) run += keys(s + lane);
    run = __builtin_amdgcn_readlane(wave_inclusive_scan(run), kWave - 1);
    if (lane == 0) s_run[w] = run;
    __syncthreads();
    int before = 0;
    for (int i = 0; i < w; ++i) before += s_run[i];
    for (int s = first + lane; s - lane < end; s += kAhead * kWave) {
      int mine[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) mine[u] = keys(s + u * kWave);
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int incl = wave_inclusive_scan(mine[u]);
        if (s + u * kWave < end) s_prefix[s + u * kWave] = before + incl - mine[u];
        before += __builtin_amdgcn_readlane(incl, kWave - 1);
      }
    }
    if (w == waves - 1 && lane == 0) s_prefix[n] = before;
    __syncthreads();
  }
  // Decode keys before sequence i (i uniform, 0 .. n).
  auto prefix = [&](int i) __attribute__((always_inline)) -> int {
    if (dense) return i * p.dense_keys;
    if (!by_lane) return __builtin_amdgcn_readfirstlane(s_prefix[i]);
    return i == 0 ? 0 : __builtin_amdgcn_readlane(upto, i - 1);
  };

  const int total = prefix(n);
  const DecodeShares shares(total, gridDim.x, p.stream_min_keys);
  if (blockIdx.x == 0 && !dense) {
    if (by_lane) {
      if (tid < n) p.seq_prefix[tid + 1] = upto;
      if (tid == 0) p.seq_prefix[0] = 0;
    } else {
      for (int s = tid; s <= n; s += blockDim.x) p.seq_prefix[s] = s_prefix[s];
    }
  }
  if (static_cast<int>(blockIdx.x) >= shares.count) return;
  const int lo = shares.begin(blockIdx.x);
  const int hi = shares.begin(blockIdx.x + 1);
  if (lo >= hi) return;

  const int wave = tid / kWave;
  const int lane = tid % kWave;
  const int g = lane / K::R;
  const int r = lane % K::R;
  int kvh = 0, h0 = 0;
  const bool active = wave_unit<GC>(p, wave, kvh, h0);
  const float score_scale = p.scale * kLog2e;

  // First sequence whose keys include `lo`: the last s with prefix[s] <= lo < prefix[s + 1].
  int seq = 0;
  if (dense) {
    seq = static_cast<int>(static_cast<uint32_t>(lo) / static_cast<uint32_t>(p.dense_keys));
  } else if (by_lane) {
    seq = __builtin_ctzll(__builtin_amdgcn_ballot_w64(upto > lo));
  } else {
    int b = n;  // invariant: prefix[seq] <= lo < prefix[b]
    while (b - seq > 1) {
      const int mid = (seq + b) >> 1;
      if (prefix(mid) <= lo) seq = mid; else b = mid;
    }
  }
  int pos = lo;
  int base = prefix(seq), next = prefix(seq + 1);  // keys before this sequence and the next one
  while (pos < hi) {
    while (next == base) next = prefix(++seq + 1);  // skip prefill / empty sequences
    const int ctx = next - base;
    const int sb = pos - base;
    const int se = min(hi, base + ctx) - base;
    // A decode-only batch (the fresh-token stream) has row s for sequence s: no load
    // ahead of the raw q/k/v reads that address by row.
    const int row = kFresh || dense ? seq : p.cu_seqlens_q[seq];
    const bool whole = sb == 0 && se == ctx;
    typename K::State st;
    if (active) {
      typename K::Q qf[GC];
      K::init(st);
      const int32_t* table = p.block_tables + static_cast<int64_t>(seq) * p.max_blocks;
      if constexpr (kFresh) {
        static_assert(K::E == 8 && K::R == 16, "the fresh-token stream takes 16-bit D = 128");
        // Loads first (all rows of the token, whether or not this run holds it: no
        // divergent loads), the arithmetic in prep() once the page ids are requested.
        const int pos = ctx - 1;
        const bool pos_ok = pos < f.max_positions;
        const int64_t trow = pos_ok ? pos : 0;  // out of range: row 0, NaN rows below
        u32x4 qraw[GC];
#pragma unroll
        for (int h = 0; h < GC; ++h) {
          qraw[h] = load16(static_cast<const char*>(f.q) +
                           (static_cast<int64_t>(row) * f.q_stride + (h0 + h) * D + r * 8) * 2);
        }
        const int64_t kvoff = (static_cast<int64_t>(row) * f.kv_stride + kvh * D + r * 8) * 2;
        const u32x4 kraw = load16(static_cast<const char*>(f.k) + kvoff);
        const u32x4 vraw = load16(static_cast<const char*>(f.v) + kvoff);
        const u32x4 wq = load16(static_cast<const char*>(f.q_weight) + r * 16);
        const u32x4 wk = load16(static_cast<const char*>(f.k_weight) + r * 16);
        float c[8], sn[8];
        Chunk<float>::unpack(load16(f.cos_t + trow * D + r * 8), c);
        Chunk<float>::unpack(load16(f.cos_t + trow * D + r * 8 + 4), c + 4);
        Chunk<float>::unpack(load16(f.sin_t + trow * D + r * 8), sn);
        Chunk<float>::unpack(load16(f.sin_t + trow * D + r * 8 + 4), sn + 4);
        const int new_page = table[pos >> p.block_shift];
        const bool has_new = se == ctx;
        typename K::Fresh fresh{-1, {}, {}};
        auto prep = [&]() {
          if (r < 8) {
#pragma unroll
            for (int e = 0; e < 8; ++e) sn[e] = -sn[e];
          }
          if (!pos_ok) {
#pragma unroll
            for (int e = 0; e < 8; ++e) c[e] = sn[e] = __int_as_float(0x7fc00000);
          }
          // The GC query rows and the key row, one per row group and pass (row group g
          // of pass i forms row 4 i + g: query heads first, then k; a row group past
          // the last row forms k again, unused), then each row's chunk r read by every
          // row group from lane 16 (row % 4) + r. One pass for up to three query heads:
          // a quarter of the arithmetic of every row group forming every row.
          constexpr int kRows = GC + 1;
          constexpr int kPasses = (kRows + K::RG - 1) / K::RG;
          u32x4 formed[kPasses];
#pragma unroll
          for (int i = 0; i < kPasses; ++i) {
            const int rix = i * K::RG + g;
            u32x4 held = kraw;
#pragma unroll
            for (int h = 0; h < GC; ++h) held = rix == h ? qraw[h] : held;
            float wf[8];
            Chunk<TQ>::unpack(rix < GC ? wq : wk, wf);
            formed[i] = norm_rope_chunk<TQ, 16>(held, wf, c, sn, f.eps);
          }
          auto row_of = [&](int rix) {
            const int src = (rix % K::RG) * 16 + r;
            const u32x4& x = formed[rix / K::RG];
            return u32x4{static_cast<uint32_t>(__shfl(static_cast<int>(x[0]), src, kWave)),
                         static_cast<uint32_t>(__shfl(static_cast<int>(x[1]), src, kWave)),
                         static_cast<uint32_t>(__shfl(static_cast<int>(x[2]), src, kWave)),
                         static_cast<uint32_t>(__shfl(static_cast<int>(x[3]), src, kWave))};
          };
#pragma unroll
          for (int h = 0; h < GC; ++h) {
            // rounded to TQ as the unfused kernel stores q
            qf[h].set(0, row_of(h));
          }
          fresh.k = row_of(GC);
          fresh.v = vraw;
          if (has_new) {
            fresh.tok = pos;
            // One wave per kv head writes the pool (the first of its query-head chunks),
            // row group 0's 16 lanes one row each of K and V.
            if (g == 0 && h0 % (p.hq / p.hk) == 0 && new_page >= 0 && new_page < f.num_blocks) {
              const int64_t slot =
                  (static_cast<int64_t>(new_page) << p.table_shift) + (pos & p.block_mask);
              const int64_t off = slot * p.kv_row_bytes + kvh * p.kv_head_bytes + r * 16;
              store16(static_cast<char*>(const_cast<void*>(p.k_pool)) + off, fresh.k);
              store16(static_cast<char*>(const_cast<void*>(p.v_pool)) + off, fresh.v);
            }
          }
        };
        K::template stream_with<true>(p, table, 0, nullptr, 0, kvh, sb, se, g, r, qf, score_scale,
                                      st, prep, fresh, EveryKey{});
      } else {
        K::load_queries(p, row, h0, r, qf);
        if constexpr (kWindow) {
          const WindowKeys keys{p.sinks, sload(p.context_lens + seq) - ctx};
          K::stream_window(p, table, keys, kvh, sb, se, g, r, qf, score_scale, st);
        } else {
          K::stream(p, dense ? nullptr : table, seq * p.dense_slots, nullptr, 0, kvh, sb, se, g, r, qf,
                    score_scale, st);
        }
      }
      if constexpr (kWindow) K::sum_row_groups(st);
      else K::merge_row_groups(st);
      if (g == 0) {
        if (whole) {
          K::write_output(p, row, h0, r, st);
        } else {
          K::write_partial(p, (static_cast<int64_t>(blockIdx.x) + seq) * p.hq + h0, 1, r, st);
        }
      }
    }
    pos = base + se;
    if (pos >= hi) break;
    base = next;
    next = prefix(++seq + 1);
  }
}

// Combine the pieces of every decode sequence cut between stream workgroups. Piece i
// of sequence s lives in slot (first + i + s), first/last being the workgroups owning
// the sequence's first and last key. Grid (sequence, block of kMergeCols float4
// columns of its H_q x D output, 512 / kMergeGroups); in a workgroup, kMergeGroups groups of threads take
// the pieces round robin (group g: pieces g, g + G, ...), each thread folding its
// pieces for one float4 column online (running max, rescaled sums) with kMergeBatch
// pieces' loads in flight at once; the groups' states then meet in LDS and are folded
// in group order. A long sequence cut into dozens of pieces so costs a few round trips
// instead of one per eight pieces, and a batch's sequences spread over H_q D / 4 /
// kMergeCols workgroups each instead of one. The fold order depends on the piece count
// alone, so a call's result does not depend on timing.
constexpr int kMergeThreads = 512;
constexpr int kMergeBatch = 8;

// kWindow: also the zeros of a decode row that has no key at all (nobody else writes it).
template <typename TQ, int D, int kMergeGroups, bool kWindow>
__global__ __launch_bounds__(kMergeThreads) void paged_decode_stream_merge_kernel(
    const PagedParams p, int wgs_i) {
  constexpr int kMergeCols = kMergeThreads / kMergeGroups;
  __shared__ float s_m[kMergeGroups][kMergeCols];
  __shared__ float s_l[kMergeGroups][kMergeCols];
  __shared__ f32x4 s_o[kMergeGroups][kMergeCols];
  const int seq = blockIdx.x;
  const bool dense = p.dense_keys > 0;
  const int total = dense ? p.num_seqs * p.dense_keys : p.seq_prefix[p.num_seqs];
  const int begin = dense ? seq * p.dense_keys : p.seq_prefix[seq];
  const int end = dense ? begin + p.dense_keys : p.seq_prefix[seq + 1];
  if (end == begin) {  // whole workgroup: no barrier follows for it
    if constexpr (kWindow) {
      const int j0 = blockIdx.y * kMergeCols + threadIdx.x;
      if (threadIdx.x < kMergeCols && j0 < p.hq * D / 4 && p.seq_lens[seq] == 1) {
        const int64_t at = static_cast<int64_t>(p.cu_seqlens_q[seq]) * p.hq * D + 4 * j0;
#pragma unroll
        for (int k = 0; k < 4; ++k) Elem<TQ>::store(p.out, at + k, 0.0f);
      }
    }
    return;
  }
  const DecodeShares shares(total, wgs_i, p.stream_min_keys);
  const int first = shares.owner(begin);
  const int last = shares.owner(end - 1);
  if (first == last) return;  // one piece: the decode kernel stored the output
  const int pieces = last - first + 1;
  const int n4 = p.hq * D / 4;
  const int local = threadIdx.x % kMergeCols;
  const int grp = threadIdx.x / kMergeCols;
  const int j = blockIdx.y * kMergeCols + local;
  const bool live = j < n4;
  const int head = live ? (4 * j) / D : 0;
  const int d = live ? 4 * j - head * D : 0;

  float m = -INFINITY, l = 0.0f;
  f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
  if (live) {
    for (int i0 = grp; i0 < pieces; i0 += kMergeGroups * kMergeBatch) {
      float mi[kMergeBatch], li[kMergeBatch];
      f32x4 oi[kMergeBatch];
#pragma unroll
      for (int u = 0; u < kMergeBatch; ++u) {
        const int i = min(i0 + u * kMergeGroups, pieces - 1);
        const int64_t pidx = static_cast<int64_t>(first + i + seq) * p.hq + head;
        mi[u] = p.part_ml[pidx * 2];
        li[u] = p.part_ml[pidx * 2 + 1];
        oi[u] = *reinterpret_cast<const f32x4*>(p.part_o + pidx * D + d);
      }
#pragma unroll
      for (int u = 0; u < kMergeBatch; ++u) {
        const int i = i0 + u * kMergeGroups;
        if (i >= pieces) continue;  // (a share is never empty: see DecodeShares)
        const float mn = fmaxf(m, mi[u]);
        const float mu = mn == -INFINITY ? 0.0f : mn;
        const float a = fast_exp2(m - mu);
        const float b = fast_exp2(mi[u] - mu);
        l = l * a + li[u] * b;
        o = o * a + oi[u] * b;
        m = mn;
      }
    }
  }
  s_m[grp][local] = m;
  s_l[grp][local] = l;
  s_o[grp][local] = o;
  __syncthreads();
  if (grp != 0 || !live) return;
  m = -INFINITY;
  l = 0.0f;
  o = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int g = 0; g < kMergeGroups; ++g) {
    const float mg = s_m[g][local];
    const float mn = fmaxf(m, mg);
    const float mu = mn == -INFINITY ? 0.0f : mn;
    const float a = fast_exp2(m - mu);
    const float b = fast_exp2(mg - mu);
    l = l * a + s_l[g][local] * b;
    o = o * a + s_o[g][local] * b;
    m = mn;
  }
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  const int row = dense ? seq : p.cu_seqlens_q[seq];
  const int64_t obase = (static_cast<int64_t>(row) * p.hq + head) * D + d;
#pragma unroll
  for (int k = 0; k < 4; ++k) Elem<TQ>::store(p.out, obase + k, o[k] * inv);
}

// -------------------------------------------------------------- grid schedule

// kWindow: a row's keys are the entries of its windowed list, page ids read from the table; a
// row without a key gets its zeros here.
template <typename TQ, typename TKV, int D, int GC, bool kWindow>
__global__ __launch_bounds__(512) void paged_decode_grid_kernel(const PagedParams p) {
  using K = Decode<TQ, TKV, D, GC>;
  __shared__ int s_pages[kWindow ? 1 : kMaxSplitPages];

  int seq, row, visible;
  if constexpr (kWindow) {
    if (!resolve_window_row(p, blockIdx.y, seq, row, visible)) return;
    if (visible <= 0) {
      if (blockIdx.x != 0 || blockIdx.z != 0) return;
      for (int j = threadIdx.x; j < p.hq * D; j += blockDim.x) {
        Elem<TQ>::store(p.out, static_cast<int64_t>(row) * p.hq * D + j, 0.0f);
      }
      return;
    }
  } else {
    if (!resolve_row(p, blockIdx.y, seq, row, visible)) return;
  }
  const int all = visible;
  if constexpr (kWindow) visible = window_keys(visible, p.window, p.sinks);

  const int nsplit = decode_num_splits(visible, p.split_tokens, p.max_splits);
  const int split = blockIdx.x;
  if (split >= nsplit) return;
  const int per_split = decode_split_len(visible, nsplit);
  const int sb = split * per_split;
  const int se = min(sb + per_split, visible);

  const int partial_row = p.by_row ? row : seq;
  const int wave = threadIdx.x / kWave;
  const int lane = threadIdx.x % kWave;
  const int g = lane / K::R;
  const int r = lane % K::R;

  const int32_t* table = p.block_tables + static_cast<int64_t>(seq) * p.max_blocks;
  const int first_page = sb >> p.block_shift;
  const int n_pages = sb < se ? ((se - 1) >> p.block_shift) - first_page + 1 : 0;
  const bool pages_in_lds = !kWindow && n_pages <= kMaxSplitPages;
  if (pages_in_lds) {
    for (int i = threadIdx.x; i < n_pages; i += blockDim.x) s_pages[i] = table[first_page + i];
  }
  if constexpr (!kWindow) __syncthreads();

  int kvh, h0;
  if (!wave_unit<GC>(p, blockIdx.z * (blockDim.x / kWave) + wave, kvh, h0)) return;

  typename K::Q qf[GC];
  K::load_queries(p, row, h0, r, qf);
  typename K::State st;
  K::init(st);
  if constexpr (kWindow) {
    const WindowKeys keys{p.sinks, all - visible};
    K::stream_window(p, table, keys, kvh, sb, se, g, r, qf, p.scale * kLog2e, st);
  } else {
    K::stream(p, table, 0, pages_in_lds ? s_pages : nullptr, first_page, kvh, sb, se, g, r, qf,
              p.scale * kLog2e, st);
  }
  if constexpr (kWindow) K::sum_row_groups(st);
  else K::merge_row_groups(st);
  if (g != 0) return;
  if (nsplit == 1) {
    K::write_output(p, row, h0, r, st);
  } else {
    K::write_partial(p, (static_cast<int64_t>(partial_row) * p.hq + h0) * p.max_splits + split,
                     p.max_splits, r, st);
  }
}

// Combine the split partials of every (row, query head) that was split:
// out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s. One wave per (row, head).
template <typename TQ, int D, bool kWindow>
__global__ __launch_bounds__(256) void paged_decode_grid_merge_kernel(const PagedParams p) {
  constexpr int kPerLane = (D + kWave - 1) / kWave;
  const int wave = threadIdx.x / kWave;
  const int lane = threadIdx.x % kWave;
  const int head = blockIdx.x * (blockDim.x / kWave) + wave;
  if (head >= p.hq) return;

  int seq, row, visible;
  if constexpr (kWindow) {
    if (!resolve_window_row(p, blockIdx.y, seq, row, visible) || visible <= 0) return;
    visible = window_keys(visible, p.window, p.sinks);
  } else {
    if (!resolve_row(p, blockIdx.y, seq, row, visible)) return;
  }
  const int nsplit = decode_num_splits(visible, p.split_tokens, p.max_splits);
  if (nsplit == 1) return;  // the decode kernel stored this row directly

  const int partial_row = p.by_row ? row : seq;
  const int64_t prow0 = (static_cast<int64_t>(partial_row) * p.hq + head) * p.max_splits;

  float mmax = -INFINITY;
  for (int s = lane; s < nsplit; s += kWave) mmax = fmaxf(mmax, p.part_ml[(prow0 + s) * 2]);
  mmax = wave_max(mmax);
  const float mu = mmax == -INFINITY ? 0.0f : mmax;

  float total_l = 0.0f;
  for (int s = lane; s < nsplit; s += kWave) {
    const float ls = p.part_ml[(prow0 + s) * 2 + 1];
    if (ls > 0.0f) total_l += __builtin_amdgcn_exp2f(p.part_ml[(prow0 + s) * 2] - mu) * ls;
  }
  total_l = wave_sum(total_l);
  const float inv = total_l > 0.0f ? 1.0f / total_l : 0.0f;

  float o[kPerLane];
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) o[i] = 0.0f;
  for (int s = 0; s < nsplit; ++s) {
    const float ls = p.part_ml[(prow0 + s) * 2 + 1];
    if (!(ls > 0.0f)) continue;  // an empty split contributes exactly nothing
    const float w = __builtin_amdgcn_exp2f(p.part_ml[(prow0 + s) * 2] - mu);
    const float* po = p.part_o + (prow0 + s) * D;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int d = lane + i * kWave;
      if (d < D) o[i] = fmaf(w, po[d], o[i]);
    }
  }
  const int64_t base = (static_cast<int64_t>(row) * p.hq + head) * D;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) {
    const int d = lane + i * kWave;
    if (d < D) Elem<TQ>::store(p.out, base + d, o[i] * inv);
  }
}

// ------------------------------------------------------------ direct schedule

// Windowed decode by a workgroup per (sequence, kv head, chunk of its query heads): its waves take
// equal runs of the sequence's list and meet in LDS, so there is one launch, and no partials or
// prefix sums in memory. A window bounds every list, so a workgroup per list is balanced enough, where
// full contexts need the stream's equal shares. The stream's second launch and its chain of
// partials cost 5 us whatever the batch: 28 lists of 128 keys 11.9 -> 6.7 us, of 700 over fp8 24 ->
// 14, 64 of 1028 48.9 -> 46.1. What bounds it, besides memory: a CU takes in about 35 GB/s (30 over
// fp8, whose rows are 128 bytes), so few lists that are long stay with the stream (one of 1028 17.0
// against 11.5). 16 waves instead of 8 measured the same.
template <typename TQ, typename TKV, int D, int GC>
__global__ __launch_bounds__(kMaxDecodeWaves * kWave) void paged_decode_direct_kernel(const PagedParams p) {
  __shared__ __align__(16) float s_o[kMaxDecodeWaves * GC * D];
  __shared__ float s_ml[2 * kMaxDecodeWaves * GC];
  decode_list<TQ, TKV, D, GC, kMaxDecodeWaves>(p, blockIdx.y, blockIdx.x, s_o, s_ml);
}

// ------------------------------------------------------------------ dispatch

namespace {

int decode_waves(const PagedParams& p, int gc) {
  const int units = p.hk * (p.hq / p.hk / gc);
  return units < 8 ? units : 8;
}

// From this many workgroups per sequence on (so about as many pieces) 16 thread groups of
// 32 columns share a sequence's pieces instead of four of 128: one 8192-key sequence 20.4 ->
// 17.4 us a call, 8 of 300-2300 keys level, 16 of 1024 (16 pieces) 19.1 -> 20.0.
constexpr int kWideMergePieces = 32;

template <typename TQ, int D, bool kWindow>
hipError_t launch_stream_merge(const PagedParams& p, hipStream_t stream) {
  const int n4 = p.hq * D / 4;
  auto grid = [&](int groups) {
    const int cols = kMergeThreads / groups;
    return dim3(p.num_seqs, (n4 + cols - 1) / cols);
  };
  if (p.stream_wgs >= kWideMergePieces * p.num_seqs) {
    paged_decode_stream_merge_kernel<TQ, D, 16, kWindow><<<grid(16), kMergeThreads, 0, stream>>>(p, p.stream_wgs);
  } else {
    paged_decode_stream_merge_kernel<TQ, D, 4, kWindow><<<grid(4), kMergeThreads, 0, stream>>>(p, p.stream_wgs);
  }
  return hipGetLastError();
}

template <typename TQ, typename TKV, int D, int GC, bool kWindow>
hipError_t launch_decode_g(const PagedParams& p, hipStream_t stream) {
  const int units = p.hk * (p.hq / p.hk / GC);
  const int waves = decode_waves(p, GC);
  constexpr int kHeadsPerMergeBlock = 4;
  if constexpr (kWindow) {
    if (p.direct != 0) {
      paged_decode_direct_kernel<TQ, TKV, D, GC>
          <<<dim3(units, p.num_seqs), kMaxDecodeWaves * kWave, 0, stream>>>(p);
      return hipGetLastError();
    }
  }
  if (p.stream_wgs > 0) {
    if (units > 8) return hipErrorInvalidValue;  // planner keeps stream mode to <= 8 units
    paged_decode_stream_kernel<TQ, TKV, D, GC, false, kWindow>
        <<<p.stream_wgs, waves * kWave, 0, stream>>>(p, FreshParams{});
    hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    return launch_stream_merge<TQ, D, kWindow>(p, stream);
  }
  const dim3 grid(p.max_splits, p.by_row ? p.num_tokens : p.num_seqs, (units + waves - 1) / waves);
  paged_decode_grid_kernel<TQ, TKV, D, GC, kWindow><<<grid, waves * kWave, 0, stream>>>(p);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess || p.max_splits == 1) return err;
  const dim3 mgrid((p.hq + kHeadsPerMergeBlock - 1) / kHeadsPerMergeBlock,
                   p.by_row ? p.num_tokens : p.num_seqs);
  paged_decode_grid_merge_kernel<TQ, D, kWindow><<<mgrid, kHeadsPerMergeBlock * kWave, 0, stream>>>(p);
  return hipGetLastError();
}

template <typename TQ, typename TKV, int D>
hipError_t launch_decode_d(const PagedParams& p, hipStream_t stream) {
  const int gc = decode_group_chunk(p.hq / p.hk);
  if (p.window > 0) {
    if (gc == 4) return launch_decode_g<TQ, TKV, D, 4, true>(p, stream);
    return gc == 2 ? launch_decode_g<TQ, TKV, D, 2, true>(p, stream)
                   : launch_decode_g<TQ, TKV, D, 1, true>(p, stream);
  }
  if (gc == 4) return launch_decode_g<TQ, TKV, D, 4, false>(p, stream);
  return gc == 2 ? launch_decode_g<TQ, TKV, D, 2, false>(p, stream)
                 : launch_decode_g<TQ, TKV, D, 1, false>(p, stream);
}

template <typename TQ, typename TKV>
hipError_t launch_decode_t(const PagedParams& p, int head_dim, hipStream_t stream) {
  switch (head_dim) {
    case 32: return launch_decode_d<TQ, TKV, 32>(p, stream);
    case 64: return launch_decode_d<TQ, TKV, 64>(p, stream);
    case 128: return launch_decode_d<TQ, TKV, 128>(p, stream);
    case 256: return launch_decode_d<TQ, TKV, 256>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace

namespace {

template <typename T, int GC>
hipError_t launch_fresh_g(const PagedParams& p, const FreshParams& f, hipStream_t stream) {
  constexpr int D = 128;
  const int units = p.hk * (p.hq / p.hk / GC);
  if (units > 8) return hipErrorInvalidValue;  // planner keeps stream mode to <= 8 units
  paged_decode_stream_kernel<T, T, D, GC, true, false>
      <<<p.stream_wgs, decode_waves(p, GC) * kWave, 0, stream>>>(p, f);
  hipError_t err = hipGetLastError();
  if (err != hipSuccess) return err;
  return launch_stream_merge<T, D, false>(p, stream);
}

template <typename T>
hipError_t launch_fresh_t(const PagedParams& p, const FreshParams& f, hipStream_t stream) {
  switch (decode_group_chunk(p.hq / p.hk)) {
    case 4: return launch_fresh_g<T, 4>(p, f, stream);
    case 2: return launch_fresh_g<T, 2>(p, f, stream);
    default: return launch_fresh_g<T, 1>(p, f, stream);
  }
}

}  // namespace

hipError_t launch_paged_decode_fresh(const PagedParams& p, const FreshParams& f, int dtype,
                                     int head_dim, hipStream_t stream) {
  if (head_dim != 128 || p.stream_wgs <= 0) return hipErrorInvalidValue;
  switch (dtype) {
    case kF16: return launch_fresh_t<f16_t>(p, f, stream);
    case kBF16: return launch_fresh_t<bf16_t>(p, f, stream);
    default: return hipErrorInvalidValue;
  }
}

hipError_t launch_paged_decode(const PagedParams& p, int q_dtype, int kv_dtype, int head_dim,
                               hipStream_t stream) {
  if (kv_dtype == kFP8E4M3) {
    if (q_dtype == kBF16) return launch_decode_t<bf16_t, fp8_t>(p, head_dim, stream);
    if (q_dtype == kF16) return launch_decode_t<f16_t, fp8_t>(p, head_dim, stream);
    if (q_dtype == kF32) return launch_decode_t<float, fp8_t>(p, head_dim, stream);
    return hipErrorInvalidValue;
  }
  if (q_dtype != kv_dtype) return hipErrorInvalidValue;
  switch (q_dtype) {
    case kF32: return launch_decode_t<float, float>(p, head_dim, stream);
    case kF16: return launch_decode_t<f16_t, f16_t>(p, head_dim, stream);
    case kBF16: return launch_decode_t<bf16_t, bf16_t>(p, head_dim, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace mvllm
