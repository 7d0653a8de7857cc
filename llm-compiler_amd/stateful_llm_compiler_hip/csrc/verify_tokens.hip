// verify_tokens: which drafted tokens the target's probabilities accept, and the
// token that follows them, from given random numbers.
//
// A sequence's nodes form a tree (node 0, the last token that stands, is its root;
// parents come first).  At a node with target row p the children are tried in
// order.  With a draft row q, from which they were drawn independently, the first
// one, x, is accepted where u q(x) < p(x); a refusal leaves w = max(p - M q, 0)
// with M = 1 and the mass m = sum w, the next child is accepted where
// u m q(x) < w(x), a refusal adds m to M, and so on (max(max(p - a q, 0) - b q, 0)
// = max(p - (a + b) q, 0)).  Without draft rows a candidate x is accepted where
// u m < p(x), m = 1 less the refused ones' probabilities, and a refusal sets
// w(x) = 0.  Where no child is accepted the next token is the first i with
// w(0) + .. + w(i) > u_0 sum w; where no w is left, p itself is drawn from.  Each
// accepted or drawn token has the target's distribution.
//
// All of it is fp64: products of two fp32 numbers are exact there, and a border
// between two tokens moves by 1e-16 of the sum with the order of additions.
//
// The bytes are one row (p) or two (p and q) of the vocabulary per sequence, and
// a call is bound by the chain of memory round trips, not by them: the nodes' own
// probabilities (all gathered at once), the row, its blocks' sums, one block again.
// So several workgroups share a sequence: each walks the tree for itself, sums
// blocks of 1024 weights, one a wave, and the last to arrive finds the block and
// the token.  Only a node whose second child is tried with a draft row needs more
// passes over its row (the mass decides the next test); the last workgroup makes
// them alone.
#include <algorithm>

#include "common.hpp"

namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kBlock = 1024;  // weights per sum, 16 a lane
constexpr int kPerLane = kBlock / 64;
constexpr int kMaxNodes = SLC_VERIFY_MAX_NODES;

struct VerifyArgs {
  const int64_t* tokens;   // [B, T], rows tok_sb apart
  const int64_t* parents;  // [B, T], rows par_sb apart; null: a chain
  const void* target;      // [B, T, V]
  const void* draft;       // [B, T - 1, V] or null
  const float* uniforms;   // [B, T], rows uni_sb apart
  int64_t* path;           // [B, T]
  int64_t* emitted;        // [B, T]
  int64_t* counts;         // [B]
  double* sums;            // [B, blocks]
  int* counters;           // [B]
  int64_t tok_sb, par_sb, uni_sb, t_sb, t_st, d_sb, d_st;
  int nodes, vocab, blocks, segments;
  bool vector_ok;  // rows start on 16 bytes
};

// The weights of a row: max(p - mass * q, 0), or p without the listed tokens.
template <typename P>
struct Row {
  const P* p;
  const P* q;  // null: no draft row
  double mass;
  const int* skip;
  int skips;

  __device__ __forceinline__ double value(float pv, float qv) const {
    const double w = static_cast<double>(pv) - mass * static_cast<double>(qv);
    return w > 0.0 ? w : 0.0;  // NaN has no weight
  }

  // Column of the lane's i-th weight of the block at `base`.  DENSE: 16 neighbours a
  // lane, for a scan in order; else as coalesced loads (16 bytes a lane, or one
  // element) have them.
  template <bool DENSE>
  static __device__ __forceinline__ int64_t index(int64_t base, int i, bool vector) {
    constexpr int kVec = 16 / sizeof(P);
    const int lane = threadIdx.x & 63;
    if constexpr (DENSE) return base + lane * kPerLane + i;
    return vector ? base + (i / kVec) * (64 * kVec) + lane * kVec + i % kVec : base + i * 64 + lane;
  }

  template <bool DENSE>
  __device__ __forceinline__ void load(int64_t base, int vocab, bool vector_ok, double (&w)[kPerLane]) const {
    constexpr int kVec = 16 / sizeof(P);
    const bool vector = vector_ok && base + kBlock <= vocab;
    float pv[kPerLane], qv[kPerLane];
    if (vector) {
      uint4 rp[kPerLane / kVec], rq[kPerLane / kVec];
#pragma unroll
      for (int j = 0; j < kPerLane / kVec; ++j)
        rp[j] = *reinterpret_cast<const uint4*>(p + index<DENSE>(base, j * kVec, true));
      if (q != nullptr) {
#pragma unroll
        for (int j = 0; j < kPerLane / kVec; ++j)
          rq[j] = *reinterpret_cast<const uint4*>(q + index<DENSE>(base, j * kVec, true));
      } else {
#pragma unroll
        for (int j = 0; j < kPerLane / kVec; ++j) rq[j] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        pv[i] = slc::to_f32(reinterpret_cast<const P*>(&rp[i / kVec])[i % kVec]);
        qv[i] = slc::to_f32(reinterpret_cast<const P*>(&rq[i / kVec])[i % kVec]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int64_t at = index<DENSE>(base, i, false);
        pv[i] = at < vocab ? slc::to_f32(p[at]) : 0.0f;
        qv[i] = at < vocab && q != nullptr ? slc::to_f32(q[at]) : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) w[i] = value(pv[i], qv[i]);
    for (int s = 0; s < skips; ++s) {
      const int64_t token = skip[s];
      if (token < base || token >= base + kBlock) continue;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i)
        if (index<DENSE>(base, i, vector) == token) w[i] = 0.0;
    }
  }
};

// A value that all lanes share, in scalar registers: the walk's branches are the wave's.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ double uniform(double v) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(bits)));
  const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(bits >> 32)));
  return __builtin_bit_cast(double, hi << 32 | lo);
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
  for (int offset = 32; offset > 0; offset >>= 1) v += __shfl_xor(v, offset, 64);
  return v;
}
// Sums over this lane and those below it.
__device__ __forceinline__ double wave_scan(double v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int offset = 1; offset < 64; offset <<= 1) {
    const double below = __shfl_up(v, offset, 64);
    if (lane >= offset) v += below;
  }
  return v;
}

template <typename P>
__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyArgs a) {
// A mass times q is rounded before it is subtracted, as the formulas' plain form does.
#pragma clang fp contract(off)
  __shared__ double prob[kMaxNodes];
  __shared__ int parent[kMaxNodes], token[kMaxNodes], path[kMaxNodes], skip[kMaxNodes];
  __shared__ unsigned char accept[kMaxNodes];
  __shared__ int arrived;
  const int64_t b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int nodes = a.nodes;
  const P* target = static_cast<const P*>(a.target) + b * a.t_sb;
  const P* draft = a.draft == nullptr ? nullptr : static_cast<const P*>(a.draft) + b * a.d_sb;
  const float* uniforms = a.uniforms + b * a.uni_sb;

  for (int c = tid; c < nodes; c += kThreads) {
    const int64_t up = a.parents == nullptr ? c - 1 : a.parents[b * a.par_sb + c];
    const int64_t t = a.tokens[b * a.tok_sb + c];
    const int above = c > 0 && up >= 0 && up < c ? static_cast<int>(up) : -1;
    const bool real = above >= 0 && t >= 0 && t < a.vocab;
    parent[c] = above;
    token[c] = real ? static_cast<int>(t) : -1;
    prob[c] = real ? static_cast<double>(slc::to_f32(target[above * a.t_st + t])) : 0.0;
    accept[c] = 0;
  }
  __syncthreads();
  // Each node's test, as if its parent was reached and every elder sibling refused.
  // Without draft rows a token that an elder sibling had too has no weight any more.
  if (draft == nullptr) {
    for (int c = tid; c < nodes; c += kThreads) {
      bool twice = false;
#pragma unroll 4
      for (int s = 1; s < c; ++s) twice |= parent[s] == parent[c] && token[s] == token[c];
      if (twice) prob[c] = 0.0;
    }
    __syncthreads();
  }
  for (int c = 1 + tid; c < nodes; c += kThreads) {
    const int above = parent[c], t = token[c];
    if (above < 0 || t < 0) continue;
    const double u = static_cast<double>(uniforms[c]);
    if (draft == nullptr) {
      double left = 1.0;
#pragma unroll 4
      for (int s = 1; s < c; ++s) left -= parent[s] == above ? prob[s] : 0.0;
      accept[c] = prob[c] > 0.0 && u * left < prob[c];
    } else {
      bool elder = false;
#pragma unroll 4
      for (int s = 1; s < c; ++s) elder |= parent[s] == above;
      accept[c] = !elder && u * static_cast<double>(slc::to_f32(draft[above * a.d_st + t])) < prob[c];
    }
  }
  __syncthreads();

  // The next child of `node` behind `after` (an accepted one), or -1; every wave
  // finds it for itself.
  auto next_child = [&](int node, int after, bool accepted) {
    for (int base = (after + 1) & ~63; base < nodes; base += 64) {
      const int c = base + lane;
      const bool hit = c > after && c < nodes && parent[c] == node && (!accepted || accept[c]);
      const uint64_t hits = __ballot(hit);
      if (hits != 0) return base + __builtin_ctzll(hits);
    }
    return -1;
  };
  int count = 0, node = 0, tried = -1;
  Row<P> row{nullptr, nullptr, 0.0, skip, 0};
  // Down the tree from `from` to the first node without an accepted child.
  auto walk = [&](int from) {
    node = from;
    path[count++] = node;  // by every thread, one value
    for (;;) {
      tried = next_child(node, node, draft == nullptr);
      if (tried < 0 || uniform(static_cast<int>(accept[tried])) == 0) break;
      node = tried;
      path[count++] = node;
    }
    row.p = target + node * a.t_st;
    row.q = draft != nullptr && tried >= 0 ? draft + node * a.d_st : nullptr;
    row.mass = row.q != nullptr ? 1.0 : 0.0;
  };
  walk(0);
  if (draft == nullptr) {
    // The refused candidates: all children of the last node.
    for (int c = next_child(node, node, false); c >= 0; c = next_child(node, c, false)) {
      skip[row.skips++] = token[c];
    }
    __syncthreads();
  }

  double* sums = a.sums + b * a.blocks;
  auto sum_blocks = [&](int first, int step) {
    for (int block = first; block < a.blocks; block += step) {
      double w[kPerLane], sum = 0.0;
      row.template load<false>(static_cast<int64_t>(block) * kBlock, a.vocab, a.vector_ok, w);
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) sum += w[i];
      sum = wave_sum(sum);
      if (lane == 0) __hip_atomic_store(&sums[block], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
  };
  sum_blocks(blockIdx.x * kWaves + wave, a.segments * kWaves);

  // The last workgroup of the sequence goes on: every wave's sums come before the
  // barrier, and the count is an agent-scope acquire-release add behind it.
  __syncthreads();
  if (tid == 0)
    arrived = __hip_atomic_fetch_add(&a.counters[b], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (uniform(arrived) != a.segments - 1) return;
  if (tid == 0) __hip_atomic_store(&a.counters[b], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

  // Sums up to and with each of 64 blocks, on the `base` of those before.
  auto scan_blocks = [&](int first, double base) {
    const double v = first + lane < a.blocks
                         ? __hip_atomic_load(&sums[first + lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                         : 0.0;
    return base + wave_scan(v);
  };
  auto total_of = [&]() {
    double total = 0.0;
    for (int first = 0; first < a.blocks; first += 64) total = __shfl(scan_blocks(first, total), 63, 64);
    return uniform(total);
  };
  auto sum_again = [&]() {
    __syncthreads();  // every wave has read the old sums
    sum_blocks(wave, kWaves);
    __syncthreads();
    return total_of();
  };
  double total = total_of();
  while (row.q != nullptr) {
    const int c = next_child(node, tried, false);
    if (c < 0) break;
    const int t = uniform(token[c]);
    const double q = t < 0 ? 0.0 : uniform(static_cast<double>(slc::to_f32(row.q[t])));
    const double rest = uniform(prob[c]) - row.mass * q;
    const bool follows = static_cast<double>(uniforms[c]) * total * q < (rest > 0.0 ? rest : 0.0);
    if (uniform(static_cast<int>(follows)) != 0) {
      walk(c);
    } else {
      row.mass += total;
      tried = c;
    }
    total = sum_again();
  }
  if (!(total > 0.0)) {
    row.mass = 0.0;
    row.q = nullptr;
    row.skips = 0;
    total = sum_again();
  }
  __syncthreads();  // the path is written

  if (wave == 0) {
    const double goal = static_cast<double>(uniforms[0]) * total;
    // The first block whose sum passes the goal; a random number outside [0, 1) or an
    // infinite sum may find none: the last block with any weight then.
    int block = -1, spare = -1;
    double before = 0.0, base = 0.0;
    for (int first = 0; first < a.blocks && block < 0; first += 64) {
      const double upto = scan_blocks(first, base);
      double prior = __shfl_up(upto, 1, 64);
      if (lane == 0) prior = base;
      const uint64_t hits = __ballot(upto > goal);
      const uint64_t any = __ballot(upto > prior);
      if (hits != 0) {
        const int hit = __builtin_ctzll(hits);
        block = first + hit;
        before = __shfl(prior, hit, 64);
      } else if (any != 0) {
        spare = first + 63 - __builtin_clzll(any);
      }
      base = __shfl(upto, 63, 64);
    }
    int64_t drawn = -1;
    if (block < 0) block = spare;
    if (block >= 0) {
      double w[kPerLane], own = 0.0;
      row.template load<true>(static_cast<int64_t>(block) * kBlock, a.vocab, a.vector_ok, w);
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) own += w[i];
      const double upto = before + wave_scan(own);
      double run = __shfl_up(upto, 1, 64);
      if (lane == 0) run = before;
      int hit = -1, last = -1;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        run += w[i];
        if (w[i] > 0.0) last = i;
        if (hit < 0 && w[i] > 0.0 && run > goal) hit = i;
      }
      // Sums of another order than the block's may end a rounding before the goal:
      // the block's last weight then.
      const uint64_t hits = __ballot(hit >= 0), lasts = __ballot(last >= 0);
      if (lasts != 0) {
        const int from = hits != 0 ? __builtin_ctzll(hits) : 63 - __builtin_clzll(lasts);
        const int at = __shfl(hits != 0 ? hit : last, from, 64);
        drawn = static_cast<int64_t>(block) * kBlock + from * kPerLane + at;
      }
    }
    for (int j = lane; j < nodes; j += 64) {
      a.path[b * nodes + j] = j < count ? path[j] : -1;
      a.emitted[b * nodes + j] = j + 1 < count ? token[path[j + 1]] : (j + 1 == count ? drawn : -1);
    }
    if (lane == 0) a.counts[b] = count;
  }
}

template <typename P>
int launch(VerifyArgs a, int64_t batch, hipStream_t stream) {
  const auto aligned = [](const void* p, int64_t sb, int64_t st) {
    return (reinterpret_cast<uintptr_t>(p) % 16 | sb * sizeof(P) % 16 | st * sizeof(P) % 16) == 0;
  };
  a.vector_ok = aligned(a.target, a.t_sb, a.t_st) && aligned(a.draft, a.d_sb, a.d_st);
  hipLaunchKernelGGL(verify_kernel<P>, dim3(a.segments, static_cast<unsigned>(batch)), dim3(kThreads), 0,
                     stream, a);
  return slc_host::check_launch("slc_hip_verify_tokens");
}

int64_t block_count(int64_t vocab) { return slc_host::ceil_div(vocab, kBlock); }

}  // namespace

extern "C" int64_t slc_hip_verify_tokens_workspace_size(int64_t batch, int64_t vocab) {
  return batch > 0 && vocab > 0 ? batch * block_count(vocab) * static_cast<int64_t>(sizeof(double)) : 0;
}

extern "C" int slc_hip_verify_tokens(
    const int64_t* tokens, const int64_t* parents, const void* target, const void* draft,
    const float* uniforms, int64_t* path, int64_t* emitted, int64_t* counts, void* workspace,
    int64_t workspace_bytes, int* counters, int64_t num_counters, int dtype, int64_t batch,
    int64_t nodes, int64_t vocab, int64_t tok_stride_b, int64_t parent_stride_b,
    int64_t uniform_stride_b, int64_t target_stride_b, int64_t target_stride_t,
    int64_t draft_stride_b, int64_t draft_stride_t, void* stream) {
  const char* what = "slc_hip_verify_tokens";
  SLC_REQUIRE(slc_host::is_float_dtype(dtype), "%s: bad dtype %d", what, dtype);
  SLC_REQUIRE(batch >= 0 && batch <= 65535, "%s: batch must be 0 to 65535", what);
  SLC_REQUIRE(nodes >= 1 && nodes <= kMaxNodes, "%s: 1 to %d nodes", what, kMaxNodes);
  SLC_REQUIRE(vocab >= 1 && vocab <= 0x7fffffff - kBlock, "%s: bad vocabulary size", what);
  if (batch == 0) return SLC_OK;
  SLC_REQUIRE(tokens && target && uniforms && path && emitted && counts && counters && workspace,
              "%s: null pointer", what);
  SLC_REQUIRE(workspace_bytes >= slc_hip_verify_tokens_workspace_size(batch, vocab) &&
                  (reinterpret_cast<uintptr_t>(workspace) & 7) == 0,
              "%s: workspace too small or not on 8 bytes", what);
  SLC_REQUIRE(num_counters >= batch, "%s: too few counters", what);
  VerifyArgs a{};
  a.tokens = tokens;
  a.parents = parents;
  a.target = target;
  a.draft = draft;
  a.uniforms = uniforms;
  a.path = path;
  a.emitted = emitted;
  a.counts = counts;
  a.sums = static_cast<double*>(workspace);
  a.counters = counters;
  a.tok_sb = tok_stride_b;
  a.par_sb = parent_stride_b;
  a.uni_sb = uniform_stride_b;
  a.t_sb = target_stride_b;
  a.t_st = target_stride_t;
  a.d_sb = draft_stride_b;
  a.d_st = draft_stride_t;
  a.nodes = static_cast<int>(nodes);
  a.vocab = static_cast<int>(vocab);
  a.blocks = static_cast<int>(block_count(vocab));
  // One block a wave while the grid stays within what the card holds a few times.
  a.segments = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>(slc_host::ceil_div(a.blocks, kWaves), 4096 / batch)));
  hipStream_t s = static_cast<hipStream_t>(stream);
  switch (dtype) {
    case SLC_BF16:
      return launch<slc::bf16_t>(a, batch, s);
    case SLC_F16:
      return launch<slc::f16_t>(a, batch, s);
    default:
      return launch<float>(a, batch, s);
  }
}
