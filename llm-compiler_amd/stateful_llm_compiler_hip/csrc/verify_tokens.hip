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
// small batches are bound by the chain of memory round trips, not by them: the nodes'
// tokens, their probabilities (all gathered at once), the row, its blocks' sums, one
// block again.  So several workgroups share a sequence: each walks the tree for itself
// and sums blocks of 1024 weights, one a wave, and the last to arrive finds the block and
// the token.  Only a node whose second child is tried with a draft row needs more
// passes over its row (the mass decides the next test); the last workgroup makes
// them alone, 19 us each at this vocabulary in fp32 (1.2 MB through one CU): 8 trees of 16 nodes,
// four children each, 65 us, of 64 nodes 65 to 104.
//
// In a graph, vocabulary 151936, fp32: a chain of 5 nodes 7.7 us, 8 trees of 64 without
// draft rows 7.7 us, of 100, from LDS, 11.6; 32 chains of 9 15.4 us, 39 MB at 2.5 TB/s: of it some
// 7 us are the round trips and the launch again, 8 us the rows at the rate of a large copy.
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace {

// The kernel's lambdas: one that is called would keep what it captures in memory.
#define SLC_INLINE __attribute__((always_inline))

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kBlock = 1024;  // weights per sum, 16 a lane
constexpr int kPerLane = kBlock / 64;
constexpr int kGroup = 4;  // neighbouring sums that a lane takes
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
  uint64_t* sums;          // [B, blocks], zero between calls
  int* counters;           // [B], zero between calls
  int64_t tok_sb, par_sb, uni_sb, t_sb, t_st, d_sb, d_st;
  int nodes, vocab, blocks, segments;
  bool vector_ok;  // rows start on 16 bytes
};

// A value that all lanes share, in scalar registers: the walk's branches are the wave's.
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ double lane_value(double v, int lane) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(bits), lane));
  const uint64_t hi = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(bits >> 32), lane));
  return __builtin_bit_cast(double, hi << 32 | lo);
}
__device__ __forceinline__ double uniform(double v) { return lane_value(v, 0); }

// A probability as a weight: none where it is NaN or negative (fmax gives its other operand
// for NaN).
template <typename P>
__device__ __forceinline__ double weight_of(P v) {
  return fmax(static_cast<double>(slc::to_f32(v)), 0.0);
}

template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double v) {
  const uint64_t bits = __builtin_bit_cast(uint64_t, v);
  const uint64_t lo = static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(bits), CTRL, ROWS, 0xf, false));
  const uint64_t hi = static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(bits >> 32), CTRL, ROWS, 0xf, false));
  return __builtin_bit_cast(double, hi << 32 | lo);
}
// Sums up to and with this lane: rows of 16 lanes by shifts, then the rows below by
// broadcasts of their last lanes.
__device__ __forceinline__ double wave_scan(double v) {
  v += dpp<0x111, 0xf>(v);  // row_shr:1
  v += dpp<0x112, 0xf>(v);
  v += dpp<0x114, 0xf>(v);
  v += dpp<0x118, 0xf>(v);
  v += dpp<0x142, 0xa>(v);  // row_bcast:15
  v += dpp<0x143, 0xc>(v);  // row_bcast:31
  return v;
}

// The nodes of a sequence.  Up to 64: one a lane, in registers of every wave.
struct LaneNodes {
  int above, token;  // parent and token, -1: none
  double prob;       // target's probability of the token behind the parent
  int place;         // lane j: the path's j-th node

  __device__ __forceinline__ int token_of(int c) const { return __builtin_amdgcn_readlane(token, c); }
  __device__ __forceinline__ double prob_of(int c) const { return lane_value(prob, c); }
  __device__ __forceinline__ int next_child(int node, int after) const {
    const uint64_t later = after >= 63 ? 0 : ~uint64_t{0} << (after + 1);
    const uint64_t hits = __ballot(above == node) & later;
    return hits != 0 ? __builtin_ctzll(hits) : -1;
  }
  // Whether an elder sibling of node c has its token.
  __device__ __forceinline__ bool again(int node, int c) const {
    return (__ballot(above == node && token == token_of(c)) & ((uint64_t{1} << c) - 1)) != 0;
  }
  __device__ __forceinline__ void put(int at, int node) { place = (threadIdx.x & 63) == static_cast<unsigned>(at) ? node : place; }
};
// More: in LDS, which the workgroup's waves fill together.
struct SharedNodes {
  int* above;
  int* token;
  double* prob;
  int* path;
  int nodes;

  __device__ __forceinline__ int token_of(int c) const { return uniform(token[c]); }
  __device__ __forceinline__ double prob_of(int c) const { return uniform(prob[c]); }
  __device__ __forceinline__ int next_child(int node, int after) const {
    const int lane = threadIdx.x & 63;
    for (int base = (after + 1) & ~63; base < nodes; base += 64) {
      const int c = base + lane;
      const uint64_t hits = __ballot(c > after && c < nodes && above[c] == node);
      if (hits != 0) return base + __builtin_ctzll(hits);
    }
    return -1;
  }
  __device__ __forceinline__ bool again(int node, int c) const {
    const int lane = threadIdx.x & 63, t = token_of(c);
    for (int base = node & ~63; base < c; base += 64) {
      const int s = base + lane;
      if (__ballot(s < c && above[s] == node && token[s] == t) != 0) return true;
    }
    return false;
  }
  __device__ __forceinline__ void put(int at, int node) { path[at] = node; }  // by every thread, one value
};

template <typename P, bool SMALL, bool DRAFT>
__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyArgs a) {
  __shared__ int arrived;
  const int64_t b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 63, wave = uniform(tid >> 6);
  const P* target = static_cast<const P*>(a.target) + b * a.t_sb;
  const P* draft = DRAFT ? static_cast<const P*>(a.draft) + b * a.d_sb : nullptr;
  const float* uniforms = a.uniforms + b * a.uni_sb;
  auto load_node = [&](int c, int& above, int& token, double& prob) SLC_INLINE {
    const int64_t up = a.parents == nullptr ? c - 1 : a.parents[b * a.par_sb + c];
    const int64_t t = a.tokens[b * a.tok_sb + c];
    above = c > 0 && up >= 0 && up < c ? static_cast<int>(up) : -1;
    const bool real = above >= 0 && t >= 0 && t < a.vocab;
    token = real ? static_cast<int>(t) : -1;
    prob = real ? weight_of(target[above * a.t_st + t]) : 0.0;
  };
  using Nodes = std::conditional_t<SMALL, LaneNodes, SharedNodes>;
  Nodes nodes;
  float u_lane = 0.0f;    // SMALL: the lane's random number,
  double q_lane = 0.0;    // and the draft's probability of its token
  if constexpr (SMALL) {
    nodes.above = nodes.token = nodes.place = -1;
    nodes.prob = 0.0;
    if (lane < a.nodes) {
      u_lane = uniforms[lane];
      load_node(lane, nodes.above, nodes.token, nodes.prob);
      if (DRAFT && nodes.token >= 0)
        q_lane = weight_of(draft[nodes.above * a.d_st + nodes.token]);
    }
  } else {
    __shared__ double prob[kMaxNodes];
    __shared__ int above[kMaxNodes], token[kMaxNodes], path[kMaxNodes];
    nodes = {above, token, prob, path, a.nodes};
    for (int c = tid; c < a.nodes; c += kThreads) load_node(c, above[c], token[c], prob[c]);
    __syncthreads();
  }
  auto random_of = [&](int c) SLC_INLINE {
    if constexpr (SMALL) return lane_value(static_cast<double>(u_lane), c);
    return uniform(static_cast<double>(uniforms[c]));
  };
  auto draft_of = [&](int node, int c) SLC_INLINE {
    if constexpr (SMALL) return lane_value(q_lane, c);
    const int t = nodes.token_of(c);
    return t < 0 ? 0.0 : uniform(weight_of(draft[node * a.d_st + t]));
  };

  // Down the tree from `node` to the first node without an accepted child; with draft
  // rows only to the first whose first child is refused, as the next test needs a mass.
  // Without, `excluded` says whether that node's children's tokens have no weight.
  int count = 0, node = 0, tried = -1;
  double mass = 0.0;
  auto walk = [&](int from) SLC_INLINE {
    node = from;
    nodes.put(count++, node);
    for (;;) {
      int next = -1;
      if constexpr (DRAFT) {
        tried = nodes.next_child(node, node);
        if (tried < 0) break;
        if (uniform(static_cast<int>(random_of(tried) * draft_of(node, tried) < nodes.prob_of(tried))) != 0) next = tried;
      } else {
        double left = 1.0;
        for (int c = nodes.next_child(node, node); c >= 0; c = nodes.next_child(node, c)) {
          const double w = nodes.again(node, c) ? 0.0 : nodes.prob_of(c);
          if (uniform(static_cast<int>(w > 0.0 && random_of(c) * left < w)) != 0) {
            next = c;
            break;
          }
          left -= w;
        }
      }
      if (next < 0) break;
      node = next;
      nodes.put(count++, node);
    }
    mass = DRAFT && tried >= 0 ? 1.0 : 0.0;
  };
  bool excluded = !DRAFT;
  walk(0);

  // The weights: max(p - mass * q, 0), or p without the children's tokens.  NaN and negative
  // probabilities have none, p's and q's.
  // The lane's 16 of a block at `base`: DENSE: neighbours, for a scan in order; else as
  // coalesced loads (16 bytes a lane, or one element) have them.
  auto column = [&](bool dense, bool vector, int i) SLC_INLINE {
    constexpr int kVec = 16 / sizeof(P);  // elements of a load
    if (dense) return lane * kPerLane + i;
    return vector ? i / kVec * (64 * kVec) + lane * kVec + i % kVec : i * 64 + lane;
  };
  constexpr int kVec = 16 / sizeof(P), kLoads = kPerLane / kVec, kWords = 4 * kLoads;
  struct Raw {
    uint32_t p[kWords], q[kWords];
  };
  auto is_vector = [&](int block) SLC_INLINE { return a.vector_ok && (block + 1) * static_cast<int64_t>(kBlock) <= a.vocab; };
  auto load_vector = [&](auto dense_tag, const P* row, int block, uint32_t (&words)[kWords]) SLC_INLINE {
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const uint4 v = *reinterpret_cast<const uint4*>(row + static_cast<int64_t>(block) * kBlock +
                                                      column(decltype(dense_tag)::value, true, j * kVec));
      words[4 * j] = v.x;
      words[4 * j + 1] = v.y;
      words[4 * j + 2] = v.z;
      words[4 * j + 3] = v.w;
    }
  };
  auto load_any = [&](auto dense_tag, const P* row, int block, uint32_t (&words)[kWords]) SLC_INLINE {
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int64_t at = static_cast<int64_t>(block) * kBlock + column(decltype(dense_tag)::value, false, i);
      const P v = row[at < a.vocab ? at : 0];
      if constexpr (sizeof(P) == 4) {
        words[i] = at < a.vocab ? __float_as_uint(v) : 0;
      } else {
        const uint32_t bits = at < a.vocab ? v.bits : 0;
        words[i / 2] = i % 2 == 0 ? bits : words[i / 2] | bits << 16;
      }
    }
  };
  // Where no mass is taken off, q's place is p's: loaded, not looked at.
  auto load = [&](auto dense_tag, int block, Raw& raw) SLC_INLINE {
    const P* p = target + node * a.t_st;
    const P* q = mass > 0.0 ? draft + node * a.d_st : p;
    if (is_vector(block)) {
      load_vector(dense_tag, p, block, raw.p);
      if constexpr (DRAFT) load_vector(dense_tag, q, block, raw.q);
    } else {
      load_any(dense_tag, p, block, raw.p);
      if constexpr (DRAFT) load_any(dense_tag, q, block, raw.q);
    }
  };
  auto element = [](const uint32_t (&words)[kWords], int i) SLC_INLINE {
    if constexpr (sizeof(P) == 4) {
      return __uint_as_float(words[i]);
    } else {
      return slc::to_f32(P{static_cast<uint16_t>(words[i / 2] >> (16 * (i % 2)))});
    }
  };
  auto weights = [&](auto dense_tag, int block, const Raw& raw, double (&w)[kPerLane]) SLC_INLINE {
    constexpr bool kDense = decltype(dense_tag)::value;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      double v = static_cast<double>(element(raw.p, i));
      if constexpr (DRAFT) v = fma(-mass, mass > 0.0 ? weight_of(element(raw.q, i)) : 0.0, v);
      w[i] = fmax(v, 0.0);  // 0 for NaN
    }
    if (!excluded) return;
    const bool vector = is_vector(block);
    for (int c = nodes.next_child(node, node); c >= 0; c = nodes.next_child(node, c)) {
      const int64_t at = nodes.token_of(c) - static_cast<int64_t>(block) * kBlock;
      if (at < 0 || at >= kBlock) continue;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i)
        if (column(kDense, vector, i) == at) w[i] = 0.0;
    }
  };

  // A block's sum is published with its sign set: a word of zeros is none yet.
  uint64_t* sums = a.sums + b * a.blocks;
  auto sum_block = [&](int block, const Raw& raw) SLC_INLINE {
    double w[kPerLane], sum = 0.0;
    weights(std::false_type{}, block, raw, w);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) sum += w[i];
    sum = wave_scan(sum);
    if (lane == 63)
      __hip_atomic_store(&sums[block], __builtin_bit_cast(uint64_t, -sum), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  };
  auto sum_blocks = [&](int first, int step) SLC_INLINE {
    // Whole blocks of 16-byte loads: a block's are in flight while the one before is
    // summed (the last one's twice, so that no branch makes the loop wait for them).
    const int whole = a.vector_ok ? a.vocab / kBlock : 0;
    const P* p = target + node * a.t_st;
    const P* q = mass > 0.0 ? draft + node * a.d_st : p;
    int block = first;
    if (block < whole) {
      Raw raw;
      load_vector(std::false_type{}, p, block, raw.p);
      if constexpr (DRAFT) load_vector(std::false_type{}, q, block, raw.q);
#pragma unroll 2
      for (; block < whole; block += step) {
        const Raw now = raw;
        const int next = block + step < whole ? block + step : block;
        load_vector(std::false_type{}, p, next, raw.p);
        if constexpr (DRAFT) load_vector(std::false_type{}, q, next, raw.q);
        sum_block(block, now);
      }
    }
#pragma unroll 1
    for (; block < a.blocks; block += step) {
      Raw raw;
      load_any(std::false_type{}, p, block, raw.p);
      if constexpr (DRAFT) load_any(std::false_type{}, q, block, raw.q);
      sum_block(block, raw);
    }
  };
  sum_blocks(blockIdx.x * kWaves + wave, a.segments * kWaves);

  // The last workgroup of the sequence goes on.  Sums that are not there yet are waited
  // for one by one, so nothing orders them and the count: a release and an acquire, whose
  // cache write-backs and invalidations delay all other workgroups' loads, make 30 us of
  // 32 chains' 15.
  __syncthreads();
  if (tid == 0)
    arrived = __hip_atomic_fetch_add(&a.counters[b], 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (uniform(arrived) != a.segments - 1) return;
  if (tid == 0) __hip_atomic_store(&a.counters[b], 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);

  // The first wave decides; the others sum blocks for it where it needs other weights.
  __shared__ int order_node, order_excluded;
  __shared__ double order_mass;
  if (wave != 0) {
    for (;;) {
      __syncthreads();  // an order is there
      node = uniform(order_node);
      if (node < 0) return;
      mass = uniform(order_mass);
      excluded = uniform(order_excluded) != 0;
      sum_blocks(wave, kWaves);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "agent");
      __syncthreads();
    }
  }
  // 256 blocks' sums, kGroup neighbours a lane, and the sums up to and with this lane's.
  auto load_group = [&](int first, double (&s)[kGroup]) SLC_INLINE {
    // The bound ends the wait whatever happens; a sum's store was issued long before.
    for (int turn = 0; turn < (1 << 20); ++turn) {
      uint64_t bits[kGroup];
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        // (A load that a branch guards would be waited for before the next.)
        const int block = first + lane * kGroup + i;
        bits[i] = __hip_atomic_load(&sums[block < a.blocks ? block : a.blocks - 1], __ATOMIC_RELAXED,
                                    __HIP_MEMORY_SCOPE_AGENT);
      }
      bool there = true;
#pragma unroll
      for (int i = 0; i < kGroup; ++i) {
        there &= bits[i] != 0;
        s[i] = first + lane * kGroup + i < a.blocks ? -__builtin_bit_cast(double, bits[i]) : 0.0;
      }
      if (__all(there)) return;
    }
  };
  auto scan_group = [&](const double (&s)[kGroup]) SLC_INLINE {
    double own = s[0];
#pragma unroll
    for (int i = 1; i < kGroup; ++i) own += s[i];
    return wave_scan(own);
  };
  double lead[kGroup], lead_scan;  // the first 256
  auto total_of = [&]() SLC_INLINE {
    load_group(0, lead);
    lead_scan = scan_group(lead);
    double total = lane_value(lead_scan, 63);
    for (int first = 64 * kGroup; first < a.blocks; first += 64 * kGroup) {
      double s[kGroup];
      load_group(first, s);
      total += lane_value(scan_group(s), 63);
    }
    return total;
  };
  auto sum_again = [&]() SLC_INLINE {
    if (lane == 0) {
      order_node = node;
      order_mass = mass;
      order_excluded = excluded;
    }
    __syncthreads();
    sum_blocks(0, kWaves);
    __syncthreads();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");  // none of the old sums
    return total_of();
  };
  double total = total_of();
  while (DRAFT && tried >= 0) {
    const int c = nodes.next_child(node, tried);
    if (c < 0) break;
    const double q = draft_of(node, c);
    const double rest = fmax(fma(-mass, q, nodes.prob_of(c)), 0.0);
    if (uniform(static_cast<int>(random_of(c) * total * q < rest)) != 0) {
      walk(c);
    } else {
      mass += total;
      tried = c;
    }
    total = sum_again();
  }
  if (!(total > 0.0)) {
    mass = 0.0;
    excluded = false;
    total = sum_again();
  }
  if (lane == 0) order_node = -1;
  __syncthreads();  // the other waves end

  // The first block with weight whose sum passes the goal.  A lane's start is a scan's sum, the
  // end of the lane before it one of neighbours: a rounding apart, the goal may lie between
  // them, and the blocks behind it weigh nothing.  A random number outside [0, 1) or an
  // infinite sum may find none: the last block with any weight then.
  const double goal = random_of(0) * total;
  int block = -1, spare = -1;
  double before = 0.0, base = 0.0;
  for (int first = 0; first < a.blocks && block < 0; first += 64 * kGroup) {
    double s[kGroup], upto;
    if (first == 0) {
#pragma unroll
      for (int i = 0; i < kGroup; ++i) s[i] = lead[i];
      upto = lead_scan;
    } else {
      load_group(first, s);
      upto = scan_group(s);
    }
    upto += base;
    double run = dpp<0x138, 0xf>(upto);  // wave_shr:1
    if (lane == 0) run = base;
    int hit = -1, some = -1;
    double start = run;
#pragma unroll
    for (int i = 0; i < kGroup; ++i) {
      const double next = run + s[i];
      if (s[i] > 0.0) some = i;
      if (hit < 0 && s[i] > 0.0 && next > goal) {
        hit = i;
        start = run;
      }
      run = next;
    }
    const uint64_t hits = __ballot(hit >= 0), any = __ballot(some >= 0);
    if (hits != 0) {
      const int from = __builtin_ctzll(hits);
      block = first + from * kGroup + __builtin_amdgcn_readlane(hit, from);
      before = lane_value(start, from);
    } else if (any != 0) {
      const int from = 63 - __builtin_clzll(any);
      spare = first + from * kGroup + __builtin_amdgcn_readlane(some, from);
    }
    base = lane_value(upto, 63);
  }
  int64_t drawn = -1;
  if (block < 0) block = spare;
  if (block >= 0) {
    Raw raw;
    double w[kPerLane], own = 0.0;
    load(std::true_type{}, block, raw);
    weights(std::true_type{}, block, raw, w);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) own += w[i];
    const double upto = before + wave_scan(own);
    double run = dpp<0x138, 0xf>(upto);
    if (lane == 0) run = before;
    int hit = -1, last = -1;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      run += w[i];
      if (w[i] > 0.0) last = i;
      if (hit < 0 && w[i] > 0.0 && run > goal) hit = i;
    }
    // Sums of another order than the block's may end a rounding before the goal: the
    // block's last weight then.
    const uint64_t hits = __ballot(hit >= 0), lasts = __ballot(last >= 0);
    if (lasts != 0) {
      const int from = hits != 0 ? __builtin_ctzll(hits) : 63 - __builtin_clzll(lasts);
      drawn = static_cast<int64_t>(block) * kBlock + from * kPerLane +
              __builtin_amdgcn_readlane(hits != 0 ? hit : last, from);
    }
  }
  for (int first = lane; first < a.blocks; first += 64)
    __hip_atomic_store(&sums[first], uint64_t{0}, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  for (int j = lane; j < a.nodes; j += 64) {
    int at, follow;
    if constexpr (SMALL) {
      at = nodes.place;
      const int next = __shfl(nodes.place, lane + 1 < 64 ? lane + 1 : 63, 64);
      follow = __shfl(nodes.token, next < 0 ? 0 : next, 64);
    } else {
      at = j < count ? nodes.path[j] : -1;
      follow = j + 1 < count ? nodes.token[nodes.path[j + 1]] : -1;
    }
    a.path[b * a.nodes + j] = j < count ? at : -1;
    a.emitted[b * a.nodes + j] = j + 1 < count ? follow : (j + 1 == count ? drawn : -1);
  }
  if (lane == 0) a.counts[b] = count;
}

template <typename P>
int launch(VerifyArgs a, int64_t batch, hipStream_t stream) {
  const auto aligned = [](const void* p, int64_t sb, int64_t st) {
    return (reinterpret_cast<uintptr_t>(p) % 16 | sb * sizeof(P) % 16 | st * sizeof(P) % 16) == 0;
  };
  a.vector_ok = aligned(a.target, a.t_sb, a.t_st) && aligned(a.draft, a.d_sb, a.d_st);
  auto kernel = a.draft != nullptr ? (a.nodes <= 64 ? verify_kernel<P, true, true> : verify_kernel<P, false, true>)
                                   : (a.nodes <= 64 ? verify_kernel<P, true, false> : verify_kernel<P, false, false>);
  hipLaunchKernelGGL(kernel, dim3(a.segments, static_cast<unsigned>(batch)), dim3(kThreads), 0, stream, a);
  return slc_host::check_launch("slc_hip_verify_tokens");
}

int64_t block_count(int64_t vocab) { return slc_host::ceil_div(vocab, kBlock); }

}  // namespace

extern "C" int64_t slc_hip_verify_tokens_counter_count(int64_t batch, int64_t vocab) {
  return batch > 0 && vocab > 0 ? (batch + 1) / 2 * 2 + 2 * batch * block_count(vocab) : 0;
}

extern "C" int slc_hip_verify_tokens(
    const int64_t* tokens, const int64_t* parents, const void* target, const void* draft,
    const float* uniforms, int64_t* path, int64_t* emitted, int64_t* counts, int* counters,
    int64_t num_counters, int dtype, int64_t batch, int64_t nodes, int64_t vocab,
    int64_t tok_stride_b, int64_t parent_stride_b, int64_t uniform_stride_b, int64_t target_stride_b,
    int64_t target_stride_t, int64_t draft_stride_b, int64_t draft_stride_t, void* stream) {
  const char* what = "slc_hip_verify_tokens";
  SLC_REQUIRE(slc_host::is_float_dtype(dtype), "%s: bad dtype %d", what, dtype);
  SLC_REQUIRE(batch >= 0 && batch <= 65535, "%s: batch must be 0 to 65535", what);
  SLC_REQUIRE(nodes >= 1 && nodes <= kMaxNodes, "%s: 1 to %d nodes", what, kMaxNodes);
  SLC_REQUIRE(vocab >= 1 && vocab <= 0x7fffffff - kBlock, "%s: bad vocabulary size", what);
  if (batch == 0) return SLC_OK;
  SLC_REQUIRE(tokens && target && uniforms && path && emitted && counts && counters, "%s: null pointer", what);
  SLC_REQUIRE(num_counters >= slc_hip_verify_tokens_counter_count(batch, vocab) &&
                  (reinterpret_cast<uintptr_t>(counters) & 7) == 0,
              "%s: too few counters, or not on 8 bytes", what);
  VerifyArgs a{};
  a.tokens = tokens;
  a.parents = parents;
  a.target = target;
  a.draft = draft;
  a.uniforms = uniforms;
  a.path = path;
  a.emitted = emitted;
  a.counts = counts;
  a.counters = counters;
  a.sums = reinterpret_cast<uint64_t*>(counters + (batch + 1) / 2 * 2);
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
  // One block a wave, but no more workgroups than CUs: with draft rows the registers (130
  // to 148 of a lane, up to 64 nodes) leave room for one each (32 chains 15 us, with twice as many
  // 21).  Without, where two fit (117 to 125), the same rule.
  a.segments = static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>(slc_host::ceil_div(a.blocks, kWaves), slc_host::device_cu_count() / batch)));
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
