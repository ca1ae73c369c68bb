// The sequence search of the packed attention (csrc/packed_attention.hip: which sequence, block of tokens and chunk of keys a workgroup
// works on) on the CPU.  Its source is included as it stands (PACKED_SOURCE, cut out by the test); the 64 lanes of a wave are
// contexts that run in turn from one exchange between lanes to the next.  Every index into the starts and lengths is checked, and so
// is every range that a kernel derives its addresses from, for consistent starts and for ones that make no sense.
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cmath>
#include <algorithm>
#include <functional>
#include <random>
#include <set>
#include <vector>
#include <ucontext.h>
#include "evlm_hip.h"

static char told[512];
[[noreturn]] static void fail(const char* what, long a = 0, long b = 0, long c = 0) {
  std::printf("FAILED: %s (%ld %ld %ld) in %s\n", what, a, b, c, told);
  std::exit(1);
}
#define CHECK(x, ...) do { if (!(x)) fail(#x, ##__VA_ARGS__); } while (0)

// ---- a wave ---------------------------------------------------------------------------------------
static ucontext_t home, lanes[64];
static char stacks[64][64 << 10];
static bool done[64];
static long exchanges[64];
static uint64_t slot[2][64];
static int now;
static std::function<void(int)> body;
struct Dim { unsigned x; };
static Dim threadIdx, blockDim = {64};
static void enter() { body(now); done[now] = true; swapcontext(&lanes[now], &home); }
static void wave(std::function<void(int)> f) {
  body = f;
  for (int i = 0; i < 64; ++i) {
    done[i] = false; exchanges[i] = 0;
    getcontext(&lanes[i]);
    lanes[i].uc_stack.ss_sp = stacks[i]; lanes[i].uc_stack.ss_size = sizeof(stacks[i]); lanes[i].uc_link = nullptr;
    makecontext(&lanes[i], enter, 0);
  }
  for (bool any = true; any;) {
    any = false;
    for (int i = 0; i < 64; ++i) {
      if (done[i]) continue;
      any = true; now = i; threadIdx.x = i;
      swapcontext(&home, &lanes[i]);
    }
    for (int i = 1; i < 64; ++i) CHECK(exchanges[i] == exchanges[0] && done[i] == done[0], i);      // all lanes at the same exchange
  }
}
static uint64_t* exchange(uint64_t mine) {
  const int me = now;
  uint64_t* s = slot[exchanges[me]++ & 1];
  s[me] = mine;
  swapcontext(&lanes[me], &home);
  return s;
}
template <typename T> static T lane_of(uint64_t* s, int l) { return (T)s[l & 63]; }
template <typename T> static T __shfl_xor(T v, int o, int) { const int me = now; auto s = exchange((uint64_t)(int64_t)v); return lane_of<T>(s, me ^ o); }
template <typename T> static T __shfl_up(T v, int o, int) { const int me = now; auto s = exchange((uint64_t)(int64_t)v); return lane_of<T>(s, me >= o ? me - o : me); }
template <typename T> static T __shfl(T v, int l, int) { auto s = exchange((uint64_t)(int64_t)v); return lane_of<T>(s, l); }
static unsigned long long __ballot(bool b) {
  auto s = exchange(b);
  unsigned long long m = 0;
  for (int i = 0; i < 64; ++i) m |= (unsigned long long)(s[i] != 0) << i;
  return m;
}
static int __builtin_amdgcn_readfirstlane(int v) { auto s = exchange((uint64_t)(int64_t)v); return lane_of<int>(s, 0); }
using std::max;
using std::min;
#define __device__
#define __forceinline__ inline

struct Starts {                      // what cu_q, cu_k and k_lens are here: every access in range
  const std::vector<int32_t>* v = nullptr;
  int32_t operator[](long i) const { CHECK(v && i >= 0 && i < (long)v->size(), i, v ? (long)v->size() : -1); return (*v)[i]; }
  explicit operator bool() const { return v != nullptr; }
};
#include PACKED_SOURCE

// ---- the checks -----------------------------------------------------------------------------------
static void check_seq(const PkArgs& a, const Seq& q) {
  CHECK(q.qs >= 0 && q.qlen >= 0 && (int64_t)q.qs + q.qlen <= a.Tq, q.qs, q.qlen, a.Tq);
  CHECK(q.ks >= 0 && q.klen >= 0 && (int64_t)q.ks + q.klen <= a.Tk, q.ks, q.klen, a.Tk);
  for (int tok : {0, q.qlen / 2, q.qlen - 1})
    if (tok >= 0 && tok < q.qlen) CHECK(vis_of(a, q, tok) >= 0 && vis_of(a, q, tok) <= q.klen, tok);
}
typedef std::set<std::pair<long, long>> Pairs;
template <bool KEYS> static void tiles(PkArgs a, int per, const std::vector<int>& lens, const std::vector<int>& from, bool sane) {
  const int T = KEYS ? a.Tk : a.Tq;
  a.per = per;
  a.tiles = T / per + a.S + 1;                               // the grid
  Pairs seen;
  std::vector<int> outside(T, 0);
  long surplus = 0;
  for (int t = 0; t < a.tiles; ++t) {
    Seq q[64]; int i[64], over[64], total[64]; bool ok[64];
    wave([&](int l) { ok[l] = find_tile<KEYS>(a, t, q[l], i[l], over[l], total[l]); });
    for (int l = 1; l < 64; ++l) CHECK(ok[l] == ok[0] && (!ok[0] || (i[l] == i[0] && q[l].qs == q[0].qs && q[l].ks == q[0].ks)), l, t);
    if (ok[0]) {
      check_seq(a, q[0]);
      const int n = KEYS ? q[0].klen : q[0].qlen;
      CHECK(i[0] >= 0 && (int64_t)i[0] * per < n, i[0], per, n);
      if (sane) CHECK(seen.insert({KEYS ? q[0].ks : q[0].qs, i[0]}).second, t);
    } else {
      ++surplus;
      CHECK(over[0] >= 0 && over[0] < a.tiles - total[0], over[0], total[0], a.tiles);
      for (unsigned w = 0; w < 4; ++w) {                     // four waves a block
        threadIdx.x = 64 * w; blockDim.x = 256;
        if constexpr (KEYS) outside_rows(a.cu_k, a.S, a.Tk, over[0], a.tiles - total[0], [&](int r) { CHECK(r >= 0 && r < T, r, T); ++outside[r]; });
        else outside_rows(a.cu_q, a.S, a.Tq, over[0], a.tiles - total[0], [&](int r) { CHECK(r >= 0 && r < T, r, T); ++outside[r]; });
        blockDim.x = 64;
      }
    }
  }
  if (!sane) return;
  size_t want = 0;
  std::vector<int> inside(T, 0);
  for (size_t s = 0; s < lens.size(); ++s) {
    want += (lens[s] + per - 1) / per;
    for (int b = 0; b * per < lens[s]; ++b) CHECK(seen.count({from[s], b}), s, b);
    for (int r = from[s]; r < from[s + 1]; ++r) inside[r] = 1;
  }
  CHECK(seen.size() == want, seen.size(), want);             // each block once, and rows outside all sequences by one wave each
  CHECK(surplus > 0);
  for (int r = 0; r < T; ++r) CHECK(outside[r] == 1 - inside[r], r, outside[r], inside[r]);
}
static void chunks(PkArgs a, const evlm_packed_attn_args& x, const std::vector<int>& lq, const std::vector<int>& lk, const std::vector<int>& from, bool sane) {
  a.per = 32 / a.gp;
  a.want = pk_want(&x, a.gp);
  if (!a.want) a.want = 7;                                   // (a size that does not ask for chunks: the arithmetic all the same)
  const long slots = (long)a.want + x.Tq / (32 / a.gp) + x.S;
  if (pk_want(&x, a.gp)) CHECK(slots == pk_chunk_slots(&x, a.gp), slots);
  a.tiles = (int)slots;
  Pairs seen;
  long keys = 0;
  for (long g = 0; g < slots; ++g) {
    Chunk c[64]; bool ok[64];
    wave([&](int l) { ok[l] = find_chunk<false>(a, (int)g, c[l]); });
    if (!ok[0]) continue;
    check_seq(a, c[0].q);
    CHECK(c[0].tile >= 0 && (int64_t)c[0].tile * a.per < c[0].q.qlen, c[0].tile);
    CHECK(c[0].keys >= PK_CHUNK && c[0].keys % 32 == 0 && c[0].chunk >= 0 && c[0].chunk < c[0].n, c[0].chunk, c[0].n);
    CHECK(c[0].first >= 0 && c[0].first + c[0].chunk == g, c[0].first, c[0].chunk, g);            // the part it writes
    keys = c[0].keys;
    if (sane) CHECK(seen.insert({((long)c[0].q.qs << 20) + c[0].tile, c[0].chunk}).second, g);
  }
  for (int t = 0; t < a.Tq; t += 1 + a.Tq / 40) {
    Chunk c[64]; bool ok[64];
    wave([&](int l) { ok[l] = find_chunk<true>(a, t, c[l]); });
    if (!ok[0]) continue;
    check_seq(a, c[0].q);
    CHECK(t >= c[0].q.qs && t - c[0].q.qs < c[0].q.qlen && c[0].tile == (t - c[0].q.qs) / a.per, t);
    for (int h = 0; h < a.gp; ++h) CHECK((t - c[0].q.qs - c[0].tile * a.per) * a.gp + h < 32, t, h);
    if (sane) CHECK(c[0].first >= 0 && c[0].first + c[0].n <= slots, c[0].first, c[0].n, slots);      // the parts it reads
  }
  if (!sane) return;
  size_t want = 0;
  for (size_t s = 0; s < lq.size(); ++s)
    want += (size_t)((lq[s] + a.per - 1) / a.per) * (keys ? std::max(1l, (lk[s] + keys - 1) / keys) : 0);
  CHECK(seen.size() == want, seen.size(), want);
}

int main(int argc, char** argv) {
  const unsigned seed = argc > 1 ? std::atoi(argv[1]) : 0;
  const int rounds = argc > 2 ? std::atoi(argv[2]) : 40;
  std::mt19937 rng(seed);
  auto any = [&](long lo, long hi) { return std::uniform_int_distribution<long>(lo, hi)(rng); };
  for (int round = 0; round < rounds; ++round) {
    const bool sane = round % 2 == 0;
    const int S = (int)(round % 7 == 0 ? any(65, 300) : any(0, 12)), G = (int)any(1, 40), longest = S > 64 ? 6 : (int)any(1, 90);
    std::vector<int> lq, lk, room;
    for (int s = 0; s < S; ++s) {
      lq.push_back((int)(any(0, 5) ? any(0, longest) : 0));
      lk.push_back((int)(any(0, 5) ? any(0, round % 3 ? 3 * longest : 30 * longest) : 0));
    }
    const bool slots = any(0, 1);
    for (int n : lk) room.push_back(n + (slots ? (int)any(0, 9) : 0));
    auto starts = [&](const std::vector<int>& n) { std::vector<int32_t> c{(int)any(0, 5)}; for (int x : n) c.push_back(c.back() + x); return c; };
    std::vector<int32_t> cu_q = starts(lq), cu_k = starts(room), lens(lk.begin(), lk.end());
    evlm_packed_attn_args x = {};
    x.S = S; x.Tq = cu_q.back() + (int)any(0, 9); x.Tk = cu_k.back() + (int)any(0, 9); x.H = G; x.Hkv = 1; x.dh = 64; x.dtype = EVLM_BF16;
    if (!sane)
      for (auto* v : {&cu_q, &cu_k, &lens})
        for (auto& e : *v) {
          const long k = any(0, 9);
          if (k == 0) e = INT32_MIN; else if (k == 1) e = INT32_MAX; else if (k < 6) e = (int32_t)any(-50, x.Tk + 50); else if (k == 6) e = (int32_t)any(INT32_MIN, INT32_MAX);
        }
    PkArgs a = {};
    a.Tq = x.Tq; a.Tk = x.Tk; a.S = S; a.H = G; a.G = G; a.dh = 64; a.causal = (int)any(0, 1);
    a.gp = largest_divisor(G, 32); a.chunks = G / a.gp; a.units = a.chunks; a.inv_gp = (65536u + a.gp - 1) / a.gp;
    a.cu_q.v = &cu_q; a.cu_k.v = &cu_k;
    if (slots) a.k_lens.v = &lens;
    std::snprintf(told, sizeof(told), "seed %u round %d: %d sequences, %d queries, %d keys, group %d, causal %d, %s", seed, round, S, x.Tq, x.Tk, G, a.causal, sane ? "consistent" : "not");
    for (unsigned r = 0; r < 256; ++r) CHECK((r * a.inv_gp >> 16) == r / a.gp, r, a.gp);
    std::vector<int> q0(cu_q.begin(), cu_q.end()), k0(cu_k.begin(), cu_k.end());
    if (sane && slots) {                                     // (keys behind the filled part of a slot are in no block: theirs is the slot)
      tiles<false>(a, 128 / a.gp, lq, q0, true);
      tiles<true>(a, 32, lk, k0, true);
    } else {
      tiles<false>(a, 32 / a.gp, lq, q0, sane);
      tiles<true>(a, any(0, 1) ? 32 : 256, lk, k0, sane);
    }
    chunks(a, x, lq, lk, q0, sane);
  }
  std::printf("ok\n");
  return 0;
}
