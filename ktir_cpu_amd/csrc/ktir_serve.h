// What the serving operators share (rotary positions, the 8-bit key / value
// cache, attention over it): the stream and device of a launch, the checks of a
// cache and a batch, and how a kernel finds its sequence.
#pragma once
#include "ktir_common.h"

namespace ktir {

constexpr int OUT_OF_RANGE = 2;      // what a kernel leaves in the device error word

// the library's device is current while this lives
class OnDevice {
 public:
  OnDevice() {
    ok_ = hipGetDevice(&before_) == hipSuccess && (before_ == device() || hipSetDevice(device()) == hipSuccess);
  }
  ~OnDevice() {
    if (ok_ && before_ != device()) (void)hipSetDevice(before_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;
  bool ok() const { return ok_; }

 private:
  int before_ = 0;
  bool ok_ = false;
};

// The shape that ktir_kv8_rows.hip gives an attention launch.
struct KV8Shape {
  int J, MT, HW, rows, splits;         // columns in 64s, rows in 16s, heads of a workgroup, most rows of a tile
  int64_t slots, part, span;           // tiles of rows for each KV head; floats of a split's part in the workspace; most keys of a tile
};
void kv8_rows_shape(const ktir_kv8_attn_t& d, KV8Shape* s);
int kv8_rows_launch(const ktir_kv8_attn_t& d, const KV8Shape& s);
bool kv8_tile_takes(const ktir_kv8_attn_t& d, int64_t* slots);       // whether ktir_kv8_tile.hip takes it instead
int kv8_tile_launch(const ktir_kv8_attn_t& d, int64_t slots);

inline hipStream_t stream_of(uint64_t s) {
  return s == 0 ? stream() : s == KTIR_STREAM_NULL ? (hipStream_t) nullptr : (hipStream_t)s;
}

// the checks of ktir_kv8.hip, for both operators on the cache
int check_kv8(const char* what, const ktir_kv8_t& c, bool written);
int check_batch(const char* what, const ktir_kv8_batch_t& b, const ktir_kv8_t& c);
int check_rows3(const char* what, const ktir_rows3_t& r, int64_t tokens, int64_t heads, int64_t columns, bool written);
int ready(const char* what);         // whether ktir_init has run

// Rows of `width` bytes, counts by counts at steps of so many bytes.
struct Strided {
  uint64_t ptr = 0;
  int64_t width = 0, count[3] = {1, 1, 1}, step[3] = {0, 0, 0};
  uint64_t end = 0;                    // behind the last byte
  Strided() = default;
  Strided(uint64_t p, int64_t w, int64_t n0 = 1, int64_t s0 = 0, int64_t n1 = 1, int64_t s1 = 0, int64_t n2 = 1, int64_t s2 = 0)
      : ptr(p), width(w), count{n0, n1, n2}, step{s0, s1, s2}, end(p + w + (uint64_t)(n0 - 1) * s0 + (uint64_t)(n1 - 1) * s1 + (uint64_t)(n2 - 1) * s2) {}
};
inline Strided rows_of(const ktir_rows3_t& r, int64_t tokens, int64_t heads, int64_t columns, int64_t bytes) {
  return {r.ptr, columns * bytes, tokens, r.tok * bytes, heads, r.head * bytes};
}
bool apart_within(Strided a, Strided b);             // for ranges that meet
// whether they share no byte; one of them is an output, whose rows do not overlap
inline bool apart(const Strided& a, const Strided& b) { return a.ptr >= b.end || b.ptr >= a.end || apart_within(a, b); }

// what a launch on the cache reads or writes of it: codes of K and V, scales of K and V
struct CacheParts {
  Strided x[4];
  explicit CacheParts(const ktir_kv8_t& c)
      : x{{c.k, c.columns, c.pages, c.k_page, c.page, c.k_tok, c.heads, c.k_head}, {c.v, c.columns, c.pages, c.v_page, c.page, c.v_tok, c.heads, c.v_head},
          {c.k_scale, 4, c.pages, c.ks_page * 4, 1, 0, c.heads, c.ks_head * 4}, {c.v_scale, 4, c.pages, c.vs_page * 4, 1, 0, c.heads, c.vs_head * 4}} {}
};
// the table (of at least one page a sequence), offsets and lengths
struct BatchParts {
  Strided x[3];
  explicit BatchParts(const ktir_kv8_batch_t& b)
      : x{{b.table, b.width * 4, b.seqs, b.table_row * 4}, {b.q_start, (b.seqs + 1) * 4}, {b.kv_len, b.seqs * 4}} {
    if (!b.width) x[0] = x[1];
  }
  bool clear_of(const Strided& out) const { return apart(out, x[0]) && apart(out, x[1]) && apart(out, x[2]); }
};
bool same(const Strided& a, const Strided& b);       // whether they are one tensor

__device__ __forceinline__ const KTIR_G(int32_t)* ints(uint64_t p) { return (const KTIR_G(int32_t)*)p; }

// A sequence of the batch: its first new token, how many are new, how many are
// cached with them, and how many of those its table has pages for.  Offsets and
// lengths that are out of range are cut to the batch and the table.
struct Seq {
  int64_t start;
  int32_t n_new, n_kv, n_held;
};

__device__ __forceinline__ Seq seq_of(const ktir_kv8_batch_t& b, int64_t page, int64_t s, int* err) {
  const int64_t a = ints(b.q_start)[s], e = ints(b.q_start)[s + 1], n = ints(b.kv_len)[s];
  const int64_t start = a < 0 ? 0 : a < b.tokens ? a : b.tokens, end = e < start ? start : e < b.tokens ? e : b.tokens;
  const int64_t kv = n < 0 ? 0 : n, held = kv < b.width * page ? kv : b.width * page;
  if (start != a || end != e || held != n) *err = OUT_OF_RANGE;
  return {start, (int32_t)(end - start), (int32_t)kv, (int32_t)held};
}

// lane i's value in every lane
__device__ __forceinline__ float lane_of(float x, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i)); }
__device__ __forceinline__ int lane_of(int x, int i) { return __builtin_amdgcn_readlane(x, i); }
__device__ __forceinline__ int64_t lane_of(int64_t x, int i) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, i), hi = __builtin_amdgcn_readlane((uint32_t)((uint64_t)x >> 32), i);
  return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ Seq lane_of(const Seq& q, int i) {
  return {lane_of(q.start, i), lane_of(q.n_new, i), lane_of(q.n_kv, i), lane_of(q.n_held, i)};
}

// The sequence that slot `w` of a launch belongs to, and its number in it, where
// sequence s has the slots from floor(q_start[s] * mul / 2^shift) + extra * s on (so
// one of n tokens has at least floor(n * mul / 2^shift) + extra): the last s whose first
// slot is not after w, with nth < 0 if there is none.  All lanes of a wavefront
// search together, 64 sequences a step.
__device__ __forceinline__ Seq seq_of_slot(const ktir_kv8_batch_t& b, int64_t page, int64_t mul, int shift, int64_t extra, int64_t w,
                                           int64_t* s, int64_t* nth, int* err) {
  const int l = threadIdx.x & 63;
  Seq found = {0, 0, 0, 0};
  *s = 0;
  *nth = -1;
  for (int64_t base = 0; base < b.seqs; base += 64) {
    int64_t at = INT64_MAX;
    Seq q = {0, 0, 0, 0};
    if (base + l < b.seqs) {
      q = seq_of(b, page, base + l, err);
      at = (q.start * mul >> shift) + extra * (base + l);
    }
    const uint64_t below = __ballot(at <= w);
    if (!below) break;
    const int last = 63 - __builtin_clzll(below);
    found = lane_of(q, last);
    *s = base + last;
    *nth = w - lane_of(at, last);
    if (last < 63) break;
  }
  return found;
}

}  // namespace ktir
