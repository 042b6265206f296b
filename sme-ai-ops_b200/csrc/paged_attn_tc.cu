// paged_attn_tc.cu -- attention of new tokens over a paged key/value cache for
// requests that bring many rows (a prompt, a chunk of one), on the sm_100a
// tensor cores.
//
// The mathematics is that of paged_attn.cu, on tiles of 256 packed rows (two
// halves of 128, the MMA's M) and blocks of 128 keys:
//   S_t = Q_t K^T      tcgen05.mma, both operands in shared memory, fp32 in TMEM
//   P_t = 2^(c (S_t - m)) in registers: a thread owns a row, so its maximum and
//                      sum need no exchange; P replaces S in TMEM as 16-bit pairs
//   O_t += P_t V       tcgen05.mma with P read from TMEM, O fp32 in TMEM
// The running maximum is only raised when it grows by more than 2^8 (P then
// stays below 2^8, or 2^15 with half's bias), so O, which has to be rescaled
// when it is, is touched rarely; the thread that owns the row does it.  P is
// rounded once to the cache's type, the only type that an MMA takes beside its
// values: the result is off by 1.4 times the rounding of the exact one (2.3e-3
// against 1.7e-3 in bf16).  The remainder as a second P would be half as many
// MMAs again in a kernel that they bound.
//
// Warp roles (12 warps, one CTA an SM):
//   warps 0-3, 4-7   softmax of half 0 and half 1 (208 registers a thread)
//   warps 8-9        load: keys and values a page (or 64 rows of one) at a time
//                    by TMA into the 128-byte-swizzled layout the MMA reads;
//                    queries, values of a block that the request ends in (whose
//                    other rows must be zeros, not what the page held before),
//                    and everything when pages are smaller than 8 tokens with
//                    16-byte cp.async
//   warp 10          allocates TMEM; one lane issues the MMAs
// A tile with rows for one half only gives both halves the same rows and deals
// them the blocks in turn; half 1's maximum, sum and context go through shared
// memory to half 0 at the end (24 requests of 64 rows over 300 to 4096 keys,
// 8 key heads of 128: 81.5 -> 77 us; 69 now, with a tile's cost on the line).
// While one half's softmax runs, the tensor core works for the other: in issue
// order PV_0(j), QK_0(j+1), PV_1(j), QK_1(j+1).  At 128 elements a block
// takes 4 x 128^3 multiply-adds for the tensor core (2048 cycles at its rate)
// and 2 x 128 x 128 exponentials (2048 cycles at 16 a cycle): the two are
// nearly in balance, and both halves' softmax has to hide behind the MMAs.
// Measured: 2 x 2048 new tokens over 8k keys, 32 query and 8 key heads of 128,
// 428 us = 1071 TFLOP/s, 3500 cycles a block; back to back for seconds 482 to
// 498 us (the board's power limit lowers the clock).  What bounds it: QK reads shared
// memory at its full 128 bytes a cycle, and the copies of keys and values have
// to fit beside that.  Slower when tried: two threads a row (16 softmax warps,
// 523 us), a part of the exponentials as polynomials on the FMA pipe (434 to
// 553 us), scores in two lots of 64 keys so that softmax and products of a half
// overlap (505 us: QK 64 keys wide reads the queries twice as often); handing P
// over in two parts and taking the exponentials before the block's maximum is
// known changed nothing.
//
// Every wait is bounded by wall time; on expiry the kernel records
// kDevErrTimeout, all roles stop, copies and MMAs in flight are drained (they
// always end, so that wait has a bound of its own, whatever the limit that ran
// out), TMEM is freed and the kernel returns.  No multicast.
#include <cuda.h>
#include <string.h>

#include "paged_attn.cuh"
#include "tcgen05.cuh"

namespace smeai {

namespace {

constexpr int kTR = 256;             // packed rows a tile
constexpr int kKB = 128;             // keys a block
constexpr int kThreads = 384;
constexpr int kLoadWarp0 = 8, kLoadWarps = 2, kMmaWarp = 10;
constexpr int kTmaMinPage = 8;       // tokens
constexpr uint64_t kDrainNs = 1000000000ull;
// 384 threads x 168 registers at launch = 256 x 208 + 128 x 88
constexpr int kAtom = 128 * 128;     // 128 rows x 128 bytes
constexpr int kTmemCols = 512;       // S0 S1 (128 columns each), O0 O1 (up to 128 each)
constexpr float kNegInf = -INFINITY;

template <int DP>
struct Tc {
  static constexpr int kCb = DP / 64;              // 64-element column blocks
  static constexpr int kItem = kCb * kAtom;        // bytes of 128 rows
  static constexpr int kSlots = DP == 128 ? 5 : 8; // ring of key and value blocks: 160 or 128 KB
  static constexpr int kQBytes = 2 * kItem;
  static constexpr size_t kSmem = 1024 + (size_t)kQBytes + (size_t)kSlots * kItem + 256 + 1024;
};

struct TcSmem {
  uint8_t* q;
  uint8_t* ring;
  uint64_t *full, *empty;            // per slot: both load warps (their threads, without TMA); one commit
  uint64_t* q_empty;                 // commit: the tile's last QK has read the queries
  uint64_t *s_full, *p_full, *o_full;  // per half: commit; 4 warps; commit
  uint64_t *x_full, *x_done;         // one half's rows on both: 4 warps have left half 1's results; 4 have taken them
  int64_t* items;                    // per load warp: ring items it has announced
  float2* x_ml;                      // [128] half 1's maximum and sum; its context lies where the queries were
  uint64_t* drain;
  uint32_t* tmem;
  int* abort;
};

template <int DP>
__device__ __forceinline__ TcSmem carve(uint8_t* base) {
  TcSmem m;
  uint8_t* p = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(base) + 1023) & ~(uintptr_t)1023);
  m.q = p;
  m.ring = p + Tc<DP>::kQBytes;
  uint64_t* b = reinterpret_cast<uint64_t*>(m.ring + (size_t)Tc<DP>::kSlots * Tc<DP>::kItem);
  m.full = b;
  m.empty = b + 8;
  m.q_empty = b + 16;
  m.s_full = b + 17;
  m.p_full = b + 19;
  m.o_full = b + 21;
  m.drain = b + 23;
  m.tmem = reinterpret_cast<uint32_t*>(b + 24);
  m.abort = reinterpret_cast<int*>(b + 25);
  m.x_full = b + 26;
  m.x_done = b + 27;
  m.items = reinterpret_cast<int64_t*>(b + 28);
  m.x_ml = reinterpret_cast<float2*>(b + 32);
  return m;
}

// Bounded wait that also gives up once another role has.  With a limit below
// the clock's step a wait that is not over at once has run out.
__device__ __forceinline__ bool wait_or_abort(const TcSmem& m, uint64_t* bar, unsigned parity, unsigned* err,
                                              uint64_t limit_ns) {
  if (mbar_test_wait(bar, parity)) return true;
  const uint64_t t0 = global_timer_ns();
  const int tries = limit_ns < 1024 ? 0 : 32;
  for (;;) {
    for (int i = 0; i < tries; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (*reinterpret_cast<volatile int*>(m.abort)) return false;
    if (global_timer_ns() - t0 > limit_ns) {
      *reinterpret_cast<volatile int*>(m.abort) = 1;
      raise_device_error(err, kDevErrTimeout);
      return false;
    }
  }
}
__device__ __forceinline__ bool wait_warp(const TcSmem& m, uint64_t* bar, unsigned parity, unsigned* err,
                                          uint64_t limit_ns) {
  return __all_sync(0xffffffffu, wait_or_abort(m, bar, parity, err, limit_ns));
}

// True in one lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
}

// D[tmem] (+)= A[tmem] * B[smem desc]^T, 16-bit inputs, fp32 accumulate.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}"
      :
      : "r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(0), "r"(0), "r"(0), "r"(0)
      : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
      "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]),
      "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]),
      "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
          addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Arrives on `bar` when this thread's cp.async copies so far have landed (the
// barrier's count includes this arrival).
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// Keeps uses of a load's registers behind the wait before it.
__device__ __forceinline__ void pin32(float* v) {
  asm volatile(""
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                 "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
                 "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                 "+f"(v[30]), "+f"(v[31]));
}

// Instruction descriptor: M = 128, fp32 accumulator, fp16 (0) or bf16 (1)
// operands; bit 16: operand B has its N dimension contiguous (the values, [key][element]).
__host__ __device__ constexpr uint32_t idesc(bool bf16, int n, bool b_n_major) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_n_major ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}

// One CTA's stretch of a tile: key blocks kb0 .. kb0 + n of it; half t works on
// the first cnt[t] of them (causal: the lower rows see fewer keys), or, with
// rows for half 0 only, on every second one.
struct Stretch {
  int kb0, n, cnt[2];
  bool last;   // reaches the tile's end
  bool dual;   // both halves hold half 0's rows
};
__device__ __forceinline__ Stretch stretch(const AttnParams& p, const AttnPos& w, int64_t left) {
  Stretch s;
  s.kb0 = w.kb;
  const int to_end = w.nkb - w.kb;
  s.n = left < to_end ? (int)left : to_end;
  s.last = s.n == to_end;
  const bool two = w.rt * kTR + 128 < w.r.rows;
  s.cnt[0] = s.n;
  s.cnt[1] = two ? s.n : 0;
  if (two) s.cnt[0] = max(0, min(s.n, attn_blocks<128, kKB>(p, w.r, 2 * w.rt) - w.kb));
  s.dual = !two && s.n > 1;
  if (s.dual) {
    s.cnt[0] = (s.n + 1) / 2;
    s.cnt[1] = s.n / 2;
  }
  return s;
}

// A TMA load of box rows x 64 elements at (element, token, head, page).
__device__ __forceinline__ void tma_load_box(uint32_t dst, const CUtensorMap* map, int x, int token, int head, int page,
                                             uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(map), "r"(x), "r"(token), "r"(head), "r"(page), "r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint64_t* bar, unsigned bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(bytes) : "memory");
}

// The cache as the TMA sees it; box_log2: log2 of the rows of a box.
struct TcMaps {
  CUtensorMap k, v;
  int box_log2;
};

template <typename T, int DP, bool kTma>
__global__ void __launch_bounds__(kThreads, 1) paged_attn_tc_kernel(const AttnParams p, const __grid_constant__ TcMaps maps,
                                                                    uint64_t limit_ns) {
  using C = Tc<DP>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ AttnShare share;
  __shared__ int64_t warp_sum[3 * kThreads / 32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const TcSmem m = carve<DP>(smem_raw);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 8; ++i) {
      mbar_init(&m.full[i], kTma ? kLoadWarps : 32 * kLoadWarps);
      mbar_init(&m.empty[i], 1);
    }
    mbar_init(m.q_empty, 1);
    for (int t = 0; t < 2; ++t) {
      mbar_init(&m.s_full[t], 1);
      mbar_init(&m.p_full[t], 4);
      mbar_init(&m.o_full[t], 1);
    }
    mbar_init(m.x_full, 4);
    mbar_init(m.x_done, 4);
    mbar_init(m.drain, 1);
    *m.abort = 0;
    mbar_fence_init();
  }
  if (warp == kMmaWarp) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(m.tmem)),
                 "r"(kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (kTma && threadIdx.x < 2)
    asm volatile("prefetch.tensormap [%0];" ::"l"(threadIdx.x ? &maps.v : &maps.k) : "memory");
  pdl_wait();
  attn_share<kTR, kKB, kThreads>(p, &share, warp_sum);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *m.tmem;
  const int64_t units = share.u1 - share.u0;
  if (threadIdx.x == 0) attn_no_parts(p);

  if (units <= 0) {
    // nothing to do
  } else if (warp >= kLoadWarp0) {
    // one instruction for the whole warpgroup: load, MMA and idle warp
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < kLoadWarp0 + kLoadWarps) {
      // ---------------- load: this warp's 64 rows of every item
      const int lw = warp - kLoadWarp0;
      AttnPos w;
      attn_open<kTR, kKB>(p, share, w);
      const int page_mask = (1 << p.kv.page_log2) - 1;
      int64_t left = units;
      int slot = 0;                  // of the next item
      unsigned round = 1;            // parity of the wait for its being free
      int64_t items = 0;             // announced: arrived on `full`
      bool ok = true;
      unsigned q_round = 1;          // parity of the wait for the queries' place
      // cp.async: 4 rows at a time, 8 lanes take 128 contiguous bytes of a row.
      // Row i * 4 + sub of 32 lands in atom row row0 + that row, its 16-byte
      // chunks XORed with the row mod 8 -- which is sub, or sub + 4 for odd i.
      const int sub = lane >> 3, col = lane & 7;
      const uint32_t even = (uint32_t)(sub * 128 + ((col ^ sub) << 4)), odd = (uint32_t)(sub * 128 + ((col ^ (sub + 4)) << 4));
      int bytes[C::kCb];                             // 0 past the head's elements
#pragma unroll
      for (int cb = 0; cb < C::kCb; ++cb) bytes[cb] = cb * 64 + col * 8 < p.kv.dim ? 16 : 0;
      // off: byte offset of row row0 + lane, -1: zeros
      auto copy_rows = [&](uint8_t* dst, const char* src, int64_t off, int row0) {
        const uint32_t d = smem_addr(dst) + row0 * 128;
        const char* from = src + col * 16;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int64_t o = __shfl_sync(0xffffffffu, off, i * 4 + sub);
#pragma unroll
          for (int cb = 0; cb < C::kCb; ++cb) {
            const int n = o >= 0 ? bytes[cb] : 0;
            cp_async16(d + i * 512 + cb * kAtom + (i & 1 ? odd : even), n ? from + o + cb * 128 : src, n);
          }
        }
      };
      auto acquire = [&]() {   // the first round over the ring finds it free
        return wait_warp(m, &m.empty[slot], round, p.err, limit_ns);
      };
      auto next_slot = [&]() {
        ++items;
        if (++slot == C::kSlots) {
          slot = 0;
          round ^= 1;
        }
      };
      // copies of this warp so far have landed: announce them
      auto landed = [&]() {
        cp_async_commit();
        cp_async_wait<0>();
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.full[slot]);
      };
      const int box_rows = 1 << maps.box_log2, boxes = 64 >> maps.box_log2;
      const int my_box = lane / C::kCb, my_cb = lane % C::kCb;
      while (left > 0 && ok) {
        const Stretch s = stretch(p, w, left);
        const int32_t* table = p.table + (int64_t)w.b * p.ld_table;
        auto page_of = [&](int key) {   // -1: no such key, or a bad page
          if (key >= w.r.kv) return -1;
          const int page = table[key >> p.kv.page_log2];
          if (page >= 0 && page < p.kv.n_pages) return page;
          raise_device_error(p.err, kDevErrBadIndex);
          return -1;
        };
        auto row_off = [&](int key) {
          const int page = page_of(key);
          return page < 0 ? (int64_t)-1
                          : page * p.kv.page_bytes + (key & page_mask) * p.kv.token_bytes + w.h * p.kv.head_bytes;
        };
        auto copy_item = [&](const char* src, int key0) {
          uint8_t* dst = m.ring + (size_t)slot * C::kItem;
          copy_rows(dst, src, row_off(key0 + lane), lw * 64);
          copy_rows(dst, src, row_off(key0 + 32 + lane), lw * 64 + 32);
        };
        // this lane's box of a TMA item: its first key's page, -1 when it has none
        const bool has_box = kTma && my_box < boxes;
        int page = has_box ? page_of(s.kb0 * kKB + lw * 64 + my_box * box_rows) : -1;
        auto load_item = [&](const CUtensorMap* map, int key0) {
          const unsigned n = __popc(__ballot_sync(0xffffffffu, page >= 0));
          if (lane == 0) mbar_expect_tx(&m.full[slot], n * box_rows * 128);
          __syncwarp();
          if (page >= 0) {
            const int row = my_box * box_rows;
            tma_load_box(smem_addr(m.ring) + slot * C::kItem + my_cb * kAtom + (lw * 64 + row) * 128, map, my_cb * 64,
                         (key0 + row) & page_mask, w.h, page, &m.full[slot]);
          }
        };
        for (int b = 0; b < s.n && ok; ++b) {
          const int key0 = (s.kb0 + b) * kKB + lw * 64;
          // the next block's pages are looked up before this block's waits
          const int next_page = has_box && b + 1 < s.n ? page_of(key0 + kKB + my_box * box_rows) : -1;
          if (!(ok = acquire())) break;
          if (kTma) load_item(&maps.k, key0);
          if (b == 0) {
            // the tile's queries land with its first keys, once the last tile's are read
            if (!(ok = wait_warp(m, m.q_empty, q_round, p.err, limit_ns))) {
              if (lane == 0) mbar_arrive(&m.full[slot]);
              ++items;
              break;
            }
            q_round ^= 1;
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
              const int row = w.rt * kTR + (s.dual ? 0 : lw * 128) + q4 * 32 + lane;
              int64_t off = -1;
              if (row < w.r.rows) {
                const int tok = row / p.group, hd = w.h * p.group + row % p.group;
                off = (int64_t)(w.r.q0 + tok) * p.ld_q + (int64_t)hd * p.kv.dim * 2;
              }
              copy_rows(m.q + lw * C::kItem, p.q, off, q4 * 32);
            }
          }
          if (!kTma) {
            copy_item(p.kv.k, key0);
            cp_async_arrive(&m.full[slot]);
          } else if (b == 0) {
            landed();
          } else if (lane == 0) {
            mbar_arrive(&m.full[slot]);
          }
          next_slot();
          if (!(ok = acquire())) break;
          if (!kTma) {
            copy_item(p.kv.v, key0);
            cp_async_arrive(&m.full[slot]);
          } else if ((s.kb0 + b + 1) * kKB > w.r.kv) {
            copy_item(p.kv.v, key0);
            landed();
          } else {
            load_item(&maps.v, key0);
            if (lane == 0) mbar_arrive(&m.full[slot]);
          }
          next_slot();
          page = next_page;
        }
        left -= s.n;
        if (left > 0) attn_next_tile<kTR, kKB>(p, w);
      }
      cp_async_commit();
      cp_async_wait<0>();
      if (lane == 0) m.items[lw] = items;
    } else if (warp == kMmaWarp) {
      // ---------------- issue the MMAs
      // The whole warp walks and waits, so that descriptors stay in uniform
      // registers; one elected lane issues.
      constexpr uint32_t kQk = idesc(Num<T>::kIsBf16, kKB, false), kPv = idesc(Num<T>::kIsBf16, DP, true);
      AttnPos w;
      attn_open<kTR, kKB>(p, share, w);
      int64_t left = units;
      unsigned it = 0;             // the stretch's first item: K, V of block b are items it + 2b, it + 2b + 1
      unsigned xc = 0;             // stretches with one half's rows on both
      unsigned pc0 = 0, pc1 = 0;   // softmax results taken, per half
      bool ok = true;
      const uint64_t q_desc = smem_desc(m.q, 16, 1024, kLayoutSw128);
      const uint64_t k_desc = smem_desc(m.ring, 16, 1024, kLayoutSw128);
      const uint64_t v_desc = smem_desc(m.ring, kAtom, 1024, kLayoutSw128);
      auto qk = [&](int t, int at) {
        if (elect_one()) {
          const uint64_t a0 = q_desc + (uint64_t)t * (C::kItem >> 4), b0 = k_desc + (uint64_t)at * (C::kItem >> 4);
#pragma unroll
          for (int ks = 0; ks < DP / 16; ++ks) {
            const uint64_t step = (uint64_t)(((ks >> 2) * kAtom + (ks & 3) * 32) >> 4);
            tc_mma_f16(tmem + t * 128, a0 + step, b0 + step, kQk, ks > 0);
          }
          tc_commit(&m.s_full[t]);
        }
        __syncwarp();
      };
      auto pv = [&](int t, int at, bool first) {
        if (elect_one()) {
          const uint64_t b0 = v_desc + (uint64_t)at * (C::kItem >> 4);
#pragma unroll
          for (int ks = 0; ks < kKB / 16; ++ks)
            tc_mma_f16_ts(tmem + 256 + t * 128, tmem + t * 128 + ks * 8, b0 + (uint64_t)((ks * 2048) >> 4), kPv,
                          !(first && ks == 0));
        }
        __syncwarp();
      };
      auto commit = [&](uint64_t* bar) {
        if (elect_one()) tc_commit(bar);
        __syncwarp();
      };
      auto tc_release = [&](int at) { commit(&m.empty[at]); };
      // the slot of an item, landed (ok says whether)
      auto take = [&](unsigned item) {
        const unsigned at = item % C::kSlots;
        ok = wait_warp(m, &m.full[at], (item / C::kSlots) & 1, p.err, limit_ns);
        fence_async_smem();      // cp.async's copies are ordinary writes; the MMA reads through the async proxy
        return (int)at;
      };
      auto weights = [&](int t) {
        unsigned& pc = t ? pc1 : pc0;
        ok = wait_warp(m, &m.p_full[t], pc & 1, p.err, limit_ns);
        ++pc;
        tc_fence_after();
        return ok;
      };
      while (left > 0) {
        const Stretch s = stretch(p, w, left);
        if (s.dual) {
          for (int b = 0; b < 2 && ok; ++b) {
            const int ik = take(it + 2 * b);
            if (!ok) break;
            tc_fence_after();
            qk(b, ik);
            tc_release(ik);
          }
          for (int b = 0; b < s.n && ok; ++b) {
            const int t = b & 1, iv = take(it + 2 * b + 1);
            if (!ok || !weights(t)) break;
            pv(t, iv, b < 2);
            tc_release(iv);
            if (b + 2 < s.n) {
              const int ik = take(it + 2 * b + 4);
              if (!ok) break;
              qk(t, ik);
              tc_release(ik);
            } else {
              commit(&m.o_full[t]);
            }
          }
          // the queries' place is free when half 0 has taken half 1's context from it
          if (!ok || !(ok = wait_warp(m, m.x_done, xc & 1, p.err, limit_ns))) break;
          ++xc;
          if (lane == 0) mbar_arrive(m.q_empty);
          __syncwarp();
        } else {
          const int k0 = take(it);
          if (!ok) break;
          tc_fence_after();
          if (s.cnt[0] > 0) qk(0, k0);
          if (s.cnt[1] > 0) qk(1, k0);
          tc_release(k0);
          if (s.n == 1) commit(m.q_empty);
          for (int b = 0; b < s.n; ++b) {
            const int iv = take(it + 2 * b + 1);
            if (!ok) break;
            const bool more = b + 1 < s.n;
            int ik = 0;
            if (more) {
              ik = take(it + 2 * b + 2);
              if (!ok) break;
            }
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              if (b >= s.cnt[t]) continue;
              if (!weights(t)) break;
              pv(t, iv, b == 0);
              if (b + 1 < s.cnt[t]) qk(t, ik);
              else commit(&m.o_full[t]);
            }
            if (!ok) break;
            tc_release(iv);
            if (more) tc_release(ik);
            if (b + 2 == s.n) commit(m.q_empty);
          }
        }
        if (!ok) break;
        it += 2 * s.n;
        left -= s.n;
        if (left > 0) attn_next_tile<kTR, kKB>(p, w);
      }
      // everything issued has finished before TMEM is freed
      commit(m.drain);
      mbar_wait_bounded(m.drain, 0, kDrainNs);
    }
    __syncwarp();
  } else {
    // ---------------- softmax of half t, one row a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp >> 2, r = (warp & 3) * 32 + lane;
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_col = tmem + lanes + t * 128, o_col = tmem + lanes + 256 + t * 128;
    AttnPos w;
    attn_open<kTR, kKB>(p, share, w);
    int64_t left = units;
    unsigned sc = 0, oc = 0, xc = 0;
    bool ok = true;
    while (left > 0 && ok) {
      const Stretch s = stretch(p, w, left);
      const int row_in = s.dual ? r : t * 128 + r;      // of the tile
      const int row = w.rt * kTR + row_in;
      const bool live = row < w.r.rows;
      const int lim = live ? min(w.r.kv, attn_limit(p, w.r, row)) : 0;
      const int lim_all = min(w.r.kv, attn_limit(p, w.r, row - r));
      const bool dead = row - lane >= w.r.rows;
      // plus: what the multiply-add adds; of a far row, or before the first maximum, so large that any score is above
      constexpr float kOpens = 3.4e38f;
      float mx = kNegInf, plus = kOpens, l = 0.f;
      const int cnt = s.cnt[t];
      for (int b = 0; b < cnt; ++b) {
        if (!(ok = wait_warp(m, &m.s_full[t], sc & 1, p.err, limit_ns))) break;
        ++sc;
        if (dead) {   // none of the warp's rows exists: whatever P holds there, nobody reads
          if (lane == 0) mbar_arrive(&m.p_full[t]);
          continue;
        }
        tc_fence_after();
        float v[128];
#pragma unroll
        for (int i = 0; i < 4; ++i) tmem_ld32(s_col + i * 32, v + i * 32);
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 4; ++i) pin32(v + i * 32);
        const int key0 = (s.kb0 + (s.dual ? 2 * b + t : b)) * kKB;
        if (key0 + kKB > lim_all) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (key0 + i >= lim) v[i] = kNegInf;
        }
        float top[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) top[i] = v[i];
#pragma unroll
        for (int i = 8; i < 120; i += 16)
#pragma unroll
          for (int k = 0; k < 8; ++k) top[k] = fmaxf(fmaxf(top[k], v[i + k]), v[i + 8 + k]);
#pragma unroll
        for (int k = 0; k < 8; ++k) top[k] = fmaxf(top[k], v[120 + k]);
        const float mn = fmaxf(fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])),
                               fmaxf(fmaxf(top[4], top[5]), fmaxf(top[6], top[7])));
        const bool open = fmaf(mn, p.scale_log2, plus) > Num<T>::kBias + kRaise;
        float add = plus;
        if (__any_sync(0xffffffffu, open)) {
          const bool raise = open && mn > mx;
          const float f = raise ? exp2_fast((mx - mn) * p.scale_log2) : 1.f;   // mx = -inf: 0
          if (raise) {
            mx = mn;
            plus = row_base(mn, p.scale_log2) == mn ? base_offset<T>(mn, p.scale_log2) : kOpens;
          }
          add = plus;
          l *= f;
          if (b > 0) {
#pragma unroll 1
            for (int i = 0; i < DP / 32; ++i) {
              float o[32];
              tmem_ld32(o_col + i * 32, o);
              tmem_ld_wait();
              pin32(o);
#pragma unroll
              for (int k = 0; k < 32; ++k) o[k] *= f;
              tmem_st32(o_col + i * 32, o);
            }
          }
          const bool far = plus == kOpens && mx > kNegInf;
          if (__any_sync(0xffffffffu, far)) {
            const float less = far ? mx : 0.f;
            if (far) add = Num<T>::kBias;
#pragma unroll
            for (int i = 0; i < 128; ++i) v[i] -= less;
          }
        }
        const uint64_t c2 = pack_f32x2(p.scale_log2, p.scale_log2), add2 = pack_f32x2(add, add);
        uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t w16[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const uint64_t x = fma_f32x2(pack_f32x2(v[i * 32 + 2 * k], v[i * 32 + 2 * k + 1]), c2, add2);
            const float e0 = exp2_fast(__uint_as_float((uint32_t)x)), e1 = exp2_fast(__uint_as_float((uint32_t)(x >> 32)));
            sum2[k & 1] = add_f32x2(sum2[k & 1], pack_f32x2(e0, e1));
            w16[k] = Num<T>::pack(e0, e1);
          }
          tmem_st16(s_col + i * 16, w16);
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&m.p_full[t]);
        sum2[0] = add_f32x2(sum2[0], sum2[1]);
        l += __uint_as_float((uint32_t)sum2[0]) + __uint_as_float((uint32_t)(sum2[0] >> 32));
      }
      if (!ok) break;
      if (cnt > 0) {
        if (!(ok = wait_warp(m, &m.o_full[t], oc & 1, p.err, limit_ns))) break;
        ++oc;
        tc_fence_after();
      }
      // one half's rows on both: half 1 leaves its results, context as
      // [4 columns][row] where the queries were (every QK of the stretch has
      // ended with its last product), half 0 adds them to its own
      float4* const x_o = reinterpret_cast<float4*>(m.q) + r;
      float f0 = 1.f, f1 = 0.f;
      if (s.dual && t == 1) {
        if (!dead) {
          m.x_ml[r] = make_float2(mx, l);
#pragma unroll 1
          for (int i = 0; i < DP / 32; ++i) {
            float o[32];
            tmem_ld32(o_col + i * 32, o);
            tmem_ld_wait();
            pin32(o);
#pragma unroll
            for (int k = 0; k < 8; ++k) x_o[(i * 8 + k) * 128] = make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(m.x_full);
      } else if (s.dual) {
        if (!(ok = wait_warp(m, m.x_full, xc & 1, p.err, limit_ns))) break;
        ++xc;
        const float2 ml = dead ? make_float2(kNegInf, 0.f) : m.x_ml[r];
        const float top = fmaxf(mx, ml.x);
        f0 = mx == kNegInf ? 0.f : exp2_fast((mx - top) * p.scale_log2);
        f1 = ml.x == kNegInf ? 0.f : exp2_fast((ml.x - top) * p.scale_log2);
        l = fmaf(ml.y, f1, l * f0);
        mx = top;
      }
      const bool mine = live && !(s.dual && t == 1);
      const bool whole = s.last && s.kb0 == 0;
      const int64_t slot = 2 * (int64_t)blockIdx.x + (s.kb0 == 0 ? 1 : 0);
      const float inv = row_scale(l);
      const int tok = row / p.group, hd = w.h * p.group + row % p.group;
      char* dst = p.out + (int64_t)(w.r.q0 + tok) * p.ld_out + (int64_t)hd * p.kv.dim * 2;
      float* part = p.part_o + (slot * kTR + row_in) * DP;
      if (cnt > 0 && !dead && !(s.dual && t == 1)) {
#pragma unroll 1
        for (int i = 0; i < DP / 32; ++i) {
          float o[32];
          tmem_ld32(o_col + i * 32, o);
          tmem_ld_wait();
          pin32(o);
          if (s.dual) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float4 x = x_o[(i * 8 + k) * 128];
              o[4 * k] = fmaf(x.x, f1, o[4 * k] * f0);
              o[4 * k + 1] = fmaf(x.y, f1, o[4 * k + 1] * f0);
              o[4 * k + 2] = fmaf(x.z, f1, o[4 * k + 2] * f0);
              o[4 * k + 3] = fmaf(x.w, f1, o[4 * k + 3] * f0);
            }
          }
          if (mine && whole) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
              if (i * 32 + k * 8 < p.kv.dim)
                *reinterpret_cast<uint4*>(dst + (i * 32 + k * 8) * 2) =
                    make_uint4(pack_mean<T>(o[8 * k] * inv, o[8 * k + 1] * inv),
                               pack_mean<T>(o[8 * k + 2] * inv, o[8 * k + 3] * inv),
                               pack_mean<T>(o[8 * k + 4] * inv, o[8 * k + 5] * inv),
                               pack_mean<T>(o[8 * k + 6] * inv, o[8 * k + 7] * inv));
          } else if (mine) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              *reinterpret_cast<float4*>(part + i * 32 + 4 * k) =
                  make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
          __syncwarp();
        }
        // the next tile's first PV, which overwrites O, waits for this warp's next arrival on p_full
        tc_fence_before();
      }
      // a half without blocks in this stretch leaves an empty sum: its context is not read
      if (!whole && mine) p.part_ml[slot * kTR + row_in] = make_float2(mx, l);
      if (s.dual && t == 0) {
        __syncwarp();
        if (lane == 0) mbar_arrive(m.x_done);
      }
      if (!whole && threadIdx.x == 0) attn_leave_part(p, w, s.kb0 == 0, s.last);
      left -= s.n;
      if (left > 0) attn_next_tile<kTR, kKB>(p, w);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (kTma && *reinterpret_cast<volatile int*>(m.abort)) {
    // A wait ran out: TMA loads that nobody waited for still write this CTA's
    // shared memory.  Their bytes complete the phases they were announced on
    // once both load warps have arrived there; the warp that left earlier is at
    // most a ring behind.
    if (threadIdx.x == 0) {
      const int64_t some = min(m.items[0], m.items[1]), all = max(m.items[0], m.items[1]);
      for (int64_t i = some; i < all; ++i) mbar_arrive(&m.full[i % C::kSlots]);
      for (int64_t i = max(all - C::kSlots, (int64_t)0); i < all; ++i)
        mbar_wait_bounded(&m.full[i % C::kSlots], (unsigned)((i / C::kSlots) & 1), kDrainNs);
    }
    __syncthreads();
  }
  pdl_trigger();
  if (warp == kMmaWarp)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static std::atomic<void*> cached{nullptr};
  void* fn = cached.load();
  if (!fn) {
    cudaDriverEntryPointQueryResult res;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &res) != cudaSuccess ||
        res != cudaDriverEntryPointSuccess) {
      cudaGetLastError();
      return nullptr;
    }
    cached.store(fn);
  }
  return reinterpret_cast<EncodeTiled>(fn);
}

// Boxes of 64 elements x up to 64 tokens of one head and page.  Elements past
// head_dim read as zeros.  Strides of dimensions of one element are never
// used, but have to be valid.
bool cache_map(const KvView& kv, const void* base, int box_rows, CUtensorMap* map) {
  const EncodeTiled encode = encode_tiled();
  if (!encode) return false;
  const cuuint64_t page = (cuuint64_t)1 << kv.page_log2;
  const cuuint64_t dims[4] = {(cuuint64_t)kv.dim, page, (cuuint64_t)kv.n_kv, (cuuint64_t)kv.n_pages};
  const cuuint64_t fill = (cuuint64_t)kv.token_bytes;
  const cuuint64_t strides[3] = {fill, kv.n_kv > 1 ? (cuuint64_t)kv.head_bytes : fill,
                                 kv.n_pages > 1 ? (cuuint64_t)kv.page_bytes : fill};
  const cuuint32_t box[4] = {64, (cuuint32_t)box_rows, 1, 1}, step[4] = {1, 1, 1, 1};
  return encode(map, kv.bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
                const_cast<void*>(base), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP, bool kTma>
int run_kernel(const AttnParams& p, const TcMaps& maps, int sms, cudaStream_t stream) {
  auto kernel = paged_attn_tc_kernel<T, DP, kTma>;
  static std::atomic<uint64_t> allowed{0};
  SMEAI_CUDA_TRY(attn_allow_smem(kernel, Tc<DP>::kSmem, allowed));
  SMEAI_CUDA_TRY(launch(kernel, dim3((unsigned)sms), dim3(kThreads), Tc<DP>::kSmem, stream, p, maps, wait_timeout_ns()));
  return kOk;
}

template <typename T, int DP>
int run_tc(AttnParams p, void* workspace, int max_kv, int sms, cudaStream_t stream) {
  const bool splits = attn_splits<kKB>(max_kv);
  attn_carve<kTR, DP>(p, splits ? workspace : nullptr, sms);
  TcMaps maps;
  memset(&maps, 0, sizeof(maps));
  maps.box_log2 = p.kv.page_log2 < 6 ? p.kv.page_log2 : 6;
  const bool tma = (1 << p.kv.page_log2) >= kTmaMinPage && cache_map(p.kv, p.kv.k, 1 << maps.box_log2, &maps.k) &&
                   cache_map(p.kv, p.kv.v, 1 << maps.box_log2, &maps.v);
  const int st = tma ? run_kernel<T, DP, true>(p, maps, sms, stream) : run_kernel<T, DP, false>(p, maps, sms, stream);
  if (st) return st;
  if (splits) SMEAI_CUDA_TRY((attn_join<T, kTR, DP>(p, sms, stream)));
  return kOk;
}

}  // namespace

size_t paged_attn_tc_workspace(int padded_dim, int max_kv, int sms) {
  if (!attn_splits<kKB>(max_kv)) return 0;
  return padded_dim == 64 ? attn_part_bytes<kTR, 64>(sms) : attn_part_bytes<kTR, 128>(sms);
}

int paged_attn_tc(const AttnParams& p, int padded_dim, void* workspace, int max_kv, int sms, cudaStream_t stream) {
  if (p.kv.bf16)
    return padded_dim == 64 ? run_tc<__nv_bfloat16, 64>(p, workspace, max_kv, sms, stream)
                            : run_tc<__nv_bfloat16, 128>(p, workspace, max_kv, sms, stream);
  return padded_dim == 64 ? run_tc<__half, 64>(p, workspace, max_kv, sms, stream)
                          : run_tc<__half, 128>(p, workspace, max_kv, sms, stream);
}

}  // namespace smeai
