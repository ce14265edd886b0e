// ce_gemm.cuh -- the matrix products of linear_ce.cu on the tensor cores: one
// kernel, C = sum over pairs of parts (i, j) of A_i B_j^T in f32, whose epilogue
// reduces a tile of logits to a maximum and a sum for each row, turns it into
// the gradient's G, or stores it.
//
// Two CTAs (a cluster) make a 256 x 256 tile with tcgen05.mma.cta_group::2: each
// holds half of A's and half of B's rows in shared memory and 128 x 256 sums in
// TMEM, so an SM reads 64 bytes of operands a clock at full rate where a CTA
// alone would read 96 and be bound by shared memory.  384 threads:
//   warp 0      TMA: K-blocks of 64 into a ring of 6 stages (128-byte swizzle,
//               zeros outside of the matrix).  An operand's rows run along K
//               (K-major) or across it (MN-major: G and x in dw, w in dx), so
//               nothing is transposed in memory;
//   warp 1      the leader's issues the MMAs, 4 to a K-block;
//   warps 4-11  epilogue, from one of two accumulators while the other fills.
// Every wait is bounded (1 s); where one runs out, the kernel records it, the
// roles leave their loops, copies in flight are waited for and TMEM is freed.
// Sums that miss a product are never handed on: the epilogue's own wait for them
// runs out, and what it has to store becomes NaN.
#pragma once

#include <cuda.h>

#include "nk_head.cuh"

namespace nk {
namespace ce {

constexpr int TM = 256, TN = 256, BK = 64;  // a pair's tile
constexpr int STAGES = 6;
constexpr int OPERAND_BYTES = 128 * BK * 2;          // a CTA's half of A or B
constexpr int STAGE_BYTES = 2 * OPERAND_BYTES;
constexpr int THREADS = 384, EPI_WARPS = 8;
constexpr int BOX_BYTES = 4096;  // GRAD, STORE: 32 rows of 128 bytes on their way out
constexpr int smem_bytes(bool boxes) { return STAGES * STAGE_BYTES + (boxes ? EPI_WARPS * BOX_BYTES : 0) + 1024 + 256; }
constexpr uint32_t TMEM_COLS = 512;
constexpr uint64_t WAIT_NS = 1000000000ull;
constexpr uint64_t TEST_WAIT_NS = 2000000ull;  // of calls under nk_linear_ce_withhold
// The tensor cores cut, not round, when they add to a sum, so a chain of products
// is off by half a step of the sum for each 16 of K, all one way (measured: 1.7e-8
// of a logit each).  Where f32 results depend on it (the loss; f32 gradients, an f32
// dw of 16-bit rows too), and in 16-bit gradients of very many terms, a chain ends
// after a few K-blocks and the epilogue's registers add the chains up.
// (f32: the low parts' products come first, as one chain: they are 2^-11 of the sum.)
// Logits of f32 rows get the shortest chains: an error of the logit is one of p, and a
// sure token's gradient is 1 - p.  (8192 x 256 x 2369, gradients from exact statistics:
// 2.7e-6 off, 5.7e-6 with chains of 4, for 2.5% of the time of 4096 x 768 x 16384.)
constexpr int chain_blocks(bool f32_logits) { return f32_logits ? 2 : 8; }
constexpr int REGS_FEW = 64, REGS_MANY = 216;  // 4 warps and 8 of 32: within 384 * 168

// What the first kernel of a call finds out, for the others (the workspace's head).
struct Head {
    uint32_t err;
    uint32_t live;     // rows that count
    float weight_max;  // the largest |row_weight| of them
    uint32_t x_max, w_max;  // f32: bits of the largest finite |x| and |w|
};

enum Mode { ROWS = 0, GRAD = 1, STORE = 2 };

struct Gemm {
    int M, N, K;  // at most: which of M and K is the number of rows that count (Head::live), `live_dim` says
    int live_dim; // 0: M, 1: K, 2: neither
    int segs;     // products of parts, small ones first
    uint32_t sa, sb;  // bit s: which part of A and B product s takes
    int b_row0;       // the first row of B (K-major) or the first of its K (MN-major)
    uint32_t idesc;
    int m_fast, group_m;  // tile order: m first within groups of group_m row blocks, else n first
    int splits, kps;      // K-blocks (of all products) a piece of a tile takes
    Head *head;
    // f32: exact powers of two that undo the parts' scales, one for each row of x and of w
    // (ROWS), or one for each matrix (nullable in STORE)
    const float *x_scale, *w_scale;
    int n_valid;                     // columns of C that exist
    // ROWS: part [2 tile + half][Mp] of (maximum, sum), zt [M]
    float2 *part;
    int64_t part_ld;
    float *zt;
    const uint32_t *target;  // of each row that counts
    // GRAD: G's parts go out through Products::c
    const float2 *stats;     // of each row that counts
    const float *weight;     // of each row that counts
    int col0;                // the piece's first token
    float g_scale;
    // STORE
    float *acc;              // [split][rows][ld_acc]
    int64_t ld_acc, acc_split;
    int add, keep;           // add what is there; keep the sum there (else it goes to out)
    void *out;
    int64_t out_ld, out_row0;
    int out_dtype, out_add;
    const uint32_t *out_row; // nullable: where a row goes
    float out_scale;         // times Head::weight_max (and the scales)
};

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ uint64_t globaltimer() {
    uint64_t t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// One lane of the warp.  (A branch on it tells the compiler that what follows is
// one thread's; a branch on the lane's number does not, and costs the MMAs and copies
// that it guards about 100 cycles each.)
__device__ __forceinline__ bool elect() {
    uint32_t r;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(r));
    return r != 0;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t at_leader(uint32_t addr) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ void pair_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint64_t limit) {
    if (mbar_try(bar, parity)) return true;
    const uint64_t t0 = globaltimer();
    while (!mbar_try(bar, parity))
        if (globaltimer() - t0 > limit) return false;
    return true;
}

// A box of a matrix into this CTA's shared memory, counted on the leader's barrier.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, uint32_t leader_bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"((uint64_t)map), "r"(leader_bar), "r"(x), "r"(y)
        : "memory");
}

// Shared memory descriptors, 128-byte swizzle.  K-major: rows of 128 bytes (64
// elements of K), groups of 8 rows 1024 bytes apart; 16 elements of K are 32
// bytes on.  MN-major: boxes of 64 rows of K, each 128 bytes (64 elements of M or
// N): groups of 8 K are 1024 bytes apart, the next 64 of M or N a box (8192
// bytes); 16 of K are 2048 bytes on.
template <bool MN>
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3FFFu) | ((uint64_t)(MN ? 8192 >> 4 : 1) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
template <bool MN>
constexpr uint64_t k_step() {
    return (MN ? 2048 : 32) >> 4;
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p; }"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate));
}
// Arrives on the barrier at this place in both CTAs when all MMAs so far are done.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
        ::"r"(bar), "h"((unsigned short)3)
        : "memory");
}

// 32 columns of this warp's 32 rows; every lane takes part.  The values are there
// after tmem_wait, which has to name them: the compiler knows of no other order.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
          "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]),
          "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]),
          "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]),
          "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
        : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void tmem_wait(float *v) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}

// Where the chain from K-block k of an item on ends; `low`: K-blocks of the low parts.
template <int CHAIN>
__device__ __forceinline__ int chain_end(int k, int k1, int low) {
    return min(k1, k < low ? low : k + CHAIN);
}

// A tile's piece: its row and column block and its K-blocks.
struct Item {
    int tm, tn, split, k0, k1;
};

struct Walk {
    int mt, nt, total, kblocks, items, M, K;
    __device__ __forceinline__ Walk() : mt(0), nt(0), total(0), kblocks(0), items(0), M(0), K(0) {}
    __device__ __forceinline__ Walk(const Gemm &p, int live) {
        M = p.live_dim == 0 ? live : p.M;
        K = p.live_dim == 1 ? live : p.K;
        mt = (M + TM - 1) / TM;
        nt = (p.N + TN - 1) / TN;
        kblocks = (K + BK - 1) / BK;
        total = kblocks * p.segs;
        items = mt * nt * p.splits;
    }
    __device__ __forceinline__ Item at(const Gemm &p, int i) const {
        Item it;
        int t = i / p.splits;
        it.split = i - t * p.splits;
        it.k0 = min(total, it.split * p.kps);
        it.k1 = min(total, it.k0 + p.kps);
        if (p.m_fast) {
            const int per = p.group_m * nt, g = t / per;
            t -= g * per;
            const int rows = min(p.group_m, mt - g * p.group_m);
            it.tn = t / rows;
            it.tm = g * p.group_m + t - it.tn * rows;
        } else {
            it.tm = t / nt;
            it.tn = t - it.tm * nt;
        }
        return it;
    }
};

// How the items of two products share the pairs, so that a last round of the one is
// filled up with the other (dx 128 tiles of 256 K-blocks and dw 256 of 128 over 74
// pairs: 896 K-blocks to a pair where each alone leaves 512 + 512).  The first's go
// round robin; the second's to the pairs that have less, until all reach one level.
// Pairs run the second's items in one order, so that neighbours share their operands.
struct Deal {
    int items[2], pairs, more;  // `more`: pairs that have one item of the first product more than the rest
    int n[2];                   // of the second, for those pairs and for the rest
    __host__ __device__ Deal(int items0, int cost0, int items1, int cost1, int pairs_) : pairs(pairs_) {
        items[0] = items0;
        items[1] = items1;
        more = items0 % pairs;
        const int q = items0 / pairs;
        const long high = (long)(q + 1) * cost0, low = (long)q * cost0;
        n[0] = n[1] = 0;
        // The least level that has room for all; from one step of a class to the next.
        long level = ((long)items0 * cost0 + (long)items1 * cost1 + pairs - 1) / pairs;
        for (;;) {
            n[0] = level > high ? (int)((level - high) / cost1) : 0;
            n[1] = level > low ? (int)((level - low) / cost1) : 0;
            if ((long)more * n[0] + (long)(pairs - more) * n[1] >= items1) break;
            const long a = high + (long)(n[0] + 1) * cost1, b = low + (long)(n[1] + 1) * cost1;
            level = more && a < b ? a : b;
        }
        if (n[1] < n[0]) n[1] = n[0];
    }
    // Item number i of a pair: the product and the item of it; false where there is none.
    __host__ __device__ bool at(int pair, int i, int &which, int &item) const {
        const int mine = items[0] / pairs + (pair < more);
        which = i >= mine;
        if (!which) {
            item = i * pairs + pair;
            return true;
        }
        const int s = i - mine, extra = n[1] - n[0];  // (first the pairs that have less of the first product)
        if (pair < more) {
            if (s >= n[0]) return false;
            item = extra * (pairs - more) + s * pairs + pair;
        } else {
            if (s >= n[1]) return false;
            item = s < extra ? s * (pairs - more) + pair - more : extra * (pairs - more) + (s - extra) * pairs + pair;
        }
        return item < items[1];
    }
};

// What a launch computes: one product (the first), or in STORE two: dx, whose A is
// K-major, and dw, whose A is MN-major (either can be empty).
struct Products {
    alignas(64) CUtensorMap a[2][2], b[2][2], c[2];  // [product][part]; c: G's parts
    Gemm g[2];
    int cost[2];  // K-blocks of an item, and what its end takes
    uint64_t wait_ns;  // bound of every wait
    int withhold;      // test control: the last K-block of the first pair's first item is never brought
};

// ---------------------------------------------------------------- epilogues
// A warp has 32 rows (lane = row) and 128 columns of its CTA's 128 x 256 sums, which
// come 64 at a time, from TMEM or (LONG) from the registers that added them up.
// `row` counts rows that count (or tokens, in dw), `col` is the first column; every
// lane of a warp calls some().

// The maximum and the sum of exponentials of 128 logits of a row.  The sum is kept
// relative to a whole power of two near the first maximum: an exponential is then one
// fma and one ex2, and 2^100 of room means that the power hardly ever moves.
template <bool SCALED>
struct RowsEpilogue {
    const Gemm &p;
    const int row, live, col, slot;
    const uint32_t t;
    float m = -INFINITY, s = 0.0f, power = -INFINITY;
    __device__ __forceinline__ RowsEpilogue(const Gemm &g, int r, int n, int c, int at)
        : p(g), row(r), live(n), col(c), slot(at), t(r < n ? g.target[r] : NO_TOKEN) {}
    __device__ __forceinline__ void some(int c, float *v) {
        if (col + c >= p.n_valid) return;  // warp-uniform
        if (SCALED) {
            // (Scales of each row of x and w; those of w run on to whole tiles.  Their
            // product first: it leaves f32's range only where the logit does.)
            const float xs = row < live ? p.x_scale[row] : 1.0f;
            const float4 *ws = reinterpret_cast<const float4 *>(p.w_scale + col + c);
#pragma unroll
            for (int j = 0; j < 64; j += 4) {
                const float4 q = ws[j / 4];
                v[j] *= xs * q.x, v[j + 1] *= xs * q.y, v[j + 2] *= xs * q.z, v[j + 3] *= xs * q.w;
            }
        }
        if (col + c + 64 > p.n_valid)
#pragma unroll
            for (int j = 0; j < 64; ++j)
                if (col + c + j >= p.n_valid) v[j] = -INFINITY;
        if (t - (uint32_t)(col + c) < 64u)
#pragma unroll
            for (int j = 0; j < 64; ++j)
                if (t == (uint32_t)(col + c + j)) p.zt[row] = v[j];
        float top[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int j = 4; j < 64; ++j) top[j & 3] = fmaxf(top[j & 3], v[j]);
        m = fmaxf(m, fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])));
        const float want = m * LOG2E;
        if (want > power + 60.0f) {
            const float now = rintf(want);
            s *= ex2(power - now);  // (s is 0 before the first)
            power = now;
        }
        const float base = power == -INFINITY ? 0.0f : power;
        float a[4] = {};
#pragma unroll
        for (int j = 0; j < 64; ++j) a[j & 3] += ex2(fmaf(v[j], LOG2E, -base));
        s += (a[0] + a[1]) + (a[2] + a[3]);
    }
    __device__ __forceinline__ void end() {
        // Relative to the maximum from here on (with the same log2(e), whose error so cancels).
        if (m > -INFINITY) s *= ex2(fmaf(-m, LOG2E, power));
        if (row < live) p.part[(int64_t)slot * p.part_ld + row] = make_float2(m, s);
    }
};

__device__ __forceinline__ void store_box(const CUtensorMap *map, uint32_t from, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"((uint64_t)map), "r"(from),
                 "r"(x), "r"(y)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// G = weight (exp(z - m - log s) - [t]) of 128 logits of a row; zeros where there
// is no row or no token, since the products that follow read whole blocks.  64
// columns of the warp's 32 rows go out at once, as a box whose 16-byte places are
// swizzled by row (a lane writing its own row to memory takes a line for each 16
// bytes: 6.3 us a tile where the box takes 3.7).
template <class T, bool SCALED>
struct GradEpilogue {
    const Gemm &p;
    const CUtensorMap *const map0, *const map1;
    uint8_t *const box;
    const bool in;
    const int row0, col;
    const uint32_t t;
    const float2 st;
    const float h, base, hp;
    __device__ __forceinline__ GradEpilogue(const Gemm &q, const CUtensorMap *a, const CUtensorMap *b, uint8_t *to, int row, int live,
                                            int c)
        : p(q), map0(a), map1(b), box(to), in(row < live), row0(row - (int)(threadIdx.x & 31)), col(c),
          t(in ? q.target[row] - (uint32_t)q.col0 : NO_TOKEN), st(in ? q.stats[row] : make_float2(0.0f, 0.0f)),
          h(in ? weight() : 0.0f), base(st.x * LOG2E),
          hp(h * ex2(-fmaf(st.y, LOG2E, fmaf(st.x, LOG2E, -base)))) {}
    __device__ __forceinline__ float weight() const { return p.weight[row0 + (int)(threadIdx.x & 31)] / p.head->weight_max * p.g_scale; }
    __device__ __forceinline__ void some(int c, float *v) {
        const int lane = threadIdx.x & 31;
        if (SCALED) {
            const float scale = *p.x_scale * *p.w_scale;
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = ex2(((v[j] * scale - st.x) - st.y) * LOG2E) * h;
        } else {
            // (One fma, whose error is of the distance to the maximum: what base lacks of it, and
            // log s, are in hp.  With both in base, p was 8e-4 off at logits of 10^4.)
#pragma unroll
            for (int j = 0; j < 64; ++j) v[j] = ex2(fmaf(v[j], LOG2E, -base)) * hp;
        }
        if (!in || col + c + 64 > p.n_valid)
#pragma unroll
            for (int j = 0; j < 64; ++j)
                if (!in || col + c + j >= p.n_valid) v[j] = 0.0f;
        if (t - (uint32_t)(col + c) < 64u) {
            const float own = SCALED ? h : weight();  // (read again: a register more and the sums spill)
#pragma unroll
            for (int j = 0; j < 64; ++j)
                if (t == (uint32_t)(col + c + j)) v[j] -= own;
        }
#pragma unroll
        for (int part = 0; part < (SCALED ? 2 : 1); ++part) {
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");  // the box is free again
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 64; j += 8) {
                uint4 q;
                T *o = reinterpret_cast<T *>(&q);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    o[e] = from_f32<T>(v[j + e]);
                    if (SCALED) v[j + e] -= to_f32(o[e]);
                }
                *reinterpret_cast<uint4 *>(box + lane * 128 + (((j >> 3) ^ (lane & 7)) << 4)) = q;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) store_box(part ? map1 : map0, smem_u32(box), col + c, row0);
        }
    }
    __device__ __forceinline__ void end() const {}
};

// N neighbouring elements of an output row at o, which is a multiple of their size.
template <class T, int N, bool ADD>
__device__ __forceinline__ void store_out(T *o, const float (&v)[N]) {
    struct __align__(N * sizeof(T)) Some {
        T e[N];
    } q;
    if (ADD) q = *reinterpret_cast<const Some *>(o);
#pragma unroll
    for (int i = 0; i < N; ++i) q.e[i] = from_f32<T>(ADD ? v[i] + to_f32(q.e[i]) : v[i]);
    *reinterpret_cast<Some *>(o) = q;
}

__device__ __forceinline__ float out_factor(const Gemm &p) {
    if (p.head->err) return NAN;  // a wait in a product before this one ran out
    float f = p.out_scale * p.head->weight_max;
    if (p.x_scale) f *= *p.x_scale;
    if (p.w_scale) f *= *p.w_scale;
    return f;
}

// Sums to memory, 32 columns of the warp's rows at a time, through its box so that 8
// lanes write 128 bytes of a row; a lane's 8 rows (lane / 8 + 4 i) are taken from the
// box together and go out together (one after the other they took 12 us a tile where
// the MMAs of 1536 of K take 6.5).  F32: the output is always f32 (f32 inputs).
template <bool F32>
struct StoreEpilogue {
    const Gemm &p;
    float *const box;
    const bool any;  // K has anything: else the accumulator holds nothing
    const int col, row0, rows;  // first column; the warp's first row; how many of its 32 rows exist
    const float factor;
    float *const acc;
    int64_t out[8];  // where the lane's rows start in the output, in elements
    __device__ __forceinline__ StoreEpilogue(const Gemm &g, uint8_t *to, bool has, int r, int n, int c, int split, float f)
        : p(g), box((float *)to), any(has), col(c), row0(r - (int)(threadIdx.x & 31)), rows(n - row0), factor(f),
          acc(g.acc ? g.acc + (int64_t)split * g.acc_split + (int64_t)(r - (int)(threadIdx.x & 31) + ((threadIdx.x & 31) >> 3)) * g.ld_acc + c
                    : nullptr) {
#pragma unroll
        for (int i = 0; i < 8; ++i) out[i] = p.keep ? 0 : start(((int)(threadIdx.x & 31) >> 3) + 4 * i);
    }
    // Where the warp's row r starts in the output (beyond the last: as the last).
    __device__ __forceinline__ int64_t start(int r) const {
        const int row = row0 + max(min(r, rows - 1), -row0);
        return (p.out_row ? (int64_t)p.out_row[row] : row + p.out_row0) * p.out_ld;
    }
    __device__ __forceinline__ float *at(int r, int c) const { return box + r * 32 + ((c >> 2) ^ (r & 7)) * 4 + (c & 3); }
    // 32 columns from c on of the warp's rows, the lane's share of which is x.
    template <class T, bool ADD>
    __device__ __forceinline__ void write(const float4 (&x)[8], int c) const {
        const int lane = threadIdx.x & 31, left = p.n_valid - (col + c);
        T *const o = (T *)p.out + col + c;
        if (left >= 32 && (((uintptr_t)p.out | (uintptr_t)(p.out_ld * sizeof(T))) & (4 * sizeof(T) - 1)) == 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if ((lane >> 3) + 4 * i < rows) {
                    const float v[4] = {x[i].x * factor, x[i].y * factor, x[i].z * factor, x[i].w * factor};
                    store_out<T, 4, ADD>(o + out[i] + (lane & 7) * 4, v);
                }
            return;
        }
        // Rows that start anywhere: through the box again, a row at a time, an element to
        // a lane.  (Pairs from 4 bytes on, with the odd ends apart, took 24 us a tile where
        // this takes 14 and the aligned form 7.6, at 256 of K.)
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float4 *>(at((lane >> 3) + 4 * i, (lane & 7) * 4)) = make_float4(x[i].x * factor, x[i].y * factor, x[i].z * factor, x[i].w * factor);
        __syncwarp();
        if (lane < left) {
#pragma unroll 8
            for (int r = 0; r < min(rows, 32); ++r) {
                const float v[1] = {*at(r, lane)};
                store_out<T, 1, ADD>(o + start(r) + lane, v);
            }
        }
        __syncwarp();
    }
    template <class T>
    __device__ __forceinline__ void write(const float4 (&x)[8], int c) const {
        if (p.out_add)
            write<T, true>(x, c);
        else
            write<T, false>(x, c);
    }
    __device__ __forceinline__ void some(int c0, float *v) {
        const int lane = threadIdx.x & 31;
#pragma unroll
        for (int h = 0; h < 64; h += 32) {
            const int c = c0 + h;
            if (col + c >= p.n_valid) return;  // warp-uniform
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; j += 4)
                *reinterpret_cast<float4 *>(box + lane * 32 + ((j >> 2) ^ (lane & 7)) * 4) =
                    any ? make_float4(v[h + j], v[h + j + 1], v[h + j + 2], v[h + j + 3]) : make_float4(0.f, 0.f, 0.f, 0.f);
            __syncwarp();
            const int cc = c + (lane & 7) * 4;
            float4 x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = (lane >> 3) + 4 * i;
                x[i] = *reinterpret_cast<const float4 *>(box + r * 32 + ((lane & 7) ^ (r & 7)) * 4);
            }
            float *a = acc + cc;
            if (p.add)
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if ((lane >> 3) + 4 * i < rows) {
                        const float4 q = *reinterpret_cast<const float4 *>(a + (int64_t)(4 * i) * p.ld_acc);
                        x[i].x += q.x, x[i].y += q.y, x[i].z += q.z, x[i].w += q.w;
                    }
            if (p.keep) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if ((lane >> 3) + 4 * i < rows) *reinterpret_cast<float4 *>(a + (int64_t)(4 * i) * p.ld_acc) = x[i];
            } else if (F32 || p.out_dtype == 0) {
                write<float>(x, c);
            } else if (p.out_dtype == 1) {
                write<__half>(x, c);
            } else {
                write<__nv_bfloat16>(x, c);
            }
        }
    }
    __device__ __forceinline__ void end() const {}
};

// ---------------------------------------------------------------- the kernel
template <int N>
__device__ __forceinline__ void more_registers() {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void fewer_registers() {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// T: the parts' type.  SCALED: f32 inputs, taken as two scaled f16 parts.  LONG:
// chains of a few K-blocks, added up in registers.
template <int MODE, class T, bool SCALED, bool LONG>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1) gemm_k(const __grid_constant__ Products ps) {
    constexpr bool B_MN = MODE == STORE;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *boxes = smem + STAGES * STAGE_BYTES;
    uint64_t *bars = (uint64_t *)(boxes + (MODE == ROWS ? 0 : EPI_WARPS * BOX_BYTES));
    uint32_t *tmem_slot = (uint32_t *)(bars + 2 * STAGES + 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, n_pairs = gridDim.x >> 1;
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[STAGES]);
    const uint32_t acc_full0 = smem_u32(&bars[2 * STAGES]), acc_empty0 = smem_u32(&bars[2 * STAGES + 2]);

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(full0 + 8 * s, 1);
            mbar_init(empty0 + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full0 + 8 * b, 1);
            mbar_init(acc_empty0 + 8 * b, 2 * EPI_WARPS);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&ps.a[0][0]) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&ps.b[0][0]) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    pair_sync();  // both CTAs' barriers exist before either signals the other
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = *tmem_slot;
    pdl_trigger();
    pdl_wait();  // (what the kernels before left is read from here on)
    Head *const head = ps.g[0].head;
    const int live = (int)head->live;
    const Walk walk0(ps.g[0], live), walk1 = MODE == STORE ? Walk(ps.g[1], live) : Walk();
    const Deal deal(walk0.items, ps.cost[0], walk1.items, ps.cost[1], n_pairs);
    // The pair's item number i.
    int which = 0, item = 0;
    auto next = [&](int i) { return deal.at(pair, i, which, item); };
    // (Gradients of 16-bit rows: as exact as their G makes them.  8192 x 1024 x 32768 with an f32 dw
    // takes 1290 us with one chain, off by up to 2e-5, 1310 with chains of 32, 1400 of 16, 1420 of 8.)
    constexpr int CHAIN = MODE == STORE && !SCALED ? 16 : chain_blocks(SCALED && MODE != STORE);
    // A wait that ran out ends the role that waited; the others' waits on it run out too.
    auto give_up = [&](uint32_t code) { atomicExch(&head->err, code); };

    if (warp < 4) {
        if constexpr (LONG) fewer_registers<REGS_FEW>();
        if (warp == 0) {
            const bool one = elect();
            int stage = 0, issued = 0;
            uint32_t phase = 0;
            bool fine = true;
            const uint32_t leader_full = at_leader(full0), ring = smem_u32(smem);
            for (int i = 0; fine && next(i); ++i) {
                const Gemm &p = ps.g[which];
                const Walk walk = MODE == STORE && which ? walk1 : walk0;
                const Item it = walk.at(p, item);
                const int m0 = it.tm * TM + (int)rank * 128, n0 = it.tn * TN + (int)rank * 128;
                int seg = it.k0 / max(1, walk.kblocks), x = (it.k0 - seg * walk.kblocks) * BK;
                const bool hold = ps.withhold && pair == 0 && i == 0;
                for (int k = it.k0; k < it.k1 - hold; ++k) {
                    fine = mbar_wait(empty0 + 8 * stage, phase ^ 1, ps.wait_ns);
                    if (!__all_sync(0xffffffffu, fine)) {
                        if (one) give_up(201);
                        fine = false;
                        break;
                    }
                    if (one) {
                        const uint32_t to = ring + stage * STAGE_BYTES, bar = leader_full + 8 * stage;
                        const CUtensorMap *ma = &ps.a[which][(p.sa >> seg) & 1], *mb = &ps.b[which][(p.sb >> seg) & 1];
                        if (rank == 0) mbar_expect_tx(full0 + 8 * stage, 2 * STAGE_BYTES);
                        if (MODE == STORE && which) {
                            tma_load(to, ma, bar, m0, x);
                            tma_load(to + OPERAND_BYTES / 2, ma, bar, m0 + 64, x);
                        } else {
                            tma_load(to, ma, bar, x, m0);
                        }
                        if (B_MN) {
                            tma_load(to + OPERAND_BYTES, mb, bar, n0, p.b_row0 + x);
                            tma_load(to + OPERAND_BYTES + OPERAND_BYTES / 2, mb, bar, n0 + 64, p.b_row0 + x);
                        } else {
                            tma_load(to + OPERAND_BYTES, mb, bar, x, p.b_row0 + n0);
                        }
                    }
                    ++issued;
                    if (++stage == STAGES) stage = 0, phase ^= 1;
                    x += BK;
                    if (x >= walk.K) x = 0, ++seg;
                }
                if (hold) fine = false;
            }
            // A stage's copies have landed once its MMAs are done: wait for the last
            // ones, so that none writes into shared memory after the CTA's end.
            stage = issued % STAGES;
            phase = (uint32_t)(issued / STAGES) & 1;
            for (int i = 0; i < min(issued, STAGES); ++i) {
                // (From the oldest of the last STAGES on: its number is issued - STAGES + i.)
                const int at = issued < STAGES ? i : (stage + i) % STAGES;
                const uint32_t ph = issued < STAGES ? 0u : (stage + i < STAGES ? phase ^ 1 : phase);
                mbar_wait(empty0 + 8 * at, ph, ps.wait_ns);
            }
        } else if (warp == 1 && rank == 0) {
            const bool one = elect();
            int stage = 0, n = 0;
            uint32_t phase = 0;
            bool fine = true;
            const uint64_t db0 = smem_desc<B_MN>(smem_u32(smem) + OPERAND_BYTES);
            for (int i = 0; fine && next(i); ++i) {
                const Gemm &p = ps.g[which];
                const Walk walk = MODE == STORE && which ? walk1 : walk0;
                const Item it = walk.at(p, item);
                const int low = SCALED ? 2 * walk.kblocks : 0;
                const bool a_mn = MODE == STORE && which;
                const uint64_t da0 = a_mn ? smem_desc<true>(smem_u32(smem)) : smem_desc<false>(smem_u32(smem));
                const uint64_t a_step = a_mn ? k_step<true>() : k_step<false>();
                const uint32_t idesc = p.idesc;
                for (int k = it.k0;;) {
                    const int end = LONG ? chain_end<CHAIN>(k, it.k1, low) : it.k1, b = n & 1;
                    fine = mbar_wait(acc_empty0 + 8 * b, (uint32_t)(((n >> 1) & 1) ^ 1), ps.wait_ns);
                    if (!__all_sync(0xffffffffu, fine)) {
                        if (one) give_up(202);
                        fine = false;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t d = tmem + b * TN;
                    uint32_t more = 0;
                    for (; k < end; ++k) {
                        fine = mbar_wait(full0 + 8 * stage, phase, ps.wait_ns);
                        if (!__all_sync(0xffffffffu, fine)) {
                            if (one) give_up(203);
                            fine = false;
                            break;
                        }
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        if (one) {
                            const uint64_t da = da0 + (uint64_t)(stage * (STAGE_BYTES >> 4)), db = db0 + (uint64_t)(stage * (STAGE_BYTES >> 4));
#pragma unroll
                            for (int kk = 0; kk < BK / 16; ++kk)
                                mma(d, da + kk * a_step, db + kk * k_step<B_MN>(), idesc, kk ? 1u : more);
                            mma_commit(empty0 + 8 * stage);
                        }
                        more = 1;
                        if (++stage == STAGES) stage = 0, phase ^= 1;
                    }
                    if (!fine) break;  // (not committed: the epilogue takes whole sums only)
                    if (one) mma_commit(acc_full0 + 8 * b);
                    ++n;
                    if (k >= it.k1) break;
                }
            }
        }
    } else {
        if constexpr (LONG) more_registers<REGS_MANY>();
        const int q = warp & 3, half = (warp - 4) >> 2;
        const uint32_t leader_empty = at_leader(acc_empty0);
        const float factor0 = MODE == STORE ? out_factor(ps.g[0]) : 1.0f, factor1 = MODE == STORE ? out_factor(ps.g[1]) : 1.0f;
        int n = 0;
        // The next accumulator: wait for it, or give it back.
        auto take = [&]() -> bool {
            const bool ok = mbar_wait(acc_full0 + 8 * (n & 1), (uint32_t)((n >> 1) & 1), ps.wait_ns);
            if (!__all_sync(0xffffffffu, ok)) {  // (every lane is here: the loads that follow are the warp's)
                if (lane == 0) give_up(204);
                return false;
            }
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            return true;
        };
        auto give = [&] {
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0)
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(leader_empty + 8 * (n & 1))
                             : "memory");
            ++n;
        };
        const uint32_t mine = tmem + ((uint32_t)(q * 32) << 16) + half * 128;
        bool fine = true;
        for (int i = 0; next(i); ++i) {
            // (After a wait that ran out, sums become NaN: this item's and those that follow.)
            if (MODE != STORE && !fine) break;
            const Gemm &p = ps.g[which];
            const Walk walk = MODE == STORE && which ? walk1 : walk0;
            const Item it = walk.at(p, item);
            const int low = SCALED ? 2 * walk.kblocks : 0;
            const int row = it.tm * TM + (int)rank * 128 + q * 32 + lane, col = it.tn * TN + half * 128;
            auto whole = [&](auto &&e) {
                if (MODE == STORE && !fine) return;
                if constexpr (LONG) {
                    float sum[128];
                    fine = take();
                    if (!fine) return;
#pragma unroll
                    for (int c = 0; c < 128; c += 32) tmem_ld32(mine + (n & 1) * TN + c, sum + c);
                    tmem_wait<128>(sum);
                    give();
#pragma unroll 1
                    for (int k = chain_end<CHAIN>(it.k0, it.k1, low); k < it.k1; k = chain_end<CHAIN>(k, it.k1, low)) {
                        fine = take();
                        if (!fine) return;
#pragma unroll
                        for (int c = 0; c < 128; c += 64) {
                            float v[64];
                            tmem_ld32(mine + (n & 1) * TN + c, v);
                            tmem_ld32(mine + (n & 1) * TN + c + 32, v + 32);
                            tmem_wait<64>(v);
#pragma unroll
                            for (int j = 0; j < 64; j += 2) {
                                const float2 t = add2(make_float2(sum[c + j], sum[c + j + 1]), make_float2(v[j], v[j + 1]));
                                sum[c + j] = t.x;
                                sum[c + j + 1] = t.y;
                            }
                        }
                        give();
                    }
                    e.some(0, sum);
                    e.some(64, sum + 64);
                } else {
                    fine = take();
                    if (!fine) return;
#pragma unroll 1
                    for (int c = 0; c < 128; c += 64) {
                        float v[64];
                        __syncwarp();
                        tmem_ld32(mine + (n & 1) * TN + c, v);
                        tmem_ld32(mine + (n & 1) * TN + c + 32, v + 32);
                        tmem_wait<64>(v);
                        e.some(c, v);
                    }
                    give();
                }
                e.end();
            };
            if constexpr (MODE == ROWS)
                whole(RowsEpilogue<SCALED>(p, row, live, col, 2 * it.tn + half));
            else if constexpr (MODE == GRAD)
                whole(GradEpilogue<T, SCALED>(p, &ps.c[0], &ps.c[1], boxes + (warp - 4) * BOX_BYTES, row, live, col));
            else {
                StoreEpilogue<SCALED> e(p, boxes + (warp - 4) * BOX_BYTES, it.k1 > it.k0, row, walk.M, col, it.split, which ? factor1 : factor0);
                whole(e);
                if (!fine) {
                    float v[64];
#pragma unroll
                    for (int j = 0; j < 64; ++j) v[j] = NAN;
                    e.some(0, v);
                    e.some(64, v);
                }
            }
        }
        if (MODE == GRAD && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    pair_sync();  // the other CTA is done with this one's barriers and TMEM
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

}  // namespace ce
}  // namespace nk
