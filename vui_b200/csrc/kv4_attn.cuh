// Attention over the paged 4-bit cache (layout: kv4_kernels.cuh).  With V and K the values that the codes stand for, row r of a
// sequence at position p and query head j:  out = sum_{i <= p} softmax_i(scale q . K_i) V_i,  K and V of kv head j / group.
#pragma once
#include "kv4_kernels.cuh"

namespace vuik {

constexpr int KA_THREADS = 128, KA_WARPS = 4;

struct Kv4AttnArgs {
    Kv4Cache c;
    const int4* entries; const int32_t* cu_units; const int32_t* cu_work; const int32_t* row_entry;
    int n, n_rows, group;
    uint32_t group_inv;                         // 2^32 / group, rounded up (group > 1)
    Kv4Split split;
    const __nv_bfloat16* q; long long q_stride;
    __nv_bfloat16* out; long long out_stride;
    float scale_log2;                          // scale * log2(e)
    bool early;                                // whether the merge lets its successor start beside it
    float* acc;                                // partial sums: (unit, column, dim), where a sequence has more than one split
    float2* ml;                                // maximum (of log2 scores) and sum: (unit, column)
};

// m16n8k16, f16 in, fp32 out: D += A B.
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// What a product of a query and a key is multiplied by to be a log2 score.  The maximum is kept of the products themselves and taken off before they
// are multiplied, so that the largest weight is 1 whatever the scores' size (as a fused multiply, scores of 2^28 would leave it at
// 2^16 or 2^-16: the maximum's rounding).  Limited to where products up to 2^38, the largest that stored keys allow, stay finite and masked
// ones -inf: products next to one another are 1e-15 apart or more, so beyond 1e26 all but the largest weigh nothing as it is.
// For a query that is not finite (`big`: the bits of its largest element) it is NaN, and so are all its weights: infinite scores have no softmax.
__device__ __forceinline__ float score_factor(float f, uint32_t big) {
    return fminf(fmaxf(f, 1e-37f), 1e26f) + (big >= 0x7f80u ? __int_as_float(0x7fffffff) : 0.f);
}

// Two scores, 15 higher, in one instruction: weights that become f16 are 2^15 times as large as the maximum's distance says, as are their sums, so
// that they keep their 11 bits down to 2^-29 of the largest and are lost below 2^-40, not 2^-14 and 2^-25: positions of little weight
// may hold large values.
__device__ __forceinline__ void lifted2(float& a, float& b, float factor_a, float factor_b) {
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%0, %1};\n\tmov.b64 y, {%2, %3};\n\tmov.b64 z, {%4, %4};\n\tfma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "+f"(a), "+f"(b) : "f"(factor_a), "f"(factor_b), "f"(15.f));
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The eight codes of a word as four pairs of the values that they stand for.  A nibble under the exponent of 1024 is 1024 + c, one
// that sits four bits higher 1024 + 16 c: both are exact in f16, and so is what is left when 1024 is taken off again.
__device__ __forceinline__ __half2 as_h2(uint32_t x) { return *reinterpret_cast<const __half2*>(&x); }
// s0, z0: scale and zero of the first two pairs, s1, z1 of the others.
__device__ __forceinline__ void kv4_values(uint32_t w, __half2 s0, __half2 z0, __half2 s1, __half2 z1, uint32_t (&r)[4]) {
    const uint32_t v = w >> 8;
    uint32_t x[4];
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(x[0]) : "r"(w));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(x[1]) : "r"(w));
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(x[2]) : "r"(v));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(x[3]) : "r"(v));
    const __half2 low = __half2half2(__ushort_as_half(0xE400)), sixteenth = __half2half2(__ushort_as_half(0x2C00)),
                  less = __half2half2(__ushort_as_half(0xD400));   // -1024, 1 / 16, -64
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __half2 h = *reinterpret_cast<const __half2*>(&x[j]);
        const __half2 code = j & 1 ? __hfma2(h, sixteenth, less) : __hadd2(h, low);
        const __half2 value = j < 2 ? __hfma2(s0, code, z0) : __hfma2(s1, code, z1);
        r[j] = *reinterpret_cast<const uint32_t*>(&value);
    }
}

// x / group for x below 2^28 (what is left over, x times less than 16, stays below 2^32).
__device__ __forceinline__ int by_group(const Kv4AttnArgs& a, int x) { return a.group == 1 ? x : (int)__umulhi((unsigned)x, a.group_inv); }

// A unit: a tile of columns of one sequence (its rows times the query heads of a kv head, COLS at a time), a kv head, a split of the
// positions.  Units lie in the order sequence, column tile, kv head, split.  What the consumers are told of one, a stage at a time:
struct __align__(16) Kv4Item {
    int flags;                                  // KI_*
    int start, rows, row0;                      // the sequence's first new position, its rows, the first of them
    int ctile, head, splits, base;              // base: position of the stage's first key
    int hi, all;                                // one past the last position that any column of the tile sees, the last that all see
    long long w;                                // number of the unit times kv heads: where its partial sums go
};
constexpr int KI_FIRST = 1, KI_LAST = 2, KI_QUERIES = 4, KI_END = 8;

struct Kv4Walk {       // the producer's place
    int entry, ctile, head, split, splits, size, base, hi;     // size: positions of a split
    int4 e, next;      // this entry and, read ahead, the one behind it
    int units, next_units;    // and their first units
    long long w, at;   // number of the unit; work of all units before it
};

template <int COLS>
__device__ __forceinline__ void walk_range(const Kv4AttnArgs& a, Kv4Walk& u) {
    u.base = u.split * u.size;
    const int end_row = by_group(a, min((u.ctile + 1) * COLS, u.e.z * a.group) - 1);
    u.hi = (int)min((long long)u.base + u.size, (long long)u.e.y + end_row + 1);
}

__device__ __forceinline__ void walk_enter(const Kv4AttnArgs& a, Kv4Walk& u, int4 e, int units) {
    u.e = e;
    u.size = a.split.of((long long)e.y + e.z);
    u.splits = a.split.parts((long long)e.y + e.z);
    u.w = (long long)units * a.c.n_kv;
    u.next = __ldcg(a.entries + min(u.entry + 1, a.n - 1));
    u.next_units = __ldcg(a.cu_units + min(u.entry + 1, a.n - 1));
}

// To the next unit.
template <int COLS>
__device__ __forceinline__ void walk_next(const Kv4AttnArgs& a, Kv4Walk& u) {
    u.at += a.split.work_of(min(u.size, u.e.y + u.e.z - u.split * u.size));
    ++u.w;
    if (++u.split == u.splits) {
        u.split = 0;
        if (++u.head == a.c.n_kv) {
            u.head = 0;
            if (++u.ctile * COLS >= u.e.z * a.group) {
                u.ctile = 0;
                while (++u.entry < a.n) {
                    walk_enter(a, u, u.next, u.next_units);
                    if (u.e.z) break;
                }
            }
        }
    }
    walk_range<COLS>(a, u);
}

// A CTA's share [from, to) of all work, and the first unit that has at least `from` work before it, found by the whole warp, 32 sequences
// at a time.  The sequences' places are read along with their work, so that n up to 32 take one read of the L2 and up to 1024 two.
template <int COLS>
__device__ __forceinline__ bool walk_begin(const Kv4AttnArgs& a, Kv4Walk& u, long long& to, int lane) {
    long long from = 0, before = 0;
    int lo = 0, hi = a.n, units = 0;      // work before lo <= from < work before hi
    int4 e = make_int4(0, 0, 0, 0);
    const int all = __ldcg(a.cu_work + a.n);
    for (bool first = true, found = false; !found; first = false) {
        const int step = (hi - lo + 31) / 32, i = lo + lane * step;
        found = step == 1;      // also where a group of one is left: its place has to be read
        const long long work = i < hi ? (long long)__ldcg(a.cu_work + i) * a.c.n_kv : 0x7fffffffffffffffll;
        if (step == 1 && i < hi) {
            e = __ldcg(a.entries + i);
            units = __ldcg(a.cu_units + i);
        }
        if (first) {
            const long long total = (long long)all * a.c.n_kv;
            from = total * blockIdx.x / gridDim.x;
            to = total * (blockIdx.x + 1) / gridDim.x;
            if (from >= to) return false;
        }
        const int k = 31 - __clz(__ballot_sync(0xffffffffu, work <= from));
        before = __shfl_sync(0xffffffffu, work, k);
        if (step == 1) {
            e.x = __shfl_sync(0xffffffffu, e.x, k); e.y = __shfl_sync(0xffffffffu, e.y, k);
            e.z = __shfl_sync(0xffffffffu, e.z, k); e.w = __shfl_sync(0xffffffffu, e.w, k);
            units = __shfl_sync(0xffffffffu, units, k);
        }
        lo += k * step;
        hi = min(hi, lo + step);
    }
    u.entry = lo;
    walk_enter(a, u, e, units);
    const int one = a.split.work((long long)e.y + e.z), full = a.split.work_of(u.size);     // of a (column tile, head), of a split
    const long long turn = (from - before) / one;
    const int into = (int)((from - before) % one);
    u.split = min((into + full - 1) / full, u.splits - 1);
    u.head = (int)(turn % a.c.n_kv);
    u.ctile = (int)(turn / a.c.n_kv);
    u.w += turn * u.splits + u.split;
    u.at = before + turn * one + u.split * full;
    walk_range<COLS>(a, u);
    if (u.at < from) walk_next<COLS>(a, u);
    return u.at < to && u.entry < a.n;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(uint32_t bar, unsigned count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, unsigned bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Waits for a phase, a bounded number of polls; false for the whole warp when they run out.
__device__ __forceinline__ bool bar_wait(uint32_t bar, unsigned parity) {
    uint32_t ok = 0;
    for (unsigned i = 0; i < KV4_POLLS && !ok; ++i)
        asm volatile(
            "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return __all_sync(0xffffffffu, ok);
}
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, unsigned bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// A wait ran out: recorded, and the CTA stays until copies that are under way have landed.
__device__ __noinline__ void give_up(int32_t* flag) {
    atomicOr(flag, KV4_TIMEOUT);
    for (int i = 0; i < 100; ++i) __nanosleep(100000);
}

// Shared memory of the mma.sync forms, in bytes.
template <int NG, int COLS>
struct KaShared {
    static constexpr int KT = NG == 2 ? 4 : 2;                                  // tiles of 16 positions a warp takes at once
    static constexpr int KEYS = KA_WARPS * KT * KV4_TILE;                         // positions of a stage
    static_assert(256 % KEYS == 0, "splits are whole stages, but for a sequence's last");
    static constexpr int TILE = NG * KV4_GT, QCOL = NG * KV4_GROUP * 2;
    static constexpr int KV = KA_WARPS * KT * TILE, Q = COLS * QCOL;
    static constexpr int STAGE = KV + Q + (int)sizeof(Kv4Item);
    static constexpr int STAGES = 2;
    static constexpr int ACC = KA_WARPS * COLS * (NG * KV4_GROUP + 4) * 4, ML = KA_WARPS * COLS * 8;
    static constexpr int TOTAL = STAGES * STAGE + ACC + ML + 8 * (2 * STAGES + 2);
};

// A CTA's shared memory and barriers: full and empty of every stage, and of the place where the consumer warps' states meet.
template <int NG, int COLS>
struct KaRing {
    using S = KaShared<NG, COLS>;
    unsigned char* smem;
    float* acc;          // [warp][column][HD + 4]
    float2* ml;          // [warp][column]
    uint32_t bars;
    __device__ __forceinline__ explicit KaRing(unsigned char* p)
        : smem(p), acc(reinterpret_cast<float*>(p + S::STAGES * S::STAGE)), ml(reinterpret_cast<float2*>(p + S::STAGES * S::STAGE + S::ACC)),
          bars(smem_addr(p + S::STAGES * S::STAGE + S::ACC + S::ML)) {}
    __device__ __forceinline__ uint32_t full(int s) const { return bars + 8 * s; }
    __device__ __forceinline__ uint32_t empty(int s) const { return bars + 8 * (S::STAGES + s); }
    __device__ __forceinline__ uint32_t acc_full() const { return bars + 16 * S::STAGES; }
    __device__ __forceinline__ uint32_t acc_empty() const { return bars + 16 * S::STAGES + 8; }
    __device__ __forceinline__ void init() const {
        if (threadIdx.x == 0) {
            for (int s = 0; s < S::STAGES; ++s) { bar_init(full(s), 1); bar_init(empty(s), KA_WARPS); }
            bar_init(acc_full(), KA_WARPS);
            bar_init(acc_empty(), KA_WARPS);
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
    }
};

// The producer warp: walks the CTA's units and brings keys, values and queries into the ring (bulk copies), a stage at a time.
template <int NG, int COLS>
__device__ __forceinline__ void ka_produce(const Kv4AttnArgs& a, const KaRing<NG, COLS>& ring, int lane) {
    using S = KaShared<NG, COLS>;
    constexpr int HD = NG * KV4_GROUP, KT = S::KT, D = S::STAGES;
    const int tiles = 1 << (a.c.block_shift - 4);     // of a block
    Kv4Walk u = {};
    int id = 0;     // the lane's tile's block
    auto block_of = [&]() {
        const int pos = u.base + lane * KV4_TILE;
        return lane < KA_WARPS * KT && pos < u.hi ? __ldcg(a.c.table + (size_t)u.e.x * a.c.max_blocks + (pos >> a.c.block_shift)) : 0;
    };
    long long last = 0;
    bool queries = true, begins = true, more = walk_begin<COLS>(a, u, last, lane);
    if (more) id = block_of();
    const int run = min(tiles, KA_WARPS * KT);    // tiles that lie behind one another
    for (unsigned k = 0;; ++k) {
        const int s = k % D;
        if (k >= D && !bar_wait(ring.empty(s), (k / D - 1) & 1)) { give_up(a.c.flag); return; }
        unsigned char* const stage = ring.smem + s * S::STAGE;
        Kv4Item* const item = reinterpret_cast<Kv4Item*>(stage + S::KV + S::Q);
        if (!more) {
            if (lane == 0) {
                item->flags = KI_END;
                bar_arrive(ring.full(s));
            }
            return;
        }
        if ((unsigned)id >= (unsigned)a.c.n_blocks) {
            atomicOr(a.c.flag, KV4_BAD_BLOCK);
            id = 0;
        }
        const bool ends = u.base + S::KEYS >= u.hi;
        const int valid = max(min((u.hi - u.base + KV4_TILE - 1) / KV4_TILE, KA_WARPS * KT), 0);   // none: a tile that does not see this split
        const int cols = min(u.e.z * a.group - u.ctile * COLS, COLS);
        if (lane == 0) {
            Kv4Item d;
            d.flags = (begins ? KI_FIRST : 0) | (ends ? KI_LAST : 0) | (queries ? KI_QUERIES : 0);
            d.start = u.e.y; d.rows = u.e.z; d.row0 = u.e.w;
            d.ctile = u.ctile; d.head = u.head; d.splits = u.splits; d.base = u.base;
            d.hi = u.hi; d.all = u.e.y + by_group(a, u.ctile * COLS); d.w = u.w;
            *item = d;
            bar_expect(ring.full(s), valid * S::TILE + (queries ? cols * S::QCOL : 0));
        }
        __syncwarp();
        const int pos = u.base + lane * KV4_TILE;
        if (lane < valid && lane % run == 0) {
            const unsigned char* src = a.c.pool + ((size_t)((long long)id * a.c.n_kv + u.head) * tiles + ((pos & ((1 << a.c.block_shift) - 1)) >> 4)) * S::TILE;
            bulk_copy(smem_addr(stage + lane * S::TILE), src, min(run, valid - lane) * S::TILE, ring.full(s));
        }
        if (queries && lane < cols) {     // the heads of a row lie behind one another
            const int c = u.ctile * COLS + lane, row = by_group(a, c), in = c - row * a.group;
            if (lane == 0 || in == 0)
                bulk_copy(smem_addr(stage + S::KV + lane * S::QCOL), a.q + (long long)(u.e.w + row) * a.q_stride + (u.head * a.group + in) * HD,
                          min(a.group - in, cols - lane) * S::QCOL, ring.full(s));
        }
        queries = false;
        begins = ends;
        u.base += S::KEYS;
        if (ends) {
            walk_next<COLS>(a, u);
            more = u.at < last && u.entry < a.n;
            queries = u.split == 0;
        }
        if (more) id = block_of();
    }
}

// The end of a unit: the four consumer warps' states, which lie in the ring's place for them, added in the order of the warps; written out,
// or kept as the split's part.
template <int NG, int COLS>
__device__ __forceinline__ void ka_finish(const Kv4AttnArgs& a, const KaRing<NG, COLS>& ring, const Kv4Item& d, int cols) {
    constexpr int HD = NG * KV4_GROUP;
    for (int i = threadIdx.x; i < min(cols, COLS) * (HD / 4); i += KA_THREADS) {
        const int col = i / (HD / 4), dim = i % (HD / 4) * 4;
        float best = -INFINITY, sum = 0.f;
#pragma unroll
        for (int k2 = 0; k2 < KA_WARPS; ++k2) best = fmaxf(best, ring.ml[k2 * COLS + col].x);
        const float now = best == -INFINITY ? 0.f : best;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int k2 = 0; k2 < KA_WARPS; ++k2) {
            const float2 part = ring.ml[k2 * COLS + col];
            const float f = ex2(part.x - now);
            const float4 v = *reinterpret_cast<const float4*>(ring.acc + (k2 * COLS + col) * (HD + 4) + dim);
            sum += f * part.y;
            o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
        }
        if (d.splits == 1) {
            const float inv = sum == 0.f ? 0.f : 1.f / sum;
            const int c = d.ctile * COLS + col, row = by_group(a, c);
            __nv_bfloat162 lo2 = __floats2bfloat162_rn(o.x * inv, o.y * inv), hi2 = __floats2bfloat162_rn(o.z * inv, o.w * inv);
            uint2 v = make_uint2(*reinterpret_cast<uint32_t*>(&lo2), *reinterpret_cast<uint32_t*>(&hi2));
            *reinterpret_cast<uint2*>(a.out + (long long)(d.row0 + row) * a.out_stride + (d.head * a.group + c - row * a.group) * HD + dim) = v;
        } else {
            *reinterpret_cast<float4*>(a.acc + (size_t)(d.w * COLS + col) * HD + dim) = o;
            if (dim == 0) a.ml[d.w * COLS + col] = make_float2(best, sum);
        }
    }
}

// Form for tiles of 8 or 16 columns: keys as the A operand, queries as the B operand (8 columns), values as f16; the scores'
// transpose for the second product is one movmatrix a fragment.  Each warp has its own positions and makes f16 of them in registers, 13
// instructions for eight codes: with 16 columns about what their products cost.  Softmax statistics and sums are fp32; the weights enter the second
// product as f16, 2^15 times as large (2^-11 of each, where bf16's 2^-8 would be as much as the output's own rounding).
template <int NG, int NT>
__global__ void __launch_bounds__(KA_THREADS + 32) k_kv4_attn(const Kv4AttnArgs a) {
    constexpr int HD = NG * KV4_GROUP, COLS = NT * 8;
    using S = KaShared<NG, COLS>;
    constexpr int KT = S::KT, D = S::STAGES;
    extern __shared__ __align__(128) unsigned char smem[];
    const KaRing<NG, COLS> ring(smem);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    ring.init();
    pdl_wait();
    pdl_launch();
    if (warp == KA_WARPS) return ka_produce<NG, COLS>(a, ring, lane);

    uint32_t qf[NT][NG][4];
    float factor[NT][2];
    int limit[NT][2];       // last position that the column sees
    float acc[NT][2 * NG][4], m[NT][2], l[NT][2];
    unsigned merged = 0;
    for (unsigned k = 0;; ++k) {
        const int s = k % D;
        if (!bar_wait(ring.full(s), (k / D) & 1)) { give_up(a.c.flag); return; }
        const unsigned char* const stage = ring.smem + s * S::STAGE;
        const Kv4Item d = *reinterpret_cast<const Kv4Item*>(stage + S::KV + S::Q);
        if (d.flags & KI_END) return;
        const int cols = d.rows * a.group - d.ctile * COLS;                 // valid ones of this tile, if fewer than COLS
        if (d.flags & KI_QUERIES) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const bool there = nt * 8 + g < cols;
                uint4 raw[NG];
                uint32_t big = 0;
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    raw[i] = make_uint4(0, 0, 0, 0);
                    if (there) raw[i] = *reinterpret_cast<const uint4*>(stage + S::KV + (nt * 8 + g) * S::QCOL + i * 64 + t * 16);
                    const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) big = max(big, max(x[j] & 0x7fffu, x[j] >> 16 & 0x7fffu));
                }
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
                big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
                // the column times a power of two, so that its largest element lies in [1, 2): exact in f16 but for elements 2^14 times smaller
                const int e = min(max((int)(big >> 7), 1), 253);
                const float down = __int_as_float((254 - e) << 23), up = __int_as_float(e << 23);
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        qf[nt][i][j] = pack_h2(__uint_as_float(x[j] << 16) * down, __uint_as_float(x[j] & 0xffff0000u) * down);
                }
                const float f = score_factor(a.scale_log2 * up, big);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int c2 = nt * 8 + 2 * t + j;
                    factor[nt][j] = __shfl_sync(0xffffffffu, f, (2 * t + j) * 4);
                    limit[nt][j] = c2 < cols ? d.start + by_group(a, d.ctile * COLS + c2) : -1;
                }
            }
        }
        if (d.flags & KI_FIRST) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                m[nt][0] = m[nt][1] = -INFINITY;
                l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * NG; ++i) acc[nt][i][0] = acc[nt][i][1] = acc[nt][i][2] = acc[nt][i][3] = 0.f;
            }
        }
        const int base = d.base + warp * KV4_TILE;                          // a warp takes every fourth tile
        const int nk = min(KT, ((d.hi - base + KV4_TILE - 1) / KV4_TILE + KA_WARPS - 1) / KA_WARPS);    // tiles that are there
        if (nk > 0) {
            constexpr int NEXT = KA_WARPS * S::TILE;
            const unsigned char* const mine = stage + warp * S::TILE;
            const bool whole = d.base + S::KEYS - 1 <= d.all;   // every column sees all of them
            float sc[KT][NT][4];
#pragma unroll
            for (int k2 = 0; k2 < KT; ++k2) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) sc[k2][nt][0] = sc[k2][nt][1] = sc[k2][nt][2] = sc[k2][nt][3] = 0.f;
                if (k2 < nk) {
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const unsigned char* p = mine + k2 * NEXT + i * KV4_GT;
                        const uint2 code = *reinterpret_cast<const uint2*>(p + lane * 8);
                        const uint2 par = *reinterpret_cast<const uint2*>(p + KV4_KPAR + g * 8);
                        uint32_t x[4], y[4];
                        kv4_values(code.x, __low2half2(as_h2(par.x)), __high2half2(as_h2(par.x)), __low2half2(as_h2(par.x)), __high2half2(as_h2(par.x)), x);
                        kv4_values(code.y, __low2half2(as_h2(par.y)), __high2half2(as_h2(par.y)), __low2half2(as_h2(par.y)), __high2half2(as_h2(par.y)), y);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816(sc[k2][nt], x[0], y[0], x[1], y[1], qf[nt][i][0], qf[nt][i][1]);
                            mma16816(sc[k2][nt], x[2], y[2], x[3], y[3], qf[nt][i][2], qf[nt][i][3]);
                        }
                    }
                }
            }
            if (!whole) {
#pragma unroll
                for (int k2 = 0; k2 < KT; ++k2) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (base + k2 * (KA_WARPS * 16) + g + (j >> 1) * 8 > limit[nt][j & 1]) sc[k2][nt][j] = -INFINITY;
                    }
                }
            }
            uint32_t p[KT][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float top[2] = {sc[0][nt][0], sc[0][nt][1]};
#pragma unroll
                for (int k2 = 0; k2 < KT; ++k2) {
                    top[0] = fmaxf(fmaxf(top[0], sc[k2][nt][0]), sc[k2][nt][2]);
                    top[1] = fmaxf(fmaxf(top[1], sc[k2][nt][1]), sc[k2][nt][3]);
                }
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
                    top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
                }
                if (d.flags & KI_FIRST) {
                    m[nt][0] = top[0];
                    m[nt][1] = top[1];
                } else if (__any_sync(0xffffffffu, top[0] > m[nt][0] || top[1] > m[nt][1])) {
                    float old[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float best = fmaxf(m[nt][j], top[j]);
                        old[j] = best == -INFINITY ? 1.f : ex2((m[nt][j] - best) * factor[nt][j]);
                        m[nt][j] = best;
                        l[nt][j] *= old[j];
                    }
#pragma unroll
                    for (int i = 0; i < 2 * NG; ++i) {
                        acc[nt][i][0] *= old[0]; acc[nt][i][1] *= old[1];
                        acc[nt][i][2] *= old[0]; acc[nt][i][3] *= old[1];
                    }
                }
                // minus the maximum; nothing seen yet: weights of exp(-inf) = 0
                const float less[2] = {m[nt][0] == -INFINITY ? 0.f : -m[nt][0], m[nt][1] == -INFINITY ? 0.f : -m[nt][1]};
#pragma unroll
                for (int k2 = 0; k2 < KT; ++k2) {
                    float e[4];
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        e[j] = sc[k2][nt][j] + less[0];
                        e[j + 1] = sc[k2][nt][j + 1] + less[1];
                        lifted2(e[j], e[j + 1], factor[nt][0], factor[nt][1]);
                        e[j] = ex2(e[j]);
                        e[j + 1] = ex2(e[j + 1]);
                        l[nt][0] += e[j];
                        l[nt][1] += e[j + 1];
                    }
                    p[k2][nt][0] = movmatrix(pack_h2(e[0], e[1]));
                    p[k2][nt][1] = movmatrix(pack_h2(e[2], e[3]));
                }
            }
#pragma unroll
            for (int k2 = 0; k2 < KT; ++k2) {
                if (k2 < nk) {
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const unsigned char* q = mine + k2 * NEXT + i * KV4_GT;
                        const uint2 code = *reinterpret_cast<const uint2*>(q + KV4_VCODE + lane * 8);
                        const uint4 par = *reinterpret_cast<const uint4*>(q + KV4_VPAR + t * 16);   // of keys 2t, 2t+8, 2t+1, 2t+9
                        const __half2 s0 = as_h2(__byte_perm(par.x, par.z, 0x5410)), z0 = as_h2(__byte_perm(par.x, par.z, 0x7632));
                        const __half2 s8 = as_h2(__byte_perm(par.y, par.w, 0x5410)), z8 = as_h2(__byte_perm(par.y, par.w, 0x7632));
                        uint32_t x[4], y[4];
                        kv4_values(code.x, s0, z0, s8, z8, x);
                        kv4_values(code.y, s0, z0, s8, z8, y);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816(acc[nt][2 * i], x[0], x[1], x[2], x[3], p[k2][nt][0], p[k2][nt][1]);
                            mma16816(acc[nt][2 * i + 1], y[0], y[1], y[2], y[3], p[k2][nt][0], p[k2][nt][1]);
                        }
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) bar_arrive(ring.empty(s));
        if (!(d.flags & KI_LAST)) continue;
        // the warps' states, added in the order of the warps
        if (merged && !bar_wait(ring.acc_empty(), (merged - 1) & 1)) { give_up(a.c.flag); return; }
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                l[nt][0] += __shfl_xor_sync(0xffffffffu, l[nt][0], o);
                l[nt][1] += __shfl_xor_sync(0xffffffffu, l[nt][1], o);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = nt * 8 + 2 * t + j;
                if (col < cols) {
                    if (g == 0) ring.ml[warp * COLS + col] = make_float2(m[nt][j] * factor[nt][j], l[nt][j]);
#pragma unroll
                    for (int i = 0; i < NG; ++i)
                        *reinterpret_cast<float4*>(ring.acc + (warp * COLS + col) * (HD + 4) + i * KV4_GROUP + 4 * g) =
                            make_float4(acc[nt][2 * i][j], acc[nt][2 * i][2 + j], acc[nt][2 * i + 1][j], acc[nt][2 * i + 1][2 + j]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) bar_arrive(ring.acc_full());
        if (!bar_wait(ring.acc_full(), merged & 1)) { give_up(a.c.flag); return; }
        ka_finish<NG, COLS>(a, ring, d, cols);
        __syncwarp();
        if (lane == 0) bar_arrive(ring.acc_empty());
        ++merged;
    }
}

// m16n8k32, bytes in, 32-bit sums out: D = A B + C, the codes A always unsigned.
#define KA_MMA8(types)                                                                                                              \
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32." types ".s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"    \
                 : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])                                                                     \
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1), "r"(c2), "r"(c3))
template <bool SIGNED>
__device__ __forceinline__ void mma16832(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1, int c0, int c1, int c2, int c3) {
    if constexpr (SIGNED) KA_MMA8("u8.s8");
    else KA_MMA8("u8.u8");
}
#undef KA_MMA8

// Form for a few columns (single tokens): what bounds it is the arithmetic a stored byte costs, not the tensor cores, so the codes enter
// the products as they are, as bytes: three logic operations for eight codes, where their f16 values take thirteen instructions, half of
// them at half rate.
//   scores:  q . K = sum over groups of scale * (q . code) + zero * (sum of the group's q)
//   outputs: sum_i w_i V_i = sum_i (w_i scale_i) code_i + sum_i w_i zero_i
// So K and V are scale * code + zero here, without the rounding to f16 (2^-11 of the value) that the other forms and k_kv4_read make.
// A query column, times a power of two, is a 15-bit whole number: exact for elements down to 2^-6 of the largest, the others to 2^-14 of
// it.  The weights times the value scales are 16-bit whole numbers in units of 2^-16 of the largest such product of the query and group
// among the warp's positions (half a unit off, each on its own): positions that a query does not see, or whose weight is nothing, take no part
// in the unit, whatever they hold.  Both are cut into two bytes that take two of the 8 columns of a product.  The tensor cores' sums are exact;
// what is added to them, statistics and outputs, is fp32.
// A product's columns hold four queries; or (HALVES, for up to two queries a tile, heads of 64 and 128) two queries twice, once for the
// even groups of 32 elements and once for the odd ones, zeros elsewhere: a lane then has one group of two to scale and to weigh.
// 256 sequences of 512 to 2048 positions, two query heads a kv head of 64: 53.5 us (219 MB: 34 us), the copies alone 52; with f16 values and a
// product's 8 columns a query each, 93.  4 sequences of 64k, four query heads of 128: 77 us (313 MB: 48).
constexpr int KA_ORIGIN = 0x4B400000;   // sums that start as the bits of 1.5 * 2^23 are that float plus the sum (below 2^22 in magnitude)
__device__ __forceinline__ float two_bytes(int high, int low) {
    return fmaf(__int_as_float(high) - 12582912.f, 256.f, __int_as_float(low) - 12582912.f);
}

// At least 4 CTAs an SM, which shared memory allows at every width: with no number the compiler kept to 72 registers and spilled at three
// of five widths (4 x 64k 78.1 us, heads of 96 17.5 for 17.2), with 5 at two (85.0).
template <int NG, bool HALVES>
__global__ void __launch_bounds__(KA_THREADS + 32, 4) k_kv4_attn_few(const Kv4AttnArgs a) {
    static_assert(!HALVES || NG % 2 == 0, "two halves of an even number of groups");
    constexpr int HD = NG * KV4_GROUP, COLS = HALVES ? 2 : 4;
    constexpr int OWN = HALVES ? NG / 2 : NG, SIDES = HALVES ? 2 : 1;      // groups that a lane scales; group i * SIDES + side
    using S = KaShared<NG, COLS>;
    constexpr int KT = S::KT, D = S::STAGES, NEXT = KA_WARPS * S::TILE;
    extern __shared__ __align__(128) unsigned char smem[];
    const KaRing<NG, COLS> ring(smem);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    ring.init();
    pdl_wait();
    pdl_launch();
    if (warp == KA_WARPS) return ka_produce<NG, COLS>(a, ring, lane);

    const int side = HALVES ? t & 1 : 0, query = HALVES ? t >> 1 : t;
    const uint32_t pick = g & 1 ? 0x6240 : 0x7351;      // low or high bytes of four 16-bit weights, in the order of a word's keys
    uint32_t qf[NG][2];         // bytes of column g: high byte (even g) or low byte of its query
    float qsum[OWN], factor;    // of the lane's query, as all below
    int limit;                  // last position that it sees
    float acc[2 * OWN][2], zsum[OWN], m, l;
    unsigned merged = 0;
    for (unsigned k = 0;; ++k) {
        const int s = k % D;
        if (!bar_wait(ring.full(s), (k / D) & 1)) { give_up(a.c.flag); return; }
        const unsigned char* const stage = ring.smem + s * S::STAGE;
        const Kv4Item& d = *reinterpret_cast<const Kv4Item*>(stage + S::KV + S::Q);
        const int flags = d.flags, base = d.base + warp * KV4_TILE;         // a warp takes every fourth tile
        if (flags & KI_END) return;
        const int left = d.hi - base;
        const bool whole = d.base + S::KEYS - 1 <= d.all;                   // every column sees all of the stage
        if (flags & KI_QUERIES) {
            const int cols = d.rows * a.group - d.ctile * COLS;
            const int col = HALVES ? g >> 2 : g >> 1;
            uint4 raw[NG];
            uint32_t big = 0;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                raw[i] = make_uint4(0, 0, 0, 0);
                if (col < cols) raw[i] = *reinterpret_cast<const uint4*>(stage + S::KV + col * S::QCOL + i * 64 + t * 16);
                big = max(big, most_bits(raw[i]));
            }
            big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
            // times a power of two, so that the largest element lies in [2^13, 2^14)
            const int e = min(max((int)(big >> 7), 1), 253);
            const float down = __int_as_float((254 - e) << 23), up = __int_as_float(e << 23);
            float total[NG];
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const uint32_t x[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                int v[8], part = 0;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    v[j] = __float2int_rn(__uint_as_float(j & 1 ? x[j >> 1] & 0xffff0000u : x[j >> 1] << 16) * down * 8192.f);
                    part += v[j];
                    const int low = (int)(signed char)(v[j] & 255);
                    v[j] = g & 1 ? low & 255 : (v[j] - low) >> 8 & 255;
                }
                qf[i][0] = v[0] | v[4] << 8 | v[1] << 16 | v[5] << 24;      // the order of a key word's low nibbles
                qf[i][1] = v[2] | v[6] << 8 | v[3] << 16 | v[7] << 24;      // and of its high ones
                if (HALVES && (g >> 1 & 1) != (i & 1)) qf[i][0] = qf[i][1] = 0;
                part += __shfl_xor_sync(0xffffffffu, part, 1);
                part += __shfl_xor_sync(0xffffffffu, part, 2);
                total[i] = (float)part;
            }
            const float f = score_factor(a.scale_log2 * up * (1.f / 8192.f), big);
            const int from = HALVES ? query * 16 : t * 8;        // a lane of the query's columns
            factor = __shfl_sync(0xffffffffu, f, from);
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                qsum[i] = __shfl_sync(0xffffffffu, total[i * SIDES], from);
                if constexpr (HALVES) {
                    const float other = __shfl_sync(0xffffffffu, total[i * SIDES + 1], from);
                    if (side) qsum[i] = other;
                }
            }
            limit = query < cols ? d.start + by_group(a, d.ctile * COLS + query) : -1;
        }
        if (flags & KI_FIRST) {
            m = -INFINITY;
            l = factor * 0.f;
#pragma unroll
            for (int i = 0; i < OWN; ++i) zsum[i] = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * OWN; ++i) acc[i][0] = acc[i][1] = 0.f;
        }
        if (left > 0) {
            const unsigned char* const mine = stage + warp * S::TILE;
            auto there = [&](int k2) { return k2 * (KA_WARPS * KV4_TILE) < left; };     // whether the warp has a tile number k2
            float sc[KT][2];      // scores of keys g and g + 8 of every tile, then weights
#pragma unroll
            for (int k2 = 0; k2 < KT; ++k2) {
                sc[k2][0] = sc[k2][1] = 0.f;
                if (there(k2)) {
#pragma unroll
                    for (int i = 0; i < OWN; ++i) {
                        const unsigned char* const p = mine + k2 * NEXT + i * SIDES * KV4_GT;
                        const uint2 par = *reinterpret_cast<const uint2*>(p + side * KV4_GT + KV4_KPAR + g * 8);
                        const float2 p0 = __half22float2(as_h2(par.x)), p1 = __half22float2(as_h2(par.y));     // scale, zero
                        int x[4];
#pragma unroll
                        for (int j = 0; j < SIDES; ++j) {
                            const uint2 code = *reinterpret_cast<const uint2*>(p + j * KV4_GT + lane * 8);
                            const uint32_t a0 = code.x & 0x0f0f0f0fu, a1 = code.y & 0x0f0f0f0fu;
                            const uint32_t a2 = code.x >> 4 & 0x0f0f0f0fu, a3 = code.y >> 4 & 0x0f0f0f0fu;
                            const uint32_t* const q = qf[i * SIDES + j];
                            if (j == 0) mma16832<true>(x, a0, a1, a2, a3, q[0], q[1], KA_ORIGIN, KA_ORIGIN, KA_ORIGIN, KA_ORIGIN);
                            else mma16832<true>(x, a0, a1, a2, a3, q[0], q[1], x[0], x[1], x[2], x[3]);
                        }
                        sc[k2][0] = fmaf(p0.x, two_bytes(x[0], x[1]), fmaf(p0.y, qsum[i], sc[k2][0]));
                        sc[k2][1] = fmaf(p1.x, two_bytes(x[2], x[3]), fmaf(p1.y, qsum[i], sc[k2][1]));
                    }
                    if constexpr (HALVES) {
                        sc[k2][0] += __shfl_xor_sync(0xffffffffu, sc[k2][0], 1);
                        sc[k2][1] += __shfl_xor_sync(0xffffffffu, sc[k2][1], 1);
                    }
                }
            }
            if (!whole) {
#pragma unroll
                for (int k2 = 0; k2 < KT; ++k2) {
                    if (base + k2 * (KA_WARPS * KV4_TILE) + g > limit) sc[k2][0] = -INFINITY;
                    if (base + k2 * (KA_WARPS * KV4_TILE) + g + 8 > limit) sc[k2][1] = -INFINITY;
                }
            }
            float top = sc[0][0];
#pragma unroll
            for (int k2 = 0; k2 < KT; ++k2) top = fmaxf(fmaxf(top, sc[k2][0]), sc[k2][1]);
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (flags & KI_FIRST) {
                m = top;
            } else if (__any_sync(0xffffffffu, top > m)) {
                const float best = fmaxf(m, top), old = best == -INFINITY ? 1.f : ex2((m - best) * factor);
                m = best;
                l *= old;
#pragma unroll
                for (int i = 0; i < OWN; ++i) zsum[i] *= old;
#pragma unroll
                for (int i = 0; i < 2 * OWN; ++i) { acc[i][0] *= old; acc[i][1] *= old; }
            }
            const float less = m == -INFINITY ? 0.f : -m;       // nothing seen yet: weights of exp(-inf) = 0
#pragma unroll
            for (int k2 = 0; k2 < KT; ++k2) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    sc[k2][j] = ex2((sc[k2][j] + less) * factor);
                    l += sc[k2][j];
                }
            }
            // weights times value scales, and the largest of each group
            float vs[KT][OWN][2], unit[OWN], units[OWN];
#pragma unroll
            for (int i = 0; i < OWN; ++i) unit[i] = 0.f;
#pragma unroll
            for (int k2 = 0; k2 < KT; ++k2) {
#pragma unroll
                for (int i = 0; i < OWN; ++i) {
                    vs[k2][i][0] = vs[k2][i][1] = 0.f;
                    if (there(k2)) {
                        const uint2 par = *reinterpret_cast<const uint2*>(mine + k2 * NEXT + (i * SIDES + side) * KV4_GT + KV4_VPAR + g * 8);
                        const float2 p0 = __half22float2(as_h2(par.x)), p1 = __half22float2(as_h2(par.y));
                        vs[k2][i][0] = sc[k2][0] * p0.x;
                        vs[k2][i][1] = sc[k2][1] * p1.x;
                        unit[i] = fmaxf(fmaxf(unit[i], vs[k2][i][0]), vs[k2][i][1]);
                        zsum[i] = fmaf(sc[k2][0], p0.y, fmaf(sc[k2][1], p1.y, zsum[i]));
                    }
                }
            }
            // Of the lane's query over all keys: two groups at a time as bf16, rounded up.  Products below 1e-30 are nothing beside the weight of 1
            // that the maximum has.
#pragma unroll
            for (int i = 0; i < OWN; i += 2) {
                const bool two = i + 1 < OWN;
                uint32_t top2 = __byte_perm(__float_as_uint(unit[i]), __float_as_uint(unit[two ? i + 1 : i]), 0x7632) + 0x00010001u;
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) top2 = __vmaxu2(top2, __shfl_xor_sync(0xffffffffu, top2, o));
                unit[i] = __uint_as_float(top2 << 16);
                if (two) unit[i + 1] = __uint_as_float(top2 & 0xffff0000u);
            }
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                units[i] = unit[i] > 1e-30f ? __fdividef(65280.f, unit[i]) : 0.f;
                unit[i] *= 1.f / 65280.f;
            }
#pragma unroll
            for (int i = 0; i < OWN; ++i) {
                int x[SIDES][2][4];
#pragma unroll
                for (int k2 = 0; k2 < KT; k2 += 2) {
                    if (k2 == 0 || there(k2)) {       // of a second tile that is not there the weights are 0
                        uint32_t b[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            // the nearest whole number in the low 16 bits, twice over, for the columns of both bytes
                            const uint32_t w0 = __float_as_uint(fmaf(vs[k2 + j][i][0], units[i], 8388608.f));
                            const uint32_t w8 = __float_as_uint(fmaf(vs[k2 + j][i][1], units[i], 8388608.f));
                            b[j] = __byte_perm(movmatrix(__byte_perm(w0, 0, 0x1010)), movmatrix(__byte_perm(w8, 0, 0x1010)), pick);
                        }
#pragma unroll
                        for (int j = 0; j < SIDES; ++j) {
                            const unsigned char* const p = mine + k2 * NEXT + (i * SIDES + j) * KV4_GT + KV4_VCODE + lane * 8;
                            const uint2 c0 = *reinterpret_cast<const uint2*>(p), c1 = *reinterpret_cast<const uint2*>(p + NEXT);
                            // elements in the high nibbles come out 16 times as large
                            int(&y)[4] = x[j][0], (&z)[4] = x[j][1];
                            if (k2 == 0) {
                                mma16832<false>(y, c0.x & 0x0f0f0f0fu, c0.x & 0xf0f0f0f0u, c1.x & 0x0f0f0f0fu, c1.x & 0xf0f0f0f0u, b[0], b[1], KA_ORIGIN, KA_ORIGIN, KA_ORIGIN, KA_ORIGIN);
                                mma16832<false>(z, c0.y & 0x0f0f0f0fu, c0.y & 0xf0f0f0f0u, c1.y & 0x0f0f0f0fu, c1.y & 0xf0f0f0f0u, b[0], b[1], KA_ORIGIN, KA_ORIGIN, KA_ORIGIN, KA_ORIGIN);
                            } else {
                                mma16832<false>(y, c0.x & 0x0f0f0f0fu, c0.x & 0xf0f0f0f0u, c1.x & 0x0f0f0f0fu, c1.x & 0xf0f0f0f0u, b[0], b[1], y[0], y[1], y[2], y[3]);
                                mma16832<false>(z, c0.y & 0x0f0f0f0fu, c0.y & 0xf0f0f0f0u, c1.y & 0x0f0f0f0fu, c1.y & 0xf0f0f0f0u, b[0], b[1], z[0], z[1], z[2], z[3]);
                            }
                        }
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    int y[4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) y[r] = HALVES && side ? x[SIDES - 1][j][r] : x[0][j][r];
                    acc[2 * i + j][0] = fmaf(unit[i], two_bytes(y[0], y[1]), acc[2 * i + j][0]);
                    acc[2 * i + j][1] = fmaf(unit[i] * 0.0625f, two_bytes(y[2], y[3]), acc[2 * i + j][1]);
                }
            }
        }
        if (!(flags & KI_LAST)) {
            __syncwarp();
            if (lane == 0) bar_arrive(ring.empty(s));
            continue;
        }
        const Kv4Item last = d;
        __syncwarp();
        if (lane == 0) bar_arrive(ring.empty(s));
        const int cols = last.rows * a.group - last.ctile * COLS;           // valid ones of this tile, if fewer than COLS
        if (merged && !bar_wait(ring.acc_empty(), (merged - 1) & 1)) { give_up(a.c.flag); return; }
        const int col = query;
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) {
            l += __shfl_xor_sync(0xffffffffu, l, o);
#pragma unroll
            for (int i = 0; i < OWN; ++i) zsum[i] += __shfl_xor_sync(0xffffffffu, zsum[i], o);
        }
        if (col < cols) {
            if (g == 0 && side == 0) ring.ml[warp * COLS + col] = make_float2(m * factor, l);
#pragma unroll
            for (int i = 0; i < OWN; ++i)
                *reinterpret_cast<float4*>(ring.acc + (warp * COLS + col) * (HD + 4) + (i * SIDES + side) * KV4_GROUP + 4 * g) =
                    make_float4(acc[2 * i][0] + zsum[i], acc[2 * i][1] + zsum[i], acc[2 * i + 1][0] + zsum[i], acc[2 * i + 1][1] + zsum[i]);
        }
        __syncwarp();
        if (lane == 0) bar_arrive(ring.acc_full());
        if (!bar_wait(ring.acc_full(), merged & 1)) { give_up(a.c.flag); return; }
        ka_finish<NG, COLS>(a, ring, last, cols);
        __syncwarp();
        if (lane == 0) bar_arrive(ring.acc_empty());
        ++merged;
    }
}

// Form for chunks of prompts: a CTA takes 128 columns, 16 a warp, and 64 positions at a time.  Codes become f16 once a CTA, one tile of 16 keys or
// values a warp, and lie in shared memory in the order in which lanes need them as the B operands of m16n8k16: 16 bytes a lane, no conflicts.
// The queries are the A operand of the first product and stay in registers; the weights, as the first product leaves them, are the A operand of
// the second.  A lane ends with eight neighbouring elements of its rows.  (Weights are 2^15 times as large here too.)
// Each step's codes are read while the step before is computed; two buffers, so that one barrier a step is enough.
// Bound: at heads of 128 a step's products take the tensor cores 2130 cycles at mma.sync's rate (8.3 a product and scheduler) and its operands
// 2050 of shared memory's; measured, about 4500 with the exponentials and the conversion in between, as two warps a scheduler overlap them
// only in part.  2 x 1000 rows of 32 query and 8 kv heads of 128 against 6000 to 9000 positions: 1061 us, 216 TFLOP/s of some 540 that mma.sync
// can do.  12 warps with 96 positions at a time (168 registers, spills) and 16 warps were slower.
constexpr int KR_COLS = 128, KR_WARPS = 8, KR_THREADS = KR_WARPS * 32, KR_STEP = 64;
template <int NG>
struct KrShared {
    static constexpr int HALF = 4 * NG * 2 * 32;            // 16-byte pieces of a step's keys, and of its values
    static constexpr int TOTAL = 2 * 2 * HALF * 16;
};

template <int NG>
__global__ void __launch_bounds__(KR_THREADS, 1) k_kv4_attn_rows(const Kv4AttnArgs a) {
    constexpr int HD = NG * KV4_GROUP, HALF = KrShared<NG>::HALF;
    extern __shared__ __align__(128) unsigned char smem[];
    uint4* const ring = reinterpret_cast<uint4*>(smem);     // [buffer][keys, values][tile][group][half][lane]
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int tile = warp & 3, tiles = 1 << (a.c.block_shift - 4);      // the tile of a step that this warp fills, keys or values
    const bool value = warp >= 4;
    pdl_wait();
    pdl_launch();
    Kv4Walk u = {};
    long long share = 0;
    int buffer = 0;
    for (bool more = walk_begin<KR_COLS>(a, u, share, lane); more; walk_next<KR_COLS>(a, u), more = u.at < share && u.entry < a.n) {
        const int first = u.ctile * KR_COLS, cols = min(u.e.z * a.group - first, KR_COLS), mine = warp * 16 + g;
        const int steps = max((u.hi - u.base + KR_STEP - 1) / KR_STEP, 0);
        const int32_t* const table = a.c.table + (size_t)u.e.x * a.c.max_blocks;
        auto block_of = [&](int j) {
            const int pos = u.base + j * KR_STEP + tile * KV4_TILE;
            return pos < u.hi ? __ldcg(table + (pos >> a.c.block_shift)) : 0;
        };
        uint2 code[NG];
        uint4 par[NG];
        auto read = [&](int j, int id) {        // what is not there is zeros
            const int pos = u.base + j * KR_STEP + tile * KV4_TILE;
            const bool there = pos < u.hi;
            if ((unsigned)id >= (unsigned)a.c.n_blocks) {
                if (lane == 0) atomicOr(a.c.flag, KV4_BAD_BLOCK);
                id = 0;
            }
            const unsigned char* const at = a.c.pool + ((size_t)((long long)id * a.c.n_kv + u.head) * tiles + ((pos & ((1 << a.c.block_shift) - 1)) >> 4)) * (NG * KV4_GT);
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                code[i] = make_uint2(0, 0);
                par[i] = make_uint4(0, 0, 0, 0);
                if (!there) continue;
                code[i] = __ldcg(reinterpret_cast<const uint2*>(at + i * KV4_GT + (value ? KV4_VCODE : 0) + lane * 8));
                if (value) {
                    par[i] = __ldcg(reinterpret_cast<const uint4*>(at + i * KV4_GT + KV4_VPAR + t * 16));      // of keys 2t, 2t+8, 2t+1, 2t+9
                } else {
                    const uint2 p = __ldcg(reinterpret_cast<const uint2*>(at + i * KV4_GT + KV4_KPAR + g * 8));
                    par[i].x = p.x;
                    par[i].y = p.y;
                }
            }
        };
        auto fill = [&](uint4* to) {
            to += (value ? HALF : 0) + tile * (NG * 64) + lane;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                uint32_t x[4], y[4];
                if (value) {
                    const __half2 s0 = as_h2(__byte_perm(par[i].x, par[i].z, 0x5410)), z0 = as_h2(__byte_perm(par[i].x, par[i].z, 0x7632));
                    const __half2 s8 = as_h2(__byte_perm(par[i].y, par[i].w, 0x5410)), z8 = as_h2(__byte_perm(par[i].y, par[i].w, 0x7632));
                    kv4_values(code[i].x, s0, z0, s8, z8, x);
                    kv4_values(code[i].y, s0, z0, s8, z8, y);
                    to[i * 64] = make_uint4(x[0], x[2], x[1], x[3]);           // elements 4 g, then 4 g + 1 of keys 2t, 2t+1 and 2t+8, 2t+9
                    to[i * 64 + 32] = make_uint4(y[0], y[2], y[1], y[3]);      // elements 4 g + 2, then 4 g + 3
                } else {
                    const __half2 s0 = __low2half2(as_h2(par[i].x)), z0 = __high2half2(as_h2(par[i].x));
                    const __half2 s8 = __low2half2(as_h2(par[i].y)), z8 = __high2half2(as_h2(par[i].y));
                    kv4_values(code[i].x, s0, z0, s0, z0, x);
                    kv4_values(code[i].y, s8, z8, s8, z8, y);
                    to[i * 64] = make_uint4(x[0], x[1], x[2], x[3]);           // elements 8 t .. 8 t + 7 of key g
                    to[i * 64 + 32] = make_uint4(y[0], y[1], y[2], y[3]);      // of key g + 8
                }
            }
        };
        int id = block_of(0);
        read(0, id);
        id = block_of(1);

        // the lane's two columns: queries (times a power of two, so that the largest element lies in [1, 2): exact in f16 but for elements 2^14
        // times smaller), the last position seen
        uint32_t q[NG][8];
        float factor[2], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[NG][4][4];
        int limit[2], row[2], head[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int c = first + mine + 8 * r;
            const bool there = mine + 8 * r < cols;
            row[r] = there ? by_group(a, c) : 0;
            head[r] = u.head * a.group + (there ? c - row[r] * a.group : 0);
            limit[r] = there ? min(u.e.y + row[r], u.hi - 1) : -1;
            const uint4* const src = reinterpret_cast<const uint4*>(a.q + (long long)(u.e.w + row[r]) * a.q_stride + head[r] * HD) + t;
            uint4 raw[NG];
            uint32_t big = 0;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                raw[i] = make_uint4(0, 0, 0, 0);
                if (there) raw[i] = __ldcg(src + i * 4);
                big = max(big, most_bits(raw[i]));
            }
            big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
            big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
            const int e = min(max((int)(big >> 7), 1), 253);
            const float down = __int_as_float((254 - e) << 23), up = __int_as_float(e << 23);
            factor[r] = score_factor(a.scale_log2 * up, big);
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const uint32_t v[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                for (int j = 0; j < 4; ++j)      // elements 8 t + 2 j: first or second half of the first (j < 2) or second product's k
                    q[i][(j >> 1) * 4 + (j & 1) * 2 + r] = pack_h2(__uint_as_float(v[j] << 16) * down, __uint_as_float(v[j] & 0xffff0000u) * down);
            }
        }
#pragma unroll
        for (int i = 0; i < NG; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j][0] = acc[i][j][1] = acc[i][j][2] = acc[i][j][3] = 0.f;
        }
        // the last position that some, and that every, column of the warp sees (a split need not end with a step)
        const int some = warp * 16 < cols ? min(u.e.y + by_group(a, first + min(warp * 16 + 15, cols - 1)), u.hi - 1) : -1;
        const int every = min(u.e.y + by_group(a, first + warp * 16), u.hi - 1);

        for (int j = 0; j < steps; ++j) {
            uint4* const at = ring + buffer * (2 * HALF);
            buffer ^= 1;
            fill(at);
            __syncthreads();
            if (j + 1 < steps) {
                read(j + 1, id);
                id = block_of(j + 2);
            }
            const int base = u.base + j * KR_STEP;
            if (base > some) continue;
            const uint4* const keys = at + lane;
            float s[4][2][4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int h = 0; h < 2; ++h) s[k][h][0] = s[k][h][1] = s[k][h][2] = s[k][h][3] = 0.f;
            }
#pragma unroll
            for (int i = 0; i < NG; ++i) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint4 b = keys[(k * NG + i) * 64], d = keys[(k * NG + i) * 64 + 32];
                    mma16816(s[k][0], q[i][0], q[i][1], q[i][2], q[i][3], b.x, b.y);
                    mma16816(s[k][1], q[i][0], q[i][1], q[i][2], q[i][3], d.x, d.y);
                    mma16816(s[k][0], q[i][4], q[i][5], q[i][6], q[i][7], b.z, b.w);
                    mma16816(s[k][1], q[i][4], q[i][5], q[i][6], q[i][7], d.z, d.w);
                }
            }
            if (base + KR_STEP - 1 > every) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            if (base + k * KV4_TILE + h * 8 + 2 * t + (x & 1) > limit[x >> 1]) s[k][h][x] = -INFINITY;
                    }
                }
            }
            float top[2] = {s[0][0][0], s[0][0][2]};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    top[0] = fmaxf(fmaxf(top[0], s[k][h][0]), s[k][h][1]);
                    top[1] = fmaxf(fmaxf(top[1], s[k][h][2]), s[k][h][3]);
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
            }
            if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float best = fmaxf(m[r], top[r]), old = best == -INFINITY ? 1.f : ex2((m[r] - best) * factor[r]);
                    m[r] = best;
                    l[r] *= old;
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            acc[i][x][2 * r] *= old;
                            acc[i][x][2 * r + 1] *= old;
                        }
                    }
                }
            }
            const float less[2] = {m[0] == -INFINITY ? 0.f : -m[0], m[1] == -INFINITY ? 0.f : -m[1]};     // nothing seen yet: weights of exp(-inf) = 0
            const uint4* const values = at + HALF + lane;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t p[4];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        float &u0 = s[k][h][2 * r], &u1 = s[k][h][2 * r + 1];
                        u0 += less[r];
                        u1 += less[r];
                        lifted2(u0, u1, factor[r], factor[r]);
                        u0 = ex2(u0);
                        u1 = ex2(u1);
                        l[r] += u0;
                        l[r] += u1;
                    }
                    p[2 * h] = pack_h2(s[k][h][0], s[k][h][1]);
                    p[2 * h + 1] = pack_h2(s[k][h][2], s[k][h][3]);
                }
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    const uint4 b = values[(k * NG + i) * 64], d = values[(k * NG + i) * 64 + 32];
                    mma16816(acc[i][0], p[0], p[1], p[2], p[3], b.x, b.y);
                    mma16816(acc[i][1], p[0], p[1], p[2], p[3], b.z, b.w);
                    mma16816(acc[i][2], p[0], p[1], p[2], p[3], d.x, d.y);
                    mma16816(acc[i][3], p[0], p[1], p[2], p[3], d.z, d.w);
                }
            }
        }
        // the lane's elements 8 t .. 8 t + 7 of every group: column 2 t of product x is element 8 t + x, column 2 t + 1 element 8 t + 4 + x
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
            if (mine + 8 * r >= cols) continue;
            const size_t place = (size_t)u.w * KR_COLS + mine + 8 * r;
            const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
            if (u.splits > 1 && t == 0) a.ml[place] = make_float2(m[r] * factor[r], l[r]);
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                if (u.splits > 1) {
                    float4* const dst = reinterpret_cast<float4*>(a.acc + place * HD + i * KV4_GROUP + t * 8);
                    dst[0] = make_float4(acc[i][0][2 * r], acc[i][1][2 * r], acc[i][2][2 * r], acc[i][3][2 * r]);
                    dst[1] = make_float4(acc[i][0][2 * r + 1], acc[i][1][2 * r + 1], acc[i][2][2 * r + 1], acc[i][3][2 * r + 1]);
                } else {
                    uint32_t w[4];
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int half = 2 * r + (x >> 1), of = x % 2 * 2;
                        const __nv_bfloat162 h = __floats2bfloat162_rn(acc[i][of][half] * inv, acc[i][of + 1][half] * inv);
                        w[x] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    *reinterpret_cast<uint4*>(a.out + (long long)(u.e.w + row[r]) * a.out_stride + head[r] * HD + i * KV4_GROUP + t * 8) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
        __syncwarp();
    }
}

// Adds up the splits of every row that has more than one: a warp, or 8, a (row, query head).  Split i belongs to class i % 32; a class adds
// its splits in order, and the classes are added in order, so that a row's bits do not depend on the number of warps, which goes by
// the cache's size: with up to 32 splits one warp, as each class then has one member at most.
// Where a row's parts lie is read from the plan before the kernel in front, the attention, has ended: that one starts its successors when
// the plan is done.  Every way out waits for it, because what comes next waits for this kernel alone.  Latency bound: 3 to 5 us.
template <int NG, int WARPS>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) k_kv4_merge(const Kv4AttnArgs a, const int cols) {
    constexpr int HD = NG * KV4_GROUP, CLASSES = 32 / WARPS;
    __shared__ float part_acc[WARPS == 1 ? 1 : 32][HD];
    __shared__ float2 part_ml[WARPS == 1 ? 1 : 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, heads = a.c.n_kv * a.group;
    const long long id = WARPS == 1 ? (long long)blockIdx.x * 4 + warp : blockIdx.x;
    if (a.early) pdl_launch();
    const int row = (int)(id / heads), head = (int)(id % heads), kv = by_group(a, head);
    const int entry = row < a.n_rows ? __ldcg(a.row_entry + row) : -1;
    const int4 e = entry >= 0 ? __ldcg(a.entries + entry) : make_int4(0, 0, 0, 0);
    const long long unit = entry >= 0 ? __ldcg(a.cu_units + entry) : 0;
    const int all = a.split.parts((long long)e.y + e.z);
    if (all <= 1) return pdl_wait();
    const int own = (e.y + row - e.w) / a.split.of((long long)e.y + e.z) + 1;        // splits that the row sees
    const int c = (row - e.w) * a.group + head - kv * a.group;
    const long long w = unit * a.c.n_kv + ((long long)(c / cols) * a.c.n_kv + kv) * all;
    const float2* ml = a.ml + w * cols + c % cols;
    const float* acc = a.acc + (size_t)(w * cols + c % cols) * HD + lane * NG;
    const size_t step = (size_t)cols * HD;
    __nv_bfloat16* dst = a.out + (long long)row * a.out_stride + head * HD;
    float best = -INFINITY, sum = 0.f, out[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) out[j] = 0.f;
    pdl_wait();
    if constexpr (WARPS == 1) {
        const float2 mine = lane < own ? __ldcg(ml + (size_t)lane * cols) : make_float2(-INFINITY, 0.f);
        float v[8][NG];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
#pragma unroll
            for (int j = 0; j < NG; ++j) v[k][j] = k < own ? __ldcg(acc + k * step + j) : 0.f;
        }
        best = mine.x;
#pragma unroll
        for (int o = 16; o; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
        const float f = ex2(mine.x - (best == -INFINITY ? 0.f : best)), l = __fmul_rn(f, mine.y);
        for (int i = 0; i < own; i += 8) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float fk = __shfl_sync(0xffffffffu, f, i + k);
                sum = __fadd_rn(sum, __shfl_sync(0xffffffffu, l, i + k));
#pragma unroll
                for (int j = 0; j < NG; ++j) out[j] = __fadd_rn(out[j], __fmul_rn(fk, v[k][j]));
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
#pragma unroll
                for (int j = 0; j < NG; ++j) v[k][j] = i + 8 + k < own ? __ldcg(acc + (i + 8 + k) * step + j) : 0.f;
            }
        }
    } else {
        float2 st[CLASSES];     // of a class: maximum and sum
        float o[CLASSES][NG];
#pragma unroll
        for (int k = 0; k < CLASSES; ++k) {
            const int i = warp * CLASSES + k;
            st[k] = i < own ? __ldcg(ml + (size_t)i * cols) : make_float2(-INFINITY, 0.f);
#pragma unroll
            for (int j = 0; j < NG; ++j) o[k][j] = i < own ? __ldcg(acc + i * step + j) : 0.f;
        }
#pragma unroll 2
        for (int first = warp * CLASSES + 32; first < own; first += 32) {
            float2 p[CLASSES];
            float v[CLASSES][NG];
#pragma unroll
            for (int k = 0; k < CLASSES; ++k) {
                const int i = first + k;
                p[k] = i < own ? __ldcg(ml + (size_t)i * cols) : make_float2(-INFINITY, 0.f);
#pragma unroll
                for (int j = 0; j < NG; ++j) v[k][j] = i < own ? __ldcg(acc + i * step + j) : 0.f;
            }
#pragma unroll
            for (int k = 0; k < CLASSES; ++k) {
                const float top = fmaxf(st[k].x, p[k].x), now = top == -INFINITY ? 0.f : top;
                const float f0 = ex2(st[k].x - now), f1 = ex2(p[k].x - now);
                st[k] = make_float2(top, f0 * st[k].y + f1 * p[k].y);
#pragma unroll
                for (int j = 0; j < NG; ++j) o[k][j] = f0 * o[k][j] + f1 * v[k][j];
            }
        }
#pragma unroll
        for (int k = 0; k < CLASSES; ++k) {
            if (lane == 0) part_ml[warp * CLASSES + k] = st[k];
#pragma unroll
            for (int j = 0; j < NG; ++j) part_acc[warp * CLASSES + k][lane * NG + j] = o[k][j];
        }
        __syncthreads();
        if (warp) return;
        const float2 mine = part_ml[lane];
        best = mine.x;
#pragma unroll
        for (int k = 16; k; k >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, k));
        const float f = ex2(mine.x - (best == -INFINITY ? 0.f : best)), l = __fmul_rn(f, mine.y);
#pragma unroll 8
        for (int k = 0; k < 32; ++k) {
            const float fk = __shfl_sync(0xffffffffu, f, k);
            sum = __fadd_rn(sum, __shfl_sync(0xffffffffu, l, k));
#pragma unroll
            for (int j = 0; j < NG; ++j) out[j] = __fadd_rn(out[j], __fmul_rn(fk, part_acc[k][lane * NG + j]));
        }
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < NG; ++j) dst[lane * NG + j] = __float2bfloat16_rn(out[j] * inv);
}

}  // namespace vuik
