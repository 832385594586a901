// Attention over the paged 4-bit cache (layout: kv4_kernels.cuh).  With V and K the values that the codes stand for, row r of a
// sequence at position p and query head j:  out = sum_{i <= p} softmax_i(scale q . K_i) V_i,  K and V of kv head j / group.
#pragma once
#include "kv4_kernels.cuh"

namespace vuik {

constexpr int KA_THREADS = 128, KA_WARPS = 4;

struct Kv4AttnArgs {
    Kv4Cache c;
    const int4* entries; const int32_t* cu_rows; const int32_t* cu_units;
    int n, n_rows, group, split;
    const __nv_bfloat16* q; long long q_stride;
    __nv_bfloat16* out; long long out_stride;
    float scale_log2;                          // scale * log2(e)
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
    asm volatile("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// The eight codes of a word as four pairs of the values that they stand for.  A nibble under the exponent of 1024 is 1024 + c, one
// that sits four bits higher 1024 + 16 c: both are exact in f16, and so is what is left when 1024 is taken off again.
__device__ __forceinline__ void kv4_values(uint32_t w, uint32_t s, uint32_t z, uint32_t (&r)[4]) {
    const uint32_t v = w >> 8;
    uint32_t x[4];
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(x[0]) : "r"(w));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(x[1]) : "r"(w));
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(x[2]) : "r"(v));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x64006400, 0xea;" : "=r"(x[3]) : "r"(v));
    const __half2 hs = *reinterpret_cast<const __half2*>(&s), hz = *reinterpret_cast<const __half2*>(&z);
    const __half2 low = __half2half2(__ushort_as_half(0xE400)), sixteenth = __half2half2(__ushort_as_half(0x2C00)),
                  less = __half2half2(__ushort_as_half(0xD400));   // -1024, 1 / 16, -64
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __half2 h = *reinterpret_cast<const __half2*>(&x[j]);
        const __half2 code = j & 1 ? __hfma2(h, sixteenth, less) : __hadd2(h, low);
        const __half2 value = __hfma2(hs, code, hz);
        r[j] = *reinterpret_cast<const uint32_t*>(&value);
    }
}

// A unit: a tile of columns of one sequence (its rows times the query heads of a kv head, COLS at a time), a kv head, a split of the
// positions.  Units lie in the order sequence, column tile, kv head, split.  What the consumers are told of one, a stage at a time:
struct __align__(16) Kv4Item {
    int flags;                                  // KI_*
    int start, rows, row0;                      // the sequence's first new position, its rows, the first of them
    int ctile, head, splits, base;              // base: position of the stage's first key
    int hi, pad;                                // one past the last position of the stage that any column of the tile sees
    long long w;                                // number of the unit times kv heads: where its partial sums go
};
constexpr int KI_FIRST = 1, KI_LAST = 2, KI_QUERIES = 4, KI_END = 8;

struct Kv4Walk {       // the producer's place
    int entry, ctile, head, split, splits, base, hi;
    int4 e, next;      // this entry and, read ahead, the one behind it
};

template <int COLS>
__device__ __forceinline__ void walk_range(const Kv4AttnArgs& a, Kv4Walk& u) {
    u.base = u.split * a.split;
    const int end_row = (min((u.ctile + 1) * COLS, u.e.z * a.group) - 1) / a.group;
    u.hi = (int)min((long long)u.base + a.split, (long long)u.e.y + end_row + 1);
}

__device__ __forceinline__ void walk_enter(const Kv4AttnArgs& a, Kv4Walk& u, int4 e) {
    u.e = e;
    u.splits = (e.y + e.z + a.split - 1) / a.split;
    u.next = __ldcg(a.entries + min(u.entry + 1, a.n - 1));
}

// The place of work item w (< cu_units[n] * n_kv), found by the whole warp, 32 sequences' first units at a time.
template <int COLS>
__device__ __forceinline__ Kv4Walk walk_at(const Kv4AttnArgs& a, long long w, int lane) {
    Kv4Walk u;
    int lo = 0, hi = a.n;      // first unit of lo <= w < first unit of hi
    long long before = 0;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const long long first = at < hi ? (long long)__ldcg(a.cu_units + at) * a.c.n_kv : 0x7fffffffffffffffll;
        const int k = 31 - __clz(__ballot_sync(0xffffffffu, first <= w));
        before = __shfl_sync(0xffffffffu, first, k);
        lo += k * step;
        hi = min(hi, lo + step);
    }
    u.entry = lo;
    walk_enter(a, u, __ldcg(a.entries + lo));
    const long long off = w - before;
    u.split = (int)(off % u.splits);
    const long long rest = off / u.splits;
    u.head = (int)(rest % a.c.n_kv);
    u.ctile = (int)(rest / a.c.n_kv);
    walk_range<COLS>(a, u);
    return u;
}

// To the next unit.
template <int COLS>
__device__ __forceinline__ void walk_next(const Kv4AttnArgs& a, Kv4Walk& u) {
    if (++u.split == u.splits) {
        u.split = 0;
        if (++u.head == a.c.n_kv) {
            u.head = 0;
            if (++u.ctile * COLS >= u.e.z * a.group) {
                u.ctile = 0;
                while (++u.entry < a.n) {
                    walk_enter(a, u, u.next);
                    if (u.e.z) break;
                }
            }
        }
    }
    walk_range<COLS>(a, u);
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

// Shared memory of the mma.sync form, in bytes.
template <int NG, int NT>
struct KaShared {
    static constexpr int KT = NG == 2 ? 4 : 2;                                  // tiles of 16 positions a warp takes at once
    static constexpr int KEYS = KA_WARPS * KT * KV4_TILE;                         // positions of a stage
    static constexpr int TILE = NG * KV4_GT, QCOL = NG * KV4_GROUP * 2;
    static constexpr int KV = KA_WARPS * KT * TILE, Q = NT * 8 * QCOL;
    static constexpr int STAGE = KV + Q + (int)sizeof(Kv4Item);
    static constexpr int STAGES = 3;
    static constexpr int ACC = KA_WARPS * NT * 8 * (NG * KV4_GROUP + 4) * 4, ML = KA_WARPS * NT * 8 * 8;
    static constexpr int TOTAL = STAGES * STAGE + ACC + ML + 8 * (2 * STAGES + 2);
};

// mma.sync form: a producer warp walks the CTA's units and brings keys, values and queries into a ring of stages (bulk copies), four
// consumer warps take KT tiles of 16 positions each.  Keys are the A operand, queries the B operand (8 columns), so that one or a few
// query heads waste nothing but columns; the scores' transpose for the second product is one movmatrix a fragment.  Softmax statistics
// and sums are fp32; the weights enter the second product as f16 (2^-11 of each, where bf16's 2^-8 would be as much as the output's own
// rounding).
template <int NG, int NT>
__global__ void __launch_bounds__(KA_THREADS + 32) k_kv4_attn(const Kv4AttnArgs a) {
    using S = KaShared<NG, NT>;
    constexpr int HD = NG * KV4_GROUP, COLS = NT * 8, KT = S::KT, D = S::STAGES;
    extern __shared__ __align__(128) unsigned char smem[];
    float* const sm_acc = reinterpret_cast<float*>(smem + D * S::STAGE);                 // [warp][column][HD + 4]
    float2* const sm_ml = reinterpret_cast<float2*>(smem + D * S::STAGE + S::ACC);       // [warp][column]
    const uint32_t bars = smem_addr(smem + D * S::STAGE + S::ACC + S::ML);
    auto full = [&](int s) { return bars + 8 * s; };
    auto empty = [&](int s) { return bars + 8 * (D + s); };
    const uint32_t acc_full = bars + 16 * D, acc_empty = acc_full + 8;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    if (threadIdx.x == 0) {
        for (int s = 0; s < D; ++s) { bar_init(full(s), 1); bar_init(empty(s), KA_WARPS); }
        bar_init(acc_full, KA_WARPS);
        bar_init(acc_empty, KA_WARPS);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    const int tiles = 1 << (a.c.block_shift - 4);     // of a block
    pdl_wait();
    pdl_launch();

    if (warp == KA_WARPS) {
        const long long total = (long long)__ldcg(a.cu_units + a.n) * a.c.n_kv;
        long long w = total * blockIdx.x / gridDim.x;
        const long long last = total * (blockIdx.x + 1) / gridDim.x;
        Kv4Walk u = {};
        int id = 0;     // the lane's tile's block
        auto block_of = [&]() {
            const int pos = u.base + lane * KV4_TILE;
            return lane < KA_WARPS * KT && pos < u.hi ? __ldcg(a.c.table + (size_t)u.e.x * a.c.max_blocks + (pos >> a.c.block_shift)) : 0;
        };
        bool queries = true, begins = true;
        if (w < last) {
            u = walk_at<COLS>(a, w, lane);
            id = block_of();
        }
        const int run = min(tiles, KA_WARPS * KT);    // tiles that lie behind one another
        for (unsigned k = 0;; ++k) {
            const int s = k % D;
            if (k >= D && !bar_wait(empty(s), (k / D - 1) & 1)) { give_up(a.c.flag); return; }
            unsigned char* const stage = smem + s * S::STAGE;
            Kv4Item* const item = reinterpret_cast<Kv4Item*>(stage + S::KV + S::Q);
            if (w >= last) {
                if (lane == 0) {
                    item->flags = KI_END;
                    bar_arrive(full(s));
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
                d.hi = u.hi; d.pad = 0; d.w = w;
                *item = d;
                bar_expect(full(s), valid * S::TILE + (queries ? cols * S::QCOL : 0));
            }
            __syncwarp();
            const int pos = u.base + lane * KV4_TILE;
            if (lane < valid && lane % run == 0) {
                const unsigned char* src = a.c.pool + ((size_t)((long long)id * a.c.n_kv + u.head) * tiles + ((pos & ((1 << a.c.block_shift) - 1)) >> 4)) * S::TILE;
                bulk_copy(smem_addr(stage + lane * S::TILE), src, min(run, valid - lane) * S::TILE, full(s));
            }
            if (queries && lane < cols) {     // the heads of a row lie behind one another
                const int c = u.ctile * COLS + lane, row = c / a.group, in = c % a.group;
                if (lane == 0 || in == 0)
                    bulk_copy(smem_addr(stage + S::KV + lane * S::QCOL), a.q + (long long)(u.e.w + row) * a.q_stride + (u.head * a.group + in) * HD,
                              min(a.group - in, cols - lane) * S::QCOL, full(s));
            }
            queries = false;
            begins = ends;
            u.base += S::KEYS;
            if (ends) {
                if (++w < last) {
                    walk_next<COLS>(a, u);
                    queries = u.split == 0;
                }
            }
            if (w < last) id = block_of();
        }
    }

    uint32_t qf[NT][NG][4];
    float factor[NT][2];
    int limit[NT][2];       // last position that the column sees
    float acc[NT][2 * NG][4], m[NT][2], l[NT][2];
    unsigned merged = 0;
    for (unsigned k = 0;; ++k) {
        const int s = k % D;
        if (!bar_wait(full(s), (k / D) & 1)) { give_up(a.c.flag); return; }
        const unsigned char* const stage = smem + s * S::STAGE;
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
                const float f = a.scale_log2 * up;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const int c2 = nt * 8 + 2 * t + j;
                    factor[nt][j] = __shfl_sync(0xffffffffu, f, (2 * t + j) * 4);
                    limit[nt][j] = c2 < cols ? d.start + (d.ctile * COLS + c2) / a.group : -1;
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
        const int base = d.base + warp * (KT * KV4_TILE);
        const int nk = min(KT, (d.hi - base + KV4_TILE - 1) / KV4_TILE);    // tiles that are there
        if (nk > 0) {
            const unsigned char* const mine = stage + warp * (KT * S::TILE);
            const bool whole = base + KT * KV4_TILE - 1 <= d.start + d.ctile * COLS / a.group;   // every column sees all of them
            float sc[KT][NT][4];
#pragma unroll
            for (int k2 = 0; k2 < KT; ++k2) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) sc[k2][nt][0] = sc[k2][nt][1] = sc[k2][nt][2] = sc[k2][nt][3] = 0.f;
                if (k2 < nk) {
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        const unsigned char* p = mine + k2 * S::TILE + i * KV4_GT;
                        const uint2 code = *reinterpret_cast<const uint2*>(p + lane * 8);
                        const uint2 par = *reinterpret_cast<const uint2*>(p + KV4_KPAR + g * 8);
                        uint32_t x[4], y[4];
                        kv4_values(code.x, __byte_perm(par.x, 0, 0x1010), __byte_perm(par.x, 0, 0x3232), x);
                        kv4_values(code.y, __byte_perm(par.y, 0, 0x1010), __byte_perm(par.y, 0, 0x3232), y);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816(sc[k2][nt], x[0], y[0], x[1], y[1], qf[nt][i][0], qf[nt][i][1]);
                            mma16816(sc[k2][nt], x[2], y[2], x[3], y[3], qf[nt][i][2], qf[nt][i][3]);
                        }
                    }
                }
            }
            uint32_t p[KT][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int k2 = 0; k2 < KT; ++k2) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        sc[k2][nt][j] *= factor[nt][j & 1];
                        if (!whole && base + k2 * 16 + g + (j >> 1) * 8 > limit[nt][j & 1]) sc[k2][nt][j] = -INFINITY;
                        top[j & 1] = fmaxf(top[j & 1], sc[k2][nt][j]);
                    }
                }
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
                    top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
                }
                float now[2];
                if (__any_sync(0xffffffffu, top[0] > m[nt][0] || top[1] > m[nt][1])) {
                    float old[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float best = fmaxf(m[nt][j], top[j]);
                        old[j] = best == -INFINITY ? 1.f : ex2(m[nt][j] - best);
                        m[nt][j] = best;
                        l[nt][j] *= old[j];
                    }
#pragma unroll
                    for (int i = 0; i < 2 * NG; ++i) {
                        acc[nt][i][0] *= old[0]; acc[nt][i][1] *= old[1];
                        acc[nt][i][2] *= old[0]; acc[nt][i][3] *= old[1];
                    }
                }
#pragma unroll
                for (int j = 0; j < 2; ++j) now[j] = m[nt][j] == -INFINITY ? 0.f : m[nt][j];    // nothing seen yet: weights of exp(-inf) = 0
#pragma unroll
                for (int k2 = 0; k2 < KT; ++k2) {
                    float e[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        e[j] = ex2(sc[k2][nt][j] - now[j & 1]);
                        l[nt][j & 1] += e[j];
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
                        const unsigned char* q = mine + k2 * S::TILE + i * KV4_GT;
                        const uint2 code = *reinterpret_cast<const uint2*>(q + KV4_VCODE + lane * 8);
                        const uint4 par = *reinterpret_cast<const uint4*>(q + KV4_VPAR + t * 16);
                        uint32_t x[4], y[4];
                        kv4_values(code.x, par.x, par.y, x);
                        kv4_values(code.y, par.z, par.w, y);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma16816(acc[nt][2 * i], x[0], x[1], y[0], y[1], p[k2][nt][0], p[k2][nt][1]);
                            mma16816(acc[nt][2 * i + 1], x[2], x[3], y[2], y[3], p[k2][nt][0], p[k2][nt][1]);
                        }
                    }
                }
            }
        }
        __syncwarp();
        if (lane == 0) bar_arrive(empty(s));
        if (!(d.flags & KI_LAST)) continue;
        // the warps' states, added in the order of the warps
        if (merged && !bar_wait(acc_empty, (merged - 1) & 1)) { give_up(a.c.flag); return; }
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
                    if (g == 0) sm_ml[warp * COLS + col] = make_float2(m[nt][j], l[nt][j]);
#pragma unroll
                    for (int i = 0; i < NG; ++i)
                        *reinterpret_cast<float4*>(sm_acc + (warp * COLS + col) * (HD + 4) + i * KV4_GROUP + 4 * g) =
                            make_float4(acc[nt][2 * i][j], acc[nt][2 * i][2 + j], acc[nt][2 * i + 1][j], acc[nt][2 * i + 1][2 + j]);
                }
            }
        }
        __syncwarp();
        if (lane == 0) bar_arrive(acc_full);
        if (!bar_wait(acc_full, merged & 1)) { give_up(a.c.flag); return; }
        for (int i = threadIdx.x; i < min(cols, COLS) * (HD / 4); i += KA_THREADS) {
            const int col = i / (HD / 4), dim = i % (HD / 4) * 4;
            float best = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k2 = 0; k2 < KA_WARPS; ++k2) best = fmaxf(best, sm_ml[k2 * COLS + col].x);
            const float now = best == -INFINITY ? 0.f : best;
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k2 = 0; k2 < KA_WARPS; ++k2) {
                const float2 part = sm_ml[k2 * COLS + col];
                const float f = ex2(part.x - now);
                const float4 v = *reinterpret_cast<const float4*>(sm_acc + (k2 * COLS + col) * (HD + 4) + dim);
                sum += f * part.y;
                o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
            }
            if (d.splits == 1) {
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
                const int c = d.ctile * COLS + col;
                __nv_bfloat162 lo2 = __floats2bfloat162_rn(o.x * inv, o.y * inv), hi2 = __floats2bfloat162_rn(o.z * inv, o.w * inv);
                uint2 v = make_uint2(*reinterpret_cast<uint32_t*>(&lo2), *reinterpret_cast<uint32_t*>(&hi2));
                *reinterpret_cast<uint2*>(a.out + (long long)(d.row0 + c / a.group) * a.out_stride + (d.head * a.group + c % a.group) * HD + dim) = v;
            } else {
                *reinterpret_cast<float4*>(a.acc + (size_t)(d.w * COLS + col) * HD + dim) = o;
                if (dim == 0) a.ml[d.w * COLS + col] = make_float2(best, sum);
            }
        }
        __syncwarp();
        if (lane == 0) bar_arrive(acc_empty);
        ++merged;
    }
}

// Adds up the splits of every row that has more than one, in the order of the positions: a warp a (row, query head).
template <int NG>
__global__ void __launch_bounds__(256) k_kv4_merge(const Kv4AttnArgs a, const int cols) {
    constexpr int HD = NG * KV4_GROUP;
    const int lane = threadIdx.x & 31, heads = a.c.n_kv * a.group;
    const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    pdl_wait();
    pdl_launch();
    const int row = (int)(id / heads), head = (int)(id % heads), kv = head / a.group;
    if (row >= a.n_rows || row >= __ldcg(a.cu_rows + a.n)) return;
    int lo = 0, hi = a.n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (__ldcg(a.cu_rows + mid) <= row) lo = mid; else hi = mid;
    }
    const int4 e = __ldcg(a.entries + lo);
    const int all = (e.y + e.z + a.split - 1) / a.split;
    if (all == 1) return;
    const int own = (e.y + row - e.w) / a.split + 1;        // splits that the row sees
    const int c = (row - e.w) * a.group + head % a.group;
    const long long w = (long long)__ldcg(a.cu_units + lo) * a.c.n_kv + ((long long)(c / cols) * a.c.n_kv + kv) * all;
    const float2* ml = a.ml + w * cols + c % cols;
    const float* acc = a.acc + (size_t)(w * cols + c % cols) * HD + lane * NG;
    float best = -INFINITY;
    for (int i = lane; i < own; i += 32) best = fmaxf(best, __ldcg(&ml[(size_t)i * cols].x));
#pragma unroll
    for (int o = 16; o; o >>= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
    const float now = best == -INFINITY ? 0.f : best;
    float sum = 0.f, out[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) out[j] = 0.f;
#pragma unroll 4
    for (int i = 0; i < own; ++i) {
        const float2 part = __ldcg(ml + (size_t)i * cols);
        const float f = ex2(part.x - now);
        sum += f * part.y;
#pragma unroll
        for (int j = 0; j < NG; ++j) out[j] += f * __ldcg(acc + (size_t)i * cols * HD + j);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int j = 0; j < NG; ++j) a.out[(long long)row * a.out_stride + head * HD + lane * NG + j] = __float2bfloat16_rn(out[j] * inv);
}

}  // namespace vuik
