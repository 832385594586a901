// Attention of many columns (chunks of prompts) over the paged 4-bit cache, on the 5th-generation tensor cores.
//
// A CTA takes 256 columns (a sequence's rows times the query heads of a kv head) of one kv head as two tiles of 128, and walks the
// positions 128 at a time:
//   * 8 warps read codes from the cache (half a step ahead, in registers) and write keys and values as f16 into a ring of shared-memory
//     tiles that both tiles of columns share: keys [position][dim], values [dim][position], both K-major with the 128-byte swizzle;
//   * one thread issues tcgen05.mma: S = Q K^T (128 x 128, K = head_dim) and O += P V (A = P from tensor memory, K = 128 positions);
//   * 4 warps a tile, one thread a column: exponentials, their sum, and P as f16 back into tensor memory over S.
// Weights are taken against a reference, the first maximum that a column meets: below 2^14 of it they fit f16 and the sums all the same, so
// that a step needs no maximum before it weighs; it looks for it meanwhile.  A step that carries a column beyond 2^14 is taken again: the
// scores are computed anew (the keys are kept until the step is accepted), the column's sums corrected, each column's by its own maximum, so
// that its bits are its own.
// While one tile's softmax runs, the tensor cores work on the other.  Per step of 128 positions and two tiles at head_dim 128 the tensor
// cores take 2048 cycles, the exponentials (16 a clock) 2048, the issue slots about 1700.
// Every wait is bounded; a role that gives up leaves its loop, and all warps meet before tensor memory is freed.
#pragma once
#include "kv4_attn.cuh"

namespace vuik {

constexpr int KC_TILE = 128;
constexpr int KC_FILL = 8, KC_WARPS = 17, KC_THREADS = KC_WARPS * 32;      // warps 0-7 fill, 8-11 and 12-15 softmax, 16 MMA

template <int NG>
struct KcShared {
    static constexpr int HD = NG * KV4_GROUP, NB = (HD + 63) / 64;
    static constexpr int BLOCK = 128 * 128;                // 128 rows of 128 bytes
    static constexpr int Q = NB * BLOCK, SLOT = NB * BLOCK; // of a tile of columns; of a tile of keys or values
    static constexpr int SLOTS = 4;
    static constexpr int BARS = 2 * Q + SLOTS * SLOT;
    static constexpr int TOTAL = BARS + 256 + 1024;        // and room to start at a multiple of 1024
    // Columns of tensor memory: the tiles' scores, 128 each; their sums, HD each; weights (two f16 a column) behind them where there is
    // room, else over the scores that they came from.
    static constexpr bool APART = HD == 64;
    __host__ __device__ static constexpr uint32_t weights(int x) { return APART ? 256 + 2 * HD + x * (KC_STEP / 2) : x * KC_TILE; }
};

// The CTAs share out all steps of all column tiles and kv heads evenly, in the order sequence, column tile, kv head, step.  A run is what a
// CTA has of one (column tile, kv head): all its steps, and the output is written; or a part, and its sums go to one of the CTA's two places
// for parts (the first if the run goes on from the CTA before, the second if it begins here).
struct KcRun {
    int entry, ctile, head, cost, from, to, steps[2];   // of the tiles: steps to take; cost: steps of the whole (tile, head)
    int4 e;
    long long at, end;      // work before the run, and where the CTA's share ends
};

__device__ __forceinline__ void kc_enter(const Kv4AttnArgs& a, KcRun& u, int from) {
    u.cost = kc_cost(u.e.y, u.e.z, a.group, u.ctile);
    u.from = from;
    u.to = (int)min((long long)u.cost, from + u.end - u.at);
    const int all = u.e.z * a.group, first = u.ctile * KC_COLS;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
        const int end = min(first + (x + 1) * KC_TILE, all);          // one past the tile's last column
        const int sees = end > first + x * KC_TILE ? (u.e.y + by_group(a, end - 1) + KC_STEP) / KC_STEP : 0;
        u.steps[x] = max(min(u.to, sees) - u.from, 0);
    }
}

// The run that begins with step number `at` of all, found by the whole warp.
__device__ __forceinline__ bool kc_find(const Kv4AttnArgs& a, KcRun& u, long long at, long long end, int lane) {
    u.at = at;
    u.end = end;
    int lo = 0, hi = a.n;      // work before lo <= at < work before hi
    long long before = 0;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, i = lo + lane * step;
        const long long work = i < hi ? (long long)__ldcg(a.cu_work + i) * a.c.n_kv : 0x7fffffffffffffffll;
        const int k = 31 - __clz(__ballot_sync(0xffffffffu, work <= u.at));
        before = __shfl_sync(0xffffffffu, work, k);
        lo += k * step;
        hi = min(hi, lo + step);
    }
    u.entry = lo;
    u.e = __ldcg(a.entries + lo);
    long long into = u.at - before;      // and now the column tile, 32 at a time
    for (u.ctile = 0;; u.ctile += 32) {
        const int t = u.ctile + lane;
        const long long mine = t * KC_COLS < u.e.z * a.group ? (long long)kc_cost(u.e.y, u.e.z, a.group, t) * a.c.n_kv : 0;
        long long sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        const unsigned past = __ballot_sync(0xffffffffu, sum > into);
        if (past) {
            const int k = __ffs(past) - 1;
            into -= __shfl_sync(0xffffffffu, sum - mine, k);
            u.ctile += k;
            break;
        }
        into -= __shfl_sync(0xffffffffu, sum, 31);
        if ((u.ctile + 32) * KC_COLS >= u.e.z * a.group) return false;      // not reached: the entry's work is the sum of its tiles'
    }
    const int cost = kc_cost(u.e.y, u.e.z, a.group, u.ctile);
    u.head = (int)(into / cost);
    kc_enter(a, u, (int)(into % cost));
    return true;
}

__device__ __forceinline__ bool kc_begin(const Kv4AttnArgs& a, KcRun& u, int lane) {
    const long long total = (long long)__ldcg(a.cu_work + a.n) * a.c.n_kv;
    const long long at = total * blockIdx.x / gridDim.x, end = total * (blockIdx.x + 1) / gridDim.x;
    return at < end && kc_find(a, u, at, end, lane);
}

__device__ __forceinline__ bool kc_next(const Kv4AttnArgs& a, KcRun& u) {
    u.at += u.to - u.from;
    if (u.at >= u.end) return false;
    if (++u.head == a.c.n_kv) {
        u.head = 0;
        if (++u.ctile * KC_COLS >= u.e.z * a.group) {
            u.ctile = 0;
            do {
                if (++u.entry >= a.n) return false;
                u.e = __ldcg(a.entries + u.entry);
            } while (u.e.z == 0);
        }
    }
    kc_enter(a, u, 0);
    return true;
}

struct KcBars {
    uint32_t at;
    __device__ __forceinline__ uint32_t q_full(int x) const { return at + 8 * x; }
    __device__ __forceinline__ uint32_t s_full(int x) const { return at + 16 + 8 * x; }
    __device__ __forceinline__ uint32_t p_full(int x) const { return at + 32 + 8 * x; }
    __device__ __forceinline__ uint32_t kv_full(int s) const { return at + 48 + 8 * s; }
    __device__ __forceinline__ uint32_t kv_empty(int s) const { return at + 80 + 8 * s; }
    __device__ __forceinline__ uint32_t tmem() const { return at + 112; }
    __device__ __forceinline__ uint32_t summed(int x) const { return at + 128 + 8 * x; }
    __device__ __forceinline__ uint32_t again(int x) const { return at + 116 + 4 * x; }     // the round of P whose step is to be taken again
};

__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}
// Low word of the descriptor of a K-major tile with the 128-byte swizzle (rows 128 bytes apart, groups of 8 rows 1024); the high word is the
// same for all.  The tensor pipe has next to no queue, so what the issuing thread spends on descriptors the pipe waits for: four MMAs (64 of
// K) are one block that adds to 32-bit words.
__device__ __forceinline__ uint32_t tile_desc(uint32_t addr) { return (addr >> 4 & 0x3FFF) | 1u << 16; }
constexpr uint32_t KC_DESC_HI = (1024u >> 4) | 1u << 14 | 2u << 29;
// f16 operands, fp32 sums, both K-major, 128 rows, n columns.
__host__ __device__ constexpr uint32_t kc_idesc(int n) { return 1u << 4 | (uint32_t)(n >> 3) << 17 | 8u << 24; }
// N (4 or 2) MMAs of 16 of K with A from shared memory; the first adds to D unless FIRST.
template <int N, bool FIRST>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#define KC_SS(off, p) "add.u32 t, %1, " off ";\n\tadd.u32 u, %2, " off ";\n\tmov.b64 x, {t, %3};\n\tmov.b64 y, {u, %3};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %4, " p ";\n\t"
    if constexpr (N == 4)
        asm volatile("{\n\t.reg .b64 x, y;\n\t.reg .b32 t, u;\n\t" KC_SS("0", "%5") KC_SS("2", "1") KC_SS("4", "1") KC_SS("6", "1") "}"
                     ::"r"(d), "r"(a), "r"(b), "r"(KC_DESC_HI), "r"(idesc), "n"(FIRST ? 0 : 1) : "memory");
    else
        asm volatile("{\n\t.reg .b64 x, y;\n\t.reg .b32 t, u;\n\t" KC_SS("0", "%5") KC_SS("2", "1") "}"
                     ::"r"(d), "r"(a), "r"(b), "r"(KC_DESC_HI), "r"(idesc), "n"(FIRST ? 0 : 1) : "memory");
#undef KC_SS
}
// Four MMAs of 16 of K with A from tensor memory (two f16 a column).
template <bool FIRST>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
#define KC_TS(aoff, boff, p) "add.u32 t, %1, " aoff ";\n\tadd.u32 u, %2, " boff ";\n\tmov.b64 y, {u, %3};\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [t], y, %4, " p ";\n\t"
    asm volatile("{\n\t.reg .b64 y;\n\t.reg .b32 t, u;\n\t" KC_TS("0", "0", "%5") KC_TS("8", "2", "1") KC_TS("16", "4", "1") KC_TS("24", "6", "1") "}"
                 ::"r"(d), "r"(a), "r"(b), "r"(KC_DESC_HI), "r"(idesc), "n"(FIRST ? 0 : 1) : "memory");
#undef KC_TS
}
#define KC_R32(r) "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), \
    "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),     \
    "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
// 32 columns of this thread's lane; they are there behind tm_wait().
__device__ __forceinline__ void tm_load32(uint32_t at, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,"
                 "%27,%28,%29,%30,%31}, [%32];" : KC_R32(r) : "r"(at));
}
__device__ __forceinline__ void tm_load16(uint32_t at, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(at));
}
// The wait names the registers, so that nothing that reads them moves in front of it.
#define KC_RW32(r) "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), \
    "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),      \
    "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
__device__ __forceinline__ void tm_wait(uint32_t (&r)[32]) { asm volatile("tcgen05.wait::ld.sync.aligned;" : KC_RW32(r)::"memory"); }
__device__ __forceinline__ void tm_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])::"memory");
}
__device__ __forceinline__ void tm_store8(uint32_t at, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ void tm_store16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tm_stored() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void sts32(uint32_t at, uint32_t v) { asm volatile("st.volatile.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ uint32_t lds32(uint32_t at) {
    uint32_t v;
    asm volatile("ld.volatile.shared.b32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t at, const uint32_t (&r)[4]) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}
// Four 8 x 8 matrices of 16-bit elements in fragment order; lane l says where row l % 8 of matrix l / 8 goes (16 bytes).
__device__ __forceinline__ void stmatrix4(uint32_t at, const uint32_t (&r)[4]) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]) : "memory");
}

// ---- the filling warps: warp w takes tile w of every 8 (of 16 positions)
template <int NG>
__device__ __forceinline__ void kc_fill(const Kv4AttnArgs& a, uint32_t ring, const KcBars bars, int w, int lane) {
    using S = KcShared<NG>;
    const int g = lane >> 2, t = lane & 3, tiles = 1 << (a.c.block_shift - 4);
    // keys: row 16 w + g of the tile (and + 8, with the same low three bits); values: element 4 g + j of a group is row 8 j + g, so that the
    // eight rows of a matrix lie in eight different banks; lane l names row l % 8 of matrix l / 8: (j = 0, keys 0-7), (1, 0-7), (0, 8-15), (1, 8-15)
    const uint32_t key_row = (w * KV4_TILE + g) * 128, key_sw = g, val_sw = ((w & 3) * 2 + (lane >> 4)) ^ (lane & 7);
    const uint32_t val_row = (w >> 2) * (S::HD * 128) + ((lane >> 3 & 1) * 8 + (lane & 7)) * 128 + (val_sw << 4);
    KcRun u;
    unsigned n = 0;        // tiles written: keys and values in turn
    for (bool more = kc_begin(a, u, lane); more; more = kc_next(a, u)) {
        const int last = max(u.steps[0], u.steps[1]), base = u.from * KC_STEP + w * KV4_TILE, len = u.e.y + u.e.z;
        const int32_t* const table = a.c.table + (size_t)u.e.x * a.c.max_blocks;
        auto block_of = [&](int j) {
            const int pos = base + j * KC_STEP;
            return j < last && pos < len ? __ldcg(table + (pos >> a.c.block_shift)) : -1;
        };
        auto place = [&](int j, int b) -> const unsigned char* {
            const int pos = base + j * KC_STEP;
            if (j >= last || pos >= len) return nullptr;
            if ((unsigned)b >= (unsigned)a.c.n_blocks) {
                if (lane == 0) atomicOr(a.c.flag, KV4_BAD_BLOCK);
                b = 0;
            }
            return a.c.pool + ((size_t)((long long)b * a.c.n_kv + u.head) * tiles + ((pos & ((1 << a.c.block_shift) - 1)) >> 4)) * (NG * KV4_GT);
        };
        // what is not there is zeros: codes, scales and values
        uint2 kc[NG], kp[NG], vc[NG];
        uint4 vp[NG];
        auto read_keys = [&](const unsigned char* at) {
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                kc[i] = kp[i] = make_uint2(0, 0);
                if (at) {
                    kc[i] = __ldcg(reinterpret_cast<const uint2*>(at + i * KV4_GT + lane * 8));
                    kp[i] = __ldcg(reinterpret_cast<const uint2*>(at + i * KV4_GT + KV4_KPAR + g * 8));
                }
            }
        };
        auto read_values = [&](const unsigned char* at) {
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                vc[i] = make_uint2(0, 0);
                vp[i] = make_uint4(0, 0, 0, 0);
                if (at) {
                    vc[i] = __ldcg(reinterpret_cast<const uint2*>(at + i * KV4_GT + KV4_VCODE + lane * 8));
                    vp[i] = __ldcg(reinterpret_cast<const uint4*>(at + i * KV4_GT + KV4_VPAR + t * 16));   // of keys 2t, 2t+8, 2t+1, 2t+9
                }
            }
        };
        auto done = [&]() {
            fence_async();
            __syncwarp();
            if (lane == 0) bar_arrive(bars.kv_full(n % S::SLOTS));
            ++n;
        };
        const unsigned char* at = place(0, block_of(0));
        int id = block_of(1);
        if (last > 0) read_keys(at);
        for (int j = 0; j < last; ++j) {
            read_values(at);
            at = place(j + 1, id);
            id = block_of(j + 2);
            if (n >= S::SLOTS && !bar_wait(bars.kv_empty(n % S::SLOTS), (n / S::SLOTS - 1) & 1)) return give_up(a.c.flag);
            uint32_t slot = ring + (n % S::SLOTS) * S::SLOT;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const uint32_t row = slot + (i >> 1) * S::BLOCK + key_row + ((((i & 1) * 4 + t) ^ key_sw) << 4);
                const __half2 s0 = __low2half2(as_h2(kp[i].x)), z0 = __high2half2(as_h2(kp[i].x));
                const __half2 s1 = __low2half2(as_h2(kp[i].y)), z1 = __high2half2(as_h2(kp[i].y));
                uint32_t r[4];
                kv4_values(kc[i].x, s0, z0, s0, z0, r);
                sts128(row, r);
                kv4_values(kc[i].y, s1, z1, s1, z1, r);
                sts128(row + 8 * 128, r);
            }
            done();
            read_keys(at);
            if (n >= S::SLOTS && !bar_wait(bars.kv_empty(n % S::SLOTS), (n / S::SLOTS - 1) & 1)) return give_up(a.c.flag);
            slot = ring + (n % S::SLOTS) * S::SLOT;
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                const uint32_t row = slot + val_row + i * (32 * 128);
                const __half2 s0 = as_h2(__byte_perm(vp[i].x, vp[i].z, 0x5410)), z0 = as_h2(__byte_perm(vp[i].x, vp[i].z, 0x7632));
                const __half2 s8 = as_h2(__byte_perm(vp[i].y, vp[i].w, 0x5410)), z8 = as_h2(__byte_perm(vp[i].y, vp[i].w, 0x7632));
                uint32_t r[4];
                kv4_values(vc[i].x, s0, z0, s8, z8, r);
                stmatrix4(row, r);
                kv4_values(vc[i].y, s0, z0, s8, z8, r);
                stmatrix4(row + 16 * 128, r);
            }
            done();
        }
    }
}

// ---- the issuing thread.  What it does between one product and the next the tensor cores wait for, and each instruction takes its turn among
// those of four busy warps: so one thread runs the whole loop, and both tiles' code is written out.
template <int NG>
__device__ __forceinline__ void kc_issue_all(const Kv4AttnArgs& a, uint32_t smem, const KcBars bars, uint32_t tmem, KcRun& u) {
    using S = KcShared<NG>;
    const uint32_t ring = smem + 2 * S::Q;
    unsigned n = 0, runs[2] = {0, 0}, rounds[2] = {0, 0}, waits[2] = {0, 0};     // tiles of keys and values, runs with steps, rounds of P, waits for sums
    auto scores = [&](int x, unsigned slot) {       // S of tile x
        const uint32_t q = tile_desc(smem + x * S::Q), k = tile_desc(ring + slot * S::SLOT), d = tmem + x * KC_TILE;
        mma_ss<4, true>(d, q, k, kc_idesc(KC_STEP));
        if constexpr (NG > 2) mma_ss<NG == 4 ? 4 : 2, false>(d, q + (S::BLOCK >> 4), k + (S::BLOCK >> 4), kc_idesc(KC_STEP));
        tc_commit(bars.s_full(x));
    };
    auto sums = [&](int x, unsigned slot, bool add) {
        const uint32_t v = tile_desc(ring + slot * S::SLOT), p = tmem + S::weights(x), d = tmem + 256 + x * S::HD;
        if (add) mma_ts<false>(d, p, v, kc_idesc(S::HD));
        else mma_ts<true>(d, p, v, kc_idesc(S::HD));
        mma_ts<false>(d, p + 32, v + (S::HD * 128 >> 4), kc_idesc(S::HD));
    };
    for (bool more = true; more; more = kc_next(a, u)) {
        const int last = max(u.steps[0], u.steps[1]);
        if (last == 0) continue;
        if (!bar_wait_one(bars.kv_full(n % S::SLOTS), (n / S::SLOTS) & 1)) return give_up(a.c.flag);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            if (!u.steps[x]) continue;
            if (!bar_wait_one(bars.q_full(x), runs[x] & 1)) return give_up(a.c.flag);
            ++runs[x];
            tc_after();
            scores(x, n % S::SLOTS);
        }
        for (int j = 0; j < last; ++j, n += 2) {
            const unsigned kslot = n % S::SLOTS, vslot = (n + 1) % S::SLOTS, next = (n + 2) % S::SLOTS;
            if (!bar_wait_one(bars.kv_full(vslot), ((n + 1) / S::SLOTS) & 1)) return give_up(a.c.flag);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                if (j >= u.steps[x]) continue;
                for (;;) {
                    if (!bar_wait_one(bars.p_full(x), rounds[x] & 1)) return give_up(a.c.flag);
                    tc_after();
                    if (lds32(bars.again(x)) != rounds[x]++) break;
                    scores(x, kslot);
                }
                sums(x, vslot, j > 0);
                if (j + 1 == u.steps[x]) {
                    tc_commit(bars.s_full(x));
                    continue;
                }
                if (!S::APART) tc_commit(bars.summed(x));
                if (!bar_wait_one(bars.kv_full(next), ((n + 2) / S::SLOTS) & 1)) return give_up(a.c.flag);
                // products of different sums are not in order by themselves: the new scores lie where the weights are read
                if (!S::APART && !bar_wait_one(bars.summed(x), waits[x]++ & 1)) return give_up(a.c.flag);
                tc_after();
                scores(x, next);
            }
            tc_commit(bars.kv_empty(kslot));
            tc_commit(bars.kv_empty(vslot));
        }
    }
}

template <int NG>
__device__ __forceinline__ void kc_issue(const Kv4AttnArgs& a, uint32_t smem, const KcBars bars, uint32_t tmem, int lane) {
    KcRun u;
    if (kc_begin(a, u, lane) && elect_one()) kc_issue_all<NG>(a, smem, bars, tmem, u);
    __syncwarp();
}

// Two numbers at a time: half the instructions.
__device__ __forceinline__ unsigned long long two(uint32_t lo, uint32_t hi) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ float2 halves(unsigned long long x) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
    return r;
}
__device__ __forceinline__ unsigned long long fma_two(unsigned long long a, unsigned long long b, unsigned long long c) {
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ unsigned long long add_two(unsigned long long a, unsigned long long b) {
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// ---- the softmax warps of tile x: thread r of 128 has column r, which is its lane of tensor memory
template <int NG>
__device__ __forceinline__ void kc_softmax(const Kv4AttnArgs& a, uint32_t smem, const KcBars bars, uint32_t tmem, int x, int r, int lane) {
    using S = KcShared<NG>;
    constexpr int HD = S::HD;
    const uint32_t lanes = tmem + ((uint32_t)(r & ~31) << 16), scores = lanes + x * KC_TILE, weights = lanes + S::weights(x), sums = lanes + 256 + x * HD;
    KcRun u;
    unsigned ns = 0, np = 0;       // rounds of S and of P
    for (bool more = kc_begin(a, u, lane); more; more = kc_next(a, u)) {
        const int mine = u.steps[x], col = u.ctile * KC_COLS + x * KC_TILE + r;
        const bool there = col < u.e.z * a.group;
        const int row = there ? by_group(a, col) : 0, head = u.head * a.group + (there ? col - row * a.group : 0);
        const int limit = there ? u.e.y + row : -1, all = u.e.y + by_group(a, u.ctile * KC_COLS + x * KC_TILE);
        float m = there ? -INFINITY : 0.f, l = 0.f;       // reference, sum
        if (mine > 0) {
            // the query times a power of two, so that its largest element lies in [1, 2): exact in f16 but for elements 2^14 times smaller
            const uint4* src = reinterpret_cast<const uint4*>(a.q + (long long)(u.e.w + row) * a.q_stride + head * HD);
            uint4 raw[HD / 8];
            uint32_t big = 0;
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                raw[i] = there ? __ldcg(src + i) : make_uint4(0, 0, 0, 0);
                big = max(big, most_bits(raw[i]));
            }
            const int e = min(max((int)(big >> 7), 1), 253);
            const float down = __int_as_float((254 - e) << 23), up = __int_as_float(e << 23);
            const float factor = fmaxf(a.scale_log2 * up, 1e-37f);       // not 0, which would make NaN of masked scores
#pragma unroll
            for (int i = 0; i < HD / 8; ++i) {
                const uint32_t v[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
                uint32_t h[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) h[j] = pack_h2(__uint_as_float(v[j] << 16) * down, __uint_as_float(v[j] & 0xffff0000u) * down);
                sts128(smem + x * S::Q + (i >> 3) * S::BLOCK + r * 128 + (((i & 7) ^ (r & 7)) << 4), h);
            }
            fence_async();
            __syncwarp();
            if (lane == 0) bar_arrive(bars.q_full(x));

            float top = -INFINITY, step = 0.f;      // of the step last weighed: maximum, and the sum that counts once it is accepted
            for (int j = 0;; ++j) {
                if (!bar_wait(bars.s_full(x), ns & 1)) return give_up(a.c.flag);
                ++ns;
                tc_after();
                if (j > 0) {
                    if (lds32(bars.again(x)) == np - 1) {       // the same step once more
                        --j;
                        const bool far = top > m + 14.f;
                        const float old = far ? ex2(m - top) : 1.f;
                        if (far) m = top;
                        l *= old;
                        if (j > 0) {
#pragma unroll 1
                            for (int i = 0; i < HD; i += 16) {
                                uint32_t v[16];
                                tm_load16(sums + i, v);
                                tm_wait(v);
#pragma unroll
                                for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * old);
                                tm_store16(sums + i, v);
                            }
                        }
                    } else {
                        l += step;
                        if (j == mine) break;
                    }
                }
                const int base = (u.from + j) * KC_STEP;
                const bool whole = base + KC_STEP - 1 <= all;        // every column sees all of the step
                top = -INFINITY;
                auto look = [&](uint32_t (&s)[16], int first) {
                    if (!whole) {
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if (base + first + i > limit) s[i] = 0xff800000u;
                    }
#pragma unroll
                    for (int i = 0; i < 16; i += 2) top = fmaxf(fmaxf(top, __uint_as_float(s[i])), __uint_as_float(s[i + 1]));
                };
                uint32_t s0[16], s1[16];
                if (__any_sync(0xffffffffu, m == -INFINITY)) {       // a column has no reference yet
#pragma unroll 1
                    for (int i = 0; i < KC_STEP; i += 16) {
                        tm_load16(scores + i, s0);
                        tm_wait(s0);
                        look(s0, i);
                    }
                    if (m == -INFINITY) m = top * factor;            // its sums are zeros so far
                    top = -INFINITY;
                }
                const float less = m == -INFINITY ? 0.f : -m;        // still nothing seen: weights of exp(-inf) = 0
                const unsigned long long factors = two(__float_as_uint(factor), __float_as_uint(factor)), lesses = two(__float_as_uint(less), __float_as_uint(less));
                unsigned long long part[2] = {0, 0};
                auto weigh = [&](uint32_t (&s)[16], int first, uint32_t (&p)[8]) {
                    look(s, first);
#pragma unroll
                    for (int i = 0; i < 16; i += 2) {
                        const float2 e = halves(fma_two(two(s[i], s[i + 1]), factors, lesses));
                        const float w0 = ex2(e.x), w1 = ex2(e.y);
                        part[i >> 1 & 1] = add_two(part[i >> 1 & 1], two(__float_as_uint(w0), __float_as_uint(w1)));
                        p[i >> 1] = pack_h2(w0, w1);
                    }
                };
                // P goes over scores that have been read, a piece behind, so that a store does not wait for the exponentials under way
                uint32_t p0[8], p1[8];
                tm_load16(scores, s0);
#pragma unroll
                for (int i = 0; i < KC_STEP; i += 32) {
                    tm_wait(s0);
                    tm_load16(scores + i + 16, s1);
                    weigh(s0, i, p0);
                    if (i > 0) tm_store8(weights + (i >> 1) - 8, p1);
                    tm_wait(s1);
                    if (i + 32 < KC_STEP) tm_load16(scores + i + 32, s0);
                    weigh(s1, i + 16, p1);
                    tm_store8(weights + (i >> 1), p0);
                }
                tm_store8(weights + KC_STEP / 2 - 8, p1);
                const float2 sum = halves(add_two(part[0], part[1]));
                step = sum.x + sum.y;
                top *= factor;
                if (__any_sync(0xffffffffu, top > m + 14.f) && lane == 0) sts32(bars.again(x), np);
                ++np;
                tm_stored();
                tc_before();
                __syncwarp();
                if (lane == 0) bar_arrive(bars.p_full(x));
            }
        }
        const bool entire = u.to - u.from == u.cost;
        const size_t place = (size_t)(2 * blockIdx.x + (u.from == 0)) * KC_COLS + x * KC_TILE + r;
        if (!entire && there) a.ml[place] = make_float2(m, l);
        if (mine > 0) {
            const float inv = l == 0.f ? 0.f : 1.f / l;
            __nv_bfloat16* dst = a.out + (long long)(u.e.w + row) * a.out_stride + head * HD;
            float* part = a.acc + place * HD;
#pragma unroll
            for (int i = 0; i < HD; i += 32) {
                uint32_t v[32];
                tm_load32(sums + i, v);
                tm_wait(v);
                if (!there) continue;
                // element 4 g + k of the group is column 8 k + g
                if (entire) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int d = k * 8 + 2 * j;
                            const __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(v[(d & 3) * 8 + (d >> 2)]) * inv, __uint_as_float(v[((d + 1) & 3) * 8 + (d >> 2)]) * inv);
                            w[j] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                        reinterpret_cast<uint4*>(dst + i)[k] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        reinterpret_cast<uint4*>(part + i)[k] = make_uint4(v[k], v[8 + k], v[16 + k], v[24 + k]);
                }
            }
        }
    }
}

template <int NG>
__global__ void __launch_bounds__(KC_THREADS, 1) k_kv4_attn_chunk(const Kv4AttnArgs a) {
    using S = KcShared<NG>;
    extern __shared__ unsigned char smem_raw[];
    const uint32_t smem = (smem_addr(smem_raw) + 1023) & ~1023u;
    const KcBars bars = {smem + S::BARS};
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) {
        for (int x = 0; x < 2; ++x) {
            bar_init(bars.q_full(x), 4);
            bar_init(bars.s_full(x), 1);
            bar_init(bars.summed(x), 1);
            bar_init(bars.p_full(x), 4);
            sts32(bars.again(x), 0xffffffffu);
        }
        for (int s = 0; s < S::SLOTS; ++s) {
            bar_init(bars.kv_full(s), KC_FILL);
            bar_init(bars.kv_empty(s), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    pdl_launch();
    if (warp == 16) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(bars.tmem()) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_before();
    __syncthreads();
    tc_after();
    uint32_t tmem;
    asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem) : "r"(bars.tmem()));
    if (warp < KC_FILL) kc_fill<NG>(a, smem + 2 * S::Q, bars, warp, lane);
    else if (warp < 16) kc_softmax<NG>(a, smem, bars, tmem, warp >= 12, threadIdx.x & 127, lane);
    else kc_issue<NG>(a, smem, bars, tmem, lane);
    tc_before();
    __syncthreads();
    tc_after();
    if (warp == 16) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

// Adds up the parts of the (column tile, kv head)s that several CTAs had, in the order of the positions.  CTA (b, i) does it for 32 columns of
// the one whose steps begin in CTA b's share of the attention and go on behind it, if there is one; its place is found in the plan
// before the attention has ended, as in k_kv4_merge.
constexpr int KC_MERGE = 32;
template <int NG>
__global__ void __launch_bounds__(256) k_kv4_chunk_merge(const Kv4AttnArgs a) {
    constexpr int HD = NG * KV4_GROUP, D4 = HD / 4;
    __shared__ float2 whole[KC_MERGE];       // of a column: reference, 1 / sum
    __shared__ int parts[1024], n_parts;
    const int lane = threadIdx.x & 31, ctas = gridDim.x, b = blockIdx.x, from = blockIdx.y * KC_MERGE;
    if (a.early) pdl_launch();
    KcRun u;
    const long long total = (long long)__ldcg(a.cu_work + a.n) * a.c.n_kv;
    auto share = [&](int i) { return total * i / ctas; };
    const long long end = share(b + 1);
    bool mine = share(b) < end && kc_find(a, u, end - 1, total, lane);
    mine = mine && u.from + 1 < u.cost && end - 1 - u.from >= share(b);     // more steps behind, and the first is this CTA's
    const int cols = mine ? min(u.e.z * a.group - u.ctile * KC_COLS - from, KC_MERGE) : 0;
    if (cols <= 0) return pdl_wait();
    // the CTA that has the last step, and of those between the ones that have any (with fewer steps than CTAs some have none)
    const int last = (int)(((end - 1 - u.from + u.cost) * ctas - 1) / total);
    if (threadIdx.x == 0) n_parts = 0;
    __syncthreads();
    if (threadIdx.x < 32)
        for (int i = b + lane; i - lane <= last; i += 32) {
            const bool has = i <= last && share(i) < share(i + 1);
            const unsigned all = __ballot_sync(0xffffffffu, has);
            if (has) parts[n_parts + __popc(all & ((1u << lane) - 1))] = (2 * i + (i == b)) * KC_COLS;
            __syncwarp();
            if (lane == 0) n_parts += __popc(all);
            __syncwarp();
        }
    __syncthreads();
    const int n = n_parts;
    pdl_wait();
    if (threadIdx.x < cols) {
        float best = -INFINITY, sum = 0.f;
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float2 part = __ldcg(a.ml + parts[i] + from + threadIdx.x);
            const float top = fmaxf(best, part.x), now = top == -INFINITY ? 0.f : top;
            sum = sum * ex2(best - now) + part.y * ex2(part.x - now);
            best = top;
        }
        whole[threadIdx.x] = make_float2(best == -INFINITY ? 0.f : best, sum == 0.f ? 0.f : 1.f / sum);
    }
    __syncthreads();
#pragma unroll 2
    for (int k = threadIdx.x; k < cols * D4; k += 256) {
        const int col = k / D4, d = k % D4, c = u.ctile * KC_COLS + from + col, row = by_group(a, c);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
        for (int i = 0; i < n; ++i) {
            const float2 part = __ldcg(a.ml + parts[i] + from + col);
            const float4 v = __ldcg(reinterpret_cast<const float4*>(a.acc + (size_t)(parts[i] + from + col) * HD) + d);
            if (part.y == 0.f) continue;        // nothing seen there: no sums were written
            const float f = ex2(part.x - whole[col].x);
            o.x += f * v.x; o.y += f * v.y; o.z += f * v.z; o.w += f * v.w;
        }
        const float inv = whole[col].y;
        const __nv_bfloat162 lo = __floats2bfloat162_rn(o.x * inv, o.y * inv), hi = __floats2bfloat162_rn(o.z * inv, o.w * inv);
        *reinterpret_cast<uint2*>(a.out + (long long)(u.e.w + row) * a.out_stride + (u.head * a.group + c - row * a.group) * HD + d * 4) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
    }
}

}  // namespace vuik
