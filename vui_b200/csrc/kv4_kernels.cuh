// Kernels of the paged KV cache held in 4 bits (host side: kv4.cu; entry points: include/vuib200.h, "Paged KV cache in 4 bits").
//
// A stored vector (one position, one kv head, keys or values) is cut into groups of 32 elements:
//   zero = f16(min x), scale = f16((max x - zero) * fl(1/15)), code = rint((x - zero) / scale) in 0 .. 15,
// and a code stands for f16(scale * code + zero).
//
// Layout of a layer's pool: [block][kv head][16 positions][32 elements] -> 640 bytes, laid out as the m16n8k16 fragments that the
// attention feeds to the tensor cores (lane = 4 g + t):
//   [  0, 256)  key codes: lane's 8 bytes = word of key g, word of key g + 8; nibble j of a word's low half is element 8 t + 2 j,
//               of its high half element 8 t + 2 j + 1
//   [256, 320)  key scale and zero: (scale, zero) of key g, of key g + 8, g = 0 .. 7
//   [320, 576)  value codes: lane's 8 bytes = keys 2t, 2t+1, 2t+8, 2t+9, 16 bits each; nibble j of a key's half is element 4 g + j
//   [576, 640)  value scales and zeros of those keys, for t = 0 .. 3: s(2t) s(2t+1) z(2t) z(2t+1) s(2t+8) s(2t+9) z(2t+8) z(2t+9)
// So a tile is read with one 8-byte load a lane and operand, without a shuffle, and a position owns whole 32-bit (keys) and 16-bit
// (values) pieces: storing one position never reads or rewrites another's.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace vuik {

constexpr int KV4_GROUP = 32;
constexpr int KV4_TILE = 16;              // positions of a tile
constexpr int KV4_GT = 640;               // bytes of a tile's group
constexpr int KV4_KPAR = 256, KV4_VCODE = 320, KV4_VPAR = 576;
constexpr float KV4_LIMIT = 60000.f;      // larger magnitudes are stored as this (f16 ends at 65504)
constexpr int KV4_MAX_SEQS = 4096;

// bits of the device flag
constexpr int KV4_BAD_SLOT = 1, KV4_BAD_LEN = 2, KV4_NO_ROWS = 4, KV4_NO_BLOCKS = 8, KV4_BAD_VALUE = 16, KV4_BAD_BLOCK = 32, KV4_TIMEOUT = 64;
constexpr unsigned KV4_POLLS = 1u << 22;  // bound of every wait

__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

struct Kv4Entry { int32_t slot, start, rows, row0; };   // as int4 in memory

struct Kv4Cache {
    unsigned char* pool;        // of the layer
    int32_t* table;             // (max_seqs, max_blocks)
    int32_t* lens;
    int32_t* free_blocks;
    int32_t* n_free;
    int32_t* flag;
    int n_kv, block_shift, n_blocks, max_seqs, max_blocks;
};

// ------------------------------------------------------------------------------------------------ tables and maps
struct Kv4PlanArgs {
    Kv4Cache c;
    const int32_t* slots; const int32_t* new_lens; const int32_t* at;
    int n, n_rows, max_new;
    int group, cols, split;     // query heads a kv head, columns of a tile, positions of a split: attention's units are counted here
    int4* entries; int32_t* cu_rows; int32_t* cu_units; int32_t* row_slot; int32_t* row_pos; long long* slot_map;
};

__device__ __forceinline__ unsigned cluster_rank() { unsigned r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ unsigned cluster_size() { unsigned r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }

// What the CTAs of the cluster (or the one CTA) wrote to global memory before is seen by all of them behind it, when read from the L2.
__device__ __forceinline__ void plan_sync(unsigned size) {
    if (size == 1) { __syncthreads(); return; }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Exclusive prefix sum over the block of one number a thread; the total comes back too.
__device__ __forceinline__ long long block_scan(long long v, long long* warp_sums, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    long long s = lane < nw ? warp_sums[lane] : 0, p = s;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(0xffffffffu, p, o);
        if (lane >= o) p += y;
    }
    total = __shfl_sync(0xffffffffu, p, 31);
    const long long before = __shfl_sync(0xffffffffu, p - s, warp);
    return before + x - v;
}

// The last i with first[i] <= x, for a non-decreasing first[0 .. n] with first[0] = 0 and x < first[n].
__device__ __forceinline__ int find_in(const int* first, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= x) lo = mid; else hi = mid;
    }
    return lo;
}

// One CTA, or one cluster whose CTAs all compute the same few prefix sums and share out what is written: a step's entries are few, its
// rows and blocks many.  Latency bound: three dependent reads (entry, length, table) and five barriers.
__global__ void __launch_bounds__(1024) k_kv4_plan(const Kv4PlanArgs a) {
    extern __shared__ int sm[];
    __shared__ long long warp_sums[32];
    const int n = a.n, per = (n + blockDim.x - 1) / blockDim.x;
    int* s_slot = sm;               // n each; slot -1: takes no part
    int* s_start = s_slot + n;
    int* s_new = s_start + n;
    int* s_have = s_new + n;
    int* s_need = s_have + n;
    int* s_cu = s_need + n;         // n + 1 each
    int* s_grow = s_cu + n + 1;
    int* s_drop = s_grow + n + 1;
    int* owner = s_drop + n + 1;    // max_seqs
    const unsigned size = cluster_size(), rank = cluster_rank();
    const int tid = threadIdx.x, first = tid * per, last = min(n, first + per);
    const int bs = 1 << a.c.block_shift;
    const long long max_len = (long long)a.c.max_blocks << a.c.block_shift;
    int bad = 0;

    for (int i = tid; i < a.c.max_seqs; i += blockDim.x) owner[i] = n;
    pdl_wait();
    pdl_launch();
    const int n_free = __ldcg(a.c.n_free);
    __syncthreads();
    for (int i = tid; i < n; i += blockDim.x) {
        const int slot = __ldcg(a.slots + i);
        s_slot[i] = slot;
        if (slot >= 0 && slot < a.c.max_seqs) atomicMin(owner + slot, i);
    }
    __syncthreads();
    for (int i = tid; i < n; i += blockDim.x) {
        int slot = s_slot[i];
        const bool there = slot >= 0 && slot < a.c.max_seqs && owner[slot] == i;   // a slot's first entry counts
        if (!there && slot != -1) bad |= KV4_BAD_SLOT;
        int len = 0, start = 0;
        long long want = 0;
        bool ok = there;
        if (there) {
            len = __ldcg(a.c.lens + slot);
            want = a.new_lens ? __ldcg(a.new_lens + i) : 1;
            start = a.at ? __ldcg(a.at + i) : len;
            if (len < 0 || len > max_len || start < 0 || start > len || want < 0 || want > a.max_new || start + want > max_len) {
                bad |= KV4_BAD_LEN;
                ok = false;
            }
        }
        s_slot[i] = ok ? slot : -1;
        s_start[i] = ok ? start : 0;
        s_new[i] = ok ? (int)want : 0;
        s_have[i] = ok ? (len + bs - 1) >> a.c.block_shift : 0;
        s_need[i] = ok ? (int)((start + want + bs - 1) >> a.c.block_shift) : 0;
    }
    __syncthreads();
    // Who is served: the rows of the entries so far have to fit, and so have the blocks that they ask for (an entry that asks for none
    // is served all the same).
    long long total, sum = 0;
    for (int i = first; i < last; ++i) sum += s_new[i];
    long long run = block_scan(sum, warp_sums, total);
    long long grow = 0, drop = 0;
    for (int i = first; i < last; ++i) {
        run += s_new[i];
        if (run > a.n_rows) {
            if (s_slot[i] >= 0) bad |= KV4_NO_ROWS;
            s_slot[i] = -1;
            s_new[i] = 0;
            s_need[i] = s_have[i];
        }
        grow += max(s_need[i] - s_have[i], 0);
        drop += max(s_have[i] - s_need[i], 0);
    }
    long long dropped;
    run = block_scan(drop, warp_sums, dropped);
    for (int i = first; i < last; ++i) {
        s_drop[i] = (int)run;
        run += max(s_have[i] - s_need[i], 0);
    }
    run = block_scan(grow, warp_sums, total);
    grow = 0;
    sum = 0;
    for (int i = first; i < last; ++i) {
        const int g = max(s_need[i] - s_have[i], 0);
        run += g;
        if (g > 0 && run > n_free + dropped) {
            bad |= KV4_NO_BLOCKS;
            s_slot[i] = -1;
            s_new[i] = 0;
            s_need[i] = s_have[i];
        } else {
            grow += g;
        }
        sum += s_new[i];
    }
    long long grown, rows, units;
    run = block_scan(grow, warp_sums, grown);
    for (int i = first; i < last; ++i) {
        s_grow[i] = (int)run;
        run += max(s_need[i] - s_have[i], 0);
    }
    run = block_scan(sum, warp_sums, rows);
    sum = 0;
    for (int i = first; i < last; ++i) {
        s_cu[i] = (int)run;
        run += s_new[i];
        const int end = s_start[i] + s_new[i];
        if (s_new[i]) sum += (long long)((s_new[i] * (long long)a.group + a.cols - 1) / a.cols) * ((end + a.split - 1) / a.split);
    }
    run = block_scan(sum, warp_sums, units);
    if (tid == 0) { s_cu[n] = (int)rows; s_grow[n] = (int)grown; s_drop[n] = (int)dropped; }
    if (bad && rank == 0) atomicOr(a.c.flag, bad);
    plan_sync(size);                   // every CTA has read the lengths and the number of free blocks
    const int step = blockDim.x * size, me = rank * blockDim.x + tid;
    if (rank == 0) {
        if (tid == 0) {
            *a.c.n_free = n_free + (int)(dropped - grown);
            a.cu_rows[n] = (int)rows;
            a.cu_units[n] = (int)units;
        }
        for (int i = first; i < last; ++i) {
            a.cu_units[i] = (int)run;
            const int end = s_start[i] + s_new[i];
            if (s_new[i]) run += (long long)((s_new[i] * (long long)a.group + a.cols - 1) / a.cols) * ((end + a.split - 1) / a.split);
            a.cu_rows[i] = s_cu[i];
            a.entries[i] = make_int4(s_slot[i], s_start[i], s_new[i], s_cu[i]);
            if (s_slot[i] >= 0) a.c.lens[s_slot[i]] = end;
        }
    }
    // Blocks given back go on the stack so that the first entry's first one is on top; those taken come off the top in entry order:
    // what was given back and is taken again in the same order gets its places again.
    const int top = n_free + (int)dropped;
    for (int r = me; r < dropped; r += step) {
        const int i = find_in(s_drop, n, r);
        int32_t* at = a.c.table + (size_t)s_slot[i] * a.c.max_blocks + s_need[i] + (r - s_drop[i]);
        if (top - 1 - r < a.c.n_blocks) a.c.free_blocks[top - 1 - r] = *at;
        *at = -1;
    }
    if (dropped) plan_sync(size);
    for (int r = me; r < grown; r += step) {
        const int i = find_in(s_grow, n, r);
        a.c.table[(size_t)s_slot[i] * a.c.max_blocks + s_have[i] + (r - s_grow[i])] = __ldcg(a.c.free_blocks + (top - 1 - r));
    }
    if (grown || dropped) plan_sync(size);
    for (int r = me; r < a.n_rows; r += step) {
        int slot = -1, pos = -1;
        long long where = -1;
        if (r < rows) {
            const int i = find_in(s_cu, n, r);
            slot = s_slot[i];
            pos = s_start[i] + (r - s_cu[i]);
            const int b = __ldcg(a.c.table + (size_t)slot * a.c.max_blocks + (pos >> a.c.block_shift));
            if (b >= 0 && b < a.c.n_blocks) where = ((long long)b << a.c.block_shift) + (pos & (bs - 1));
            else atomicOr(a.c.flag, KV4_BAD_BLOCK);
        }
        a.row_slot[r] = slot;
        a.row_pos[r] = pos;
        a.slot_map[r] = where;
    }
}

__global__ void k_kv4_reset(Kv4Cache c) {
    const long long n = (long long)c.max_seqs * c.max_blocks, step = (long long)gridDim.x * blockDim.x;
    const long long me = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    pdl_wait();
    for (long long i = me; i < n; i += step) c.table[i] = -1;
    for (long long i = me; i < c.n_blocks; i += step) c.free_blocks[i] = (int)i;
    for (long long i = me; i < c.max_seqs; i += step) c.lens[i] = 0;
    if (me == 0) { *c.n_free = c.n_blocks; *c.flag = 0; }
}

// ------------------------------------------------------------------------------------------------ rows in and out
// Byte offset of the tile of position `where` (block * block size + offset in it), kv head h, in a layer's pool.
template <int NG>
__device__ __forceinline__ size_t tile_at(const Kv4Cache& c, long long where, int h) {
    const int tiles = 1 << (c.block_shift - 4);
    const long long b = where >> c.block_shift;
    const int tile = (int)(where & ((1 << c.block_shift) - 1)) >> 4;
    return ((size_t)(b * c.n_kv + h) * tiles + tile) * (NG * KV4_GT);
}

struct Kv4RowsArgs {
    Kv4Cache c;
    const __nv_bfloat16* k; const __nv_bfloat16* v;      // append: rows in
    __nv_bfloat16* k_out; __nv_bfloat16* v_out;          // read: rows out
    long long k_stride, v_stride;                        // elements between rows
    const long long* slot_map;                           // append
    const int32_t* row_slot; const int32_t* row_pos;     // read
    int n_rows;
};

// A thread quantises 8 elements of a row; the four threads of a group share its extremes.  blockIdx.y: keys or values.
template <int NG>
__global__ void __launch_bounds__(256) k_kv4_append(const Kv4RowsArgs a) {
    constexpr int CH = NG * 4;   // threads of a vector
    const bool value = blockIdx.y != 0;
    const long long id = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int ch = (int)(id % CH);
    const long long rest = id / CH;
    const int h = (int)(rest % a.c.n_kv);
    const long long row = rest / a.c.n_kv;
    pdl_wait();
    pdl_launch();
    long long where = -1;
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (row < a.n_rows) {
        where = __ldcg(a.slot_map + row);
        const __nv_bfloat16* src = (value ? a.v + row * a.v_stride : a.k + row * a.k_stride) + (size_t)h * (NG * KV4_GROUP) + ch * 8;
        raw = __ldcg(reinterpret_cast<const uint4*>(src));
    }
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float x[8];
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = __uint_as_float(j & 1 ? w[j >> 1] & 0xffff0000u : w[j >> 1] << 16);
        odd |= !(fabsf(x[j]) <= KV4_LIMIT);
        x[j] = x[j] == x[j] ? fminf(fmaxf(x[j], -KV4_LIMIT), KV4_LIMIT) : 0.f;   // so that what is stored is finite
    }
    float lo = x[0], hi = x[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) { lo = fminf(lo, x[j]); hi = fmaxf(hi, x[j]); }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    if (where < 0) return;
    if (odd) atomicOr(a.c.flag, KV4_BAD_VALUE);
    const __half zero = __float2half_rn(lo);
    const float z = __half2float(zero);
    const __half scale = __float2half_rn(__fmul_rn(__fsub_rn(hi, z), 1.f / 15.f));
    const float s = __half2float(scale);
    uint32_t code[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
        code[j] = s > 0.f ? (uint32_t)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(x[j], z), s)), 0.f), 15.f) : 0u;
    const int key = (int)(where & 15), key8 = key & 7, upper = key >> 3, grp = ch >> 2, t = ch & 3;
    unsigned char* tile = a.c.pool + tile_at<NG>(a.c, where, h) + grp * KV4_GT;
    if (!value) {
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) word |= code[j] << (4 * (j >> 1) + 16 * (j & 1));
        *reinterpret_cast<uint32_t*>(tile + (key8 * 4 + t) * 8 + upper * 4) = word;
        if (t == 0)
            *reinterpret_cast<__half2*>(tile + KV4_KPAR + key8 * 8 + upper * 4) = __halves2half2(scale, zero);
    } else {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t half = code[4 * q] | code[4 * q + 1] << 4 | code[4 * q + 2] << 8 | code[4 * q + 3] << 12;
            *reinterpret_cast<uint16_t*>(tile + KV4_VCODE + ((2 * t + q) * 4 + (key8 >> 1)) * 8 + upper * 4 + (key8 & 1) * 2) = (uint16_t)half;
        }
        if (t == 0) {
            __half* par = reinterpret_cast<__half*>(tile + KV4_VPAR + (key8 >> 1) * 16 + upper * 8) + (key8 & 1);
            par[0] = scale;
            par[2] = zero;
        }
    }
}

// The reverse: 8 elements a thread, bf16 out.  Rows whose slot or position is out of range, or whose block the table lacks, come out as zeros.
template <int NG>
__global__ void __launch_bounds__(256) k_kv4_read(const Kv4RowsArgs a) {
    constexpr int CH = NG * 4;
    const bool value = blockIdx.y != 0;
    const long long id = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const int ch = (int)(id % CH);
    const long long rest = id / CH;
    const int h = (int)(rest % a.c.n_kv);
    const long long row = rest / a.c.n_kv;
    pdl_wait();
    pdl_launch();
    if (row >= a.n_rows) return;
    const int slot = __ldcg(a.row_slot + row), pos = __ldcg(a.row_pos + row);
    long long where = -1;
    if (slot >= 0 && slot < a.c.max_seqs && pos >= 0 && (pos >> a.c.block_shift) < a.c.max_blocks) {
        const int b = __ldcg(a.c.table + (size_t)slot * a.c.max_blocks + (pos >> a.c.block_shift));
        if (b >= 0 && b < a.c.n_blocks) where = ((long long)b << a.c.block_shift) + (pos & ((1 << a.c.block_shift) - 1));
    }
    if (where < 0 && slot != -1) atomicOr(a.c.flag, KV4_BAD_SLOT);
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (where >= 0) {
        const int key = (int)(where & 15), key8 = key & 7, upper = key >> 3, grp = ch >> 2, t = ch & 3;
        const unsigned char* tile = a.c.pool + tile_at<NG>(a.c, where, h) + grp * KV4_GT;
        float s, z;
        uint32_t code[8];
        if (!value) {
            const uint32_t word = __ldcg(reinterpret_cast<const uint32_t*>(tile + (key8 * 4 + t) * 8 + upper * 4));
            const uint32_t par = __ldcg(reinterpret_cast<const uint32_t*>(tile + KV4_KPAR + key8 * 8 + upper * 4));
            s = __half2float(__ushort_as_half((unsigned short)(par & 0xffff)));
            z = __half2float(__ushort_as_half((unsigned short)(par >> 16)));
#pragma unroll
            for (int j = 0; j < 8; ++j) code[j] = word >> (4 * (j >> 1) + 16 * (j & 1)) & 15;
        } else {
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const uint32_t half = __ldcg(reinterpret_cast<const unsigned short*>(tile + KV4_VCODE + ((2 * t + q) * 4 + (key8 >> 1)) * 8 + upper * 4 + (key8 & 1) * 2));
#pragma unroll
                for (int j = 0; j < 4; ++j) code[4 * q + j] = half >> (4 * j) & 15;
            }
            const unsigned short* par = reinterpret_cast<const unsigned short*>(tile + KV4_VPAR + (key8 >> 1) * 16 + upper * 8) + (key8 & 1);
            s = __half2float(__ushort_as_half(__ldcg(par)));
            z = __half2float(__ushort_as_half(__ldcg(par + 2)));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = __half2float(__float2half_rn(__fmaf_rn(s, (float)code[j], z)));   // the product is exact
    }
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 p = __floats2bfloat162_rn(x[2 * j], x[2 * j + 1]);
        w[j] = *reinterpret_cast<const uint32_t*>(&p);
    }
    __nv_bfloat16* dst = (value ? a.v_out + row * a.v_stride : a.k_out + row * a.k_stride) + (size_t)h * (NG * KV4_GROUP) + ch * 8;
    *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
}

}  // namespace vuik
