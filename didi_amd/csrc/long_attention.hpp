// Kernels of the attention of any lengths (long_attention.hip) and their launches, instantiated by one unit per element type.
// Attention of any lengths: queries over keys / values of another length (an encoder's states), forward and backward, with right
// padding, key masks, a causal limit, keys shared by groups of heads, a learned relative position bias by buckets, and dropout.
//
//   visible(b, i, j) = j < count[b] and mask[b, j] != 0 and (not causal or j <= q_start + i)
//   (count[b] < 0: mask and scores do not count in that dialog, t = 0 at all keys that causal leaves: what additive masks of the lowest value come to)
//   t_ij  = scale q_i . k_j + table[bucket(j - q_start - i)][head]          p_ij = exp(t_ij - lse_i) over the visible j, 0 elsewhere
//   o_i   = sum_j drop(p_ij) v_j           lse_i = log sum_j exp(t_ij)
//   ds_ij = p_ij (drop(do_i . v_j) - do_i . o_i)
//   dq_i  = scale sum_j ds_ij k_j     dk_j = scale sum_i ds_ij q_i     dv_j = sum_i drop(p_ij) do_i     dtable[t][h] = sum of ds of bucket t
// A row that sees no key gives o = 0, lse = -inf and no gradients, whatever its query and its do hold; keys and values that no row of a dialog
// sees are never multiplied (their LDS rows are zeros), so whatever lies there -- infinities, NaN -- stays there.  What the causal limit hides from
// some rows only is multiplied by zeros for those, as in the products' plain form: it has to be finite.
//
// One online softmax pass (running maximum and sum per row, fp32).  Everything is laid out so that one lane owns one row's statistics:
//   S^T = K Q^T   v_mfma_f32_32x32x16 (32x32x2 in fp32), A = K rows out of LDS, B = Q rows in registers
//                 -> lane holds t[q = lane & 31][key = (r & 3) + 8 (r >> 2) + 4 (lane >> 5)], r = 0..15
//   O^T += V^T P^T   the 16-bit probabilities a lane holds ARE its B operand (the contraction runs over the lane's own keys); the
//                 matching V^T operand comes out of the row-major V image by transposing LDS reads (fp32: plain row reads)
// so the rescale by exp(m_old - m_new) and every per-row constant of the backward is one register of the lane.
// The backward's dK / dV kernel is the mirror image (lane = key), its dQ kernel the forward's arrangement: two deterministic passes
// (14 products per pair and head-dim element against 10 with atomics, whose order would change the result).
#pragma once
#include <math.h>

#include <algorithm>
#include <atomic>

#include "common.hpp"
#include "philox.hpp"

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef short v4s __attribute__((ext_vector_type(4)));

namespace la {

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int PADB = 96;  // a tile that touches the bias's changing distances reaches at most 64 + 31 beyond them

struct LaParams {
    int B, H, Hk, G, Sq, Sk, D;
    int HG, Gr;  // row groups of the grid: Hk groups of G heads' rows packed together, or (bias) H groups of one head
    int causal, q_start;
    float scale, sc;  // sc = scale * log2(e): the softmax runs in base 2
    const int32_t *mask, *count;
    const void *Q, *K, *V, *dO, *O[2];
    void *Ow[2], *dQ, *dK, *dV;
    int64_t qb, kb, vb, ob, dob, dqb, dkb, dvb;  // elements between dialogs
    int ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;
    float* lse;
    float* rows;    // backward, per row: [3][B][H][Sq]: -lse log2(e) (-inf: sees nothing), do . o, |do| (fp16)
    const void* table;  // [nb][H]
    const int32_t* map; // [2 maxd + 1]
    int nb, maxd;
    float on, rest;  // factors of a kept probability and of the sums over them (drop4)
    uint32_t thr;
    uint64_t seed, offset;
    uint32_t images;  // bytes of LDS before the bias
    int ns, nrt, per;  // splits of the contraction, row (key) tiles, contraction tiles of a split
    float *part, *ml, *part2, *tpart;
    void* dtable;  // la_backward_kv: written by the workgroups behind the keys', from tparts arrays per (dialog, head)
    int tparts;
};

// ---- element types: how operands lie in memory, what multiplies them
template <bool F16_>
struct E16 {
    static constexpr bool F32 = false, F16 = F16_;
    static constexpr int ES = 2, EPC = 8;  // elements per 16-byte LDS chunk
    __device__ static uint4 load(const void* p, int64_t off) { return *reinterpret_cast<const uint4*>(static_cast<const u16*>(p) + off); }
    __device__ static float to_f32(u16 x) { return F16 ? f16_to_f32(x) : bf16_to_f32(x); }
    __device__ static void store4(void* const* p, int64_t off, const float v[4]) {
        uint2 hi, lo;
        split4(v, hi, lo, F16);
        *reinterpret_cast<uint2*>(static_cast<u16*>(p[0]) + off) = hi;
        if (p[1]) *reinterpret_cast<uint2*>(static_cast<u16*>(p[1]) + off) = lo;
    }
    // the attention's output, a mean of the values: beyond fp16's largest number by no more than the 16-bit probabilities may have put it there (2^-11
    // of it, and fp32's rest), it is that number
    __device__ static void store4_mean(void* const* p, int64_t off, float v[4]) {
        if constexpr (F16) {
            if (fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3]))) > 65504.f) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = fabsf(v[e]) <= 65568.f ? fminf(fmaxf(v[e], -65504.f), 65504.f) : v[e];
            }
        }
        store4(p, off, v);
    }
    __device__ static float elem(const void* p, int64_t off) { return to_f32(static_cast<const u16*>(p)[off]); }
};
struct EF32 {
    static constexpr bool F32 = true, F16 = false;
    static constexpr int ES = 4, EPC = 4;
    __device__ static uint4 load(const void* p, int64_t off) { return *reinterpret_cast<const uint4*>(static_cast<const float*>(p) + off); }
    __device__ static void store4(void* const* p, int64_t off, const float v[4]) {
        *reinterpret_cast<float4*>(static_cast<float*>(p[0]) + off) = make_float4(v[0], v[1], v[2], v[3]);
    }
    __device__ static void store4_mean(void* const* p, int64_t off, float v[4]) { store4(p, off, v); }
    __device__ static float elem(const void* p, int64_t off) { return static_cast<const float*>(p)[off]; }
};
// ---- LDS images [rows][DP] in 16-byte chunks, XOR-swizzled within a row so that the reads use all 64 banks: 16 neighbouring rows at one chunk
// (MFMA A rows) fall into 16 different chunks of 256 bytes, and 4 neighbouring rows at 4 neighbouring chunks (what 32 lanes of a transposing
// read fetch) into 4 different quarters.  With the rows' low bits alone a transposing read took two turns.
template <int CH>
__device__ __forceinline__ int swz(int row) {
    if constexpr (CH % 16 == 0) return (row & 3) << 2 | ((row >> 2) & 3);
    else if constexpr (CH % 8 == 0) return (row & 2) << 1 | ((row >> 1) & 2) | ((row >> 3) & 1);
    else return (row >> 2) & 3;
}
template <int CH>
__device__ __forceinline__ int lds_off(int row, int ch) { return (row * CH + (ch ^ swz<CH>(row))) * 16; }

__device__ __forceinline__ v4s tr_read(const char* p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)p); }

template <bool F16>
__device__ __forceinline__ f32x16 mma32(uint4 a, uint4 b, f32x16 c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// B operand fragments of one lane's row, the whole head dim: 16-bit: chunk 2 ks + h (8 elements); fp32: chunk 2 c + h (4)
template <class T, int DP>
struct Frag {
    static constexpr int N = DP / (2 * T::EPC);
    uint4 x[N];
    __device__ void load(const void* p, int64_t off, bool ok, int D, int h) {
#pragma unroll
        for (int c = 0; c < N; ++c) {
            const int col = (2 * c + h) * T::EPC;
            x[c] = make_uint4(0, 0, 0, 0);
            if (ok && col < D) x[c] = T::load(p, off + col);
        }
    }
    __device__ void clear() {
#pragma unroll
        for (int c = 0; c < N; ++c) x[c] = make_uint4(0, 0, 0, 0);
    }
    // The loads have landed.  Said once before a loop that counts its copies: the compiler would otherwise wait for them -- and with them for
    // every copy on its way -- at their first use in each of its turns.
    __device__ void settle() {
#pragma unroll
        for (int c = 0; c < N; ++c) asm volatile("" : "+v"(x[c].x), "+v"(x[c].y), "+v"(x[c].z), "+v"(x[c].w));
    }
};

// Nothing is moved across: the LDS reads before it are issued together, ahead of what uses them (left alone, the compiler puts each read
// right before its product and waits for every one of them).
template <class T>
__device__ __forceinline__ void keep_order() {
    if constexpr (!T::F32) __builtin_amdgcn_sched_barrier(0);
}

// The lane number, made anew where it is asked for: the swizzled addresses that follow from it are then computed next to their reads (an
// instruction each) instead of being kept in up to 64 registers across the loop.
template <bool ANEW>
__device__ __forceinline__ int lane_of(int lane) {
    if constexpr (ANEW) asm volatile("" : "+v"(lane));
    return lane;
}

// A operand for dot products over the head dim: lane = row row0 + (lane & 31) of the image, chunk 2 c + h.  16 bits: all chunks are read at once;
// fp32: each when its products are issued (a product takes 64 cycles, about a read's latency: held all at once they only cost registers)
template <class T, int DP>
struct Rows {
    static constexpr int N = DP / (2 * T::EPC), CH = DP / T::EPC;
    uint4 x[T::F32 ? 1 : N];
    const char* at;
    int lane;
    __device__ __forceinline__ void read(const char* img, int row0, int lane_) {
        at = img + row0 * CH * 16;  // row0 % 32 == 0: the swizzle repeats
        lane = lane_of<T::F32>(lane_);
        if constexpr (!T::F32) {
#pragma unroll
            for (int c = 0; c < N; ++c) x[c] = chunk(c);
        }
    }
    __device__ __forceinline__ uint4 chunk(int c) const { return *reinterpret_cast<const uint4*>(at + lds_off<CH>(lane & 31, 2 * c + (lane >> 5))); }
};

// rows . frag -> [32 rows][32 lanes]
template <class T, int DP>
__device__ __forceinline__ f32x16 dot(const Rows<T, DP>& a, const Frag<T, DP>& f, int D) {
    f32x16 acc;
#pragma unroll
    for (int e = 0; e < 16; ++e) acc[e] = 0.f;
#pragma unroll
    for (int c = 0; c < Frag<T, DP>::N; ++c) {
        if constexpr (T::F32) {
            if (c > 0 && c * 2 * T::EPC >= D) break;  // 256 cycles each: columns of padding are left out
            const float4 af = __builtin_bit_cast(float4, a.chunk(c)), bf = __builtin_bit_cast(float4, f.x[c]);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(af.x, bf.x, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(af.y, bf.y, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(af.z, bf.z, acc, 0, 0, 0);
            acc = __builtin_amdgcn_mfma_f32_32x32x2f32(af.w, bf.w, acc, 0, 0, 0);
        } else {
            acc = mma32<T::F16>(a.x[c], f.x[c], acc);
        }
    }
    return acc;
}

// A operand for sums over 32 rows row0 .. of the image: lane = column, the rows in the order in which the lanes of a 32x32 result hold them.
// 16 bits: transposing reads, fragment [16-row step][32 columns]; fp32: one value for each product, read when it is issued
template <class T, int DP>
struct Cols {
    static constexpr int CH = DP / T::EPC;
    uint4 x[T::F32 ? 1 : DP / 32 * 2];
    const char* at;
    int lane;
    __device__ __forceinline__ void read(const char* img, int row0, int lane_) {
        at = img + row0 * CH * 16;
        lane = lane_of<T::F32>(lane_);
        if constexpr (!T::F32) {
            const int h = lane >> 5, i = lane & 15, dh = (lane >> 4) & 1;  // the lane's address in its 16 lanes' 4 x 16 block; which half of the 32 columns
#pragma unroll
            for (int s = 0; s < 2; ++s)
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt) {
                    const int ra = 16 * s + 4 * h + (i >> 2), ch = dt * 4 + dh * 2 + ((i & 3) >> 1), sub = (i & 1) * 8;
                    const uint2 lo = __builtin_bit_cast(uint2, tr_read(at + lds_off<CH>(ra, ch) + sub));
                    const uint2 hi = __builtin_bit_cast(uint2, tr_read(at + lds_off<CH>(ra + 8, ch) + sub));
                    x[s * (DP / 32) + dt] = make_uint4(lo.x, lo.y, hi.x, hi.y);
                }
        }
    }
    __device__ __forceinline__ float value(int r, int dt) const {
        const int row = 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3), d = dt * 32 + (lane & 31);
        return *reinterpret_cast<const float*>(at + lds_off<CH>(row, d >> 2) + (d & 3) * 4);
    }
};

// w minus its 16-bit rounding
template <class T>
__device__ __forceinline__ f32x16 remainder16(const f32x16& w) {
    f32x16 r;
#pragma unroll
    for (int e = 0; e < 16; ++e) r[e] = w[e] - (T::F16 ? f16_to_f32(f16_bits(w[e])) : bf16_to_f32(bf16_bits(w[e])));
    return r;
}

// acc[dt][d = 32 dt + ..][lane] += sum over the 32 rows k of cols[k][d] * w[k][lane]
template <class T, int DP>
__device__ __forceinline__ void add(const Cols<T, DP>& a, const f32x16& w, f32x16 acc[DP / 32]) {
    if constexpr (T::F32) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.value(r, dt), w[r], acc[dt], 0, 0, 0);
    } else {
        typedef float f2 __attribute__((ext_vector_type(2)));
        uint32_t pk[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            const f2 v = {w[2 * r], w[2 * r + 1]};
            if constexpr (T::F16) {
                typedef _Float16 h2 __attribute__((ext_vector_type(2)));
                pk[r] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
            } else {
                typedef __bf16 b2 __attribute__((ext_vector_type(2)));
                pk[r] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, b2));
            }
        }
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
                acc[dt] = mma32<T::F16>(a.x[s * (DP / 32) + dt], make_uint4(pk[4 * s], pk[4 * s + 1], pk[4 * s + 2], pk[4 * s + 3]), acc[dt]);
    }
}

typedef __attribute__((address_space(3))) void lds_void;
typedef int i32x4 __attribute__((ext_vector_type(4)));

// Asynchronous copy global -> LDS, 16 (4) bytes a lane to lds + 16 (4) lane; a lane whose offset lies at or past the resource's end writes
// zeros.  Out of the compiler's sight (it would wait for every one before the next LDS read): every use is followed by a counted wait and a
// barrier before the first read.
__device__ __forceinline__ i32x4 resource(const void* base, uint32_t bytes) {
    const uint64_t a = reinterpret_cast<uint64_t>(base);
    return i32x4{__builtin_amdgcn_readfirstlane((int)(uint32_t)a), __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32)),
                 __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000};
}
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void copy16(uint32_t off, i32x4 rsrc, uint32_t lds) {
    const uint32_t m = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(rsrc), "s"(m) : "memory", "m0");
}
__device__ __forceinline__ void copy4(uint32_t off, i32x4 rsrc, uint32_t lds) {
    const uint32_t m = __builtin_amdgcn_readfirstlane(lds);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(off), "s"(rsrc), "s"(m) : "memory", "m0");
}
#pragma clang diagnostic pop
template <int N>
__device__ __forceinline__ void wait_copies() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
// every wave's LDS reads and writes are done and its counted copies have landed; others stay in flight (__syncthreads would drain them)
__device__ __forceinline__ void barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

constexpr uint32_t NOWHERE = 0x80000000u;  // beyond every resource: zeros

// one operand's tiles [ROWS][DP], global -> LDS images; rows at or past `n`, columns past D and rows without a `keep` bit become zeros
template <class T, int DP, int ROWS>
struct Tile {
    static constexpr int CH = DP / T::EPC, NC = ROWS * CH / 256;
    static_assert(ROWS * CH % 256 == 0, "whole copies");
    uint32_t off[NC];  // byte offset of this lane's chunks from the tile's first row
    __device__ __forceinline__ static int row(int j, int tid) { return (tid + j * 256) / CH; }
    __device__ __forceinline__ void init(int64_t ld, int D, int tid) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int r = row(j, tid), col = (((tid + j * 256) % CH) ^ swz<CH>(r)) * T::EPC;  // the image is written in order: the lane picks its chunk
            off[j] = col < D ? (uint32_t)(r * ld + col) * T::ES : NOWHERE;
        }
    }
    // base: element offset of the tile's first row; n: rows of it that exist; masked: bit r of word r / 64 of keep
    __device__ __forceinline__ void copy(const void* p, int64_t base, int64_t ld, int n, bool masked, const uint64_t* keep, int keep_shift, char* smem,
                                         uint32_t img, int tid) const {
        const i32x4 rs = resource(static_cast<const char*>(p) + base * T::ES, (uint32_t)max(min(n, ROWS), 0) * (uint32_t)(ld * T::ES));
        const uint32_t dst = (uint32_t)(uintptr_t)(lds_void*)smem + img + (tid >> 6) * 1024;
        if (masked) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const int r = row(j, tid) + keep_shift;
                copy16((keep[r >> 6] >> (r & 63)) & 1 ? off[j] : NOWHERE, rs, dst + j * 4096);
            }
        } else {
#pragma unroll
            for (int j = 0; j < NC; ++j) copy16(off[j], rs, dst + j * 4096);
        }
    }
};

__device__ __forceinline__ uint64_t low_bits(int n) { return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1; }

// x where bit n of `bits` is set, y elsewhere (two VALU instructions, no compare)
__device__ __forceinline__ float where_bit(uint32_t bits, int n, float x, float y) {
    const uint32_t m = (uint32_t)((int32_t)(bits << (31 - n)) >> 31);
    return __builtin_bit_cast(float, (__builtin_bit_cast(uint32_t, x) & m) | (__builtin_bit_cast(uint32_t, y) & ~m));
}

// the larger of a row's two halves (lanes l and l + 32)
__device__ __forceinline__ float max_halves(float x) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x), false, false);
    return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

// Workgroups: x = dialog and head group, y = block of rows (keys), z = split.  They go round the eight XCDs one by one, so where the number of
// (dialog, head) pairs is a multiple of eight all blocks of a pair share one XCD's L2.

// a packed row's head within the group, and its query
__device__ __forceinline__ int row_group(const LaParams& p, int r) { return p.Gr > 1 ? (int)((unsigned)r / (unsigned)p.Sq) : 0; }

// keys of a dialog; `even`: its count is negative, every key weighs the same
__device__ __forceinline__ int visible_end(const LaParams& p, int b, bool& even) {
    even = false;
    if (!p.count) return p.Sk;
    const int n = __builtin_amdgcn_readfirstlane(p.count[b]);
    even = n < 0;
    return even ? p.Sk : min(n, p.Sk);
}

// Which keys of a dialog a workgroup's rows may see, 64 a word: the key mask is turned into bits ahead of the tiles, 64 words at a time into a
// ring of 128 in LDS; without a mask the padding alone decides and nothing is kept.  Where the first window holds more than four words a wave asks
// for eight at once: one after the other their latencies were 2 us of a launch over 777 keys (127 keys: 25 us with the loop, 27 with the longer code).
struct Keys {
    const int32_t* row;  // the dialog's key mask or null
    uint64_t* ring;
    int end, window;
    __device__ __forceinline__ void fill(int w, int tid) const {
        const int lane = tid & 63;
        for (int k = tid >> 6; k < 64; k += 4) {
            const int64_t word = (int64_t)w * 64 + k, key = word * 64 + lane;
            if (word * 64 >= end) break;
            const uint64_t bits = __ballot(key < end && row[key] != 0);
            if (lane == 0) ring[word & 127] = bits;
        }
    }
    __device__ __forceinline__ void start(const LaParams& p, int b, bool even, int end_, uint64_t* ring_, int key0, int tid) {
        row = p.mask && end_ > 0 && !even ? p.mask + (int64_t)b * p.Sk : nullptr;
        ring = ring_;
        end = end_;
        window = key0 >> 12;
        if (row) {
            if (end - (window << 12) <= 256) {
                fill(window, tid);
            } else {
#pragma unroll 1
                for (int w = window * 64; w < window * 64 + 64 && w * 64 < end; w += 32) {
                    const int lane = tid & 63, w0 = w + (tid >> 6);
                    int m[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) m[j] = row[min((w0 + 4 * j) * 64 + lane, end - 1)];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int word = w0 + 4 * j;
                        const uint64_t bits = __ballot(word * 64 + lane < end && m[j] != 0);
                        if (lane == 0 && word * 64 < end) ring[word & 127] = bits;
                    }
                }
                fill(window + 1, tid);
            }
            barrier();
        }
    }
    // called between barriers as the tiles advance: the window before the current one is no longer read by anyone
    __device__ __forceinline__ void advance(int key0, int tid) {
        if (row && (key0 >> 12) != window) {
            window = key0 >> 12;
            fill(window + 1, tid);
        }
    }
    __device__ __forceinline__ const uint64_t* words(int key0) const { return ring + ((key0 >> 6) & 127); }
    // N = 32 or 64 keys from key0 on (key0 % N == 0)
    template <int N>
    __device__ __forceinline__ uint64_t bits(int key0) const {
        uint64_t x = low_bits(end - key0);
        if (row) {
            const uint64_t m = ring[(key0 >> 6) & 127] >> (key0 & 63);
            x &= (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)m) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(m >> 32)) << 32;
        }
        return N == 32 ? x & 0xffffffffull : x;
    }
};

// The bias as a function of the distance alone, for one head, in base-2 units: bv[d + maxd + PADB] for |d| <= maxd + PADB.  A bucket outside the
// table gives NaN.  Bucket and value are two loads that wait for one another, so a kernel asks for the buckets first, for the values after its index
// arithmetic, and stores them behind its other loads (512 distances at once; done in one place they took 2 us of a launch).
template <class T>
struct Bias {
    int t[2];
    float f[2];
    bool even = false;  // no bias at all
    __device__ __forceinline__ void ask(const LaParams& p, int x0, int tid) {
#pragma unroll
        for (int k = 0; k < 2; ++k) t[k] = p.map[min(max(x0 + tid + 256 * k - PADB, 0), 2 * p.maxd)];
    }
    __device__ __forceinline__ void gather(const LaParams& p, int head) {
#pragma unroll
        for (int k = 0; k < 2; ++k) f[k] = T::elem(p.table, (int64_t)min(max(t[k], 0), p.nb - 1) * p.H + head);
    }
    __device__ __forceinline__ void store(const LaParams& p, float* v, int x0, int tid) const {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int x = x0 + tid + 256 * k;
            if (x < 2 * p.maxd + 1 + 2 * PADB) v[x] = even ? 0.f : t[k] >= 0 && t[k] < p.nb ? f[k] * LOG2E : __builtin_nanf("");
        }
    }
    // stores what was asked for and the rest; [lo, hi]: outside these distances the buckets are those of the ends (sh: 8 ints)
    __device__ __forceinline__ void finish(const LaParams& p, int head, float* v, int* sh, int tid, int& lo, int& hi) {
        const int a = p.map[0], z = p.map[2 * p.maxd];
        int l = p.maxd + 1, h = -p.maxd - 1;
        for (int x0 = 0; x0 < 2 * p.maxd + 1 + 2 * PADB; x0 += 512) {
            if (x0 > 0) {
                ask(p, x0, tid);
                gather(p, head);
            }
            store(p, v, x0, tid);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int d = min(max(x0 + tid + 256 * k - PADB, 0), 2 * p.maxd) - p.maxd;
                if (t[k] != a) l = min(l, d);
                if (t[k] != z) h = max(h, d);
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            l = min(l, __shfl_xor(l, o, 64));
            h = max(h, __shfl_xor(h, o, 64));
        }
        if ((tid & 63) == 0) {
            sh[tid >> 6] = l;
            sh[4 + (tid >> 6)] = h;
        }
        barrier();
        lo = min(min(sh[0], sh[1]), min(sh[2], sh[3]));
        hi = max(max(sh[4], sh[5]), max(sh[6], sh[7]));
        // one bucket throughout (or two that meet): everything left of lo is the left end's, everything from lo on the right end's
        hi = max(hi, lo - 1);
        lo = min(lo, hi + 1);
    }
};
template <class T>
__device__ __forceinline__ void bias_fill(const LaParams& p, int head, bool even, float* v, int tid) {
    for (int x0 = 0; x0 < 2 * p.maxd + 1 + 2 * PADB; x0 += 512) {
        Bias<T> b;
        b.even = even;
        b.ask(p, x0, tid);
        b.gather(p, head);
        b.store(p, v, x0, tid);
    }
}

// keep (the factor `on`) or drop (0) of the 4 probabilities of keys j0 .. j0 + 3 (j0 % 4 == 0) of one row: the stream of
// didi_attention_train_forward: element (b, h, i, j) is dropped iff word j & 3 of Philox(offset + ((b H + h) Sq + i) ceil(Sk / 4) + j / 4) < p 2^32.
// 1 / (1 - p) = on rest: what fp16's range leaves no room for on the 16-bit probabilities -- up to 1 in the backward, up to 2^8 in the forward, whose
// running maximum lags -- goes onto the fp32 sums.
__device__ __forceinline__ void drop4(const LaParams& p, uint64_t row, int j0, float k[4]) {
    uint32_t w[4];
    philox4x32_10(p.offset + row * (uint64_t)((p.Sk + 3) >> 2) + (uint64_t)(j0 >> 2), p.seed, w);
#pragma unroll
    for (int e = 0; e < 4; ++e) k[e] = w[e] < p.thr ? 0.f : p.on;
}

// Tiles of the contraction in LDS: 32 rows (16 bits, unshared: 64) for each wave that takes a part of them, and as many tiles -- the current one
// and those on their way -- as leave room for two workgroups of 16-bit types on a CU.
constexpr int tile_rows(bool f32, int share) { return 32 * share * (share == 1 && !f32 ? 2 : 1); }
constexpr int image_bytes(bool f32, int DP, int share) { return tile_rows(f32, share) * DP * (f32 ? 4 : 2); }
constexpr int stages(int image) { return image <= 8 * 1024 ? 3 : 2; }
constexpr int MAX_LDS = 158 * 1024;  // dynamic: 160 KB less the kernels' static words
// the waves of a workgroup can share a block of rows four ways where two tiles of 128 fp32 rows fit the LDS
constexpr int max_share(bool f32, int DP) { return f32 && DP > 64 ? 2 : 4; }

// ------------------------------------------------------------------ forward
// A workgroup's four waves are 4 / WK groups of 32 rows times WK parts of every key tile.  WK = 1: 128 rows share each key tile; WK = 2, 4:
// fewer rows, the waves' shares are joined through LDS at the end (small batches, one token per dialog).
// What bounds it: one token per dialog, the reading of keys and values -- 32 dialogs x 12 heads to 4096 keys, fp16: 48 us, 4.3 TB/s; 4 x 32 heads
// over 8 of 128, 33001 keys, bf16: 100 us and 5 to join the splits, 5.1 TB/s.  Many rows, the products with the softmax between them (a wave's
// products wait for its exponentials; other waves fill in): 2 x 16 heads of 128, 2048 x 8192, bf16: 315 us, 728 TFLOP/s.  Between them latency: a
// launch over 500 keys is a prologue of 4 us and eight tiles that come one behind the other (64 x 12 heads, 63 x 512, fp16: 19 us).
template <class T, int DP, int WK>
struct FwdCfg {
    static constexpr int BN = tile_rows(T::F32, WK), NT = BN / (32 * WK);  // 32-key blocks a wave takes of a tile
    static constexpr int ROWS = 128 / WK;
    static constexpr int IMG = image_bytes(T::F32, DP, WK);  // bytes of one operand's image
    static constexpr int NS = stages(IMG);  // key tiles in LDS: the current one and those on their way
    static constexpr int BYTES = 2 * NS * IMG;
    static constexpr int JOIN = WK == 1 ? 0 : 4 * 32 * (DP + 4) * 4 + 4 * 32 * 8;
    static constexpr int LDS = BYTES > JOIN ? BYTES : JOIN;
    static constexpr int WAVES = T::F32 ? (DP > 64 ? 1 : 2) : DP <= 64 ? 3 : 2;  // per SIMD
};

template <class T, int DP, int WK, bool BIAS>
__global__ void __launch_bounds__(256, (FwdCfg<T, DP, WK>::WAVES)) la_forward(LaParams p) {
    using C = FwdCfg<T, DP, WK>;
    using KV = Tile<T, DP, C::BN>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ uint64_t ring[128];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    Bias<T> bias;
    if constexpr (BIAS) bias.ask(p, 0, tid);
    const int rt = blockIdx.y, split = blockIdx.z, b = (int)(blockIdx.x / (unsigned)p.HG), hg = (int)blockIdx.x - b * p.HG;
    const int head0 = p.Gr > 1 ? hg * p.Gr : hg, kvh = p.Gr > 1 ? hg : p.G > 1 ? hg / p.G : hg;
    const int R = p.Gr * p.Sq, rbase = rt * C::ROWS, wr = wave / WK, wk = wave % WK, rw = rbase + wr * 32;
    bool even;
    int kend = visible_end(p, b, even);
    if (p.causal) {
        const int last = min(R, rbase + C::ROWS) - 1;
        const int g0 = row_group(p, rbase), g1 = row_group(p, last);
        kend = min(kend, p.q_start + (g0 == g1 ? last - g1 * p.Sq : p.Sq - 1) + 1);  // up to the last row's position
    }
    const int tiles = (kend + C::BN - 1) / C::BN;
    const int t0 = split * p.per, t1 = min(tiles, t0 + p.per);

    const int r = rw + (lane & 31), g = r < R ? row_group(p, r) : 0, i = r < R ? r - g * p.Sq : 0, head = head0 + g, pos = p.q_start + i;
    const int64_t rowid = ((int64_t)b * p.H + head) * p.Sq + i;
    if constexpr (BIAS) {
        bias.even = even;
        bias.gather(p, head0);
    }
    Frag<T, DP> q;
    q.load(p.Q, (int64_t)b * p.qb + (int64_t)i * p.ldq + head * p.D, r < R, p.D, h);
    const int64_t kbase = (int64_t)b * p.kb + kvh * p.D, vbase = (int64_t)b * p.vb + kvh * p.D;
    KV tk, tv;
    tk.init(p.ldk, p.D, tid);
    tv.init(p.ldv, p.D, tid);
    Keys keys;
    keys.start(p, b, even, kend, ring, t0 * C::BN, tid);
    int slot = 0;  // where the next tile goes
    auto issue = [&](int t) {
        const uint32_t img = slot * 2 * C::IMG;
        slot = slot + 1 == C::NS ? 0 : slot + 1;
        const int k0 = t * C::BN, shift = C::BN < 64 ? k0 & 63 : 0;
        const uint64_t* keep = keys.words(k0);
        tk.copy(p.K, kbase + (int64_t)k0 * p.ldk, p.ldk, kend - k0, keys.row != nullptr, keep, shift, smem, img, tid);
        tv.copy(p.V, vbase + (int64_t)k0 * p.ldv, p.ldv, kend - k0, keys.row != nullptr, keep, shift, smem, img + C::IMG, tid);
    };
#pragma unroll
    for (int k = 0; k < C::NS - 1; ++k)
        if (t0 + k < t1) issue(t0 + k);

    float* bv = reinterpret_cast<float*>(smem + p.images);
    int blo = 0, bhi = -1;
    if constexpr (BIAS) bias.finish(p, head0, bv, reinterpret_cast<int*>(bv + 2 * p.maxd + 1 + 2 * PADB), tid, blo, bhi);

    f32x16 o[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[dt][e] = 0.f;
    float m = -INFINITY, l = 0.f;  // maximum in units of t (base 2: with the bias) or of q . k; this lane's half of the row's sum
    if (even) q.clear();
    q.settle();
    const float mul = BIAS ? 1.f : p.sc;

    int cur = 0;
    for (int t = t0; t < t1; ++t) {
        // this tile has landed; the later ones may be on their way
        if (C::NS > 2 && t + 1 < t1) wait_copies<(C::NS > 2 ? 1 : 0) * 2 * KV::NC>();
        else wait_copies<0>();
        barrier();
        keys.advance(t * C::BN, tid);
        if (t + C::NS - 1 < t1) issue(t + C::NS - 1);
        const char *Ks = smem + cur * 2 * C::IMG, *Vs = Ks + C::IMG;
        cur = cur + 1 == C::NS ? 0 : cur + 1;
        if (rw >= R) continue;
#pragma unroll
        for (int nt = 0; nt < C::NT; ++nt) {
            const int krow = (wk * C::NT + nt) * 32, k0 = t * C::BN + krow;
            const uint32_t bits = (uint32_t)keys.template bits<32>(k0);  // the keys of this block that the dialog sees
            if (!bits) continue;
            Rows<T, DP> ak;
            ak.read(Ks, krow, lane);
            keep_order<T>();
            f32x16 s = dot<T, DP>(ak, q, p.D);
            Cols<T, DP> cv;  // the values are on their way while the softmax is computed
            cv.read(Vs, krow, lane);
            keep_order<T>();
            if constexpr (BIAS) {
                const int pmin = p.q_start + rw, dmin = k0 - pmin - 31, dmax = k0 + 31 - pmin;
                if (dmax < blo || dmin > bhi) {
                    const float c = dmax < blo ? bv[0] : bv[2 * p.maxd + 2 * PADB];
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = fmaf(s[e], p.sc, c);
                } else {
                    asm volatile("");  // keeps the reads out of the other blocks
                    const float* at = bv + (k0 - pmin - (lane & 31) + p.maxd + PADB + 4 * h);
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = fmaf(s[e], p.sc, at[8 * (e >> 2) + (e & 3)]);
                }
            }
            uint32_t mine = bits;
            if (p.causal) mine &= (uint32_t)low_bits(pos - k0 + 1);
            if (!__all(mine == ~0u)) {
                mine >>= 4 * h;
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = where_bit(mine, 8 * (e >> 2) + (e & 3), s[e], -INFINITY);
            }
            float top = s[0];
#pragma unroll
            for (int e = 0; e < 16; ++e) top = fmaxf(top, s[e]);
            top = max_halves(top);
            // the sums are kept relative to a maximum that is moved only when a row's has grown by more than 2^8: rare after the first blocks
            if (__any(top * mul > m * mul + 8.f)) {
                const float mn = fmaxf(m, top);
                const float a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - mn) * mul);
                m = mn;
                l *= a;
#pragma unroll
                for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[dt][e] *= a;
            }
            const float sub = m == -INFINITY ? 0.f : -m * mul;
            float ls[2] = {0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], mul, sub));
                ls[e & 1] += s[e];
            }
            l += ls[0] + ls[1];
            if (p.thr) {
                asm volatile("");  // a branch: speculated, the random numbers would cost more than all the rest
#pragma unroll
                for (int gq = 0; gq < 4; ++gq) {
                    float k[4];
                    drop4(p, (uint64_t)rowid, k0 + 8 * gq + 4 * h, k);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[4 * gq + e] *= k[e];
                }
            }
            // 16 bits: the probabilities are rounded once to the type that the matrix instructions take, which leaves outputs 1.3 to 1.4 times as far off as
            // the rounding of the result alone; a product with their remainders besides would be half the forward's products again
            add<T, DP>(cv, s, o);
            if constexpr (!T::F32) {
                // D = do . o of the backward wants an output without the rounding of the probabilities, so their remainders are multiplied too where
                // the output's remainder is asked for and it tells: with a bias (the table's gradient sums p (dp - D) over many pairs that cancel),
                // and over few keys (the rounding of n probabilities is 1 / sqrt(n) of that of a score gradient) or narrow heads, whose scores spread
                // more and leave a row few keys that count.  dq and dk against one rounding of theirs: 1.5 to 1.7 without, 1.41 to 1.47 with;
                // everywhere it would be 5 % of a training step of 2048 x 8192 positions of 128.
                if (p.Ow[1] && (BIAS || DP <= 32 || kend <= 64)) add<T, DP>(cv, remainder16<T>(s), o);
            }
        }
    }

    const int64_t rows_all = (int64_t)p.B * p.H * p.Sq;
    l += __shfl_xor(l, 32, 64);
    const float m2 = m * mul;  // base-2 maximum
    if constexpr (WK == 1) {
        if (r >= R) return;
        const float inv = p.ns > 1 ? 1.f : p.rest / l;  // only l == 0 has seen nothing: a sum that is not a number stays one, and so does the row
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                const int d = dt * 32 + gq * 8 + 4 * h;
                if (d >= p.D) continue;
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = l == 0.f ? 0.f : o[dt][4 * gq + e] * inv;
                if (p.ns > 1) *reinterpret_cast<float4*>(p.part + ((int64_t)split * rows_all + rowid) * p.D + d) = make_float4(v[0], v[1], v[2], v[3]);
                else T::store4_mean(p.Ow, (int64_t)b * p.ob + (int64_t)i * p.ldo + head * p.D + d, v);
            }
        if (h == 0) {
            if (p.ns > 1) *reinterpret_cast<float2*>(p.ml + ((int64_t)split * rows_all + rowid) * 2) = make_float2(m2, l);
            else if (p.lse) p.lse[rowid] = l == 0.f ? -INFINITY : (m2 + __builtin_amdgcn_logf(l)) * LN2;
        }
    } else {
        // join the waves of a row group: O^T to LDS as [wave][row][d], maxima and sums beside it
        barrier();
        constexpr int LD = DP + 4;
        float* ox = reinterpret_cast<float*>(smem);
        float2* mx = reinterpret_cast<float2*>(ox + 4 * 32 * LD);
        const int at = wave * 32 + (lane & 31);
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq)
                *reinterpret_cast<float4*>(ox + at * LD + dt * 32 + gq * 8 + 4 * h) = make_float4(o[dt][4 * gq], o[dt][4 * gq + 1], o[dt][4 * gq + 2], o[dt][4 * gq + 3]);
        if (h == 0) mx[at] = make_float2(m2, l);
        barrier();
        for (int x = tid; x < C::ROWS * (DP / 4); x += 256) {
            const int row = x / (DP / 4), d = x % (DP / 4) * 4, rr = rbase + row;
            if (rr >= R || d >= p.D) continue;
            const int w0 = (row >> 5) * WK * 32 + (row & 31);  // the row in the group's first wave; in its next one: 32 on
            float top = -INFINITY;
#pragma unroll
            for (int k = 0; k < WK; ++k) top = fmaxf(top, mx[w0 + k * 32].x);
            float sum = 0.f, v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < WK; ++k) {
                const float2 e = mx[w0 + k * 32];
                if (e.y == 0.f) continue;  // saw nothing; a sum that is not a number is not left out
                const float a = __builtin_amdgcn_exp2f(e.x - top);
                sum += a * e.y;
                const float4 ov = *reinterpret_cast<const float4*>(ox + (w0 + k * 32) * LD + d);
                v[0] = fmaf(a, ov.x, v[0]);
                v[1] = fmaf(a, ov.y, v[1]);
                v[2] = fmaf(a, ov.z, v[2]);
                v[3] = fmaf(a, ov.w, v[3]);
            }
            const int gg = row_group(p, rr), ii = rr - gg * p.Sq, hd = head0 + gg;
            const int64_t id = ((int64_t)b * p.H + hd) * p.Sq + ii;
            if (p.ns > 1) {
                *reinterpret_cast<float4*>(p.part + ((int64_t)split * rows_all + id) * p.D + d) = make_float4(v[0], v[1], v[2], v[3]);
                if (d == 0) *reinterpret_cast<float2*>(p.ml + ((int64_t)split * rows_all + id) * 2) = make_float2(top, sum);
            } else {
                const float inv = sum == 0.f ? 0.f : p.rest / sum;
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] *= inv;
                T::store4_mean(p.Ow, (int64_t)b * p.ob + (int64_t)ii * p.ldo + hd * p.D + d, v);
                if (d == 0 && p.lse) p.lse[id] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
            }
        }
    }
}

// Joins the splits of the forward: 5 us behind the longest (latency: it reads a few MB).  A workgroup takes 256 / (32 SL) rows: 32 lanes of four head-dim elements each, SL of them take the splits
// in turn and are added in LDS (few rows, many splits: one token over a long context would otherwise wait for one split after the other).
template <class T, int SL>
__global__ void __launch_bounds__(256) la_join(LaParams p) {
    __shared__ float4 acc[SL > 1 ? 256 : 1];
    __shared__ float part_sum[SL > 1 ? 8 * SL : 1];
    const int64_t rows = (int64_t)p.B * p.H * p.Sq;
    const int tid = threadIdx.x, d = (tid & 31) * 4, sl = (tid >> 5) % SL;
    const int64_t row = (int64_t)blockIdx.x * (8 / SL) + (tid >> 5) / SL;
    float top = -INFINITY, sum = 0.f;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (row < rows) {
#pragma unroll 8
        for (int s = 0; s < p.ns; ++s) top = fmaxf(top, reinterpret_cast<const float2*>(p.ml)[s * rows + row].x);
#pragma unroll 4
        for (int s = sl; s < p.ns; s += SL) {
            const float2 e = reinterpret_cast<const float2*>(p.ml)[s * rows + row];
            const float4 o = d < p.D ? *reinterpret_cast<const float4*>(p.part + (s * rows + row) * p.D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
            const float a = e.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(e.x - top);  // a split that saw nothing wrote zeros and -inf
            sum = fmaf(a, e.y, sum);
            v.x = fmaf(a, o.x, v.x);
            v.y = fmaf(a, o.y, v.y);
            v.z = fmaf(a, o.z, v.z);
            v.w = fmaf(a, o.w, v.w);
        }
    }
    if constexpr (SL > 1) {
        acc[tid] = v;
        if ((tid & 31) == 0) part_sum[tid >> 5] = sum;
        __syncthreads();
        if (sl != 0) return;
#pragma unroll
        for (int k = 1; k < SL; ++k) {
            const float4 o = acc[tid + 32 * k];
            v.x += o.x;
            v.y += o.y;
            v.z += o.z;
            v.w += o.w;
            sum += part_sum[(tid >> 5) + k];
        }
    }
    if (row >= rows || d >= p.D) return;
    const float inv = sum == 0.f ? 0.f : p.rest / sum;
    float out[4] = {v.x * inv, v.y * inv, v.z * inv, v.w * inv};
    const int i = (int)(row % p.Sq);
    const int64_t bh = row / p.Sq;
    T::store4_mean(p.Ow, bh / p.H * p.ob + (int64_t)i * p.ldo + bh % p.H * p.D + d, out);
    if (d == 0 && p.lse) p.lse[row] = sum == 0.f ? -INFINITY : (top + __builtin_amdgcn_logf(sum)) * LN2;
}

// ------------------------------------------------------------------ backward: dQ, D = do . o, and the sums of ds by distance
// fp16: ds is scaled by a power of two before it is rounded to 16 bits, so that small gradients keep their bits and none overflows.  Here it
// belongs to a row (undone at the end: the lane owns the row): 32 .. 64 / |do_i| at first, which keeps probabilities down to 1e-6 of a row normal
// numbers, and less from the first block on whose score gradients would leave the range.  In la_backward_kv it belongs to a key, and what bounds
// its gradients is known beforehand: |ds_ij| <= max_i |do_i| |v_j| / (1 - drop_p) + max_i |do_i . o_i| is brought to 2^14 .. 2^15.  Results that
// lie beyond fp16 are infinite, as any rounding to fp16 makes them (a loss scaler looks for that).  Watching the gradients costs nothing without a
// bias (8 x 12 heads of 64, 512 x 512: the backward 48 us with and without) and 4 of 79 us with one, whose sums want them unscaled.
// the power of two that brings norm into [2^to, 2^(to + 1)); 1 if there is none
__device__ __forceinline__ float pow2_scale(float norm, int to) {
    if (!(norm > 0.f) || !(norm < INFINITY)) return 1.f;
    const int e = (int)((__builtin_bit_cast(uint32_t, norm) >> 23) & 0xff) - 127;  // norm >= 2^e
    return __builtin_bit_cast(float, (uint32_t)(127 + min(max(to - e, -100), 100)) << 23);
}

// Bound by the products: 2 x 16 heads of 128, 2048 x 8192, bf16: 373 us for its three, 921 TFLOP/s.  Short ones by latency: causal fp32 128 x 128,
// 96 heads of 64: 21 us, a third of it before the first tile (rows, bias, the sums' zeros), the rest two tiles of 6000 cycles.
template <class T, int DP, int WK, bool BIAS>
struct BwdQCfg {
    static constexpr int BN = tile_rows(T::F32, WK), NT = BN / (32 * WK);
    static constexpr int ROWS = 128 / WK;
    static constexpr int IMG = image_bytes(T::F32, DP, WK);
    static constexpr int NS = stages(IMG);
    static constexpr int BYTES = 2 * NS * IMG;
    static constexpr int JOIN = WK == 1 ? 0 : 4 * 32 * (DP + 4) * 4;
    static constexpr int LDS = BYTES > JOIN ? BYTES : JOIN;
    static constexpr int WAVES = T::F32 ? (DP > 64 ? 1 : 2) : DP <= 64 && !BIAS ? 3 : DP > 96 && (BIAS || WK == 4) ? 1 : 2;
};

// Where the table's gradient is accumulated: one array of distances per wave, index d + maxd + PADB.  A 32x32 block's diagonals are summed through a
// wave's own [32][64] words of LDS: lane q writes its row shifted by q, so a diagonal becomes a column, and lane t adds column t (63 of them; the
// corners that no row reaches stay zero).  LDS float adds would do it in place, but take three cycles a lane: 12 times the time of the block's
// products, measured.
__host__ __device__ constexpr int dist_len(int maxd) { return 2 * maxd + 1 + 2 * PADB; }

template <class T, int DP, int WK, bool BIAS>
__global__ void __launch_bounds__(256, (BwdQCfg<T, DP, WK, BIAS>::WAVES)) la_backward_q(LaParams p) {
    using C = BwdQCfg<T, DP, WK, BIAS>;
    using KV = Tile<T, DP, C::BN>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ uint64_t ring[128];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    Bias<T> bias;
    if constexpr (BIAS) bias.ask(p, 0, tid);
    const int rt = blockIdx.y, split = blockIdx.z, b = (int)(blockIdx.x / (unsigned)p.HG), hg = (int)blockIdx.x - b * p.HG;
    const int head0 = p.Gr > 1 ? hg * p.Gr : hg, kvh = p.Gr > 1 ? hg : p.G > 1 ? hg / p.G : hg;
    const int R = p.Gr * p.Sq, rbase = rt * C::ROWS, wk = wave % WK, rw = rbase + wave / WK * 32;
    const int r = rw + (lane & 31);
    const bool rok = r < R;
    const int g = rok ? row_group(p, r) : 0, i = rok ? r - g * p.Sq : 0, head = head0 + g, pos = p.q_start + i;
    const int64_t rowid = ((int64_t)b * p.H + head) * p.Sq + i;
    bool even;
    int kend = visible_end(p, b, even);
    if (p.causal) {
        const int last = min(R, rbase + C::ROWS) - 1;
        const int g0 = row_group(p, rbase), g1 = row_group(p, last);
        kend = min(kend, p.q_start + (g0 == g1 ? last - g1 * p.Sq : p.Sq - 1) + 1);  // up to the last row's position
    }
    const int tiles = (kend + C::BN - 1) / C::BN;
    const int t0 = split * p.per, t1 = min(tiles, t0 + p.per);

    if constexpr (BIAS) {
        bias.even = even;
        bias.gather(p, head0);
    }
    const int64_t oo = (int64_t)b * p.ob + (int64_t)i * p.ldo + head * p.D;
    Frag<T, DP> q, go, o;
    q.load(p.Q, (int64_t)b * p.qb + (int64_t)i * p.ldq + head * p.D, rok, p.D, h);
    go.load(p.dO, (int64_t)b * p.dob + (int64_t)i * p.lddo + head * p.D, rok, p.D, h);
    o.load(p.O[0], oo, rok, p.D, h);
    const float lse = rok ? p.lse[rowid] : -INFINITY;
    if (__any(lse == -INFINITY)) {  // rows that saw nothing: whatever their gradient holds, it is not multiplied
        if (lse == -INFINITY) {
            go.clear();
            o.clear();
        }
    }

    const int64_t kbase = (int64_t)b * p.kb + kvh * p.D, vbase = (int64_t)b * p.vb + kvh * p.D;
    KV tk, tv;
    tk.init(p.ldk, p.D, tid);
    tv.init(p.ldv, p.D, tid);
    Keys keys;
    keys.start(p, b, even, kend, ring, t0 * C::BN, tid);
    auto issue = [&](int t) {
        const uint32_t img = (t - t0) % C::NS * 2 * C::IMG;
        const int k0 = t * C::BN, shift = C::BN < 64 ? k0 & 63 : 0;
        const uint64_t* keep = keys.words(k0);
        tk.copy(p.K, kbase + (int64_t)k0 * p.ldk, p.ldk, kend - k0, keys.row != nullptr, keep, shift, smem, img, tid);
        tv.copy(p.V, vbase + (int64_t)k0 * p.ldv, p.ldv, kend - k0, keys.row != nullptr, keep, shift, smem, img + C::IMG, tid);
    };
#pragma unroll
    for (int k = 0; k < C::NS - 1; ++k)
        if (t0 + k < t1) issue(t0 + k);

    float delta = 0.f, norm = 0.f;
    {
#pragma unroll
        for (int c = 0; c < Frag<T, DP>::N; ++c) {
            if constexpr (T::F32) {
                const float4 a = __builtin_bit_cast(float4, o.x[c]), e = __builtin_bit_cast(float4, go.x[c]);
                delta = fmaf(a.x, e.x, fmaf(a.y, e.y, fmaf(a.z, e.z, fmaf(a.w, e.w, delta))));
            } else {
                const uint32_t a[4] = {o.x[c].x, o.x[c].y, o.x[c].z, o.x[c].w}, e[4] = {go.x[c].x, go.x[c].y, go.x[c].z, go.x[c].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float e0 = T::to_f32((u16)e[k]), e1 = T::to_f32((u16)(e[k] >> 16));
                    delta = fmaf(T::to_f32((u16)a[k]), e0, fmaf(T::to_f32((u16)(a[k] >> 16)), e1, delta));
                    norm = fmaf(e0, e0, fmaf(e1, e1, norm));
                }
            }
        }
        if constexpr (!T::F32) {
            if (p.O[1]) {  // the output's remainder: the sums of ds by distance cancel, so D wants more than the output's 8 or 11 bits
                o.load(p.O[1], oo, lse != -INFINITY, p.D, h);
#pragma unroll
                for (int c = 0; c < Frag<T, DP>::N; ++c) {
                    const uint32_t a[4] = {o.x[c].x, o.x[c].y, o.x[c].z, o.x[c].w}, e[4] = {go.x[c].x, go.x[c].y, go.x[c].z, go.x[c].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        delta = fmaf(T::to_f32((u16)a[k]), T::to_f32((u16)e[k]), fmaf(T::to_f32((u16)(a[k] >> 16)), T::to_f32((u16)(e[k] >> 16)), delta));
                }
            }
        }
        delta += __shfl_xor(delta, 32, 64);
        norm += __shfl_xor(norm, 32, 64);
    }
    norm = __builtin_amdgcn_sqrtf(norm);
    float fs = T::F16 ? pow2_scale(norm, 5) : 1.f;
    const float sub = lse == -INFINITY ? -INFINITY : -lse * LOG2E;  // a row that sees nothing: p = exp2(-inf) = 0
    if (split == 0 && wk == 0 && rok && h == 0) {  // for la_backward_kv
        const int64_t rows_all = (int64_t)p.B * p.H * p.Sq;
        p.rows[rowid] = sub;
        p.rows[rows_all + rowid] = delta;
        if constexpr (T::F16) p.rows[2 * rows_all + rowid] = norm;
    }

    float* bv = reinterpret_cast<float*>(smem + p.images) + 4 * 2048;  // behind the four waves' blocks of diagonals
    int blo = 0, bhi = -1;
    const int len = dist_len(p.maxd);
    float* acc_d = bv + len + 8;  // [4 waves][len]
    float* skew = reinterpret_cast<float*>(smem + p.images) + wave * 2048;
    if constexpr (BIAS) {
        if (p.tpart) {
            for (int x = lane * 4; x < 2048; x += 256) *reinterpret_cast<float4*>(skew + x) = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int x = tid; x < 4 * len; x += 256) acc_d[x] = 0.f;
        }
        bias.finish(p, head0, bv, reinterpret_cast<int*>(bv + len), tid, blo, bhi);
    }
    float* mine_d = acc_d + wave * len;
    float far_l = 0.f, far_r = 0.f;

    f32x16 dq[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) dq[dt][e] = 0.f;

    if (even) q.clear();
    q.settle();
    go.settle();
    for (int t = t0; t < t1; ++t) {
        if (C::NS > 2 && t + 1 < t1) wait_copies<(C::NS > 2 ? 1 : 0) * 2 * KV::NC>();
        else wait_copies<0>();
        barrier();
        keys.advance(t * C::BN, tid);
        if (t + C::NS - 1 < t1) issue(t + C::NS - 1);
        const char *Ks = smem + (t - t0) % C::NS * 2 * C::IMG, *Vs = Ks + C::IMG;
        const int krow = wk * 32 * C::NT, k0 = t * C::BN + krow;
        uint64_t bits = keys.template bits<32 * C::NT>(k0);
        constexpr uint64_t ALL = C::NT == 1 ? 0xffffffffull : ~0ull;
        bool full = bits == ALL;
        if (bits && rw < R) {
            if (p.causal) {
                const uint64_t mine = low_bits(pos - k0 + 1) & ALL;
                full = full && __all(mine == ALL);
                bits &= mine;
            }
            const int pmin = p.q_start + rw, dmin = k0 - pmin - 31, dmax = k0 + 32 * C::NT - 1 - pmin;
            const bool left = dmax < blo, near = BIAS && !left && dmin <= bhi;
            const float fc = BIAS ? (left ? bv[0] : bv[len - 1]) : 0.f;
            const int at = k0 - (p.q_start + r) + p.maxd + PADB + 4 * h;
            constexpr int UNROLL = DP > 64 ? 1 : C::NT;  // head dims past 64: unrolled, it no longer fits the registers of two waves
#pragma unroll UNROLL
            for (int nt = 0; nt < C::NT; ++nt) {
                Rows<T, DP> a;
                a.read(Ks, krow + nt * 32, lane);
                keep_order<T>();
                f32x16 s = dot<T, DP>(a, q, p.D);
                keep_order<T>();
                a.read(Vs, krow + nt * 32, lane);
                keep_order<T>();
                f32x16 dp = dot<T, DP>(a, go, p.D);
                if (near) {
                    asm volatile("");
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], p.sc, bv[at + nt * 32 + 8 * (e >> 2) + (e & 3)] + sub));
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], p.sc, fc + sub));
                }
                if (!full) {
                    const uint32_t mine = (uint32_t)(bits >> (32 * nt)) >> (4 * h);
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] = where_bit(mine, 8 * (e >> 2) + (e & 3), s[e], 0.f);
                }
                if (p.thr) {
                    asm volatile("");  // a branch: speculated, the random numbers would cost more than all the rest
#pragma unroll
                    for (int gq = 0; gq < 4; ++gq) {
                        float k[4];
                        drop4(p, (uint64_t)rowid, k0 + nt * 32 + 8 * gq + 4 * h, k);
#pragma unroll
                        for (int e = 0; e < 4; ++e) dp[4 * gq + e] *= k[e];
                    }
                }
                const float ds_scale = T::F16 && !BIAS ? fs : 1.f;  // a bias wants its sums unscaled
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] *= fmaf(dp[e], p.rest * ds_scale, -delta * ds_scale);
                if constexpr (T::F16) {
                    const float rest_scale = BIAS ? fs : 1.f;
                    float top = 0.f;
#pragma unroll
                    for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(s[e]));
                    if (__any(top * rest_scale > 49152.f)) {
                        asm volatile("");
                        top = max_halves(top) * rest_scale;  // both halves of a row keep one scale
                        const float less = top > 49152.f && top < INFINITY ? pow2_scale(top, 12) : 1.f;
#pragma unroll
                        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                            for (int e = 0; e < 16; ++e) dq[dt][e] *= less;
                        if constexpr (!BIAS) {
#pragma unroll
                            for (int e = 0; e < 16; ++e) s[e] *= less;
                        }
                        fs *= less;
                    }
                }
                if (BIAS && p.tpart) {
                    if (near) {
                        float* to = skew + (lane & 31) * 63 + 31 + 4 * h;
#pragma unroll
                        for (int e = 0; e < 16; ++e) to[8 * (e >> 2) + (e & 3)] = s[e];
                        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int x = 0; x < 32; ++x) sum[x & 3] += skew[x * 64 + lane];
                        // column t is distance k0 + 32 nt - pmin - 31 + t; column 63 holds nothing
                        if (lane < 63) mine_d[k0 + nt * 32 - pmin - 31 + lane + p.maxd + PADB] += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                    } else {
                        float sum = 0.f;
#pragma unroll
                        for (int e = 0; e < 16; ++e) sum += s[e];
                        if (left) far_l += sum;
                        else far_r += sum;
                    }
                }
                if constexpr (T::F16 && BIAS) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) s[e] *= fs;
                }
                keep_order<T>();
                Cols<T, DP> ck;
                ck.read(Ks, krow + nt * 32, lane);
                add<T, DP>(ck, s, dq);
            }
        }
    }
    const float out = p.scale / fs;
    void* dqp[2] = {p.dQ, nullptr};
    if constexpr (WK == 1) {
        if (rok) {
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int gq = 0; gq < 4; ++gq) {
                    const int d = dt * 32 + gq * 8 + 4 * h;
                    if (d >= p.D) continue;
                    const float v[4] = {dq[dt][4 * gq] * out, dq[dt][4 * gq + 1] * out, dq[dt][4 * gq + 2] * out, dq[dt][4 * gq + 3] * out};
                    if (p.ns > 1) *reinterpret_cast<float4*>(p.part + ((int64_t)split * p.B * p.H * p.Sq + rowid) * p.D + d) = make_float4(v[0], v[1], v[2], v[3]);
                    else T::store4(dqp, (int64_t)b * p.dqb + (int64_t)i * p.lddq + head * p.D + d, v);
                }
        }
    } else {
        // add the waves of a row group: dQ^T to LDS as [wave][row][d]
        constexpr int LD = DP + 4;
        float* ox = reinterpret_cast<float*>(smem);
        barrier();
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq)
                *reinterpret_cast<float4*>(ox + (wave * 32 + (lane & 31)) * LD + dt * 32 + gq * 8 + 4 * h) =
                    make_float4(dq[dt][4 * gq] * out, dq[dt][4 * gq + 1] * out, dq[dt][4 * gq + 2] * out, dq[dt][4 * gq + 3] * out);
        barrier();
        for (int x = tid; x < C::ROWS * (DP / 4); x += 256) {
            const int row = x / (DP / 4), d = x % (DP / 4) * 4, rr = rbase + row, w0 = (row >> 5) * WK * 32 + (row & 31);
            if (rr >= R || d >= p.D) continue;
            float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < WK; ++k) {
                const float4 a = *reinterpret_cast<const float4*>(ox + (w0 + k * 32) * LD + d);
                v[0] += a.x;
                v[1] += a.y;
                v[2] += a.z;
                v[3] += a.w;
            }
            const int gg = row_group(p, rr), ii = rr - gg * p.Sq, hd = head0 + gg;
            const int64_t id = ((int64_t)b * p.H + hd) * p.Sq + ii;
            if (p.ns > 1) *reinterpret_cast<float4*>(p.part + ((int64_t)split * p.B * p.H * p.Sq + id) * p.D + d) = make_float4(v[0], v[1], v[2], v[3]);
            else T::store4(dqp, (int64_t)b * p.dqb + (int64_t)ii * p.lddq + hd * p.D + d, v);
        }
    }
    if (BIAS && p.tpart) {
        // this workgroup's sums by distance: the eight arrays joined in a fixed order; what lies beyond the map's ends joins the far tiles
        float* fx = bv;  // the bias is no longer needed
        far_l = wave_sum(far_l);
        far_r = wave_sum(far_r);
        __syncthreads();
        if (lane == 0) {
            fx[wave] = far_l;
            fx[4 + wave] = far_r;
        }
        for (int x = tid; x < len; x += 256) {
            float sum = 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) sum += acc_d[k * len + x];
            acc_d[x] = sum;
        }
        __syncthreads();
        const int nd = 2 * p.maxd + 1;
        float* out = p.tpart + ((((int64_t)hg * p.B + b) * gridDim.y + rt) * gridDim.z + split) * (nd + 2);
        for (int x = tid; x < nd; x += 256) out[x] = acc_d[PADB + x];
        if (wave < 2) {
            float sum = 0.f;
            for (int x = lane; x < PADB; x += 64) sum += acc_d[wave == 0 ? x : len - PADB + x];
            sum = wave_sum(sum);
            if (lane == 0) out[nd + wave] = sum + fx[4 * wave] + fx[4 * wave + 1] + fx[4 * wave + 2] + fx[4 * wave + 3];
        }
    }
}

// dtable[t][h] from the sums by distance of `parts` workgroups per (dialog, head) -- tpart [H][B][parts][2 maxd + 1 distances, left, right] --
// added in a fixed order by one workgroup of N threads per head.  Latency is all there is to it, so sixteen loads are in flight at a time, and the
// attention's backward gives these workgroups a place in la_backward_kv's launch (a launch of their own took 7 us).
constexpr int table_lds(int maxd, int threads) { return (threads / 256 + 1) * (2 * maxd + 3) * 4; }
template <class T, int N>
__device__ __forceinline__ void table_sum(const float* tpart, const int32_t* map, int B, int H, int parts, int nb, int maxd, void* out, int h, float* dist) {
    constexpr int G = N / 256;
    const int nd = 2 * maxd + 1, n = nd + 2, tid = threadIdx.x, grp = tid >> 8, total = B * parts;
    int* bucket = reinterpret_cast<int*>(dist + G * n);  // dist: [G][n], then the map
    for (int x = tid; x < nd; x += N) bucket[x] = map[x];
    for (int x = tid & 255; x < n; x += 256) {
        float sum = 0.f;
        for (int e0 = grp; e0 < total; e0 += 16 * G) {
            float v[16];
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                v[u] = tpart[((int64_t)h * total + min(e0 + u * G, total - 1)) * n + x];
            }
#pragma unroll
            for (int u = 0; u < 16; ++u) sum += e0 + u * G < total ? v[u] : 0.f;
        }
        dist[grp * n + x] = sum;
    }
    __syncthreads();
    if constexpr (G == 4) {
        for (int x = tid; x < n; x += N) dist[x] = (dist[x] + dist[n + x]) + (dist[2 * n + x] + dist[3 * n + x]);
        __syncthreads();
    }
    // one wave per bucket: its lanes take the distances in turn
    const int lane = tid & 63;
    for (int t = tid >> 6; t < nb; t += N / 64) {
        float sum = 0.f;
#pragma unroll 4
        for (int x = lane; x < nd; x += 64) sum += bucket[x] == t ? dist[x] : 0.f;
        if (lane == 0 && bucket[0] == t) sum += dist[nd];
        if (lane == 1 && bucket[2 * maxd] == t) sum += dist[nd + 1];
        sum = wave_sum(sum);
        if (lane == 0) {
            if constexpr (T::F32) static_cast<float*>(out)[(int64_t)t * H + h] = sum;
            else static_cast<u16*>(out)[(int64_t)t * H + h] = T::F16 ? f16_bits(sum) : bf16_bits(sum);
        }
    }
}
template <class T>
__global__ void __launch_bounds__(1024) la_table_sum(const float* tpart, const int32_t* map, int B, int H, int parts, int nb, int maxd, void* out) {
    extern __shared__ float dist[];
    table_sum<T, 1024>(tpart, map, B, H, parts, nb, maxd, out, blockIdx.x, dist);
}

// out row = sum of the splits' partial rows
template <class T>
__global__ void __launch_bounds__(256) la_sum_parts(const float* part, int ns, int64_t rows, int per_bh, int heads, int D, void* out, int64_t batch, int ld) {
    const int64_t x = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int d4 = D / 4;
    const int64_t row = x / d4;
    if (row >= rows) return;
    const int d = (int)(x - row * d4) * 4;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < ns; ++s) {
        const float4 a = *reinterpret_cast<const float4*>(part + (s * rows + row) * D + d);
        v[0] += a.x;
        v[1] += a.y;
        v[2] += a.z;
        v[3] += a.w;
    }
    const int64_t bh = row / per_bh;
    void* o[2] = {out, nullptr};
    T::store4(o, bh / heads * batch + (row % per_bh) * ld + bh % heads * D + d, v);
}

// ------------------------------------------------------------------ backward: dK, dV
// A workgroup owns 128 keys of one key head, its waves 32 each (lane = key: K and V rows live in registers); it walks tiles of BQ rows of
// Q and dO of every head of the group.  Bound by its four products and what they wait for: head dims past 64 (16 bits) hold dK, dV, K and V of a wave's
// keys in 400 registers, so one wave a SIMD is all there is to hide an LDS read behind: 2 x 16 heads of 128, 2048 x 8192, bf16: 736 us, 622
// TFLOP/s.  One launch for dK and one for dV have two waves a SIMD, but five products: 800 us.
template <class T, int DP, int WQ>
struct BwdKCfg {
    static constexpr int BQ = tile_rows(T::F32, WQ), NT = BQ / (32 * WQ);  // 32-row blocks a wave takes of a tile
    static constexpr int KEYS = 128 / WQ;
    static constexpr int IMG = image_bytes(T::F32, DP, WQ);
    static constexpr int NS = stages(IMG);
    static constexpr int STAT = 4 * 2 * 64 * 4;  // each wave's own copy of its rows' constants
    static constexpr int BYTES = NS * (2 * IMG + STAT);
    static constexpr int JOIN = WQ == 1 ? 0 : 4 * 32 * (DP + 4) * 4;
    static constexpr int LDS = BYTES > JOIN ? BYTES : JOIN;
    static constexpr int WAVES = DP > 64 ? 1 : 2;
};

template <class T, int DP, int WQ, bool BIAS>
__global__ void __launch_bounds__(256, (BwdKCfg<T, DP, WQ>::WAVES)) la_backward_kv(LaParams p) {
    using C = BwdKCfg<T, DP, WQ>;
    using QT = Tile<T, DP, C::BQ>;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    __shared__ float top4[2][4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    if constexpr (BIAS) {
        if ((int)blockIdx.x >= p.B * p.Hk) {
            if (blockIdx.y == 0 && blockIdx.z == 0)
                table_sum<T, 256>(p.tpart, p.map, p.B, p.H, p.tparts, p.nb, p.maxd, p.dtable, (int)blockIdx.x - p.B * p.Hk, reinterpret_cast<float*>(smem));
            return;
        }
    }
    Bias<T> bias;
    if constexpr (BIAS) bias.ask(p, 0, tid);
    const int kt = blockIdx.y, split = blockIdx.z, b = (int)(blockIdx.x / (unsigned)p.Hk), kvh = (int)blockIdx.x - b * p.Hk;
    const int kbase = kt * C::KEYS, wq = wave % WQ, kw = kbase + wave / WQ * 32, key = kw + (lane & 31);
    bool even;
    int kend = visible_end(p, b, even);
    if (p.causal) kend = min(kend, p.q_start + p.Sq);  // the last row's position: what lies behind it is visible to no row
    const int seen = key < kend ? p.mask && !even ? p.mask[(int64_t)b * p.Sk + key] : 1 : 0;
    const int64_t kvrow = (int64_t)b * p.kb + (int64_t)key * p.ldk + kvh * p.D, vrow = (int64_t)b * p.vb + (int64_t)key * p.ldv + kvh * p.D;
    const int64_t rows_all = (int64_t)p.B * p.H * p.Sq;

    const int qt0 = p.causal ? min(max(0, kbase - p.q_start), p.Sq) / C::BQ : 0, nq = (p.Sq + C::BQ - 1) / C::BQ - qt0;
    const int tiles = kbase < kend ? p.G * max(nq, 0) : 0;
    const int t0 = split * p.per, t1 = min(tiles, t0 + p.per);
    int gcur = t0 < t1 ? t0 / nq : 0;
    if constexpr (BIAS) {
        bias.even = even;
        bias.gather(p, kvh * p.G + gcur);
    }
    QT tq, tg;
    tq.init(p.ldq, p.D, tid);
    tg.init(p.lddo, p.D, tid);
    auto issue = [&](int t) {
        const int head = kvh * p.G + t / nq, i0 = (qt0 + t % nq) * C::BQ;
        const uint32_t img = (t - t0) % C::NS * (2 * C::IMG + C::STAT);
        tq.copy(p.Q, (int64_t)b * p.qb + (int64_t)i0 * p.ldq + head * p.D, p.ldq, p.Sq - i0, false, nullptr, 0, smem, img, tid);
        tg.copy(p.dO, (int64_t)b * p.dob + (int64_t)i0 * p.lddo + head * p.D, p.lddo, p.Sq - i0, false, nullptr, 0, smem, img + C::IMG, tid);
        const int i1 = i0 + wq * 32 * C::NT;  // this wave's rows
        const int64_t rowid = ((int64_t)b * p.H + head) * p.Sq + i1;
        const uint32_t st = (uint32_t)(uintptr_t)(lds_void*)smem + img + 2 * C::IMG + wave * 512;
        copy4(lane * 4, resource(p.rows + rowid, (uint32_t)max(p.Sq - i1, 0) * 4u), st);
        copy4(lane * 4, resource(p.rows + rows_all + rowid, (uint32_t)max(p.Sq - i1, 0) * 4u), st + 256);
    };
#pragma unroll
    for (int k = 0; k < C::NS - 1; ++k)
        if (t0 + k < t1) issue(t0 + k);

    Frag<T, DP> kf, vf;
    kf.load(p.K, kvrow, key < kend && !even, p.D, h);  // for the scores alone
    vf.load(p.V, vrow, key < kend, p.D, h);
    f32x16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[dt][e] = dv[dt][e] = 0.f;

    float* bv = reinterpret_cast<float*>(smem + p.images);
    const int len = dist_len(p.maxd);
    int blo = 0, bhi = -1;
    if constexpr (BIAS) bias.finish(p, kvh * p.G + gcur, bv, reinterpret_cast<int*>(bv + len), tid, blo, bhi);
    float fs = 1.f;
    const bool vis = seen != 0;
    if constexpr (T::F16) {
        float top[2] = {0.f, 0.f};  // of D and of |do|
        const float* of = p.rows + rows_all + ((int64_t)b * p.H + kvh * p.G) * p.Sq;
        const int n = p.G * p.Sq;
        for (int x = tid; x < n; x += 1024)
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int w = 0; w < 2; ++w) top[w] = fmaxf(top[w], fabsf(of[w * rows_all + min(x + 256 * k, n - 1)]));
#pragma unroll
        for (int w = 0; w < 2; ++w) {
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) top[w] = fmaxf(top[w], __shfl_xor(top[w], o, 64));
            if (lane == 0) top4[w][wave] = top[w];
        }
        barrier();
#pragma unroll
        for (int w = 0; w < 2; ++w) top[w] = fmaxf(fmaxf(top4[w][0], top4[w][1]), fmaxf(top4[w][2], top4[w][3]));
        float vv = 0.f;  // |v_j|^2: a masked key's gradients are zeros, whatever the scale
#pragma unroll
        for (int c = 0; c < Frag<T, DP>::N; ++c) {
            const uint32_t a[4] = {vf.x[c].x, vf.x[c].y, vf.x[c].z, vf.x[c].w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float e0 = T::to_f32((u16)a[k]), e1 = T::to_f32((u16)(a[k] >> 16));
                vv = fmaf(e0, e0, fmaf(e1, e1, vv));
            }
        }
        vv += __shfl_xor(vv, 32, 64);
        fs = pow2_scale(fmaf(top[1] * __builtin_amdgcn_sqrtf(vv), p.on * p.rest, top[0]), 14);
    }
    if (!vis) {  // whatever a masked key holds, it is not multiplied
        kf.clear();
        vf.clear();
    }
    const bool some = __any(vis);
    kf.settle();
    vf.settle();
    for (int t = t0; t < t1; ++t) {
        const int g = t / nq, i0 = (qt0 + t % nq) * C::BQ, head = kvh * p.G + g, qrow = wq * 32 * C::NT;
        if (C::NS > 2 && t + 1 < t1) wait_copies<(C::NS > 2 ? 1 : 0) * (2 * QT::NC + 2)>();
        else wait_copies<0>();
        barrier();
        if (BIAS && g != gcur) {  // another head of the group: its bias
            bias_fill<T>(p, head, even, bv, tid);
            barrier();
            gcur = g;
        }
        if (t + C::NS - 1 < t1) issue(t + C::NS - 1);
        const char *Qs = smem + (t - t0) % C::NS * (2 * C::IMG + C::STAT), *Gs = Qs + C::IMG;
        const float* rc = reinterpret_cast<const float*>(Gs + C::IMG + wave * 512);  // -lse log2(e) of the wave's rows, 64 on D
        // a wave none of whose keys is seen, or seen by the tile's last row, has nothing to add
        if (some && (!p.causal || kw <= p.q_start + min(i0 + qrow + 32 * C::NT, p.Sq) - 1)) {
            // Rows that saw nothing are not multiplied either (their constants D and |do| are zeros): a wave clears what it is about to read itself, others
            // that read the same rows do so too.  Without a causal limit and a bias every row of a dialog sees what its keys show, and looking for such
            // rows would cost 2 % (2048 x 8192 of 128, one wave a SIMD: 30 of 1010 us).
            uint64_t none = BIAS || p.causal ? __ballot(rc[lane & (32 * C::NT - 1)] == -INFINITY) & (C::NT == 2 ? ~0ull : 0xffffffffull) : 0;
            if (none) {
                constexpr int CH = DP / T::EPC;
                char* at = smem + (Qs - smem) + qrow * CH * 16 + lane * 16;
                for (; none; none &= none - 1)
                    if (lane < CH) {
                        const int to = __builtin_ctzll(none) * CH * 16;
                        *reinterpret_cast<uint4*>(at + to) = make_uint4(0, 0, 0, 0);
                        *reinterpret_cast<uint4*>(at + to + C::IMG) = make_uint4(0, 0, 0, 0);
                    }
                asm volatile("" ::: "memory");
            }
            constexpr int UNROLL = DP > 64 ? 1 : C::NT;
#pragma unroll UNROLL
            for (int nt = 0; nt < C::NT; ++nt) {
                const int i1 = i0 + qrow + nt * 32;
                Rows<T, DP> a;
                Cols<T, DP> c;
                a.read(Qs, qrow + nt * 32, lane);
                keep_order<T>();
                f32x16 s = dot<T, DP>(a, kf, p.D);
                keep_order<T>();
                a.read(Gs, qrow + nt * 32, lane);
                c.read(Gs, qrow + nt * 32, lane);
                const int p0 = p.q_start + i1, dmin = kw - p0 - 31, dmax = kw + 31 - p0;
                const bool near = BIAS && dmax >= blo && dmin <= bhi;
                const float fc = vis ? (BIAS ? (dmax < blo ? bv[0] : bv[len - 1]) : 0.f) : -INFINITY;
                const int at = key - p0 + p.maxd + PADB - 4 * h;
                float ls[16];  // -lse log2(e) of the lane's rows, then with the bias
#pragma unroll
                for (int gq = 0; gq < 4; ++gq) {
                    const float4 l4 = *reinterpret_cast<const float4*>(rc + nt * 32 + 8 * gq + 4 * h);
                    ls[4 * gq] = l4.x;
                    ls[4 * gq + 1] = l4.y;
                    ls[4 * gq + 2] = l4.z;
                    ls[4 * gq + 3] = l4.w;
                }
                if (near) {
                    asm volatile("");
#pragma unroll
                    for (int e = 0; e < 16; ++e) ls[e] += vis ? bv[at - 8 * (e >> 2) - (e & 3)] : -INFINITY;
                } else {
#pragma unroll
                    for (int e = 0; e < 16; ++e) ls[e] += fc;
                }
                // a wave issues in order and a product that waits for the one before it holds everything behind it up: the exponentials go between
                // the products of do . v, the score gradients between those of dV
                keep_order<T>();
                f32x16 dp = dot<T, DP>(a, vf, p.D);
#pragma unroll
                for (int e = 0; e < 16; ++e) s[e] = __builtin_amdgcn_exp2f(fmaf(s[e], p.sc, ls[e]));
                if constexpr (!T::F32) {
#pragma unroll
                    for (int x = 0; x < DP / 16; ++x) {
                        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x2, 256 / DP, 0);
                        __builtin_amdgcn_sched_group_barrier(0x400, 256 / DP, 0);
                    }
                }
                keep_order<T>();
                if (p.causal && kw + 31 > p0) {
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (key > p0 + 8 * (e >> 2) + 4 * h + (e & 3)) s[e] = 0.f;
                }
                if (i1 + 32 > p.Sq) {  // rows behind the last: their operands and constants are zeros
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (i1 + 8 * (e >> 2) + 4 * h + (e & 3) >= p.Sq) s[e] = 0.f;
                }
                f32x16 pd = s;  // the probabilities behind the dropout
                if (p.thr) {
                    asm volatile("");  // a branch: speculated, the random numbers would cost more than all the rest
                    const int t4 = lane & 3;
#pragma unroll
                    for (int gq = 0; gq < 4; ++gq) {
                        // lane t of a quad (four neighbouring keys: one Philox counter) draws for row 8 gq + 4 h + t; word t of row e
                        // comes from lane e
                        const int i = i1 + 8 * gq + 4 * h + t4;
                        float k[4];
                        drop4(p, ((uint64_t)b * p.H + head) * p.Sq + i, key & ~3, k);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int src = (lane & ~3) | e;
                            const float w0 = __shfl(k[0], src, 64), w1 = __shfl(k[1], src, 64), w2 = __shfl(k[2], src, 64), w3 = __shfl(k[3], src, 64);
                            const float mk = t4 == 0 ? w0 : t4 == 1 ? w1 : t4 == 2 ? w2 : w3;
                            pd[4 * gq + e] *= mk;
                            dp[4 * gq + e] *= mk;
                        }
                    }
                }
                Cols<T, DP> cq;
                cq.read(Qs, qrow + nt * 32, lane);
                float dl[16];
#pragma unroll
                for (int gq = 0; gq < 4; ++gq) {
                    const float4 d4 = *reinterpret_cast<const float4*>(rc + 64 + nt * 32 + 8 * gq + 4 * h);
                    dl[4 * gq] = d4.x;
                    dl[4 * gq + 1] = d4.y;
                    dl[4 * gq + 2] = d4.z;
                    dl[4 * gq + 3] = d4.w;
                }
                keep_order<T>();
                add<T, DP>(c, pd, dv);
                f32x16 ds;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    ds[e] = s[e] * fmaf(dp[e], p.rest, -dl[e]);
                    if constexpr (T::F16) ds[e] *= fs;
                }
                if constexpr (!T::F32) {
                    __builtin_amdgcn_sched_group_barrier(0x2, 8, 0);  // the probabilities' roundings
#pragma unroll
                    for (int x = 0; x < DP / 16; ++x) {
                        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x2, 768 / DP, 0);
                    }
                }
                keep_order<T>();
                add<T, DP>(cq, ds, dk);
            }
        }
    }
    if (!__all(vis)) {  // keys that nobody saw: nothing, whatever the queries and their gradients hold
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                dk[dt][e] = vis ? dk[dt][e] : 0.f;
                dv[dt][e] = vis ? dv[dt][e] : 0.f;
            }
    }
    const float out = p.scale / fs;
    void *dkp[2] = {p.dK, nullptr}, *dvp[2] = {p.dV, nullptr};
    const int64_t rows = (int64_t)p.B * p.Hk * p.Sk;
    auto write = [&](int ky, int d, const float v[4], bool is_k) {
        const int64_t row = ((int64_t)b * p.Hk + kvh) * p.Sk + ky;
        if (p.ns > 1) *reinterpret_cast<float4*>((is_k ? p.part : p.part2) + ((int64_t)split * rows + row) * p.D + d) = make_float4(v[0], v[1], v[2], v[3]);
        else if (is_k) T::store4(dkp, (int64_t)b * p.dkb + (int64_t)ky * p.lddk + kvh * p.D + d, v);
        else T::store4(dvp, (int64_t)b * p.dvb + (int64_t)ky * p.lddv + kvh * p.D + d, v);
    };
    if constexpr (WQ == 1) {
        if (key >= p.Sk) return;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
            for (int gq = 0; gq < 4; ++gq) {
                const int d = dt * 32 + gq * 8 + 4 * h;
                if (d >= p.D) continue;
                const float a[4] = {dk[dt][4 * gq] * out, dk[dt][4 * gq + 1] * out, dk[dt][4 * gq + 2] * out, dk[dt][4 * gq + 3] * out};
                const float c[4] = {dv[dt][4 * gq] * p.rest, dv[dt][4 * gq + 1] * p.rest, dv[dt][4 * gq + 2] * p.rest, dv[dt][4 * gq + 3] * p.rest};
                write(key, d, a, true);
                write(key, d, c, false);
            }
    } else {
        constexpr int LD = DP + 4;
        float* ox = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int pass = 0; pass < 2; ++pass) {
            barrier();
#pragma unroll
            for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
                for (int gq = 0; gq < 4; ++gq) {
                    const f32x16& x = pass == 0 ? dk[dt] : dv[dt];
                    const float f = pass == 0 ? out : p.rest;
                    *reinterpret_cast<float4*>(ox + (wave * 32 + (lane & 31)) * LD + dt * 32 + gq * 8 + 4 * h) =
                        make_float4(x[4 * gq] * f, x[4 * gq + 1] * f, x[4 * gq + 2] * f, x[4 * gq + 3] * f);
                }
            barrier();
            for (int x = tid; x < C::KEYS * (DP / 4); x += 256) {
                const int row = x / (DP / 4), d = x % (DP / 4) * 4, w0 = (row >> 5) * WQ * 32 + (row & 31);
                if (kbase + row >= p.Sk || d >= p.D) continue;
                float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < WQ; ++k) {
                    const float4 a = *reinterpret_cast<const float4*>(ox + (w0 + k * 32) * LD + d);
                    v[0] += a.x;
                    v[1] += a.y;
                    v[2] += a.z;
                    v[3] += a.w;
                }
                write(kbase + row, d, v, pass == 0);
            }
        }
    }
}

// ------------------------------------------------------------------ launches
// How a launch is cut: `wk` of the four waves of a workgroup share a block of rows (keys in la_backward_kv) and take a part of every tile
// each, so a workgroup has 128 / wk rows; `ns` workgroups share them and are joined through the workspace.
struct Cut {
    int wk, nrt, ns, per;
};
// la_backward_q beside its images: the bias, the four arrays of sums by distance, the blocks whose diagonals are summed
constexpr int sums_lds(int maxd) { return (5 * dist_len(maxd) + 8 + 4 * 2048) * 4; }

struct Plan {
    Cut f, q, k;
    size_t fwd_bytes, rows, part, tpart, bwd_bytes;
};

// more than 64 KB of dynamic LDS is asked for once per kernel and device
template <class F>
bool lds_opt_in(F* fn, size_t bytes, std::atomic<uint64_t>& done) {
    if (bytes <= 64 * 1024) return true;
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return false;
    const uint64_t bit = 1ull << (dev & 63);
    if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return true;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, MAX_LDS) != hipSuccess) return false;
    done.fetch_or(bit, std::memory_order_release);
    return true;
}
inline int pad_dim(int D) { return (D + 31) / 32 * 32; }

inline void set_cut(LaParams& p, const Cut& c) {
    p.nrt = c.nrt;
    p.ns = c.ns;
    p.per = c.per;
}
inline size_t bias_lds(const LaParams& p) { return p.table ? (size_t)(2 * p.maxd + 1 + 2 * PADB + 8) * 4 : 0; }

// a short contraction does not fill the stages: what it leaves lets another workgroup onto the CU
template <class C>
uint32_t used_lds(const LaParams& p) {
    return (uint32_t)std::max(C::BYTES / C::NS * std::min(C::NS, p.per), C::JOIN);
}

template <class T, int DP, int WK>
int launch_forward(LaParams p, hipStream_t st) {
    static_assert(FwdCfg<T, DP, WK>::LDS + 8 * 1024 <= MAX_LDS, "the widest bias fits beside it");
    p.images = used_lds<FwdCfg<T, DP, WK>>(p);
    const size_t lds = p.images + bias_lds(p);
    auto* fn = p.table ? &la_forward<T, DP, WK, true> : &la_forward<T, DP, WK, false>;
    static std::atomic<uint64_t> done[2];
    if (!lds_opt_in(fn, lds, done[p.table != nullptr])) return DIDI_ERR_LAUNCH;
    fn<<<dim3(p.B * p.HG, p.nrt, p.ns), 256, lds, st>>>(p);
    DIDI_LAUNCH_CHECK();
    return DIDI_OK;
}
template <class T, int DP>
int run_forward(const LaParams& p, const Cut& c, hipStream_t st) {
    const int rc = c.wk == 1 ? launch_forward<T, DP, 1>(p, st) : c.wk == 2 ? launch_forward<T, DP, 2>(p, st) : launch_forward<T, DP, max_share(T::F32, DP)>(p, st);
    if (rc || p.ns == 1) return rc;
    const int64_t rows = (int64_t)p.B * p.H * p.Sq;
    if (p.ns <= 4) la_join<T, 1><<<(unsigned)((rows + 7) / 8), 256, 0, st>>>(p);
    else la_join<T, 8><<<(unsigned)rows, 256, 0, st>>>(p);
    DIDI_LAUNCH_CHECK();
    return DIDI_OK;
}
template <class T>
int run_forward_t(const LaParams& p, const Cut& c, hipStream_t st) {
    switch (pad_dim(p.D)) {
        case 32: return run_forward<T, 32>(p, c, st);
        case 64: return run_forward<T, 64>(p, c, st);
        case 96: return run_forward<T, 96>(p, c, st);
        default: return run_forward<T, 128>(p, c, st);
    }
}

template <class T, int DP, int WK>
int launch_backward_q(LaParams p, hipStream_t st) {
    p.images = used_lds<BwdQCfg<T, DP, WK, false>>(p);
    const size_t lds = p.images + (p.table ? sums_lds(p.maxd) : 0);
    auto* fn = p.table ? &la_backward_q<T, DP, WK, true> : &la_backward_q<T, DP, WK, false>;
    static std::atomic<uint64_t> done[2];
    if (!lds_opt_in(fn, lds, done[p.table != nullptr])) return DIDI_ERR_LAUNCH;
    fn<<<dim3(p.B * p.HG, p.nrt, p.ns), 256, lds, st>>>(p);
    DIDI_LAUNCH_CHECK();
    return DIDI_OK;
}
template <class T, int DP, int WQ>
int launch_backward_kv(LaParams p, hipStream_t st) {
    static_assert(BwdKCfg<T, DP, WQ>::LDS + 8 * 1024 <= MAX_LDS, "the widest bias fits beside it");
    p.images = used_lds<BwdKCfg<T, DP, WQ>>(p);
    const size_t lds = std::max<size_t>(p.images + bias_lds(p), p.dtable ? table_lds(p.maxd, 256) : 0);
    auto* fn = p.table ? &la_backward_kv<T, DP, WQ, true> : &la_backward_kv<T, DP, WQ, false>;
    static std::atomic<uint64_t> done[2];
    if (!lds_opt_in(fn, lds, done[p.table != nullptr])) return DIDI_ERR_LAUNCH;
    fn<<<dim3(p.B * p.Hk + (p.dtable ? p.H : 0), p.nrt, p.ns), 256, lds, st>>>(p);
    DIDI_LAUNCH_CHECK();
    return DIDI_OK;
}

template <class T, int DP>
int run_backward(LaParams p, const Plan& z, void* dtable, hipStream_t st) {
    const int64_t rows = (int64_t)p.B * p.H * p.Sq, krows = (int64_t)p.B * p.Hk * p.Sk;
    if (rows > 0) {
        set_cut(p, z.q);
        if (const int rc = z.q.wk == 1 ? launch_backward_q<T, DP, 1>(p, st) : z.q.wk == 2 ? launch_backward_q<T, DP, 2>(p, st) : launch_backward_q<T, DP, max_share(T::F32, DP)>(p, st))
            return rc;
        if (p.ns > 1) {
            la_sum_parts<T><<<(unsigned)((rows * (p.D / 4) + 255) / 256), 256, 0, st>>>(p.part, p.ns, rows, p.Sq, p.H, p.D, p.dQ, p.dqb, p.lddq);
            DIDI_LAUNCH_CHECK();
        }
    }
    if (dtable && (krows == 0 || rows == 0)) {  // nothing to sum, or no launch to do it in
        la_table_sum<T><<<p.H, 1024, table_lds(p.maxd, 1024), st>>>(p.tpart, p.map, rows > 0 ? p.B : 0, p.H, z.q.nrt * z.q.ns, p.nb, p.maxd, dtable);
        DIDI_LAUNCH_CHECK();
    }
    if (krows > 0) {
        set_cut(p, z.k);
        p.dtable = rows > 0 ? dtable : nullptr;
        p.tparts = z.q.nrt * z.q.ns;
        p.part2 = p.part + (int64_t)p.ns * krows * p.D;
        if (const int rc = z.k.wk == 1 ? launch_backward_kv<T, DP, 1>(p, st) : z.k.wk == 2 ? launch_backward_kv<T, DP, 2>(p, st) : launch_backward_kv<T, DP, max_share(T::F32, DP)>(p, st))
            return rc;
        if (p.ns > 1) {
            const unsigned grid = (unsigned)((krows * (p.D / 4) + 255) / 256);
            la_sum_parts<T><<<grid, 256, 0, st>>>(p.part, p.ns, krows, p.Sk, p.Hk, p.D, p.dK, p.dkb, p.lddk);
            la_sum_parts<T><<<grid, 256, 0, st>>>(p.part2, p.ns, krows, p.Sk, p.Hk, p.D, p.dV, p.dvb, p.lddv);
            DIDI_LAUNCH_CHECK();
        }
    }
    return DIDI_OK;
}
template <class T>
int run_backward_t(const LaParams& p, const Plan& z, void* dtable, hipStream_t st) {
    switch (pad_dim(p.D)) {
        case 32: return run_backward<T, 32>(p, z, dtable, st);
        case 64: return run_backward<T, 64>(p, z, dtable, st);
        case 96: return run_backward<T, 96>(p, z, dtable, st);
        default: return run_backward<T, 128>(p, z, dtable, st);
    }
}

// one definition of each per unit: long_attention_{bf16,fp16,fp32}_{forward,backward}.hip
int forward_bf16(const LaParams& p, const Cut& c, hipStream_t st);
int forward_fp16(const LaParams& p, const Cut& c, hipStream_t st);
int forward_fp32(const LaParams& p, const Cut& c, hipStream_t st);
int backward_bf16(const LaParams& p, const Plan& z, void* dtable, hipStream_t st);
int backward_fp16(const LaParams& p, const Plan& z, void* dtable, hipStream_t st);
int backward_fp32(const LaParams& p, const Plan& z, void* dtable, hipStream_t st);

}  // namespace la
