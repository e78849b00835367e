// What the attention kernels share: arguments, tiles in LDS, matrix-instruction fragments, scores and masks.
//
// Every product is made with the 32 x 32 matrix instructions (16-bit types: 32x32x16, fp32: 32x32x2), whose result has, in lane l, column l % 32
// and rows 8 (r / 4) + 4 (l / 32) + r % 4 for its registers r = 0 .. 15.  The kernels are laid out so that the index a softmax runs over is
// the ROW of such a result: a lane then owns whole columns (one query, or one key), its maximum and sum need one exchange with the other
// half of the wave, and -- since the order of a contraction is free -- the result's registers are, converted, the right-hand operand of
// the next product as they stand:  registers 8 s .. 8 s + 7 are the contraction indexes {16 s + 4 half + 0 .. 3, 16 s + 8 + 4 half + 0 .. 3},
// and the left-hand operand is fetched for those same indexes (ds_read_b64_tr_b16: four consecutive rows of a row-major tile, one column
// per lane).  Probabilities and score gradients never leave the registers.
#pragma once
#include "relbias.h"

#define ATTN_MAX_D 128
#define ATTN_LOG2E 1.44269504088896340736f
#define ATTN_LN2 0.69314718055994530942f

#ifdef __HIPCC__
namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef re_bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef re_f16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));

#define ATTN_INF __builtin_inff()

struct args {
    const void *q, *k, *v;
    int64_t qs[3], ks[3], vs[3];       // strides in elements: batch, head, row (adjacent inside a row)
    int32_t B, Hq, Hkv, Sq, Sk, D, group;
    float scale;
    int32_t causal, mkind;             // mkind: 0 none, 1 truth values, 2 / 3 / 4 additive fp32 / bf16 / fp16
    const void* mask;
    int64_t ms[4];                     // batch, head, query, key
    const int64_t *lens, *offs;
    int64_t off;
    const void* table;
    const int32_t* map;
    int32_t tdtype, R, buckets;
};

// ---------------------------------------------------------------------------------------------------------- matrix instructions
// A fragment is 16 bytes a lane: KS contraction indexes of a 32-wide operand, the lane's own KS / 2 of them at 16 bytes * half.
template <class T>
struct mm;
template <>
struct mm<re_bf16> {
    typedef bf16x8 frag;
    static constexpr int KS = 16;
    static __device__ __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct mm<re_f16> {
    typedef f16x8 frag;
    static constexpr int KS = 16;
    static __device__ __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};
template <>
struct mm<float> {
    typedef f32x4 frag;
    static constexpr int KS = 8;
    static __device__ __forceinline__ f32x16 mul(frag a, frag b, f32x16 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
        return c;
    }
};

// ---------------------------------------------------------------------------------------------------------- tiles
// A tile is ROWS rows of a tensor in LDS, row-major in 16-byte chunks.  16-bit types: the chunk of a row is moved by an exclusive or with
// a value of the row such that both kinds of reads -- 16 rows at one chunk (row fragments) and 4 rows at 4 chunks (transposed
// fragments) -- fall on distinct banks; fp32: rows are padded by one chunk (its column reads meet two-fold conflicts).
template <class T, int DP>
struct tile {
    static constexpr int EPC = 16 / (int)sizeof(T);                  // elements of a chunk
    static constexpr int CH = DP / EPC;                              // chunks of a row
    static constexpr int CHP = sizeof(T) == 4 ? CH + 1 : CH <= 4 ? 4 : CH <= 8 ? 8 : 16;      // ... as laid out
    static constexpr int ROW = CHP * EPC;                            // elements between rows
    static __device__ __forceinline__ int swz(int row) {
        if constexpr (sizeof(T) == 4) return 0;
        else if constexpr (CHP == 16) return ((row & 3) << 2) | ((row >> 2) & 3);
        else if constexpr (CHP == 8) return (((row >> 1) & 1) << 2) | ((row >> 2) & 3);
        else return (row >> 2) & 3;
    }
    static __device__ __forceinline__ int at(int row, int chunk) { return row * ROW + ((chunk ^ swz(row)) * EPC); }
    static constexpr size_t bytes(int rows) { return (size_t)rows * CHP * 16; }
};

// 16 bytes a lane from base + at (bytes) to 64 consecutive pieces of LDS, as the bare instruction (nothing is returned in registers; the wait is the
// caller's re_sync_full).  Behind the builtin the transposed reads wait for all loads in flight: the tile that was just asked for is then
// waited for in the middle of the one before, which a kernel of two waves a SIMD hides and a stream over a cache does not.
__device__ __forceinline__ void to_lds(const void* base, uint32_t at, const void* lds) {
    const uint32_t to = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)lds;
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(__builtin_amdgcn_readfirstlane(to)), "v"(at), "s"(base) : "memory", "m0");
}

// ROWS x DP elements of a tensor into a tile, in two steps: fetch() starts the loads, land() ends them in LDS; a barrier that waits for
// memory (re_sync_full) comes behind land().
// 16-bit types on whole 16-byte chunks (VEC) go straight from memory to LDS, the tile's exclusive or applied to the source; no
// register holds them.  Rows from `rows` on are copies of the last one and columns from D on of the row's last chunk: finite wherever the rows
// themselves are, and every use of them is multiplied by zero or thrown away: the other operand of a contraction over columns is zero from D on.
// PLAIN: by the bare instruction.  Otherwise (ZEROS: asked for) through registers, missing rows and columns zero; VEC: chunk by chunk, else element by element.
template <class T, int DP, int ROWS, int THREADS, bool VEC, bool ZEROS = false, bool PLAIN = false>
struct stage {
    typedef tile<T, DP> tl;
    static constexpr bool DIRECT = VEC && !ZEROS && sizeof(T) == 2;
    static constexpr int CH = DIRECT ? tl::CHP : tl::CH;
    static constexpr int N = (ROWS * CH + THREADS - 1) / THREADS;
    static_assert(!DIRECT || ROWS * CH % THREADS == 0, "whole waves of chunks");
    uint4 r[DIRECT ? 1 : N];
    __device__ __forceinline__ void fetch(const T* base, int64_t stride, int rows, int D, T* lds) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = n * THREADS + (int)threadIdx.x, row = c / CH;
            if constexpr (DIRECT) {
                const int e = min(((c % CH) ^ tl::swz(row)) * tl::EPC, D - tl::EPC);
                const uint32_t at = (uint32_t)min(row, rows - 1) * ((uint32_t)stride * 2u) + (uint32_t)e * 2u;      // bytes (vec: below 2^31)
                const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
                T* const to = lds + (n * THREADS + wave * 64) * tl::EPC;
                if constexpr (PLAIN) {
                    to_lds(base, at, to);
                    continue;
                }
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) uint32_t*)(reinterpret_cast<const char*>(base) + at),
                                                 (__attribute__((address_space(3))) uint32_t*)(to), 16, 0, 0);
            } else {
                const int e = (c % CH) * tl::EPC;
                r[n] = make_uint4(0, 0, 0, 0);
                if constexpr (VEC) {
                    if (row < rows && row < ROWS && e < D) r[n] = *reinterpret_cast<const uint4*>(base + row * stride + e);
                } else {
                    union { uint4 u; T t[tl::EPC]; } x;
                    x.u = r[n];
#pragma unroll
                    for (int i = 0; i < tl::EPC; ++i)
                        if (row < rows && row < ROWS && e + i < D) x.t[i] = base[row * stride + e + i];
                    r[n] = x.u;
                }
            }
        }
    }
    __device__ __forceinline__ void land(T* lds) const {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = n * THREADS + (int)threadIdx.x;
                if (ROWS * CH % THREADS == 0 || c < ROWS * CH) *reinterpret_cast<uint4*>(lds + tl::at(c / CH, c % CH)) = r[n];
            }
        }
    }
};

// a row's own fragments straight from memory (the operand that a wave keeps): 16 bytes at KS * step + KS / 2 * half
template <class T, int DP, bool VEC>
__device__ __forceinline__ void load_row_frags(const T* row, bool live, int D, int half, typename mm<T>::frag* f) {
    typedef typename mm<T>::frag frag;
    constexpr int EPC = 16 / (int)sizeof(T);
#pragma unroll
    for (int s = 0; s < DP / mm<T>::KS; ++s) {
        const int e = s * mm<T>::KS + half * EPC;
        union { frag f; uint4 u; T t[EPC]; } x;
        x.u = make_uint4(0, 0, 0, 0);
        if constexpr (VEC) {
            if (live && e < D) x.u = *reinterpret_cast<const uint4*>(row + e);
        } else {
#pragma unroll
            for (int i = 0; i < EPC; ++i)
                if (live && e + i < D) x.t[i] = row[e + i];
        }
        f[s] = x.f;
    }
}

// left-hand operand, rows of a tile: lane l holds row row0 + l % 32
template <class T, int DP>
__device__ __forceinline__ typename mm<T>::frag row_frag(const T* lds, int row, int step, int half) {
    typedef tile<T, DP> tl;
    return *reinterpret_cast<const typename mm<T>::frag*>(lds + tl::at(row, 2 * step + half));
}

// left-hand operand, COLUMNS of a tile: lane l holds column col0 + l % 32; the contraction runs over the rows that registers
// PR s .. PR s + PR - 1 of a 32 x 32 result stand for (PR = 8, fp32: 4); row0: the block's first row
template <class T, int DP>
__device__ __forceinline__ typename mm<T>::frag col_frag(const T* lds, int row0, int s, int col0, int lane) {
    typedef tile<T, DP> tl;
    const int half = lane >> 5;
    if constexpr (sizeof(T) == 4) {
        f32x4 f;
        const int c = col0 + (lane & 31);
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = lds[(row0 + 8 * s + 4 * half + i) * tl::ROW + c];
        return f;
    } else {
        // a group of 16 lanes reads 4 rows x 16 columns, 4 elements a lane, and gets 4 rows of one column a lane
        const int i = lane & 15;
        const int chunk = (col0 >> 3) + ((lane >> 4) & 1) * 2 + ((i >> 1) & 1);
        union { s16x4 h[2]; typename mm<T>::frag f; } x;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const int row = row0 + 16 * s + 8 * p + 4 * half + (i >> 2);
            const T* at = lds + tl::at(row, chunk) + (i & 1) * 4;
            x.h[p] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)(at));
        }
        return x.f;
    }
}

// registers PR s .. of a result as the right-hand operand of the next product (16-bit types: one rounding, to nearest)
template <class T>
__device__ __forceinline__ typename mm<T>::frag reg_frag(const f32x16& x, int s) {
    typename mm<T>::frag f;
    constexpr int PR = sizeof(T) == 4 ? 4 : 8;
#pragma unroll
    for (int i = 0; i < PR; ++i) f[i] = (T)x[PR * s + i];
    return f;
}
template <class T>
constexpr int frags_of_block() { return sizeof(T) == 4 ? 4 : 2; }
// fp16 has its eleven bits between 2^-14 and 2^16 only (bf16 has fp32's range), and what is rounded to it here can be of any size: it is multiplied by a
// power of two first, and the product's fp32 sums by its inverse in the end
template <class T>
constexpr bool narrow() { return re_type<T>::CODE == RE_F16; }

__device__ __forceinline__ float other_half(float v) { return __shfl_xor(v, 32, 64); }
__device__ __forceinline__ int row_of(int r, int half) { return 8 * (r >> 2) + 4 * half + (r & 3); }

// Workgroup -> (unit, tile): a unit is what shares keys and values (a sequence's head), its tiles are work of one kind, with a triangle the
// longest first.  Workgroups are dealt to the eight XCDs in turn: where eight divides the groups of `chunk` units that share keys and values, a
// group stays on one XCD (its L2 holds what they share), neighbouring groups on neighbouring XCDs (a ragged batch has its long sequence on all
// of them); and there `set` units run side by side, tile by tile, so that the long tiles of all of them start before the short ones of any
// (2 x 16 heads x 4096 x 128, causal, forward: 238 us a head at a time, 185 so).
struct order {
    int32_t xcd, units, tiles, set, chunk;      // xcd: 8, or 1; units per XCD (the last set may be smaller)
};
__device__ __forceinline__ void place(const order& o, int id, int& unit, int& tile) {
    const int x = id % o.xcd;
    id /= o.xcd;
    const int per = o.set * o.tiles, first = id / per * o.set, r = id % per, wide = min(o.set, o.units - first);
    tile = r / wide;
    const int l = first + r % wide;
    unit = (l / o.chunk * o.xcd + x) * o.chunk + l % o.chunk;
}

// What rounding took from a 16-bit output, in that type, for the backward's delta = rowsum(dO O): a row's probabilities sum to one, so an error of delta
// is common to the whole row of dS, and in sums over it (a bias's gradient) it does not average out.  Rows of low_len(D) elements.
__host__ __device__ inline int low_len(int D) { return (D + 7) / 8 * 8; }
template <class T>
__device__ __forceinline__ T* low_row(const args& a, void* low, int b, int h, int i) {
    return static_cast<T*>(low) + (((int64_t)b * a.Hq + h) * a.Sq + i) * low_len(a.D);
}

// ---------------------------------------------------------------------------------------------------------- lengths, masks, bias
__device__ __forceinline__ int seq_len(const args& a, int b) {
    if (!a.lens) return a.Sk;
    const int64_t n = a.lens[b];
    return n < 0 ? 0 : n > a.Sk ? a.Sk : (int)n;
}
// the position of query 0 among the keys; clipped where nothing changes any more (keys and queries are below 2^30)
__device__ __forceinline__ int seq_off(const args& a, int b) {
    const int64_t o = a.offs ? a.offs[b] : a.off;
    return o < -(1 << 30) ? -(1 << 30) : o > (1 << 30) - 1 ? (1 << 30) - 1 : (int)o;
}
// additive value of the mask; a truth value that is false and -inf shut the place
__device__ __forceinline__ float mask_add(const args& a, int64_t at) {
    if (a.mkind == 1) return static_cast<const uint8_t*>(a.mask)[at] ? 0.f : -ATTN_INF;
    return re_load_as_float(a.mask, at, a.mkind - 2);
}
__device__ __forceinline__ int clip_distance(int d, int R) { return d < -R ? -R : d > R ? R : d; }

// A head's bias by distance in LDS: distances -R - 31 .. R + 31, the ends repeated.  A lane's 32 distances in a block then need one clamp, of their
// lowest, and sixteen constant offsets from it.  `line` points to distance -R.
__host__ __device__ inline int line_len(int R) { return 2 * R + 63; }
template <int THREADS>
__device__ __forceinline__ void load_lines(const args& a, int h0, int heads, float* line) {
    const int n = line_len(a.R);
    for (int x = threadIdx.x; x < heads * n; x += THREADS)
        line[x - 31] = rb_entry(a.table, a.tdtype, a.map, clip_distance(x % n - 31 - a.R, a.R) + a.R, a.buckets, a.Hq, h0 + x / n);
}

// Does the mask depend on the key alone (within a sequence)?  Then a tile's part of it is one bit a key.
__device__ __forceinline__ bool mask_by_key(const args& a) { return a.mkind == 1 && a.ms[1] == 0 && a.ms[2] == 0; }

template <class T>
__device__ __forceinline__ float dot_rows(const T* x, const T* y, int D) {
    float s = 0.f;
    for (int d = 0; d < D; ++d) s += (float)x[d] * (float)y[d];
    return s;
}
// One score, outside the matrix path, of query row q and key row k; vis = false, and neither row touched, where the row may not see the key
template <class T>
__device__ __forceinline__ float score_of(const args& a, const T* q, const T* k, int b, int h, int i, int j, int len, int off, const float* line, bool& vis) {
    vis = j < len && !(a.causal && j > off + i);
    if (!vis) return -ATTN_INF;
    float m = 0.f;
    if (a.mkind) {
        m = mask_add(a, b * a.ms[0] + h * a.ms[1] + i * a.ms[2] + j * a.ms[3]);
        vis = m != -ATTN_INF;
        if (!vis) return -ATTN_INF;
    }
    float s = dot_rows(q, k, a.D) * a.scale;
    if (a.table && line) s += line[clip_distance(j - (off + i), a.R) + a.R];
    return a.mkind ? s + m : s;
}
// ... with the bias straight from its table
template <class T>
__device__ __forceinline__ float score_from_table(const args& a, const T* q, const T* k, int b, int h, int i, int j, int len, int off, bool& vis) {
    const float s = score_of(a, q, k, b, h, i, j, len, off, nullptr, vis);
    if (!vis || !a.table) return s;
    return s + rb_entry(a.table, a.tdtype, a.map, clip_distance(j - (off + i), a.R) + a.R, a.buckets, a.Hq, h);
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
    return v;
}
// The row-by-row forms stop where every sum is NaN, which no further term changes: a batch that is NaN throughout would otherwise be made again place by
// place (2 x 16 x 4096 x 128, all of q NaN, training: 536 ms)
template <class... F>
__device__ __forceinline__ bool all_nan(bool live, F... v) { return __all(!live || (... && (v != v))); }
__device__ __forceinline__ bool not_finite(float v) { return !(fabsf(v) < ATTN_INF); }

// s[r] += the bias at distance d0 + SIGN * row_of(r)
template <int SIGN>
__device__ __forceinline__ void add_bias(f32x16& s, const float* line, int d0, int half, int R) {
    const int lo = SIGN > 0 ? d0 : d0 - 31;
    const float* at = line + ((lo < -R - 31 ? -R - 31 : lo > R ? R : lo) + R + (SIGN > 0 ? 4 * half : 31 - 4 * half));
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] += at[SIGN * row_of(r, 0)];
}

// A 32 x 32 block of raw products -> scores (MOD: with a bias, or with a mask that is additive or differs between rows) or the products as they
// are (otherwise: lengths, the triangle, truth values by key), shut places -inf.  Scores stay
// in natural units: a mask of the type's lowest value would overflow as a multiple of log2 e, and a row that holds nothing else has
// to come out even.
// The lane's column is query (i, h) and rows are keys j0 + row_of (BY_KEY = false), or the column is key j and rows are queries (true).
// bits: the tile's keys that are there (length and by-key mask), bit 0 = key j0; only with keys as rows.
template <bool MOD>
__device__ __forceinline__ void apply_keys(const args& a, f32x16& s, int b, int h, int i, int j0, int half, int off, uint32_t bits, bool diag,
                                           const float* line) {
    if constexpr (MOD) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= a.scale;
        if (a.table) add_bias<1>(s, line, j0 - (off + i), half, a.R);
    }
    if constexpr (MOD) {
        if (a.mkind && !mask_by_key(a)) {
            int64_t at = b * a.ms[0] + h * a.ms[1] + (int64_t)i * a.ms[2] + (int64_t)j0 * a.ms[3];
            asm volatile("" : "+v"(at));               // (sixteen addresses carried from tile to tile would not fit the registers)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = row_of(r, half);
                if (bits >> row & 1) {                  // (a key that is there: its mask may be read)
                    const float m = mask_add(a, at + row * a.ms[3]);
                    s[r] = m == -ATTN_INF ? -ATTN_INF : s[r] + m;
                }
            }
        }
    }
    if (bits != 0xffffffffu) {
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = bits >> row_of(r, half) & 1 ? s[r] : -ATTN_INF;
    }
    if (diag) {
        const int last = off + i - j0;                  // the last key that the query sees, within the block
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = row_of(r, half) > last ? -ATTN_INF : s[r];
    }
}
// 2^x as the one instruction: x <= 8 here, and below -126 the result is taken as 0 (the library's form pays four more instructions for denormals)
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// A row's exponentials, and with them its sum and its output until it is divided by the sum, are 2^p_lift times exp(s - m).  fp16: the reference may lag by
// 2^8 (attn_fwd.inc), so 2^7 more is what fits, and a key has its eleven bits down to 2^-21 of the reference's (64 x 700 x 128, a first key
// that takes nearly all and adds nothing, the others about 2^-19 of it: the output was off by 1.2e-3 of its norm, its own rounding is 2e-4); the other
// types need none.
template <class T>
constexpr float p_lift() { return narrow<T>() ? 7.f : 0.f; }
template <class T>
constexpr float p_drop() { return narrow<T>() ? 0x1p-7f : 1.f; }
// 2^lift exp(s - m) of a block's score; mu: m in natural units (MOD) or m * scale * log2 e - lift, of the products' units
template <class T, bool MOD>
__device__ __forceinline__ float exp_of(float s, float mu, float c1) {
    if constexpr (!MOD) return exp2_fast(s * c1 - mu);
    else if constexpr (narrow<T>()) return exp2_fast((s - mu) * ATTN_LOG2E + p_lift<T>());
    else return exp2_fast((s - mu) * ATTN_LOG2E);
}
// May anything see key j (length, by-key mask)?  Not 0: yes.  A wave's answers for 64 keys are the bits of apply_keys; asked for a tile ahead, and
// kept as the byte that was loaded, so that the load is not waited for before it is used.
__device__ __forceinline__ int key_there(const args& a, int b, int j, int len, bool by_key) {
    int there = j < len;
    if (there && by_key) there = static_cast<const uint8_t*>(a.mask)[b * a.ms[0] + j * a.ms[3]];
    return there;
}

}  // namespace attn

// ---------------------------------------------------------------------------------------------------------- host
#include <initializer_list>

static inline int attn_args(const re_attention* d, attn::args& a) {
    if (!d || !re_dtype_size(d->dtype)) return RE_EINVAL;
    if (d->B < 0 || d->Hq < 0 || d->Hkv < 1 || d->Sq < 0 || d->Sk < 0 || d->D < 1 || d->Hq % d->Hkv) return RE_EINVAL;
    if (d->D > ATTN_MAX_D || d->Sq > (1 << 30) - 1 || d->Sk > (1 << 30) - 1 || d->B > (1 << 24) || d->Hq > (1 << 16)) return RE_EUNSUPPORTED;
    if (!(d->scale > 0.f) || d->scale > 1e30f) return RE_EINVAL;
    if (d->mask ? d->mask_kind < 1 || d->mask_kind > 4 : d->mask_kind != 0) return RE_EINVAL;
    if (d->table) {
        if (!d->bucket_map || !re_dtype_size(d->table_dtype)) return RE_EINVAL;
        if (!rb_sizes_ok(d->max_distance, d->buckets)) return RE_EUNSUPPORTED;
    }
    a = attn::args{d->q, d->k, d->v, {d->q_stride[0], d->q_stride[1], d->q_stride[2]}, {d->k_stride[0], d->k_stride[1], d->k_stride[2]},
                   {d->v_stride[0], d->v_stride[1], d->v_stride[2]}, (int32_t)d->B, (int32_t)d->Hq, (int32_t)d->Hkv, (int32_t)d->Sq, (int32_t)d->Sk,
                   (int32_t)d->D, (int32_t)(d->Hq / d->Hkv), d->scale, d->causal != 0, d->mask_kind, d->mask,
                   {d->mask_stride[0], d->mask_stride[1], d->mask_stride[2], d->mask_stride[3]}, d->key_lengths, d->q_offsets, d->q_offset, d->table,
                   d->bucket_map, d->table_dtype, d->table ? (int32_t)d->max_distance : 0, d->table ? (int32_t)d->buckets : 0};
    return RE_OK;
}
static inline bool attn_empty(const attn::args& a) { return a.B == 0 || a.Hq == 0 || a.Sq == 0; }

// the kernels' general form: scores are formed place by place
static inline bool attn_mod(const attn::args& a) { return a.table || a.mkind >= 2 || (a.mkind == 1 && (a.ms[1] || a.ms[2])); }

static inline attn::order attn_order(int64_t units, int64_t tiles, int chunk) {
    attn::order o;
    o.chunk = chunk;
    o.xcd = units / chunk % 8 == 0 ? 8 : 1;
    o.units = (int32_t)(units / o.xcd);
    o.tiles = (int32_t)tiles;
    // a set fills an XCD's 32 units of two workgroups each twice over
    const int64_t set = re_cdiv(128 * (8 / o.xcd), tiles);
    o.set = (int32_t)(set < o.units ? set : o.units);
    return o;
}

struct attn_tensor {
    const void* p;
    const int64_t* stride;
};
// every row of every tensor starts on 16 bytes and is whole 16-byte chunks, and rows follow each other upwards and are not gigabytes apart (what is not
// so goes through the form that reads element by element at 64-bit addresses)
static inline bool attn_aligned(const attn::args& a, int32_t dtype, std::initializer_list<attn_tensor> ts) {
    const int64_t epc = 16 / (int64_t)re_dtype_size(dtype);
    if (a.D % epc) return false;
    for (const attn_tensor& t : ts) {
        if (reinterpret_cast<uintptr_t>(t.p) & 15) return false;
        for (int x = 0; x < 3; ++x)
            if (t.stride[x] % epc) return false;
        if (t.stride[2] < 0 || t.stride[2] > (1 << 22)) return false;      // (a tile's rows lie within 2^31 bytes of its first: unsigned 32-bit offsets)
    }
    return true;
}
#endif
