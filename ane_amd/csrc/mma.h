// mma.h — operand tiles of the matrix instructions, for the kernels that multiply channel-first tensors.
//
// An operand lies in LDS as a panel: rows of 128 bytes (64 bfloat16 or 32 fp32 values), the positions of a tensor [channel][position]
// along the row, one channel to a row.  A panel is read in two ways:
//   columns: a lane takes one position and the values of several channels (products over the channels: scores from Q and K).  In
//            bfloat16 that is gfx950's transposing LDS read, which hands 4 rows x 16 columns around among 16 lanes; fp32 needs one
//            value per lane and instruction.
//   rows:    a lane takes one channel and several positions (products over the positions: P V, dS K, and the gradients).
// The result of a 32 x 32 product, C[i][j], has column j = lane % 32 in every lane and rows i = 8 * (r / 4) + 4 * (lane / 32) + r % 4
// in its 16 registers r.  A product over those rows takes the registers as they are for its second operand when the first one is
// read in the same order of positions: no score and no gradient of one ever passes through LDS.
//
// Chunk c (16 bytes) of row r is kept in place c ^ panel_swz(r).  Of the 64 banks (256 bytes: two rows) a transposing read then
// touches each at most twice with 512 bytes, a row read of 8 bytes per lane all of them with 16 rows, one of 16 bytes no bank twice
// with 8 rows.
#pragma once
#include "panel_walk.h"
#include "tile.h"

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

constexpr int PANEL_ROW = 128;      // bytes

__device__ __forceinline__ int panel_at(int row, int chunk) { return row * PANEL_ROW + ((chunk ^ panel_swz(row)) << 4); }

// row of register r of a 32 x 32 product, less the 4 that lanes 32..63 add
__device__ __forceinline__ constexpr int acc_row(int r) { return 8 * (r >> 2) + (r & 3); }

__device__ __forceinline__ bool is_finite(float v) { return (__float_as_uint(v) & 0x7f800000u) != 0x7f800000u; }
__device__ __forceinline__ v16f v16_zero() {
    v16f z;
#pragma unroll
    for (int r = 0; r < 16; r++) z[r] = 0.f;
    return z;
}

template <typename T> struct Mma;

template <> struct Mma<bf16_t> {
    static constexpr int COLS = 64, SUBS = 2, EPC = 8;      // columns of a panel, groups of 32 of them, values per 16 bytes
    static constexpr int STEP = 16;                         // rows of a panel that one product over the channels takes
    typedef bf16x8 Frag;
    typedef v4u_any Any16;                                  // 16 bytes of global memory at any value
    // Values of rows step*16 + 8*(lane/32) .. +7 at column sub*32 + lane%32.
    static __device__ __forceinline__ Frag columns(const char *panel, int sub, int step) {
        const int lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4 & 1, h = lane >> 5;
        const int row = 8 * h + (i >> 2), chunk = sub * 4 + 2 * g + (i >> 1 & 1);
        const char *at = panel + step * (16 * PANEL_ROW) + ((i & 1) << 3);
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(at + panel_at(row, chunk)));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s *)(at + panel_at(row + 4, chunk)));
        const v8s v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        return __builtin_bit_cast(Frag, v);
    }
    static __device__ __forceinline__ v16f mul(Frag a, Frag b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    // For products over the positions whose result rows are the panel's: columns step*16 + 8*(lane/32) .. +7 of row block*32 + lane%32.
    static __device__ __forceinline__ Frag along(const char *panel, int block, int step) {
        const int lane = threadIdx.x & 63;
        return *reinterpret_cast<const Frag *>(panel + block * (32 * PANEL_ROW) + panel_at(lane & 31, step * 2 + (lane >> 5)));
    }

    // A product's registers as the second operand of a product over its rows: each value's upper half, and what that leaves of it rounded
    // to bfloat16, so that the pair is off by 2^-15 of the value at most.  (One bfloat16 value, 2^-8, shows in results of that type: error
    // of a batch's attention against 64 bits 0.0019 where the rounding of the results alone is 0.0016, of its gradients 0.0026 for 0.0017.)
    // An infinity leaves NaN; WILD: nothing.
    struct Packed { Frag hi[2], lo[2]; };
    template <bool WILD>
    static __device__ __forceinline__ Packed pack(const v16f &p) {
        Packed out;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            v4u hi, lo;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const unsigned a = __float_as_uint(p[8 * j + 2 * i]), b = __float_as_uint(p[8 * j + 2 * i + 1]);
                hi[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
                float ra = p[8 * j + 2 * i] - __uint_as_float(a & 0xffff0000u), rb = p[8 * j + 2 * i + 1] - __uint_as_float(b & 0xffff0000u);
                if (WILD) {
                    ra = is_finite(p[8 * j + 2 * i]) ? ra : 0.f;
                    rb = is_finite(p[8 * j + 2 * i + 1]) ? rb : 0.f;
                }
                lo[i] = f2_to_bf2(ra, rb);
            }
            out.hi[j] = __builtin_bit_cast(Frag, hi);
            out.lo[j] = __builtin_bit_cast(Frag, lo);
        }
        return out;
    }
    // The values of the panel's 32 columns `sub` at rows block*32 + lane%32, in the order of a product's registers.
    struct Row { v8s v[2]; };
    static __device__ __forceinline__ Row row(const char *panel, int block, int sub) {
        const int lane = threadIdx.x & 63, row = lane & 31, h = lane >> 5;
        const char *at = panel + block * (32 * PANEL_ROW) + (h << 3);
        Row out;
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const v4s lo = *reinterpret_cast<const v4s *>(at + panel_at(row, sub * 4 + 2 * j));
            const v4s hi = *reinterpret_cast<const v4s *>(at + panel_at(row, sub * 4 + 2 * j + 1));
            out.v[j] = v8s{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        }
        return out;
    }
    // acc[row][column] += sum over them of row[.] * p[.][column]; FINITE: infinities and NaNs of the panel count as zero.
    template <bool FINITE>
    static __device__ __forceinline__ v16f mul_row(const Row &r, const Packed &p, v16f acc) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            v8s v = r.v[j];
            if constexpr (FINITE) {
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = (v[e] & 0x7f80) == 0x7f80 ? (short)0 : v[e];
            }
            acc = mul(__builtin_bit_cast(Frag, v), p.lo[j], acc);
            acc = mul(__builtin_bit_cast(Frag, v), p.hi[j], acc);
        }
        return acc;
    }
    static __device__ __forceinline__ float value(const char *panel, int row, int col) {
        return bf_to_f(*reinterpret_cast<const bf16_t *>(panel + panel_at(row, col >> 3) + ((col & 7) << 1)));
    }
    // c + the sum of a lane's products
    static __device__ __forceinline__ float dot(Frag a, Frag b, float c) {
#pragma unroll
        for (int j = 0; j < 8; j++) c = __builtin_fmaf((float)a[j], (float)b[j], c);
        return c;
    }
};

template <> struct Mma<float> {
    static constexpr int COLS = 32, SUBS = 1, EPC = 4;
    static constexpr int STEP = 2;
    typedef float Frag;
    typedef unsigned Any16 __attribute__((ext_vector_type(4), aligned(4)));
    static __device__ __forceinline__ Frag columns(const char *panel, int, int step) {
        const int lane = threadIdx.x & 63, col = lane & 31;
        return *reinterpret_cast<const float *>(panel + panel_at(2 * step + (lane >> 5), col >> 2) + ((col & 3) << 2));
    }
    static __device__ __forceinline__ v16f mul(Frag a, Frag b, v16f c) { return __builtin_amdgcn_mfma_f32_32x32x2f32(a, b, c, 0, 0, 0); }
    typedef v16f Packed;
    template <bool WILD>
    static __device__ __forceinline__ Packed pack(const v16f &p) { return p; }
    struct Row { v4f v[4]; };
    static __device__ __forceinline__ Row row(const char *panel, int block, int) {
        const int lane = threadIdx.x & 63, row = lane & 31, h = lane >> 5;
        const char *at = panel + block * (32 * PANEL_ROW);
        Row out;
#pragma unroll
        for (int j = 0; j < 4; j++) out.v[j] = *reinterpret_cast<const v4f *>(at + panel_at(row, 2 * j + h));
        return out;
    }
    template <bool FINITE>
    static __device__ __forceinline__ v16f mul_row(const Row &r, const Packed &p, v16f acc) {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc = mul(FINITE && !is_finite(r.v[j][e]) ? 0.f : r.v[j][e], p[4 * j + e], acc);
        return acc;
    }
    static __device__ __forceinline__ float value(const char *panel, int row, int col) {
        return *reinterpret_cast<const float *>(panel + panel_at(row, col >> 2) + ((col & 3) << 2));
    }
    static __device__ __forceinline__ float dot(Frag a, Frag b, float c) { return __builtin_fmaf(a, b, c); }
};

// acc + sum over the channels of panel[channel][sub*32 + .] * own[channel][.]: what a group of products takes is read while the group before
// it is multiplied.  (Left alone, the compiler reads right before each product, or so far ahead that registers spill.)
template <typename T, int STEPS>
__device__ __forceinline__ v16f over_channels(const char *panel, int sub, const typename Mma<T>::Frag (&own)[STEPS], v16f acc) {
    constexpr int GROUP = sizeof(T) == 2 ? 2 : 16, GROUPS = STEPS / GROUP;
    static_assert(GROUPS * GROUP == STEPS, "whole groups");
    typename Mma<T>::Frag f[2][GROUP];
#pragma unroll
    for (int i = 0; i < GROUP; i++) f[0][i] = Mma<T>::columns(panel, sub, i);
#pragma unroll
    for (int g = 0; g < GROUPS; g++) {
        if (g + 1 < GROUPS) {
#pragma unroll
            for (int i = 0; i < GROUP; i++) f[(g + 1) & 1][i] = Mma<T>::columns(panel, sub, (g + 1) * GROUP + i);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < GROUP; i++) acc = Mma<T>::mul(f[g & 1][i], own[g * GROUP + i], acc);
    }
    return acc;
}
// acc[channel][.] += sum over the panel's 32 columns `sub` of panel[channel][.] * p[.][.], for all channels
template <typename T, int HDB, bool FINITE>
__device__ __forceinline__ void over_positions(v16f (&acc)[HDB], const char *panel, int sub, const typename Mma<T>::Packed &p) {
    typename Mma<T>::Row r[2];
    r[0] = Mma<T>::row(panel, 0, sub);
#pragma unroll
    for (int d = 0; d < HDB; d++) {
        if (d + 1 < HDB) {
            r[(d + 1) & 1] = Mma<T>::row(panel, d + 1, sub);
            __builtin_amdgcn_sched_barrier(0);
        }
        acc[d] = Mma<T>::template mul_row<FINITE>(r[d & 1], p, acc[d]);
    }
}

// ---- from memory straight into LDS ----
// 16 bytes a lane, the lanes of an instruction one after the other (eight rows of a panel), so what panel_at() would put elsewhere is
// fetched by another lane instead: lane l reads chunk (l & 7) ^ panel_swz(row) of row l / 8.  Addresses are multiples of 16 bytes.  A read
// outside of the buffer gives zero.
typedef int rsrc_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ rsrc_t buffer_at(const void *p, unsigned long long bytes) {
    const unsigned long long a = (unsigned long long)p;
    return rsrc_t{(int)a, (int)(a >> 32) & 0xffff, (int)(unsigned)(bytes < 0xffffff00ull ? bytes : 0xffffff00ull), 0x00027000};
}
// Place in LDS, as loads to it are told: taken once from the array, then counted on as a number (each conversion of a pointer would compare
// it with null).
__device__ __forceinline__ unsigned lds_place(const char *array) {
    return (unsigned)(unsigned long long)(__attribute__((address_space(3))) const char *)array;
}
// LDS[place + 16 * lane] = 16 bytes of the buffer at voffset + soffset.  Counts in vmcnt, and nothing but that counter tells when it is there.
// (With the builtin for it the compiler waits for all loads under way before every transposing read of LDS.)  It has no result register.
// m0, which it sets, is reserved: the compiler keeps nothing there, refuses to have it named as clobbered, and sets it right before an instruction
// of its own that needs it; these kernels have none.
// The compiler does not look into the asm, so its wait states are here: five between a vector instruction that writes a scalar register
// (readfirstlane, where the compiler does not see by itself that a value is the same in all lanes) and a load that reads it, one between m0 and
// a load into LDS.  (tests/test_wait_states.py looks the library's code over for both.  They are in every load, where the values are known to be
// the same too, at up to 1 %: gradients of 4096 positions 398 -> 401 us, 32000 x 4096 results of 768 terms 282 -> 285, the others of ten cases
// no difference.)
__device__ __forceinline__ void load_to_lds(rsrc_t r, unsigned voffset, unsigned soffset, unsigned place) {
    auto uni = [](int v) { return __builtin_amdgcn_readfirstlane(v); };        // (nothing, where the compiler sees it by itself)
    const rsrc_t u = {uni(r[0]), uni(r[1]), uni(r[2]), uni(r[3])};
    asm volatile("s_mov_b32 m0, %3\n\ts_nop 3\n\tbuffer_load_dwordx4 %0, %1, %2 offen lds"
                 :: "v"(voffset), "s"(u), "s"(uni((int)soffset)), "s"(uni((int)place)) : "memory");
}
// All but the newest LEFT of the wave's loads are there and all but its newest READS reads of LDS done, and so are the other waves'.
template <int LEFT, int READS>
__device__ __forceinline__ void loads_and_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(%1)\n\ts_barrier" :: "n"(LEFT), "n"(READS) : "memory");
}
