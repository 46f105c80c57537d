// fa2_product.h -- matrix product tiles, D[m, n] = sum_k A[m, k] B[n, k], on the
// 32x32x16 MFMAs: operands by direct global->LDS transfers, in stages of 64 k.
//
// Operands are 16-bit matrices in either order: ROWS are stored [m][k] (n for B),
// the others [k][m].  A tile's operand is a number of panels of 64 x 64 elements (8
// KB, rows of 128 bytes): 64 of its rows by 64 k, or 64 k rows by 64 columns.  Both
// kinds are moved by the same transfers; they differ in the swizzle (16-byte chunk
// ch of row r sits at ch ^ swz(r)) and in the read: ROWS fragments are 16-byte
// reads, the others the transposing 8-byte reads, in the same k order (lane 32 g2 +
// c holds k = 8 g2 .. 8 g2 + 7 of each step of 16), so that any two orders can meet
// in one product.
#pragma once

#include "fa2_token.h"

namespace fa2 {

__device__ __forceinline__ f16x mfma(h8 a, h8 b, f16x c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f16x mfma(b8 a, b8 b, f16x c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }

// Row of element r of a 32x32 accumulator (its column is lane & 31).
__device__ __forceinline__ int acc_row(int r, int g2) { return 8 * (r >> 2) + 4 * g2 + (r & 3); }

// A 64-bit value that is the same in every lane, in scalar registers.
__device__ __forceinline__ uint64_t uniform64(uint64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)v);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return ((uint64_t)hi << 32) | lo;
}

constexpr int PANEL = 8192;    // bytes
constexpr int PK = 64;         // k of a stage

// An operand in panels: a matrix of [rows / 64][columns / 64] panels, each 64 x 64
// elements in one piece of 8 KB, read by its rows or its columns.  Every transfer of a
// panel is one contiguous kilobyte, where rows of a matrix a large power of two wide meet
// in few channels of the memory: 16384 tokens x 32000 x 768, forward and backward, took
// 3155 us with P by rows and takes 3089 in panels.
template <bool ROWS, int NP>
struct PanelFeed {
    uint64_t base;         // the tile's first panel, k = 0
    uint32_t jstep, kstep; // bytes between the tile's panels, and between 64 k
    uint32_t off;          // this lane's bytes in a panel

    // per_row: panels in a row of panels; first: the tile's first row (column), a multiple of 64.
    __device__ __forceinline__ void init(const void *p, int per_row, int first) {
        const int lane = threadIdx.x & 63, row = 8 * (threadIdx.x >> 6) + (lane >> 3);
        off = (uint32_t)(row * 128 + (((lane & 7) ^ (ROWS ? swz_rows(row) : swz_tr(row))) << 4));
        jstep = ROWS ? (uint32_t)per_row * PANEL : PANEL;
        kstep = ROWS ? PANEL : (uint32_t)per_row * PANEL;
        base = uniform64((uint64_t)(uintptr_t)p + (uint64_t)(uint32_t)(first >> 6) * jstep);
    }

    __device__ __forceinline__ void issue(int k0, uint32_t lds) const {
        lds += __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
        const uint64_t b = base + (uint64_t)(uint32_t)(k0 >> 6) * kstep;
#pragma unroll
        for (int j = 0; j < NP; ++j) lds_dma16_at(b + (uint64_t)(uint32_t)j * jstep, off, lds + j * PANEL);
    }
};

enum Source {
    CLAMPED,   // the operand may end inside the tile
    RAGGED,    // and its stored rows inside a panel
    PADDED,    // it has every row of the tile
    PANELED,   // it is stored in panels
};

// One operand of a tile: where the transfers of this thread read.  Eight waves
// move a panel, wave w its rows 8 w .. 8 w + 7.
template <bool ROWS, Source S, int NP>
struct Feed {
    uint64_t base;                 // ROWS: first row, k = 0; else k = 0, column 0
    uint32_t ld;                   // bytes of a row, below 2^24
    uint32_t row, chunk;           // this lane's row of a panel; byte in the row
    int last;                      // last row there is (k row, if not ROWS), from base
    uint32_t end;                  // RAGGED: bytes of a row
    uint32_t col[ROWS ? 1 : NP];   // not ROWS: bytes of each panel's first column

    // p: the matrix; first: the tile's first row (column); limit: rows (columns) there
    // are; klimit: k there are.  Rows (columns) past the limit are read from the last there
    // are, and so are k rows; k columns past theirs become zeros, whatever stands
    // behind them.  Columns: a multiple of 8 where RAGGED, else of 64.
    __device__ __forceinline__ void init(const void *p, int64_t ld_elems, int first, int limit, int klimit) {
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
        row = 8 * w + (lane >> 3);
        ld = (uint32_t)ld_elems * 2;
        if constexpr (ROWS) {
            const int f0 = min(first, limit - 1);
            base = uniform64((uint64_t)(uintptr_t)p + (uint64_t)f0 * (uint64_t)ld);
            last = limit - 1 - f0;
            end = (uint32_t)klimit * 2;
            chunk = (uint32_t)((lane & 7) ^ swz_rows(row)) << 4;
        } else {
            base = uniform64((uint64_t)(uintptr_t)p);
            last = klimit - 1;
            end = (uint32_t)limit * 2;
            chunk = (uint32_t)((lane & 7) ^ swz_tr(row)) << 4;
#pragma unroll
            for (int j = 0; j < NP; ++j)
                col[j] = (uint32_t)(S == RAGGED ? first + 64 * j : min(first + 64 * j, limit - 64)) * 2;
        }
    }

    // Starts the transfers of stage k0 / PK into the panels at LDS address `lds`.  Rows are
    // held to the last one at every issue: offsets kept for each panel cost the registers
    // that make the forward's kernel reload some from scratch memory, behind the
    // transfers in flight.
    __device__ __forceinline__ void issue(int k0, uint32_t lds) const {
        lds += __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
        if constexpr (ROWS) {
            const uint64_t b = base + (uint64_t)(uint32_t)k0 * 2;
            int r = (int)row;
            if (S != PADDED) asm volatile("" : "+v"(r));   // no offset leaves the loop
            auto panels = [&]() FA2_INLINE {
#pragma unroll
                for (int j = 0; j < NP; ++j)
                    if (S == PADDED)
                        lds_dma16_at(b + (uint64_t)(64 * j) * ld, mul_u24(ld, (uint32_t)r) + chunk, lds + j * PANEL);
                    else
                        lds_dma16_at(b, mul_u24(ld, (uint32_t)min(64 * j + r, last)) + chunk, lds + j * PANEL);
            };
            const uint32_t left = end - (uint32_t)k0 * 2;
            if (S != RAGGED || left >= 2 * PK) {
                panels();
            } else {   // every wave has lanes on both sides: it starts as many transfers as ever
                FA2_COLD_BRANCH();
                if (chunk < left) {
                    panels();
                } else {
                    typedef __attribute__((address_space(3))) f4 lds_f4;
#pragma unroll
                    for (int j = 0; j < NP; ++j) *(lds_f4 *)(lds + j * PANEL + (threadIdx.x & 63) * 16) = f4{0.f, 0.f, 0.f, 0.f};
                }
            }
        } else {
            const uint32_t o = mul_u24(ld, (uint32_t)min((int)row, last - k0));
            const uint64_t b = base + (uint64_t)(uint32_t)k0 * ld;
#pragma unroll
            for (int j = 0; j < NP; ++j)
                if (S == RAGGED)
                    lds_dma16_at(b, o + min(col[j] + chunk, end - 16), lds + j * PANEL);
                else
                    lds_dma16_at(b + col[j], o + chunk, lds + j * PANEL);
        }
    }
};

// Fragment reads of one operand: 32 rows (columns) from `at` (a multiple of 32) of
// the tile, k step ks of the stage.  W: rows (columns) that a wave reads in all.
template <typename T, bool ROWS, int W>
struct Frag {
    typedef typename vec_of<T>::v8 v8;
    uint32_t off[4];   // ROWS: of k step 0..3; else: column 0 / 32 of a panel, first / second read

    // first: the first row (column) that the wave reads.
    __device__ __forceinline__ void init(int first) {
        const int lane = threadIdx.x & 63;
        if constexpr (ROWS) {
            const int c = lane & 31, g2 = lane >> 5;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) off[ks] = (uint32_t)(c * 128 + (((2 * ks + g2) ^ swz_rows(c)) << 4));
        } else {
            const int G = lane >> 4, s = lane & 15;
#pragma unroll
            for (int q = 0; q < (W == 32 ? 2 : 4); ++q) {
                const int half = W == 32 ? first & 32 : 32 * (q >> 1);
                const int row = 8 * (G >> 1) + (s >> 2) + 4 * (q & 1), col = half + 16 * (G & 1) + 4 * (s & 3);
                off[q] = (uint32_t)(row * 128 + (((col >> 3) ^ swz_tr(row)) << 4) + 2 * (col & 7));
            }
        }
    }

    __device__ __forceinline__ v8 read(const char *stage, int at, int ks) const {
        typedef __attribute__((address_space(3))) const char lds_char;
        lds_char *p = (lds_char *)stage + (at >> 6) * PANEL;
        if constexpr (ROWS) {
            return *(__attribute__((address_space(3))) const v8 *)(p + (at & 32) * 128 + off[ks]);
        } else {
            const int q = W == 32 ? 0 : (at & 32) >> 4;
            const s4v r0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v *)(p + ks * 2048 + off[q]));
            const s4v r1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4v *)(p + ks * 2048 + off[q + 1]));
            return __builtin_bit_cast(v8, __builtin_shufflevector(r0, r1, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// Tile of 64 MP x 64 NP by eight waves in WM x WN, each (64 MP / WM) x (64 NP / WN),
// with NS stages in LDS.
template <typename T, bool AROWS, bool BROWS, Source AS, Source BS, int MP, int NP, int WM, int WN, int NS = 2>
struct Product {
    static_assert(WM * WN == 8, "eight waves");
    static constexpr int TM = 64 * MP, TN = 64 * NP;
    static constexpr int MI = TM / WM / 32, NI = TN / WN / 32;   // a wave's 32x32 blocks
    static constexpr int STAGE = (MP + NP) * PANEL;
    static constexpr int LDS = NS * STAGE;

    typename std::conditional<AS == PANELED, PanelFeed<AROWS, MP>, Feed<AROWS, AS, MP>>::type A;
    typename std::conditional<BS == PANELED, PanelFeed<BROWS, NP>, Feed<BROWS, BS, NP>>::type B;
    Frag<T, AROWS, TM / WM> fa;
    Frag<T, BROWS, TN / WN> fb;
    char *mem;
    uint32_t lds;
    int wm, wn;        // the wave's first row and column of the tile

    __device__ __forceinline__ void init(char *m) {
        const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        mem = m;
        lds = lds_addr(m);
        wm = (w % WM) * (TM / WM);
        wn = (w / WM) * (TN / WN);
        fa.init(wm);
        fb.init(wn);
    }

    // Starts the transfers of stage k0 / PK into buffer buf.
    __device__ __forceinline__ void issue(int k0, int buf) const {
        A.issue(k0, lds + buf * STAGE);
        B.issue(k0, lds + buf * STAGE + MP * PANEL);
    }

    typedef typename vec_of<T>::v8 v8;
    struct Frags {
        v8 a[MI], b[NI];
    };

    __device__ __forceinline__ void read(Frags &f, int buf, int ks) const {
        const char *s = mem + buf * STAGE;
#pragma unroll
        for (int i = 0; i < MI; ++i) f.a[i] = fa.read(s, wm + 32 * i, ks);
#pragma unroll
        for (int j = 0; j < NI; ++j) f.b[j] = fb.read(s + MP * PANEL, wn + 32 * j, ks);
    }

    static __device__ __forceinline__ void multiply(const Frags &f, f16x (&acc)[MI][NI]) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = mfma(f.a[i], f.b[j], acc[i][j]);
    }

    static __device__ __forceinline__ void zero(f16x (&acc)[MI][NI]) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = zero16();
    }

    // Holds the scheduler to the order of a k step: its products, with the reads of the
    // next step's fragments spread over the first of them (left to itself it moves the
    // reads to their use, and every step waits for LDS).
    static __device__ __forceinline__ void interleave() {
        constexpr int R = MI * (AROWS ? 1 : 2) + NI * (BROWS ? 1 : 2), M = MI * NI;
        constexpr int PER = (R + M - 1) / M;   // reads a product
#pragma unroll
        for (int i = 0; i < M; ++i) {
            if (i * PER < R) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);   // LDS reads
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                      // MFMA
        }
    }

    // A stream of stages.  begin() starts the first NS and reads the first
    // fragments; steps() consumes n stages (at least one) into a tile's accumulators.  next(buf) starts the following stage's
    // transfers into buffer buf and returns whether there was one left.
    //
    // The fragments of each k step are read while the step before is multiplied.
    // The one barrier of a stage stands before its last step: by then every wave
    // holds that step's fragments, so the stage's buffer is free for the stage NS
    // later, and the next stage has landed, so its first fragments can be read
    // behind the last step's products.
    struct Stream {
        Frags f0;
        int buf, ahead;   // the current stage's buffer; stages started after it
    };

    template <typename N>
    __device__ __forceinline__ void begin(Stream &st, N next) const {
        int ahead = -1;
#pragma unroll
        for (int s = 0; s < NS; ++s) ahead += next(s) ? 1 : 0;
        landed<NS - 1>(ahead);
        st.buf = 0;
        st.ahead = ahead;
        read(st.f0, 0, 0);
    }

    // Every wave's transfers of all but the last `F` stages started have landed, if all
    // those are under way (a wave's loads complete in order); else all of them.
    template <int F>
    static __device__ __forceinline__ void landed(int ahead) {
        if (F > 0 && ahead == F)
            vm_wait<F *(MP + NP)>();
        else
            vm_wait<0>();
        lds_barrier();
    }

    // FIRST: the accumulators start from zero, as the constant operand of their first
    // products (cleared registers cost 2% at K = 768).
    template <bool FIRST, typename N>
    __device__ __forceinline__ void step(Stream &st, f16x (&acc)[MI][NI], N &next) const {
        Frags f1;
        read(f1, st.buf, 1);
        if (FIRST) zero(acc);
        multiply(st.f0, acc);
        interleave();
        read(st.f0, st.buf, 2);
        multiply(f1, acc);
        interleave();
        read(f1, st.buf, 3);
        multiply(st.f0, acc);
        interleave();
        landed<NS - 2>(--st.ahead);   // counted from the next stage on
        st.ahead += next(st.buf) ? 1 : 0;
        st.buf = NS == 2 ? st.buf ^ 1 : st.buf == NS - 1 ? 0 : st.buf + 1;
        read(st.f0, st.buf, 0);
        multiply(f1, acc);
        interleave();
    }

    template <typename N>
    __device__ __forceinline__ void steps(Stream &st, int n, f16x (&acc)[MI][NI], N next) const {
        step<true>(st, acc, next);
        for (int t = 1; t < n; ++t) step<false>(st, acc, next);
    }

    // k from kbeg to kend, multiples of PK, of the operands as they are.  Leaves no
    // transfer in flight and every wave past its last read.
    __device__ __forceinline__ void run(int kbeg, int kend, f16x (&acc)[MI][NI]) const {
        int k = kbeg;
        auto next = [&](int b) FA2_INLINE {
            const bool more = k < kend;
            if (more) issue(k, b);
            k += PK;
            return more;
        };
        Stream st;
        begin(st, next);
        if (kbeg < kend)
            steps(st, (kend - kbeg) / PK, acc, next);
        else
            zero(acc);
        lds_barrier();
    }
};

// Swizzle of store_rows: 16 consecutive rows' 8-byte writes of one column group, and two
// rows' 16-byte reads, touch distinct banks.
__device__ __forceinline__ int swz_out(int r) { return (r ^ (r >> 3)) & 7; }

// store_rows_f16 for either 16-bit type: a wave's 32 x 64 block in two
// accumulators (acc0: columns 0..31, acc1: 32..63, row = lane & 31), times mul, as
// rows dst + r * stride for r < nrows, through 4 KB of LDS that only this wave
// touches.  Columns from ncols on are left out (a multiple of 8 for whole 16-byte stores).
template <typename T>
__device__ __forceinline__ void store_rows(const f16x &acc0, const f16x &acc1, float mul, char *blk, T *dst, int64_t stride,
                                           int nrows, int ncols, bool vec16) {
    typedef typename vec_of<T>::v4 v4;
    typedef typename vec_of<T>::v8 v8;
    const int lane = threadIdx.x & 63, c = lane & 31, g2 = lane >> 5;
#pragma unroll
    for (int db = 0; db < 2; ++db)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f4 x;
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] = (db ? acc1 : acc0)[4 * i + j] * mul;
            *reinterpret_cast<v4 *>(blk + c * 128 + (((4 * db + i) ^ swz_out(c)) << 4) + 8 * g2) = __builtin_convertvector(x, v4);
        }
    const int ch = lane & 7;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int r = 8 * k + (lane >> 3);
        const v8 v = *reinterpret_cast<const v8 *>(blk + r * 128 + ((ch ^ swz_out(r)) << 4));
        if (r < nrows) {
            T *p = dst + r * stride + 8 * ch;
            if (vec16 && 8 * ch + 8 <= ncols) {
                *reinterpret_cast<v8 *>(p) = v;
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (8 * ch + e < ncols) p[e] = v[e];
            }
        }
    }
}

}  // namespace fa2
