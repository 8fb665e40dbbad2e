// Shared parts of the gated delta rule kernels.
//
// The rule, per value head, with a state S [D, DV]:
//     S_t = a_t S_{t-1} + k_t u_t^T,   u_t = b_t (v_t - a_t S_{t-1}^T k_t),   o_t = scale S_t^T q_t,   a_t = exp(g_t).
// Over a chunk of 64 positions that starts from S0, with G the running sum of g inside the chunk, E_ts = exp(G_t - G_s),
// L the strictly lower part of E * (K K^T) and T = (I + L diag(b))^-1:
//     Y = V - e^G K S0,   X = T Y,   U = b X,   O = scale e^G Q S0 + P U,   P = scale tril(E * Q K^T),
//     S1 = e^{G_63} S0 + K^T (e^{G_63 - G} U).
// T depends on K, g and b alone, so one parallel kernel forms T and P of every chunk (delta_prepare.cu) and only products
// with the state are left to the chain of chunks (delta_forward.cu).  T = I - (products of contractions), so for key
// vectors of length one its entries stay within one: the inverse is well conditioned and survives a bf16 rounding.
//
// A fragment notation used throughout: mma.m16n8k16 keeps its 16 x 8 accumulator as (row lane/4 and lane/4 + 8, columns
// 2 (lane%4) and +1); two neighbouring accumulators, rounded to bf16 and packed in pairs, are the 16 x 16 left operand of
// the next product.  Everything that depends on the state is computed transposed ([dv, position] and [dv, d]), so a warp
// owns 16 columns of the state for the whole sequence and the chain of products never leaves its registers.
#pragma once
#include <atomic>

#include "dism_common.cuh"

namespace dism {

// Opts a kernel into its dynamic shared memory, once per device (the call costs a microsecond of host time).
template <auto* KERNEL>
cudaError_t allow_shared(int bytes) {
    static std::atomic<uint64_t> done{0};
    int device = 0;
    if (cudaError_t status = cudaGetDevice(&device)) return status;
    const uint64_t bit = device < 64 ? uint64_t(1) << device : 0;
    if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
    if (cudaError_t status = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)) return status;
    done.fetch_or(bit, std::memory_order_relaxed);
    return cudaSuccess;
}

constexpr int CHUNK = 64;
// Per chunk and head: e^G, b, e^{G_63 - G}, the product of the last two, and G as a pair of floats.
constexpr int ROW_DECAY = 0, ROW_BETA = CHUNK, ROW_TAIL = 2 * CHUNK, ROW_WRITE = 3 * CHUNK, ROW_HIGH = 4 * CHUNK, ROW_LOW = 5 * CHUNK, ROW_VALUES = 6 * CHUNK;
constexpr int MATRIX = 10 * 256;           // elements of T and P of one chunk and head: the 16 x 16 tiles up to the diagonal
#define NOT_A_NUMBER __int_as_float(0x7fc00000)

__device__ __forceinline__ void mma16816(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned smem_address(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void ldsm4(unsigned (&r)[4], unsigned address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void ldsm4_trans(unsigned (&r)[4], unsigned address) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(address) : "memory");
}
__device__ __forceinline__ void stsm4_trans(unsigned address, unsigned r0, unsigned r1, unsigned r2, unsigned r3) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(address), "r"(r0), "r"(r1), "r"(r2),
                 "r"(r3) : "memory");
}
__device__ __forceinline__ unsigned pack2(float lo, float hi) {
    __nv_bfloat162 pair = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<unsigned*>(&pair);
}
__device__ __forceinline__ float low_half(unsigned x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float high_half(unsigned x) { return __uint_as_float(x & 0xffff0000u); }
// What the rounding to bf16 left out, as bf16 again: value and remainder carry 16 bits between them.
__device__ __forceinline__ unsigned pack2_rest(float lo, float hi, unsigned rounded) {
    return pack2(lo - low_half(rounded), hi - high_half(rounded));
}
// Two neighbouring accumulators (columns 16 j .. 16 j + 15) as the left operand of the next product.
__device__ __forceinline__ void to_operand(unsigned (&a)[4], const float (&c0)[4], const float (&c1)[4]) {
    a[0] = pack2(c0[0], c0[1]), a[1] = pack2(c0[2], c0[3]), a[2] = pack2(c1[0], c1[1]), a[3] = pack2(c1[2], c1[3]);
}
__device__ __forceinline__ void to_operand_rest(unsigned (&r)[4], const unsigned (&a)[4], const float (&c0)[4], const float (&c1)[4]) {
    r[0] = pack2_rest(c0[0], c0[1], a[0]), r[1] = pack2_rest(c0[2], c0[3], a[1]);
    r[2] = pack2_rest(c1[0], c1[1], a[2]), r[3] = pack2_rest(c1[2], c1[3], a[3]);
}

// Byte offsets a lane passes to ldmatrix / stmatrix for a 16 x 16 tile of a row-major matrix with `pitch` bytes a row.
// rows_first: matrices in the order (rows 0-7, cols 0-7), (rows 8-15, cols 0-7), (rows 0-7, cols 8-15), (rows 8-15, cols 8-15);
// cols_first: the two middle ones exchanged.
__device__ __forceinline__ unsigned rows_first(int lane, int pitch) { return ((lane & 7) + (lane & 8)) * pitch + (lane >> 4) * 16; }
__device__ __forceinline__ unsigned cols_first(int lane, int pitch) { return ((lane & 7) + ((lane >> 4) << 3)) * pitch + ((lane >> 3) & 1) * 16; }
// The kernels hand T, P and the states to one another as 8 x 8 blocks of 128 contiguous bytes: fragments leave and enter in whole
// lines and no access has a bank conflict.  States: `width` blocks to a row of blocks.  T and P: 16 x 16 tiles of four blocks, by
// rows, the tiles on and below the diagonal one after the other.
__device__ __forceinline__ unsigned rows_first_blocked(int lane, int width) { return (((lane >> 3) & 1) * width + (lane >> 4)) * 128 + (lane & 7) * 16; }
__device__ __forceinline__ unsigned cols_first_blocked(int lane, int width) { return ((lane >> 4) * width + ((lane >> 3) & 1)) * 128 + (lane & 7) * 16; }
__device__ __forceinline__ unsigned rows_first_tile(int lane) { return rows_first_blocked(lane, 2); }
__device__ __forceinline__ unsigned cols_first_tile(int lane) { return lane * 16; }
__host__ __device__ constexpr int tile_at(int row_tile, int column_tile) { return (row_tile * (row_tile + 1) / 2 + column_tile) * 512; }

// Zeros in the rows of no document, before the first and behind the last: `pieces` of 16 bytes from `tensor` on in each row.
template <int THREADS>
__device__ __forceinline__ void clear_rows(char* tensor, int64_t stride, int pieces, int64_t first, int64_t last, int thread) {
    for (int64_t i = thread; i < (last - first) * pieces; i += THREADS)
        *reinterpret_cast<uint4*>(tensor + (first + i / pieces) * stride + i % pieces * 16) = make_uint4(0, 0, 0, 0);
}

// Where the sequences lie.  Fixed layout: `sequences` rows of n positions.  Packed: one row of n positions, document i at
// [cu[i], cu[i+1]).  Every chunk has a slot of its own: in a pack, document i starts at slot cu[i] / 64 + i, which leaves
// room for its last, partly filled chunk and needs no running sum over the documents.  Entries of cu are clamped to the
// pack, so whatever they hold, every access stays inside the tensors.
struct DeltaLayout {
    const int* cu;
    int sequences, n;
    __host__ __device__ int chunks() const { return (n + CHUNK - 1) / CHUNK; }
    __host__ __device__ int64_t slots() const { return cu ? int64_t(n / CHUNK) + sequences : int64_t(sequences) * chunks(); }
    __device__ int start(int i) const { return min(max(__ldg(cu + i), 0), n); }
    __device__ void span(int sequence, int64_t& row, int& length, int64_t& slot) const {
        if (!cu) {
            row = int64_t(sequence) * n, length = n, slot = int64_t(sequence) * chunks();
            return;
        }
        const int begin = start(sequence);
        row = begin, length = max(start(sequence + 1) - begin, 0), slot = begin / CHUNK + sequence;
    }
    // Row and number of positions of the chunk in a slot; zero positions when the slot is not used.
    __device__ void chunk(int64_t slot, int64_t& row, int& count) const {
        int64_t first;
        int length, sequence;
        if (!cu) {
            sequence = int(unsigned(slot) / unsigned(chunks()));  // slots fit 31 bits
        } else {
            int lo = 0, hi = sequences - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (start(mid) / CHUNK + mid <= slot) lo = mid;
                else hi = mid - 1;
            }
            sequence = lo;
        }
        span(sequence, row, length, first);
        const int64_t before = (slot - first) * CHUNK;
        count = before < 0 ? 0 : int(min(int64_t(CHUNK), max(int64_t(length) - before, int64_t(0))));
        row += max(before, int64_t(0));
    }
};

// A chain of chunks is cut into segments of `length` chunks (0: not cut) when there are too few chains to fill the device.  The state is
// linear in the state at the segment's start, S_end = M S_start + B, so a first launch finds M (the chain applied to the unit matrix
// without values) and B (the chain from zero) of all segments but the last of a sequence at once, and a second one runs every segment
// from its true start, which it puts together from the M and B before it.  CTAs are numbered like chunks: in a pack, document i
// begins at segment slot / length + i.  What is kept of segments lies closer: of a sequence of c chunks only the first (c - 1) / length segments
// are (the last has no successor; in the reverse chain, the first no predecessor, and the others move up by one), so they fit from place
// slot / length on without meeting the next sequence's, and short documents take no room.
struct DeltaSegments {
    int length;
    float* ends;                  // B as accumulator fragments, [stored, H, D * DV]
    __nv_bfloat16 *m, *m_rest;    // M, transposed, in 8 x 8 blocks, as pairs, [stored, H, D * D]
    __host__ __device__ int64_t stored(const DeltaLayout& layout) const { return length ? layout.slots() / length : 0; }
    // The place of the segment that begins with the chunk in this slot; that of the next one of the sequence is one further.
    __device__ int64_t place(int64_t slot) const { return slot / length; }
    __host__ __device__ int64_t count(const DeltaLayout& layout) const {
        if (!length) return layout.sequences;
        if (!layout.cu) return int64_t(layout.sequences) * ((layout.chunks() + length - 1) / length);
        return layout.slots() / length + layout.sequences;
    }
    // Sequence and number in it of a segment; a negative number before the first document, a too large one behind a sequence's end.
    __device__ void find(const DeltaLayout& layout, int64_t segment, int& sequence, int& number) const {
        number = 0;
        if (!length) {
            sequence = int(segment);
        } else if (!layout.cu) {
            const unsigned each = (layout.chunks() + length - 1) / length;
            sequence = int(unsigned(segment) / each), number = int(unsigned(segment) % each);
        } else {
            int lo = 0, hi = layout.sequences - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if ((layout.start(mid) / CHUNK + mid) / length + mid <= segment) lo = mid;
                else hi = mid - 1;
            }
            sequence = lo, number = int(segment - ((layout.start(lo) / CHUNK + lo) / length + lo));
        }
    }
};

// Chains of equal sequences that would leave the device partly empty at the end are walked in equal shares instead (length 0: they are not):
// with all chains laid end to end, place i takes the chunks from i * length on.  A share is no shorter than a chain, so no more than
// one chain is cut at its end; that one is walked first and its state, in 32 bits, handed to the next place, which walks the rest of it last.
struct DeltaShares {
    int length, places;
    float* states;    // accumulator fragments, [places, D * 64]
    unsigned* flags;  // tickets drawn; then one for each place: its state is there.  Zeros before the launch.
    size_t flag_bytes() const { return size_t(places + 1) * 4; }
};
// What one walk covers: a segment (or sequence), value head and block of columns; with shares, chunks begin .. end - 1 in walking order,
// from the state at `from` (null: the sequence's first) and leaving the state at `to` (null: the sequence ends).
struct DeltaPart {
    unsigned segment, head, block;
    int begin, end;
    const float* from;
    float* to;
    bool lost;  // what stands at `from` was not waited for
};

struct DeltaShape {
    DeltaLayout layout;
    DeltaSegments segments;
    DeltaShares shares;
    int key_heads, heads, d, dv;
    bool gates_bf16;
    float scale;
    unsigned wait_tries;  // limit of the bounded waits: polls of a barrier, by up to 20 microseconds each; 64 times as many of a share's flag
};

// The parts of a CTA's share.  Places are drawn in the order in which CTAs start, so the one before has started, and what it hands on comes
// first and waits for nobody: no wait depends on CTAs that are not resident.  It is bounded all the same, by about two seconds; then `code`
// is recorded in `fault` and the walk goes on from a state of NaN.  STATE: floats of a state that is handed on.
template <int STATE>
struct ShareWalk {
    int64_t chain, lowest, highest;
    int first, last, chunks;  // the lowest chain's first chunk, the end of the highest one's
    unsigned blocks;
    float* states;
    unsigned* flag;
    __device__ __forceinline__ bool draw(const DeltaShape& shape, unsigned columns) {  // false: more CTAs than places
        __shared__ int drawn;
        if (threadIdx.x == 0) drawn = int(atomicAdd(shape.shares.flags, 1u));
        __syncthreads();
        const int place = drawn;
        chunks = shape.layout.chunks(), blocks = shape.dv / columns;
        const int64_t all = int64_t(shape.layout.sequences) * shape.heads * blocks * chunks, begin = int64_t(place) * shape.shares.length;
        const int64_t end = min(begin + shape.shares.length, all);
        lowest = begin / chunks, highest = chain = (end - 1) / chunks;
        first = int(begin - lowest * chunks), last = int(end - highest * chunks);
        states = shape.shares.states + int64_t(place) * STATE, flag = shape.shares.flags + 1 + place;
        return place < shape.shares.places;
    }
    __device__ __forceinline__ DeltaPart part(const DeltaShape& shape, int* fault, int code) const {
        const int begin = chain == lowest ? first : 0, end = chain == highest ? last : chunks;
        bool lost = false;
        if (begin > 0) {
            unsigned there = threadIdx.x;
            if (threadIdx.x == 0) {
                for (unsigned tries = 0; tries < 64 * shape.wait_tries && !there; ++tries) {
                    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(there) : "l"(flag - 1) : "memory");
                    if (!there) __nanosleep(500);
                }
                if (!there) atomicCAS(fault, 0, code);
            }
            lost = __syncthreads_or(!there);
        }
        const int64_t sequence = chain / blocks;
        return DeltaPart{unsigned(sequence / shape.heads), unsigned(sequence % shape.heads), unsigned(chain % blocks), begin, end,
                         begin > 0 ? states - STATE : nullptr, end < chunks ? states : nullptr, lost};
    }
    __device__ __forceinline__ bool next(const DeltaPart& walked) {  // false: that was the last part
        __syncthreads();  // the stages are free, and a state that is handed on is written
        if (walked.to && threadIdx.x == 0) {
            __threadfence();
            asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(flag), "r"(1u) : "memory");
        }
        return --chain >= lowest;
    }
};

// Zeros in the gradients' rows of no document; CTA `index` of `count` takes every count-th row.
template <int THREADS>
__device__ __forceinline__ void clear_gradients(const DeltaShape& shape, __nv_bfloat16* dq, __nv_bfloat16* dk, void* dg, void* dbeta, int64_t index,
                                                int64_t count, int thread) {
    const int64_t begin = shape.layout.start(0), end = shape.layout.start(shape.layout.sequences), outside = begin + max(int64_t(shape.layout.n) - end, int64_t(0));
    const int width = shape.key_heads * shape.d;
    for (int64_t i = index; i < outside; i += count) {
        const int64_t row = i < begin ? i : end + i - begin;
        for (int j = thread * 8; j < width; j += THREADS * 8) {
            *reinterpret_cast<uint4*>(dq + row * width + j) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(dk + row * width + j) = make_uint4(0, 0, 0, 0);
        }
        for (int j = thread; j < shape.heads; j += THREADS) {
            const int64_t at = row * shape.heads + j;
            if (shape.gates_bf16) static_cast<__nv_bfloat16*>(dg)[at] = static_cast<__nv_bfloat16*>(dbeta)[at] = __float2bfloat16(0.f);
            else static_cast<float*>(dg)[at] = static_cast<float*>(dbeta)[at] = 0.f;
        }
    }
}

// What the kernels hand to one another, per slot and value head.  The backward needs all of it.
struct DeltaSaved {
    float* rows;               // [slots, H, ROW_VALUES]
    __nv_bfloat16 *t, *t_rest; // [slots, H, MATRIX] blocked; t_rest only for an exact state
    __nv_bfloat16* p;
    __nv_bfloat16 *states, *x; // S0 [slots, H, DV, D] and X, transposed, [slots, H, DV, CHUNK], both blocked; only for a backward
};

__device__ __forceinline__ float gate(const void* gates, int64_t index, bool is_bf16) {
    return is_bf16 ? bf2f(static_cast<const __nv_bfloat16*>(gates)[index]) : static_cast<const float*>(gates)[index];
}

// Tiles of 64 rows of BYTES bytes in shared memory: the 16-byte pieces of a row are exchanged by the row number, so that the eight
// rows of an ldmatrix fall into different banks without padding.
template <int BYTES>
__device__ __forceinline__ int piece_key(int row) { return BYTES >= 128 ? row & 7 : (row >> 1) & 3; }
// A lane's view of such a tile for ldmatrix / stmatrix: `at` + its row, and what its pieces are exchanged by.  A 16 x 16 part that
// starts at row 16 i and piece 2 j is at row + 16 i * BYTES + ((32 j) ^ flip).
struct TileLane {
    unsigned row, flip;
    __device__ __forceinline__ unsigned at(int bytes) const { return row + (unsigned(bytes) ^ flip); }
};
template <int BYTES>
__device__ __forceinline__ TileLane tile_rows_first(unsigned tile, int lane) {
    const int row = (lane & 7) + (lane & 8);
    return {tile + row * BYTES, unsigned(((lane >> 4) ^ piece_key<BYTES>(row)) * 16)};
}
template <int BYTES>
__device__ __forceinline__ TileLane tile_cols_first(unsigned tile, int lane) {
    const int row = (lane & 7) + ((lane >> 4) << 3);
    return {tile + row * BYTES, unsigned((((lane >> 3) & 1) ^ piece_key<BYTES>(row)) * 16)};
}
// Copies `count` rows from a strided tensor into such a tile; the rest is zeros.  A full chunk takes the unrolled path with one
// running pointer: addresses worked out ahead of the loop over the chunks would cost the chains their registers.
template <int BYTES, int THREADS>
__device__ __forceinline__ void load_tile(unsigned tile, const char* global, int64_t stride, int count, int thread) {
    constexpr int PIECES = BYTES / 16, STEP = THREADS / PIECES;  // rows that the threads take at a time
    static_assert(THREADS % PIECES == 0 && CHUNK % STEP == 0 && (STEP % 8 == 0 || 8 % STEP == 0), "rows are dealt out evenly");
    const int first = thread / PIECES, piece = thread % PIECES;
    const char* from = global + first * stride + piece * 16;
    const unsigned to = tile + first * BYTES;
    if (count == CHUNK) {
#pragma unroll
        for (int row = 0; row < CHUNK; row += STEP) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + row * BYTES + ((piece ^ piece_key<BYTES>(first + row)) * 16)), "l"(from) : "memory");
            from += STEP * stride;
        }
    } else {
#pragma unroll 1
        for (int row = 0; row < CHUNK; row += STEP) {
            const bool inside = first + row < count;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + row * BYTES + ((piece ^ piece_key<BYTES>(first + row)) * 16)),
                         "l"(inside ? from : global), "r"(inside ? 16 : 0) : "memory");
            from += STEP * stride;
        }
    }
}
// The same with padded rows of `pitch` bytes.
template <int BYTES, int THREADS>
__device__ __forceinline__ void load_rows(unsigned tile, int pitch, const char* global, int64_t stride, int count, int thread) {
    constexpr int PIECES = BYTES / 16;
#pragma unroll
    for (int i = thread; i < CHUNK * PIECES; i += THREADS) {
        const int row = i / PIECES, piece = i % PIECES;
        const bool inside = row < count;
        const char* from = global + (inside ? row * stride : 0) + piece * 16;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tile + row * pitch + piece * 16), "l"(from),
                     "r"(inside ? 16 : 0));
    }
}
template <int BYTES, int THREADS>
__device__ __forceinline__ void load_block(unsigned tile, const char* global, int thread) {
#pragma unroll
    for (int i = thread * 16; i < BYTES; i += THREADS * 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(tile + i), "l"(global + i));
}

DeltaShares delta_shares(const DeltaLayout& layout, int heads, int d, int dv);
// Chunks to a segment, 0 for whole sequences.
int delta_segment_length(const DeltaLayout& layout, int heads, int d, int dv);
struct DeltaGradients {
    const __nv_bfloat16 *q, *k, *dout;
    const float* dfinal;  // gradient of the last states, or null
    __nv_bfloat16* dstates;  // scratch: dS1 [slots, H, DV, D] blocked
    float* dbeta_parts;      // scratch: [DV / 16, slots, H, CHUNK]
    float* ends;             // scratch: the reverse chain's B, as DeltaSegments has the forward's
    __nv_bfloat16 *dq, *dk, *dv;
    void *dg, *dbeta;        // in the gates' type
    float* dinitial;         // gradient of the first states, or null
};

cudaError_t launch_delta_prepare(const DeltaShape& shape, const __nv_bfloat16* q, const __nv_bfloat16* k, const void* g,
                                 const void* beta, const DeltaSaved& saved, cudaStream_t stream);
cudaError_t launch_delta_chain(const DeltaShape& shape, const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* v,
                               const float* initial, const DeltaSaved& saved, __nv_bfloat16* out, float* final_state,
                               cudaStream_t stream);
cudaError_t launch_delta_backward(const DeltaShape& shape, const DeltaGradients& gradients, const DeltaSaved& saved, cudaStream_t stream);
// The last stage of the backward on tcgen05, for D and DV of 64 or 128.
cudaError_t launch_delta_gradient_tensor(const DeltaShape& shape, const DeltaGradients& gradients, const DeltaSaved& saved, cudaStream_t stream);
// First bounded wait that ran out on the current device, of the tensor-memory pipeline (1 to 11) or between shares (12, 13), 0 if none; reading clears it.
cudaError_t read_delta_fault(int* code);
cudaError_t read_chain_fault(int* code);
cudaError_t read_reverse_fault(int* code);
cudaError_t launch_delta_step(const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* v, const void* g, const void* beta,
                              bool gates_bf16, float scale, float* state, const int* slots, int64_t pool, int batch, int key_heads,
                              int heads, int d, int dv, __nv_bfloat16* out, cudaStream_t stream);

}  // namespace dism
