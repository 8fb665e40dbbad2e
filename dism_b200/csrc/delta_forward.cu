// Chain of chunks of the gated delta rule, forward.
//
// A warp owns 16 columns of the state of one value head of one sequence and walks the chunks with the state, transposed, in
// its accumulators.  Per chunk: S0 K^T and S0 Q^T (S0 rounded to bf16 straight from the accumulators), Y = V - e^G K S0,
// X = T Y, U = b X, O = scale e^G Q S0 + P U, S1 = e^{G_63} S0 + K^T (e^{G_63 - G} U).  Warps share K, Q, T and P of the
// chunk in shared memory, double-buffered with cp.async; nothing else passes between them.
//
// Why a warp per 16 columns: the chain of products has to be short, and with the accumulators of one product as the left operand of the
// next nothing goes through memory between them.  The same chain on tcgen05 (a thread per column, three round trips through tensor
// memory a chunk) was built in full and took 2.8 to 3.1 us a chunk, where this chain (then with single operands) took 2.66 for a CTA alone on its SM and 4.7
// for two.  In us, that one against this: 16 x 2048, 10 heads of 128: 228 / 232; 4 x 8192, 16 heads of 128: 402 / 340; 2 x 8192, 16 heads of
// 64, uncut: 279 / 209; prompt of 16384, 16 heads of 128, uncut: 850 / 762; 500, 4 heads: 38 to 45 / 27.
// What bounds it: with four warps a CTA and two CTAs an SM, latency of dependent instructions (one or two warps to a scheduler; the main
// stall is the fixed latency of an instruction, with one CTA an SM the tensor pipe is 47 % busy).  16 x 2048 positions, 10 heads of 128
// (320 chains for 296 places): 175 us in shares, 250 as 320 CTAs; as segments 2 x 8192, 16 heads of 64: 62 + 76 us (66 with joins of single operands).
//
// What is rounded: products take bf16, so every operand that is not one already is rounded, once, or kept as a pair (value and
// remainder, 16 bits) for a second product.  Y and what is added to the state are pairs always: these roundings would reach every
// later position (with slow decays each alone costs the gradients 2e-3 of their norm, as much as their own rounding to bf16).
// EXACT: the state is wanted at the end.  S0 in S0 K^T and T are pairs as well then, which holds the state to a few 1e-6 (2e-5 over
// thousands of positions with decays of 1e-4).
#include "delta_common.cuh"

namespace dism {
namespace {

template <int D, int WARPS, bool EXACT>
struct ForwardStage {
    static constexpr int PITCH = 2 * D, VALUE_PITCH = 32 * WARPS;
    static constexpr int K = 0, Q = K + CHUNK * PITCH, T = Q + CHUNK * PITCH, T_REST = T + 2 * MATRIX;
    static constexpr int P = T_REST + (EXACT ? 2 * MATRIX : 0), V = P + 2 * MATRIX, ROWS = V + CHUNK * VALUE_PITCH;
    static constexpr int BYTES = ROWS + 3 * CHUNK * 4;
};

__device__ int delta_chain_fault;

// LOCAL: the first launch over segments (see DeltaSegments): neither Q nor outputs, B from the first CTAs of a head and M from the others.
// SHARES: a part of an uncut chain, from a neighbour's state or to one (see DeltaShares).
template <int D, int WARPS, bool EXACT, bool SAVE, bool LOCAL, bool SHARES>
__global__ void __launch_bounds__(WARPS * 32, 2) delta_chain_kernel(DeltaShape shape, const __nv_bfloat16* __restrict__ q,
                                                                    const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ v,
                                                                    const float* __restrict__ initial, DeltaSaved saved,
                                                                    __nv_bfloat16* __restrict__ out, float* __restrict__ final_state) {
    using Stage = ForwardStage<D, WARPS, EXACT>;
    constexpr int THREADS = WARPS * 32, TILES = CHUNK / 8;
    extern __shared__ __align__(128) unsigned char shared[];
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31;
    ShareWalk<D * 16 * WARPS> share;
    if (SHARES && !share.draw(shape, WARPS * 16)) return;
    bool more = false;
    do {
        const DeltaPart part = SHARES ? share.part(shape, &delta_chain_fault, 12) : DeltaPart{blockIdx.x, blockIdx.y, blockIdx.z, 0, 0, nullptr, nullptr, false};
        const int head = part.head, dv = shape.dv, key_head = head / (shape.heads / shape.key_heads);
        const bool unit = LOCAL && part.block * WARPS * 16 >= dv;  // this CTA's columns are the unit matrix's
        const int column = (part.block * WARPS + warp) * 16 - (unit ? dv : 0);
        int64_t row, slot;
        int length, sequence, number;
        if (SHARES) sequence = part.segment, number = 0;
        else shape.segments.find(shape.layout, part.segment, sequence, number);
        if (number < 0) return;  // segments before the first document
        shape.layout.span(sequence, row, length, slot);
        const unsigned base = smem_address(shared);
        if (!LOCAL && !SHARES && shape.layout.cu && number == 0) {
            char* to = reinterpret_cast<char*>(out + int64_t(head) * dv + part.block * WARPS * 16);
            const int64_t stride = int64_t(shape.heads) * dv * 2;
            if (sequence == 0) clear_rows<WARPS * 32>(to, stride, WARPS * 2, 0, row, thread);
            if (sequence == shape.layout.sequences - 1) clear_rows<WARPS * 32>(to, stride, WARPS * 2, row + length, shape.layout.n, thread);
        }
        int chunks = (length + CHUNK - 1) / CHUNK;
        bool last = true;
        if (SHARES) {
            chunks = part.end - part.begin;
            slot += part.begin, row += int64_t(part.begin) * CHUNK, length -= part.begin * CHUNK;
        } else if (shape.segments.length) {
            const int before = min(number * shape.segments.length, chunks);
            last = chunks - before <= shape.segments.length;
            if (number && before == chunks) return;  // no such segment
            if (LOCAL && last) return;
            chunks = min(chunks - before, shape.segments.length);
            slot += before, row += int64_t(before) * CHUNK, length -= before * CHUNK;
        }

        const int64_t key_stride = int64_t(shape.key_heads) * D * 2, value_stride = int64_t(shape.heads) * dv * 2;
        auto load = [&](int c) {
            const unsigned stage = base + (c & 1) * Stage::BYTES;
            const int count = min(CHUNK, length - c * CHUNK);
            const int64_t at = row + int64_t(c) * CHUNK, place = (slot + c) * shape.heads + head;
            const int64_t key = (at * shape.key_heads + key_head) * D * 2;
            load_tile<2 * D, THREADS>(stage + Stage::K, reinterpret_cast<const char*>(k) + key, key_stride, count, thread);
            if (!unit) load_tile<32 * WARPS, THREADS>(stage + Stage::V,
                                           reinterpret_cast<const char*>(v) + ((at * shape.heads + head) * dv + part.block * WARPS * 16) * 2,
                                           value_stride, count, thread);
            load_block<3 * CHUNK * 4, THREADS>(stage + Stage::ROWS, reinterpret_cast<const char*>(saved.rows + place * ROW_VALUES), thread);
            load_block<2 * MATRIX, THREADS>(stage + Stage::T, reinterpret_cast<const char*>(saved.t + place * MATRIX), thread);
            if (EXACT) load_block<2 * MATRIX, THREADS>(stage + Stage::T_REST, reinterpret_cast<const char*>(saved.t_rest + place * MATRIX), thread);
            if (!LOCAL) load_tile<2 * D, THREADS>(stage + Stage::Q, reinterpret_cast<const char*>(q) + key, key_stride, count, thread);
            if (!LOCAL) load_block<2 * MATRIX, THREADS>(stage + Stage::P, reinterpret_cast<const char*>(saved.p + place * MATRIX), thread);
            cp_async_commit();
        };

        float s[D / 8][4];  // the state, transposed: 16 columns of S by D
        const int64_t state_at = (int64_t(sequence) * shape.heads + head) * D * dv + column + (lane >> 2);
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = 8 * n + 2 * (lane & 3) + (e & 1);
                if (LOCAL) s[n][e] = unit && d == column + (lane >> 2) + (e >> 1) * 8 ? 1.f : 0.f;
                else if (!SHARES || !part.from) s[n][e] = initial ? __ldg(initial + state_at + int64_t(d) * dv + (e >> 1) * 8) : 0.f;
            }
        if (SHARES && part.from) {
            const float4* from = reinterpret_cast<const float4*>(part.from) + warp * (D / 8) * 32 + lane;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
                *reinterpret_cast<float4*>(s[n]) = part.lost ? make_float4(NOT_A_NUMBER, NOT_A_NUMBER, NOT_A_NUMBER, NOT_A_NUMBER) : __ldcg(from + n * 32);
        }
        // The state at a later segment's start: S <- M S + B over the segments before it.  M and S are pairs here whatever is wanted at the end: a
        // rounding at a join stays in the state, and with slow decays and weak writes (M close to one) single bf16 left 1.1 to 2.2 % of the output's norm
        // after 32 joins.
        if constexpr (!LOCAL && !SHARES && D >= 64 && WARPS == 4)
            for (int before = 0; before < number; ++before) {
                const int64_t place = (shape.segments.place(slot) - number + before) * shape.heads + head;
                load_block<2 * D * D, THREADS>(base, reinterpret_cast<const char*>(shape.segments.m + place * D * D), thread);
                load_block<2 * D * D, THREADS>(base + 2 * D * D, reinterpret_cast<const char*>(shape.segments.m_rest + place * D * D), thread);
                cp_async_commit();
                float x[D / 8][4];
                const float4* end = reinterpret_cast<const float4*>(shape.segments.ends + place * D * dv) + column / 16 * (D / 8) * 32 + lane;
#pragma unroll
                for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float4*>(x[n]) = __ldg(end + n * 32);
                cp_async_wait<0>();
                __syncthreads();
#pragma unroll
                for (int kb = 0; kb < D / 16; ++kb) {
                    unsigned a[4], rest[4];
                    to_operand(a, s[2 * kb], s[2 * kb + 1]);
                    to_operand_rest(rest, a, s[2 * kb], s[2 * kb + 1]);
                    const unsigned m = base + kb * 2 * (D / 8) * 128 + rows_first_blocked(lane, D / 8);
#pragma unroll
                    for (int np = 0; np < D / 16; ++np) {
                        unsigned b[4];
                        ldsm4_trans(b, m + np * 256);
                        mma16816(x[2 * np], a, b[0], b[1]);
                        mma16816(x[2 * np + 1], a, b[2], b[3]);
                        mma16816(x[2 * np], rest, b[0], b[1]);
                        mma16816(x[2 * np + 1], rest, b[2], b[3]);
                        ldsm4_trans(b, m + 2 * D * D + np * 256);
                        mma16816(x[2 * np], a, b[0], b[1]);
                        mma16816(x[2 * np + 1], a, b[2], b[3]);
                    }
                }
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = x[n][e];
                __syncthreads();
            }
        if (chunks > 0) load(0);
        for (int c = 0; c < chunks; ++c) {
            cp_async_wait<0>();
            __syncthreads();  // chunk c is in, and every warp has left chunk c - 1
            if (c + 1 < chunks) load(c + 1);
            const unsigned stage = base + (c & 1) * Stage::BYTES;
            const float* rows = reinterpret_cast<const float*>(shared + (c & 1) * Stage::BYTES + Stage::ROWS);
            const int64_t place = (slot + c) * shape.heads + head;

            float ks[TILES][4], qs[TILES][4];
#pragma unroll
            for (int n = 0; n < TILES; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) ks[n][e] = qs[n][e] = 0.f;
            const TileLane keys = tile_cols_first<Stage::PITCH>(stage + Stage::K, lane);
#pragma unroll
            for (int kb = 0; kb < D / 16; ++kb) {
                unsigned a[4], rest[4];
                to_operand(a, s[2 * kb], s[2 * kb + 1]);
                if (EXACT) to_operand_rest(rest, a, s[2 * kb], s[2 * kb + 1]);
                if (SAVE) {
                    unsigned* to = reinterpret_cast<unsigned*>(saved.states + place * dv * D) + (int64_t(column / 8) * (D / 8) + 2 * kb) * 32 + lane;
                    to[0] = a[0], to[D / 8 * 32] = a[1], to[32] = a[2], to[D / 8 * 32 + 32] = a[3];
                }
#pragma unroll
                for (int np = 0; np < TILES / 2; ++np) {
                    unsigned b[4];
                    ldsm4(b, keys.at(kb * 32) + np * 16 * Stage::PITCH);
                    mma16816(ks[2 * np], a, b[0], b[1]);
                    mma16816(ks[2 * np + 1], a, b[2], b[3]);
                    if (EXACT) {
                        mma16816(ks[2 * np], rest, b[0], b[1]);
                        mma16816(ks[2 * np + 1], rest, b[2], b[3]);
                    }
                    if (!LOCAL) {
                        ldsm4(b, keys.at(kb * 32) + Stage::Q - Stage::K + np * 16 * Stage::PITCH);
                        mma16816(qs[2 * np], a, b[0], b[1]);
                        mma16816(qs[2 * np + 1], a, b[2], b[3]);
                    }
                }
            }
            // Y, as the left operand of X = T Y
            const unsigned values = tile_cols_first<Stage::VALUE_PITCH>(stage + Stage::V, lane).at(warp * 32);
            unsigned y[TILES / 2][4], y_rest[TILES / 2][4];
#pragma unroll
            for (int np = 0; np < TILES / 2; ++np) {
                unsigned vv[4] = {0, 0, 0, 0};
                if (!unit) ldsm4_trans(vv, values + np * 16 * Stage::VALUE_PITCH);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float(&tile)[4] = ks[2 * np + h];
                    const float2 decay = *reinterpret_cast<const float2*>(rows + 16 * np + 8 * h + 2 * (lane & 3));
                    tile[0] = low_half(vv[2 * h]) - decay.x * tile[0], tile[1] = high_half(vv[2 * h]) - decay.y * tile[1];
                    tile[2] = low_half(vv[2 * h + 1]) - decay.x * tile[2], tile[3] = high_half(vv[2 * h + 1]) - decay.y * tile[3];
                    const float sx = shape.scale * decay.x, sy = shape.scale * decay.y;
                    float(&o)[4] = qs[2 * np + h];
                    o[0] *= sx, o[1] *= sy, o[2] *= sx, o[3] *= sy;
                }
                to_operand(y[np], ks[2 * np], ks[2 * np + 1]);
                to_operand_rest(y_rest[np], y[np], ks[2 * np], ks[2 * np + 1]);
            }
            float(&x)[TILES][4] = ks;
#pragma unroll
            for (int n = 0; n < TILES; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) x[n][e] = 0.f;
            const unsigned inverse = stage + Stage::T + cols_first_tile(lane), inside = inverse + Stage::P - Stage::T;
#pragma unroll
            for (int np = 0; np < TILES / 2; ++np)
#pragma unroll
                for (int kb = 0; kb <= np; ++kb) {
                    unsigned b[4];
                    ldsm4(b, inverse + tile_at(np, kb));
                    mma16816(x[2 * np], y[kb], b[0], b[1]);
                    mma16816(x[2 * np + 1], y[kb], b[2], b[3]);
                    mma16816(x[2 * np], y_rest[kb], b[0], b[1]);
                    mma16816(x[2 * np + 1], y_rest[kb], b[2], b[3]);
                    if (EXACT) {
                        ldsm4(b, inverse + Stage::T_REST - Stage::T + tile_at(np, kb));
                        mma16816(x[2 * np], y[kb], b[0], b[1]);
                        mma16816(x[2 * np + 1], y[kb], b[2], b[3]);
                    }
                }
            const int count = min(CHUNK, length - c * CHUNK);
            // the warp's 16 columns of the value tile are its own: O leaves through them in rows of 32 bytes
            auto leave = [&](const float(&tiles)[TILES][4], char* to, int64_t stride, int rows_out) {
                __syncwarp();
#pragma unroll
                for (int np = 0; np < TILES / 2; ++np) {
                    const float(&t0)[4] = tiles[2 * np], (&t1)[4] = tiles[2 * np + 1];
                    stsm4_trans(values + np * 16 * Stage::VALUE_PITCH, pack2(t0[0], t0[1]), pack2(t0[2], t0[3]), pack2(t1[0], t1[1]), pack2(t1[2], t1[3]));
                }
                __syncwarp();
#pragma unroll
                for (int i = 0; i < CHUNK * 2 / 32; ++i) {
                    const int t = i * 16 + (lane >> 1);
                    const uint4 piece = *reinterpret_cast<const uint4*>(shared + (c & 1) * Stage::BYTES + Stage::V + t * Stage::VALUE_PITCH + ((warp * 2 + (lane & 1)) ^ piece_key<Stage::VALUE_PITCH>(t)) * 16);
                    if (t < rows_out) *reinterpret_cast<uint4*>(to + t * stride + (lane & 1) * 16) = piece;
                }
            };
            if (SAVE) {
                unsigned* to = reinterpret_cast<unsigned*>(saved.x + place * CHUNK * dv) + column / 8 * TILES * 32 + lane;
#pragma unroll
                for (int n = 0; n < TILES; ++n) to[n * 32] = pack2(x[n][0], x[n][1]), to[(TILES + n) * 32] = pack2(x[n][2], x[n][3]);
            }
            // U, as left operand of P U; then with the decay to the chunk's end, of the state's update
            unsigned u[TILES / 2][4], u_rest[TILES / 2][4];
#pragma unroll
            for (int np = 0; np < TILES / 2; ++np) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 b = *reinterpret_cast<const float2*>(rows + CHUNK + 16 * np + 8 * h + 2 * (lane & 3));
                    float(&tile)[4] = x[2 * np + h];
                    tile[0] *= b.x, tile[1] *= b.y, tile[2] *= b.x, tile[3] *= b.y;
                }
                if (!LOCAL) to_operand(u[np], x[2 * np], x[2 * np + 1]);
            }
            if (!LOCAL) {
#pragma unroll
            for (int np = 0; np < TILES / 2; ++np)
#pragma unroll
                for (int kb = 0; kb <= np; ++kb) {
                    unsigned b[4];
                    ldsm4(b, inside + tile_at(np, kb));
                    mma16816(qs[2 * np], u[kb], b[0], b[1]);
                    mma16816(qs[2 * np + 1], u[kb], b[2], b[3]);
                }
            leave(qs, reinterpret_cast<char*>(out + ((row + int64_t(c) * CHUNK) * shape.heads + head) * dv + column), value_stride, count);
            }
            const float kept = rows[CHUNK - 1];
#pragma unroll
            for (int np = 0; np < TILES / 2; ++np) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 tail = *reinterpret_cast<const float2*>(rows + 2 * CHUNK + 16 * np + 8 * h + 2 * (lane & 3));
                    float(&tile)[4] = x[2 * np + h];
                    tile[0] *= tail.x, tile[1] *= tail.y, tile[2] *= tail.x, tile[3] *= tail.y;
                }
                to_operand(u[np], x[2 * np], x[2 * np + 1]);
                to_operand_rest(u_rest[np], u[np], x[2 * np], x[2 * np + 1]);
            }
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[n][e] *= kept;
            const TileLane keys_trans = tile_rows_first<Stage::PITCH>(stage + Stage::K, lane);
#pragma unroll
            for (int kb = 0; kb < TILES / 2; ++kb)
#pragma unroll
                for (int np = 0; np < D / 16; ++np) {
                    unsigned b[4];
                    ldsm4_trans(b, keys_trans.at(np * 32) + kb * 16 * Stage::PITCH);
                    mma16816(s[2 * np], u[kb], b[0], b[1]);
                    mma16816(s[2 * np + 1], u[kb], b[2], b[3]);
                    mma16816(s[2 * np], u_rest[kb], b[0], b[1]);
                    mma16816(s[2 * np + 1], u_rest[kb], b[2], b[3]);
                }
        }
        if (LOCAL) {
            const int64_t place = shape.segments.place(slot) * shape.heads + head;
            if (unit) {
                unsigned* to = reinterpret_cast<unsigned*>(shape.segments.m + place * D * D) + int64_t(column / 8) * (D / 8) * 32 + lane;
                unsigned* to_rest = reinterpret_cast<unsigned*>(shape.segments.m_rest + place * D * D) + int64_t(column / 8) * (D / 8) * 32 + lane;
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const unsigned value = pack2(s[n][2 * h], s[n][2 * h + 1]);
                        to[(h * (D / 8) + n) * 32] = value;
                        to_rest[(h * (D / 8) + n) * 32] = pack2_rest(s[n][2 * h], s[n][2 * h + 1], value);
                    }
            } else {
                float4* to = reinterpret_cast<float4*>(shape.segments.ends + place * D * dv) + column / 16 * (D / 8) * 32 + lane;
#pragma unroll
                for (int n = 0; n < D / 8; ++n) to[n * 32] = *reinterpret_cast<float4*>(s[n]);
            }
        } else if (SHARES && part.to) {
            float4* to = reinterpret_cast<float4*>(part.to) + warp * (D / 8) * 32 + lane;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) to[n * 32] = *reinterpret_cast<float4*>(s[n]);
        } else if (final_state && last) {
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    final_state[state_at + int64_t(8 * n + 2 * (lane & 3) + (e & 1)) * dv + (e >> 1) * 8] = s[n][e];
        }
        more = SHARES && share.next(part);
    } while (more);
}

template <int D, int WARPS, bool EXACT, bool SAVE, bool LOCAL = false>
cudaError_t launch(const DeltaShape& shape, const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* v,
                   const float* initial, const DeltaSaved& saved, __nv_bfloat16* out, float* final_state, cudaStream_t stream) {
    constexpr int BYTES = 2 * ForwardStage<D, WARPS, EXACT>::BYTES;
    constexpr auto* kernel = delta_chain_kernel<D, WARPS, EXACT, SAVE, LOCAL, false>;
    if (cudaError_t status = allow_shared<kernel>(BYTES)) return status;
    if constexpr (!LOCAL && D >= 64 && WARPS == 4)
        if (shape.shares.length) {
            constexpr auto* shared_kernel = delta_chain_kernel<D, WARPS, EXACT, SAVE, false, true>;
            if (cudaError_t status = allow_shared<shared_kernel>(BYTES)) return status;
            if (cudaError_t status = cudaMemsetAsync(shape.shares.flags, 0, shape.shares.flag_bytes(), stream)) return status;
            KernelTimer timer("delta_chain", stream);
            shared_kernel<<<shape.shares.places, WARPS * 32, BYTES, stream>>>(shape, q, k, v, initial, saved, out, final_state);
            return cudaGetLastError();
        }
    KernelTimer timer(LOCAL ? "delta_segments" : "delta_chain", stream);
    const dim3 grid(unsigned(shape.segments.count(shape.layout)), shape.heads, (shape.dv + (LOCAL ? D : 0)) / (16 * WARPS));
    kernel<<<grid, WARPS * 32, BYTES, stream>>>(shape, q, k, v, initial, saved, out, final_state);
    return cudaGetLastError();
}

template <int D, int WARPS>
cudaError_t choose(const DeltaShape& shape, const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* v,
                   const float* initial, const DeltaSaved& saved, __nv_bfloat16* out, float* final_state, cudaStream_t stream) {
    const bool exact = saved.t_rest != nullptr, save = saved.states != nullptr;
    if constexpr (D >= 64 && WARPS == 4) {
        if (shape.segments.length) {
            cudaError_t status = exact ? launch<D, WARPS, true, false, true>(shape, q, k, v, initial, saved, out, final_state, stream)
                                       : launch<D, WARPS, false, false, true>(shape, q, k, v, initial, saved, out, final_state, stream);
            if (status) return status;
        }
    }
    if (exact && save) return launch<D, WARPS, true, true>(shape, q, k, v, initial, saved, out, final_state, stream);
    if (exact) return launch<D, WARPS, true, false>(shape, q, k, v, initial, saved, out, final_state, stream);
    if (save) return launch<D, WARPS, false, true>(shape, q, k, v, initial, saved, out, final_state, stream);
    return launch<D, WARPS, false, false>(shape, q, k, v, initial, saved, out, final_state, stream);
}

template <int D>
cudaError_t by_width(const DeltaShape& shape, const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* v,
                     const float* initial, const DeltaSaved& saved, __nv_bfloat16* out, float* final_state, cudaStream_t stream) {
    if (shape.dv % 64 == 0) return choose<D, 4>(shape, q, k, v, initial, saved, out, final_state, stream);
    return choose<D, 2>(shape, q, k, v, initial, saved, out, final_state, stream);
}
}  // namespace

// A segment costs two CTA walks forward (one of them for B and M, without outputs) and two backward, so cutting pays when the walks
// get at least four times shorter; the chunks are divided by the places of two CTAs per SM (what the chains' registers and shared memory
// allow), but a segment has no fewer than eight, below which putting the starts together costs what it saves.  Every sequence rounds up to whole segments, so
// the second launch may have a few more CTAs than places: 320 on 296 at the first two shapes below.  Measured, forward and
// backward chain with single operands, uncut / for one / for two CTAs per SM (us): 2 x 8192, 16 heads of 64: 426 / 281 / 211; prompt of 16384, 16 heads of
// 128: 761 / 523 / 439; pack of 7019, 8 heads: 166 / 152 / 120.  4 x 2048, 10 heads of 128 (32 chunks to 9): 204 / - / 212.
int delta_segment_length(const DeltaLayout& layout, int heads, int d, int dv) {
    if (d < 64 || dv < 64) return 0;
    const int64_t chains = int64_t(heads) * (dv / 64), room = 2 * int64_t(device_sm_count());
    if (room <= 0) return 0;
    const int64_t even = (layout.slots() * chains + room - 1) / room, length = even < 8 ? 8 : even;
    return 4 * length <= layout.chunks() ? int(length) : 0;
}

// Chains that fill the device's places some times over and at most half of them once more are walked in equal shares (DeltaShares).  Measured
// on 296 places, walked one by one / in shares, forward and backward chain (us): 320 chains of 32 chunks, 128 x 128: 252 + 236 / 177 + 167; of
// 8 chunks 72 + 66 / 56 + 54; 440 of 8, 64 x 64: 48 + 60 / 52 + 52; 600 of 32, 64 x 64: 252 + 260 / 222 + 222.  With more left over the last
// round is nearly full: 560 of 8, 64 x 64: 60 + 62 / 62 + 66; 580 of 32: 203 + 207 / 215 + 216.  Chains of four chunks gain nothing: 300,
// 64 x 64: 27 + 29 / 27 + 35.
DeltaShares delta_shares(const DeltaLayout& layout, int heads, int d, int dv) {
    DeltaShares shares{};
    if (layout.cu || d < 64 || dv < 64) return shares;
    const int64_t chains = int64_t(layout.sequences) * heads * (dv / 64), room = 2 * int64_t(device_sm_count()), chunks = layout.chunks();
    if (room <= 0 || chains <= room || chains % room == 0 || chains % room > room / 2 || chunks < 8) return shares;
    const int64_t length = (chains * chunks + room - 1) / room;
    if (length > INT_MAX) return shares;
    shares.length = int(length), shares.places = int((chains * chunks + length - 1) / length);
    return shares;
}

cudaError_t read_chain_fault(int* code) {
    if (cudaError_t status = cudaMemcpyFromSymbol(code, delta_chain_fault, sizeof(int))) return status;
    const int zero = 0;
    return cudaMemcpyToSymbol(delta_chain_fault, &zero, sizeof(int));
}

cudaError_t launch_delta_chain(const DeltaShape& shape, const __nv_bfloat16* q, const __nv_bfloat16* k, const __nv_bfloat16* v,
                               const float* initial, const DeltaSaved& saved, __nv_bfloat16* out, float* final_state,
                               cudaStream_t stream) {
    if (shape.d == 32) return by_width<32>(shape, q, k, v, initial, saved, out, final_state, stream);
    if (shape.d == 64) return by_width<64>(shape, q, k, v, initial, saved, out, final_state, stream);
    return by_width<128>(shape, q, k, v, initial, saved, out, final_state, stream);
}

}  // namespace dism
