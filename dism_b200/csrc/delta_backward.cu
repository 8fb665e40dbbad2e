// Gated delta rule, backward.  With dS1 the gradient of a chunk's last state (notation of delta_common.cuh):
//     dU = P^T dO + e^{G_63 - G} K dS1,   dX = b dU,   dY = T^T dX = dV,
//     dS0 = e^{G_63} dS1 + (scale e^G Q)^T dO - (e^G K)^T dY.
// delta_reverse_kernel walks the chunks from the last to the first with dS, transposed, in its accumulators (a warp owns 16
// columns, as in the forward chain), writes dV, keeps every dS1 and the part of db that needs dU.
// As the forward chain it is bound by latency: 167 us at 16 x 2048 positions, 10 heads of 128 (in shares); segments of 2 x 8192, 16 heads of 64: 39 + 68.
// delta_gradient_kernel then takes all chunks at once (here for D or DV of 32; delta_gradient.cu has the others).  With Z1 = dO X^T and Z2 = dY X^T,
//     dP~ = scale E b_s Z1 (s <= t),   dL~ = -E b_s Z2 (s < t),
//     dQ = scale e^G dO S0^T + dP~ K,
//     dK = -e^G dY S0^T + e^{G_63 - G} b X dS1^T + dL~ K + dL~^T K + dP~^T Q,
//     db_s = dU_s.X_s - sum_t E_ts (k_t.k_s) Z2_ts.
// Every exponent is a difference of G: M = dP~ * (Q K^T) + dL~ * (K K^T) adds its row sums to dG and takes its column sums
// away; the products with the states add q.dQ, k.dK and take k.dK of the three state terms; dG_63 gets the state's own
// e^{G_63} <dS1, S0> and the sum of the last of these.  dg is the reverse running sum of dG in the chunk.  Row and column
// sums come from one matrix in 32 bits, so the pairs that cancel in dg cancel exactly.
#include "delta_common.cuh"

namespace dism {
namespace {

template <int D, int WARPS>
struct ReverseStage {
    static constexpr int PITCH = 2 * D, VALUE_PITCH = 32 * WARPS;
    static constexpr int K = 0, Q = K + CHUNK * PITCH, T = Q + CHUNK * PITCH, P = T + 2 * MATRIX;
    static constexpr int DOUT = P + 2 * MATRIX, ROWS = DOUT + CHUNK * VALUE_PITCH, BYTES = ROWS + 3 * CHUNK * 4;
    static constexpr int X = 2 * BYTES, TOTAL = X + CHUNK * VALUE_PITCH;  // one X for both stages: its columns belong to a warp each
};

__device__ int delta_reverse_fault;

// LOCAL: the first launch over segments: from a zero gradient behind the segment to the one before it, no outputs.
// SHARES: a part of an uncut chain (see DeltaShares), its chunks counted from the end.
template <int D, int WARPS, bool LOCAL, bool SHARES>
__global__ void __launch_bounds__(WARPS * 32, 2) delta_reverse_kernel(DeltaShape shape, const __nv_bfloat16* __restrict__ q,
                                                                      const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ dout,
                                                                      const float* __restrict__ dfinal, DeltaSaved saved,
                                                                      __nv_bfloat16* __restrict__ dstates, float* __restrict__ dbeta_parts,
                                                                      __nv_bfloat16* __restrict__ dv_out, float* __restrict__ dinitial, float* __restrict__ ends) {
    using Stage = ReverseStage<D, WARPS>;
    constexpr int THREADS = WARPS * 32, TILES = CHUNK / 8;
    extern __shared__ __align__(128) unsigned char shared[];
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31;
    ShareWalk<D * 16 * WARPS> share;
    if (SHARES && !share.draw(shape, WARPS * 16)) return;
    bool more = false;
    do {
        const DeltaPart part = SHARES ? share.part(shape, &delta_reverse_fault, 13) : DeltaPart{blockIdx.x, blockIdx.y, blockIdx.z, 0, 0, nullptr, nullptr, false};
        const int head = part.head, dv = shape.dv;
        const int key_head = head / (shape.heads / shape.key_heads), column = (part.block * WARPS + warp) * 16;
        int64_t row, slot;
        int length, sequence, number;
        if (SHARES) sequence = part.segment, number = 0;
        else shape.segments.find(shape.layout, part.segment, sequence, number);
        if (number < 0) return;  // segments before the first document
        shape.layout.span(sequence, row, length, slot);
        const unsigned base = smem_address(shared);
        if (!LOCAL && !SHARES && shape.layout.cu && number == 0) {
            char* to = reinterpret_cast<char*>(dv_out + int64_t(head) * dv + part.block * WARPS * 16);
            const int64_t stride = int64_t(shape.heads) * dv * 2;
            if (sequence == 0) clear_rows<WARPS * 32>(to, stride, WARPS * 2, 0, row, thread);
            if (sequence == shape.layout.sequences - 1) clear_rows<WARPS * 32>(to, stride, WARPS * 2, row + length, shape.layout.n, thread);
        }
        int chunks = (length + CHUNK - 1) / CHUNK, behind = 0;  // segments behind this one
        if (SHARES) {
            const int before = chunks - part.end;
            chunks = part.end - part.begin;
            slot += before, row += int64_t(before) * CHUNK, length -= before * CHUNK;
        } else if (shape.segments.length) {
            const int before = min(number * shape.segments.length, chunks);
            if (number && before == chunks) return;  // no such segment
            if (LOCAL && number == 0) return;
            behind = (chunks - 1 - before) / shape.segments.length;
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
            load_tile<32 * WARPS, THREADS>(stage + Stage::DOUT,
                                           reinterpret_cast<const char*>(dout) + ((at * shape.heads + head) * dv + part.block * WARPS * 16) * 2,
                                           value_stride, count, thread);
            load_block<3 * CHUNK * 4, THREADS>(stage + Stage::ROWS, reinterpret_cast<const char*>(saved.rows + place * ROW_VALUES), thread);
            load_block<2 * MATRIX, THREADS>(stage + Stage::P, reinterpret_cast<const char*>(saved.p + place * MATRIX), thread);
            load_block<2 * MATRIX, THREADS>(stage + Stage::T, reinterpret_cast<const char*>(saved.t + place * MATRIX), thread);
            load_tile<2 * D, THREADS>(stage + Stage::Q, reinterpret_cast<const char*>(q) + key, key_stride, count, thread);
            cp_async_commit();
        };

        float ds[D / 8][4];
        const int64_t state_at = (int64_t(sequence) * shape.heads + head) * D * dv + column + (lane >> 2);
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                // the gradient behind the sequence; a segment that is not the last starts from zero in the first launch
                if (!SHARES || !part.from) ds[n][e] = dfinal && (!LOCAL || behind == 0) ? __ldg(dfinal + state_at + int64_t(8 * n + 2 * (lane & 3) + (e & 1)) * dv + (e >> 1) * 8) : 0.f;
        if (SHARES && part.from) {
            const float4* from = reinterpret_cast<const float4*>(part.from) + warp * (D / 8) * 32 + lane;
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
                *reinterpret_cast<float4*>(ds[n]) = part.lost ? make_float4(NOT_A_NUMBER, NOT_A_NUMBER, NOT_A_NUMBER, NOT_A_NUMBER) : __ldcg(from + n * 32);
        }
        // the gradient behind an earlier segment: dS <- M^T dS + B over the segments behind it, M and dS as pairs as in the forward.  The last one's B already has dfinal.
        if constexpr (!LOCAL && !SHARES && D >= 64 && WARPS == 4)
            for (int later = behind; later > 0; --later) {
                const int64_t place = (shape.segments.place(slot) + later) * shape.heads + head;  // of M; B lies one before
                const float4* end = reinterpret_cast<const float4*>(ends + (place - shape.heads) * D * dv) + column / 16 * (D / 8) * 32 + lane;
                float x[D / 8][4];
#pragma unroll
                for (int n = 0; n < D / 8; ++n) *reinterpret_cast<float4*>(x[n]) = __ldg(end + n * 32);
                if (later < behind) {
                    load_block<2 * D * D, THREADS>(base, reinterpret_cast<const char*>(shape.segments.m + place * D * D), thread);
                    load_block<2 * D * D, THREADS>(base + 2 * D * D, reinterpret_cast<const char*>(shape.segments.m_rest + place * D * D), thread);
                    cp_async_commit();
                    cp_async_wait<0>();
                    __syncthreads();
#pragma unroll
                    for (int kb = 0; kb < D / 16; ++kb) {
                        unsigned a[4], rest[4];
                        to_operand(a, ds[2 * kb], ds[2 * kb + 1]);
                        to_operand_rest(rest, a, ds[2 * kb], ds[2 * kb + 1]);
                        const unsigned m = base + kb * 2 * 128 + cols_first_blocked(lane, D / 8);
#pragma unroll
                        for (int np = 0; np < D / 16; ++np) {
                            unsigned b[4];
                            ldsm4(b, m + np * 2 * (D / 8) * 128);
                            mma16816(x[2 * np], a, b[0], b[1]);
                            mma16816(x[2 * np + 1], a, b[2], b[3]);
                            mma16816(x[2 * np], rest, b[0], b[1]);
                            mma16816(x[2 * np + 1], rest, b[2], b[3]);
                            ldsm4(b, m + 2 * D * D + np * 2 * (D / 8) * 128);
                            mma16816(x[2 * np], a, b[0], b[1]);
                            mma16816(x[2 * np + 1], a, b[2], b[3]);
                        }
                    }
                    __syncthreads();
                }
#pragma unroll
                for (int n = 0; n < D / 8; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) ds[n][e] = x[n][e];
            }
        if (chunks > 0) load(chunks - 1);
        for (int c = chunks - 1; c >= 0; --c) {
            cp_async_wait<0>();
            __syncthreads();  // chunk c is in, and every warp has left chunk c + 1
            if (!LOCAL) {  // X of this chunk, transposed: the warp's own rows, two kilobytes, needed only after dU
                const char* from = reinterpret_cast<const char*>(saved.x + ((slot + c) * shape.heads + head) * CHUNK * dv + column * CHUNK);
#pragma unroll
                for (int i = lane * 16; i < 2048; i += 512)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(base + Stage::X + warp * 2048 + i), "l"(from + i));
                cp_async_commit();
            }
            if (c > 0) load(c - 1);
            else cp_async_commit();
            const unsigned stage = base + (c & 1) * Stage::BYTES;
            const float* rows = reinterpret_cast<const float*>(shared + (c & 1) * Stage::BYTES + Stage::ROWS);
            const int64_t place = (slot + c) * shape.heads + head;

            float du[TILES][4];
#pragma unroll
            for (int n = 0; n < TILES; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) du[n][e] = 0.f;
            const TileLane keys = tile_cols_first<Stage::PITCH>(stage + Stage::K, lane);
            unsigned* state_out = reinterpret_cast<unsigned*>(dstates + place * dv * D) + int64_t(column / 8) * (D / 8) * 32 + lane;
#pragma unroll
            for (int kb = 0; kb < D / 16; ++kb) {
                unsigned a[4];
                to_operand(a, ds[2 * kb], ds[2 * kb + 1]);
                if (!LOCAL) {
                    unsigned* to = state_out + 2 * kb * 32;
                    to[0] = a[0], to[D / 8 * 32] = a[1], to[32] = a[2], to[D / 8 * 32 + 32] = a[3];
                }
#pragma unroll
                for (int np = 0; np < TILES / 2; ++np) {
                    unsigned b[4];
                    ldsm4(b, keys.at(kb * 32) + np * 16 * Stage::PITCH);
                    mma16816(du[2 * np], a, b[0], b[1]);
                    mma16816(du[2 * np + 1], a, b[2], b[3]);
                }
            }
            const unsigned own = tile_cols_first<Stage::VALUE_PITCH>(0, lane).at(warp * 32);
            unsigned grad[TILES / 2][4];  // dO, transposed, as a left operand
#pragma unroll
            for (int np = 0; np < TILES / 2; ++np) {
                ldsm4_trans(grad[np], stage + Stage::DOUT + own + np * 16 * Stage::VALUE_PITCH);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 tail = *reinterpret_cast<const float2*>(rows + 2 * CHUNK + 16 * np + 8 * h + 2 * (lane & 3));
                    float(&tile)[4] = du[2 * np + h];
                    tile[0] *= tail.x, tile[1] *= tail.y, tile[2] *= tail.x, tile[3] *= tail.y;
                }
            }
            const unsigned inside = stage + Stage::P + rows_first_tile(lane), inverse = inside + Stage::T - Stage::P;
#pragma unroll
            for (int np = 0; np < TILES / 2; ++np)
#pragma unroll
                for (int kb = np; kb < TILES / 2; ++kb) {
                    unsigned b[4];
                    ldsm4_trans(b, inside + tile_at(kb, np));
                    mma16816(du[2 * np], grad[kb], b[0], b[1]);
                    mma16816(du[2 * np + 1], grad[kb], b[2], b[3]);
                }
            // the part of db that needs dU: this warp's 16 columns of dU.X
            float* part = dbeta_parts + (int64_t(column / 16) * shape.layout.slots() * shape.heads + place) * CHUNK;
            unsigned dx[TILES / 2][4], dx_rest[TILES / 2][4];  // a pair: its rounding would be one more in dV and in all that follows
            cp_async_wait<1>();  // all but the next chunk
            __syncwarp();
#pragma unroll
            for (int np = 0; np < TILES / 2; ++np) {
                unsigned xx[4] = {0, 0, 0, 0};
#pragma unroll
                for (int e = 0; e < 4 && !LOCAL; ++e) xx[e] = *reinterpret_cast<const unsigned*>(shared + Stage::X + warp * 2048 + ((e & 1) * TILES + 2 * np + (e >> 1)) * 128 + lane * 4);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float(&tile)[4] = du[2 * np + h];
                    if (!LOCAL) {
                        float even = tile[0] * low_half(xx[2 * h]) + tile[2] * low_half(xx[2 * h + 1]);
                        float odd = tile[1] * high_half(xx[2 * h]) + tile[3] * high_half(xx[2 * h + 1]);
#pragma unroll
                        for (int m = 4; m < 32; m <<= 1) even += __shfl_xor_sync(FULL, even, m), odd += __shfl_xor_sync(FULL, odd, m);
                        if (lane < 4) *reinterpret_cast<float2*>(part + 16 * np + 8 * h + 2 * lane) = make_float2(even, odd);
                    }
                    const float2 b = *reinterpret_cast<const float2*>(rows + CHUNK + 16 * np + 8 * h + 2 * (lane & 3));
                    tile[0] *= b.x, tile[1] *= b.y, tile[2] *= b.x, tile[3] *= b.y;
                }
                to_operand(dx[np], du[2 * np], du[2 * np + 1]);
                to_operand_rest(dx_rest[np], dx[np], du[2 * np], du[2 * np + 1]);
            }
            float(&dy)[TILES][4] = du;
#pragma unroll
            for (int n = 0; n < TILES; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) dy[n][e] = 0.f;
#pragma unroll
            for (int np = 0; np < TILES / 2; ++np)
#pragma unroll
                for (int kb = np; kb < TILES / 2; ++kb) {
                    unsigned b[4];
                    ldsm4_trans(b, inverse + tile_at(kb, np));
                    mma16816(dy[2 * np], dx[kb], b[0], b[1]);
                    mma16816(dy[2 * np + 1], dx[kb], b[2], b[3]);
                    mma16816(dy[2 * np], dx_rest[kb], b[0], b[1]);
                    mma16816(dy[2 * np + 1], dx_rest[kb], b[2], b[3]);
                }
            if (!LOCAL) {
                // dV leaves through the warp's room of X: rows of 32 bytes, the halves of rows 4-7 of every eight exchanged
                const unsigned values = base + Stage::X + warp * 2048 + ((lane & 7) + ((lane >> 4) << 3)) * 32 + ((((lane >> 3) ^ (lane >> 2)) & 1) * 16);
                __syncwarp();
#pragma unroll
                for (int np = 0; np < TILES / 2; ++np)
                    stsm4_trans(values + np * 512, pack2(dy[2 * np][0], dy[2 * np][1]), pack2(dy[2 * np][2], dy[2 * np][3]),
                                pack2(dy[2 * np + 1][0], dy[2 * np + 1][1]), pack2(dy[2 * np + 1][2], dy[2 * np + 1][3]));
                __syncwarp();
                const int count = min(CHUNK, length - c * CHUNK);
                char* to = reinterpret_cast<char*>(dv_out + ((row + int64_t(c) * CHUNK) * shape.heads + head) * dv + column);
#pragma unroll
                for (int i = 0; i < CHUNK * 2 / 32; ++i) {
                    const int t = i * 16 + (lane >> 1);
                    const uint4 piece = *reinterpret_cast<const uint4*>(shared + Stage::X + warp * 2048 + t * 32 + (((lane & 1) ^ ((t >> 2) & 1)) * 16));
                    if (t < count) *reinterpret_cast<uint4*>(to + t * value_stride + (lane & 1) * 16) = piece;
                }
                __syncwarp();  // the room is free for the next chunk's X
            }
            // scale e^G dO and -e^G dY, the left operands of the state's step
#pragma unroll
            for (int np = 0; np < TILES / 2; ++np) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 decay = *reinterpret_cast<const float2*>(rows + 16 * np + 8 * h + 2 * (lane & 3));
                    const float sx = shape.scale * decay.x, sy = shape.scale * decay.y;
                    float(&tile)[4] = dy[2 * np + h];
                    tile[0] *= -decay.x, tile[1] *= -decay.y, tile[2] *= -decay.x, tile[3] *= -decay.y;
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        grad[np][2 * h + e] = pack2(low_half(grad[np][2 * h + e]) * sx, high_half(grad[np][2 * h + e]) * sy);
                }
                to_operand(dx[np], dy[2 * np], dy[2 * np + 1]);
            }
            const float kept = rows[CHUNK - 1];
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) ds[n][e] *= kept;
            const TileLane keys_trans = tile_rows_first<Stage::PITCH>(stage + Stage::K, lane);
#pragma unroll
            for (int kb = 0; kb < TILES / 2; ++kb)
#pragma unroll
                for (int np = 0; np < D / 16; ++np) {
                    unsigned b[4];
                    ldsm4_trans(b, keys_trans.at(np * 32) + kb * 16 * Stage::PITCH);
                    mma16816(ds[2 * np], dx[kb], b[0], b[1]);
                    mma16816(ds[2 * np + 1], dx[kb], b[2], b[3]);
                    ldsm4_trans(b, keys_trans.at(np * 32) + Stage::Q - Stage::K + kb * 16 * Stage::PITCH);
                    mma16816(ds[2 * np], grad[kb], b[0], b[1]);
                    mma16816(ds[2 * np + 1], grad[kb], b[2], b[3]);
                }
        }
        if (LOCAL) {
            float4* to = reinterpret_cast<float4*>(ends + ((shape.segments.place(slot) - 1) * shape.heads + head) * D * dv) + column / 16 * (D / 8) * 32 + lane;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) to[n * 32] = *reinterpret_cast<float4*>(ds[n]);
        } else if (SHARES && part.to) {
            float4* to = reinterpret_cast<float4*>(part.to) + warp * (D / 8) * 32 + lane;
#pragma unroll
            for (int n = 0; n < D / 8; ++n) to[n * 32] = *reinterpret_cast<float4*>(ds[n]);
        } else if (dinitial && number == 0) {
#pragma unroll
            for (int n = 0; n < D / 8; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    dinitial[state_at + int64_t(8 * n + 2 * (lane & 3) + (e & 1)) * dv + (e >> 1) * 8] = ds[n][e];
        }
        more = SHARES && share.next(part);
    } while (more);
}

constexpr int GRADIENT_THREADS = 256;

template <int D, int DV>
struct GradientShared {
    static constexpr int PITCH = 2 * D + 16, VALUE_PITCH = 2 * DV + 16, MATRIX_PITCH = 2 * CHUNK + 16;
    static constexpr int K = 0, Q = K + CHUNK * PITCH, DOUT = Q + CHUNK * PITCH, DY = DOUT + CHUNK * VALUE_PITCH, X = DY + CHUNK * VALUE_PITCH;
    static constexpr int S0 = X + CHUNK * 2 * DV, DS = S0 + 2 * D * DV, DP = DS + 2 * D * DV, DL = DP + CHUNK * MATRIX_PITCH;
    static constexpr int ROWS = DL + CHUNK * MATRIX_PITCH, SUMS = ROWS + ROW_VALUES * 4;
    // sums: rows of M [2][64], columns of M [4][2][64], columns of b [4][64], state terms of dG [2][64] and dG_63 [2][64], <dS1, S0> [8]
    static constexpr int ROW_SUM = 0, COLUMN_SUM = ROW_SUM + 2 * CHUNK, BETA_SUM = COLUMN_SUM + 8 * CHUNK, STATE_SUM = BETA_SUM + 4 * CHUNK;
    static constexpr int LAST_SUM = STATE_SUM + 2 * CHUNK, DOT = LAST_SUM + 2 * CHUNK, BYTES = SUMS + (DOT + 8) * 4;
};

template <int D, int DV>
__global__ void __launch_bounds__(GRADIENT_THREADS, 1) delta_gradient_kernel(DeltaShape shape, const __nv_bfloat16* __restrict__ q,
                                                                             const __nv_bfloat16* __restrict__ k, const __nv_bfloat16* __restrict__ dout,
                                                                             const __nv_bfloat16* __restrict__ dy, DeltaSaved saved,
                                                                             const __nv_bfloat16* __restrict__ dstates, const float* __restrict__ dbeta_parts,
                                                                             __nv_bfloat16* __restrict__ dq, __nv_bfloat16* __restrict__ dk,
                                                                             void* __restrict__ dg, void* __restrict__ dbeta) {
    using Shared = GradientShared<D, DV>;
    constexpr int TILES = CHUNK / 8, NT = D / 16;  // a warp takes 16 rows and half of the D columns: NT tiles of 8
    extern __shared__ __align__(128) unsigned char shared[];
    const int thread = threadIdx.x, warp = thread >> 5, lane = thread & 31, g = lane >> 2, c = lane & 3;
    const int part = warp & 3, half = warp >> 2, key_head = blockIdx.y, group = shape.heads / shape.key_heads;
    int64_t row;
    int count;
    const int64_t slot = blockIdx.x;
    if (shape.layout.cu && key_head == 0) clear_gradients<GRADIENT_THREADS>(shape, dq, dk, dg, dbeta, blockIdx.x, gridDim.x, thread);
    shape.layout.chunk(slot, row, count);
    if (count == 0) return;
    const unsigned base = smem_address(shared);
    float* rows = reinterpret_cast<float*>(shared + Shared::ROWS);
    float* sums = reinterpret_cast<float*>(shared + Shared::SUMS);
    const int64_t key_stride = int64_t(shape.key_heads) * D * 2, value_stride = int64_t(shape.heads) * DV * 2;
    const int64_t key = (row * shape.key_heads + key_head) * D * 2;
    load_rows<2 * D, GRADIENT_THREADS>(base + Shared::K, Shared::PITCH, reinterpret_cast<const char*>(k) + key, key_stride, count, thread);
    load_rows<2 * D, GRADIENT_THREADS>(base + Shared::Q, Shared::PITCH, reinterpret_cast<const char*>(q) + key, key_stride, count, thread);

    float dq_sum[NT][4], dk_sum[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) dq_sum[n][e] = dk_sum[n][e] = 0.f;

    for (int head = key_head * group; head < (key_head + 1) * group; ++head) {
        const int64_t place = slot * shape.heads + head;
        const int64_t value = (row * shape.heads + head) * DV * 2;
        load_block<2 * CHUNK * DV, GRADIENT_THREADS>(base + Shared::X, reinterpret_cast<const char*>(saved.x + place * CHUNK * DV), thread);
        load_rows<2 * DV, GRADIENT_THREADS>(base + Shared::DOUT, Shared::VALUE_PITCH, reinterpret_cast<const char*>(dout) + value, value_stride, count, thread);
        load_rows<2 * DV, GRADIENT_THREADS>(base + Shared::DY, Shared::VALUE_PITCH, reinterpret_cast<const char*>(dy) + value, value_stride, count, thread);
        load_block<ROW_VALUES * 4, GRADIENT_THREADS>(base + Shared::ROWS, reinterpret_cast<const char*>(saved.rows + place * ROW_VALUES), thread);
        cp_async_commit();
        load_block<2 * D * DV, GRADIENT_THREADS>(base + Shared::S0, reinterpret_cast<const char*>(saved.states + place * D * DV), thread);
        load_block<2 * D * DV, GRADIENT_THREADS>(base + Shared::DS, reinterpret_cast<const char*>(dstates + place * D * DV), thread);
        cp_async_commit();
        cp_async_wait<1>();
        __syncthreads();
        {  // warps 0-3: Z1 and Q K^T; warps 4-7: Z2 and K K^T; sixteen rows each, columns up to the diagonal
            float z[TILES][4], y[TILES][4];
#pragma unroll
            for (int n = 0; n < TILES; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) z[n][e] = y[n][e] = 0.f;
            const unsigned own = base + (half ? Shared::DY : Shared::DOUT) + part * 16 * Shared::VALUE_PITCH + rows_first(lane, Shared::VALUE_PITCH);
            const unsigned xs = base + Shared::X + rows_first_blocked(lane, TILES);
#pragma unroll
            for (int kb = 0; kb < DV / 16; ++kb) {
                unsigned a[4];
                ldsm4(a, own + kb * 32);
#pragma unroll
                for (int np = 0; np < TILES / 2; ++np) {
                    if (np > part) continue;
                    unsigned b[4];
                    ldsm4_trans(b, xs + (kb * 2 * TILES + np * 2) * 128);
                    mma16816(z[2 * np], a, b[0], b[1]);
                    mma16816(z[2 * np + 1], a, b[2], b[3]);
                }
            }
            const unsigned own_key = base + (half ? Shared::K : Shared::Q) + part * 16 * Shared::PITCH + rows_first(lane, Shared::PITCH);
            const unsigned keys = base + Shared::K + cols_first(lane, Shared::PITCH);
#pragma unroll
            for (int kb = 0; kb < D / 16; ++kb) {
                unsigned a[4];
                ldsm4(a, own_key + kb * 32);
#pragma unroll
                for (int np = 0; np < TILES / 2; ++np) {
                    if (np > part) continue;
                    unsigned b[4];
                    ldsm4(b, keys + np * 16 * Shared::PITCH + kb * 32);
                    mma16816(y[2 * np], a, b[0], b[1]);
                    mma16816(y[2 * np + 1], a, b[2], b[3]);
                }
            }
            const float *high = rows + ROW_HIGH, *low = rows + ROW_LOW, *beta = rows + ROW_BETA;
            float row_sum[2] = {0.f, 0.f};
#pragma unroll
            for (int n = 0; n < TILES; ++n) {
                float column_sum[2] = {0.f, 0.f}, beta_sum[2] = {0.f, 0.f};
                const int s = 8 * n + 2 * c;
                if (n <= 2 * part + 1) {
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const int t = 16 * part + 8 * r + g;
                        float d[2];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float between = ex2((high[t] - high[s + e]) + (low[t] - low[s + e]));
                            const bool counts = half ? s + e < t : s + e <= t;
                            const float w = counts ? (half ? -between : shape.scale * between) * z[n][2 * r + e] : 0.f;
                            d[e] = w * beta[s + e];
                            const float m = d[e] * y[n][2 * r + e];
                            row_sum[r] += m, column_sum[e] += m;
                            beta_sum[e] += w * y[n][2 * r + e];
                        }
                        *reinterpret_cast<unsigned*>(shared + (half ? Shared::DL : Shared::DP) + t * Shared::MATRIX_PITCH + s * 2) = pack2(d[0], d[1]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int m = 4; m < 32; m <<= 1) {
                        column_sum[e] += __shfl_xor_sync(FULL, column_sum[e], m);
                        beta_sum[e] += __shfl_xor_sync(FULL, beta_sum[e], m);
                    }
                    if (g == 0) {
                        sums[Shared::COLUMN_SUM + (part * 2 + half) * CHUNK + s + e] = column_sum[e];
                        if (half) sums[Shared::BETA_SUM + part * CHUNK + s + e] = beta_sum[e];
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                row_sum[r] += __shfl_xor_sync(FULL, row_sum[r], 1);
                row_sum[r] += __shfl_xor_sync(FULL, row_sum[r], 2);
                if (c == 0) sums[Shared::ROW_SUM + half * CHUNK + 16 * part + 8 * r + g] = row_sum[r];
            }
        }
        cp_async_wait<0>();
        __syncthreads();
        {
            float dot = 0.f;  // <dS1, S0>
            const uint4 *s0 = reinterpret_cast<const uint4*>(shared + Shared::S0), *ds = reinterpret_cast<const uint4*>(shared + Shared::DS);
#pragma unroll
            for (int i = thread; i < D * DV / 8; i += GRADIENT_THREADS) {
                const uint4 x = s0[i], y = ds[i];
                dot += low_half(x.x) * low_half(y.x) + high_half(x.x) * high_half(y.x) + low_half(x.y) * low_half(y.y) + high_half(x.y) * high_half(y.y);
                dot += low_half(x.z) * low_half(y.z) + high_half(x.z) * high_half(y.z) + low_half(x.w) * low_half(y.w) + high_half(x.w) * high_half(y.w);
            }
#pragma unroll
            for (int m = 16; m; m >>= 1) dot += __shfl_xor_sync(FULL, dot, m);
            if (lane == 0) sums[Shared::DOT + warp] = dot;
        }
        const int t0 = 16 * part + g;  // this lane's rows: t0 and t0 + 8
        const float decay[2] = {rows[t0], rows[t0 + 8]};
        float state_sum[2] = {0.f, 0.f}, last_sum[2] = {0.f, 0.f};
        float tile[NT][4];
        // 16 rows of a value-wide operand times half of a state
        auto state_product = [&](int operand, int state, bool transposed) {
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) tile[n][e] = 0.f;
            const unsigned left = transposed ? base + operand + cols_first_blocked(lane, TILES) + part * 256
                                             : base + operand + part * 16 * Shared::VALUE_PITCH + rows_first(lane, Shared::VALUE_PITCH);
            const unsigned right = base + state + rows_first_blocked(lane, D / 8) + half * (D / 16) * 128;
#pragma unroll
            for (int kb = 0; kb < DV / 16; ++kb) {
                unsigned a[4];
                if (transposed) ldsm4_trans(a, left + kb * 2 * TILES * 128);
                else ldsm4(a, left + kb * 32);
#pragma unroll
                for (int np = 0; np < NT / 2; ++np) {
                    unsigned b[4];
                    ldsm4_trans(b, right + (kb * 2 * (D / 8) + np * 2) * 128);
                    mma16816(tile[2 * np], a, b[0], b[1]);
                    mma16816(tile[2 * np + 1], a, b[2], b[3]);
                }
            }
        };
        // scales the product's rows, adds it to a gradient and its dot with the rows of q or k to the sums
        auto take = [&](float (&to)[NT][4], int factor, float f0, float f1, float (&dots)[2]) {
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int d = half * (D / 2) + 8 * n + 2 * c;
                const unsigned x0 = *reinterpret_cast<const unsigned*>(shared + factor + t0 * Shared::PITCH + d * 2);
                const unsigned x1 = *reinterpret_cast<const unsigned*>(shared + factor + (t0 + 8) * Shared::PITCH + d * 2);
                const float v0 = tile[n][0] * f0, v1 = tile[n][1] * f0, v2 = tile[n][2] * f1, v3 = tile[n][3] * f1;
                to[n][0] += v0, to[n][1] += v1, to[n][2] += v2, to[n][3] += v3;
                dots[0] += v0 * low_half(x0) + v1 * high_half(x0);
                dots[1] += v2 * low_half(x1) + v3 * high_half(x1);
            }
        };
        state_product(Shared::DOUT, Shared::S0, false);
        take(dq_sum, Shared::Q, shape.scale * decay[0], shape.scale * decay[1], state_sum);
        state_product(Shared::DY, Shared::S0, false);
        take(dk_sum, Shared::K, -decay[0], -decay[1], state_sum);
        state_product(Shared::X, Shared::DS, true);
        take(dk_sum, Shared::K, rows[ROW_WRITE + t0], rows[ROW_WRITE + t0 + 8], last_sum);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int m = 1; m < 4; m <<= 1) {
                state_sum[r] += __shfl_xor_sync(FULL, state_sum[r], m);
                last_sum[r] += __shfl_xor_sync(FULL, last_sum[r], m);
            }
            if (c == 0) {
                sums[Shared::STATE_SUM + half * CHUNK + t0 + 8 * r] = state_sum[r];
                sums[Shared::LAST_SUM + half * CHUNK + t0 + 8 * r] = last_sum[r];
            }
        }
        // dP~ K and dL~ K take the columns up to the diagonal, dL~^T K and dP~^T Q the rows from it
        {
            const unsigned left = base + Shared::DP + part * 16 * Shared::MATRIX_PITCH + rows_first(lane, Shared::MATRIX_PITCH);
            const unsigned left_trans = base + Shared::DP + part * 32 + cols_first(lane, Shared::MATRIX_PITCH);
            const unsigned keys = base + Shared::K + rows_first(lane, Shared::PITCH) + half * D, queries = keys + Shared::Q - Shared::K;
            constexpr int DL = Shared::DL - Shared::DP;
#pragma unroll
            for (int kb = 0; kb < TILES / 2; ++kb) {
                unsigned p[4], l[4], pt[4], lt[4];
                if (kb <= part) {
                    ldsm4(p, left + kb * 32);
                    ldsm4(l, left + DL + kb * 32);
                }
                if (kb >= part) {
                    ldsm4_trans(pt, left_trans + kb * 16 * Shared::MATRIX_PITCH);
                    ldsm4_trans(lt, left_trans + DL + kb * 16 * Shared::MATRIX_PITCH);
                }
#pragma unroll
                for (int np = 0; np < NT / 2; ++np) {
                    unsigned b[4];
                    ldsm4_trans(b, keys + kb * 16 * Shared::PITCH + np * 32);
                    if (kb <= part) {
                        mma16816(dq_sum[2 * np], p, b[0], b[1]);
                        mma16816(dq_sum[2 * np + 1], p, b[2], b[3]);
                        mma16816(dk_sum[2 * np], l, b[0], b[1]);
                        mma16816(dk_sum[2 * np + 1], l, b[2], b[3]);
                    }
                    if (kb >= part) {
                        mma16816(dk_sum[2 * np], lt, b[0], b[1]);
                        mma16816(dk_sum[2 * np + 1], lt, b[2], b[3]);
                        ldsm4_trans(b, queries + kb * 16 * Shared::PITCH + np * 32);
                        mma16816(dk_sum[2 * np], pt, b[0], b[1]);
                        mma16816(dk_sum[2 * np + 1], pt, b[2], b[3]);
                    }
                }
            }
        }
        __syncthreads();
        if (warp == 0) {
            float here[2], last = 0.f;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int t = 2 * lane + e;
                const float tail = sums[Shared::LAST_SUM + t] + sums[Shared::LAST_SUM + CHUNK + t];
                float value = sums[Shared::ROW_SUM + t] + sums[Shared::ROW_SUM + CHUNK + t];
#pragma unroll
                for (int i = 0; i < 8; ++i) value -= sums[Shared::COLUMN_SUM + i * CHUNK + t];
                here[e] = value + (sums[Shared::STATE_SUM + t] + sums[Shared::STATE_SUM + CHUNK + t]) - tail;
                last += tail;
                float b = 0.f;
                const int64_t stride = shape.layout.slots() * shape.heads * CHUNK;
                for (int i = 0; i < DV / 16; ++i) b += __ldg(dbeta_parts + i * stride + place * CHUNK + t);
#pragma unroll
                for (int i = 0; i < 4; ++i) b += sums[Shared::BETA_SUM + i * CHUNK + t];
                if (t < count) {
                    const int64_t index = (row + t) * shape.heads + head;
                    if (shape.gates_bf16) static_cast<__nv_bfloat16*>(dbeta)[index] = __float2bfloat16(b);
                    else static_cast<float*>(dbeta)[index] = b;
                }
            }
#pragma unroll
            for (int m = 16; m; m >>= 1) last += __shfl_xor_sync(FULL, last, m);
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) dot += sums[Shared::DOT + i];
            last += rows[CHUNK - 1] * dot;
            if (lane == 31) here[1] += last;
            here[0] += here[1];
            float after = here[0];
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const float other = __shfl_down_sync(FULL, after, s);
                if (lane + s < 32) after += other;
            }
            after -= here[0];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int t = 2 * lane + e;
                if (t < count) {
                    const int64_t index = (row + t) * shape.heads + head;
                    // a decay that is zero in 32 bits has no gradient; the sum would leave the roundings of terms that cancel
                    const float *high = rows + ROW_HIGH, *low = rows + ROW_LOW;
                    const float step = t ? (high[t] - high[t - 1]) + (low[t] - low[t - 1]) : high[0];
                    const float value = step < -149.f ? 0.f : after + here[e];
                    if (shape.gates_bf16) static_cast<__nv_bfloat16*>(dg)[index] = __float2bfloat16(value);
                    else static_cast<float*>(dg)[index] = value;
                }
            }
        }
        __syncthreads();  // the tiles and sums are free for the next head
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const int t = 16 * part + 8 * r + g;
        if (t >= count) continue;
        const int64_t at = ((row + t) * shape.key_heads + key_head) * D + half * (D / 2) + 2 * c;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            *reinterpret_cast<unsigned*>(dq + at + 8 * n) = pack2(dq_sum[n][2 * r], dq_sum[n][2 * r + 1]);
            *reinterpret_cast<unsigned*>(dk + at + 8 * n) = pack2(dk_sum[n][2 * r], dk_sum[n][2 * r + 1]);
        }
    }
}

template <int D, int WARPS, bool LOCAL = false>
cudaError_t launch_reverse(const DeltaShape& shape, const DeltaGradients& x, const DeltaSaved& saved, cudaStream_t stream) {
    if constexpr (!LOCAL && D >= 64 && WARPS == 4)
        if (shape.segments.length)
            if (cudaError_t status = launch_reverse<D, WARPS, true>(shape, x, saved, stream)) return status;
    constexpr int BYTES = ReverseStage<D, WARPS>::TOTAL;
    constexpr auto* kernel = delta_reverse_kernel<D, WARPS, LOCAL, false>;
    if (cudaError_t status = allow_shared<kernel>(BYTES)) return status;
    if constexpr (!LOCAL && D >= 64 && WARPS == 4)
        if (shape.shares.length) {
            constexpr auto* shared_kernel = delta_reverse_kernel<D, WARPS, false, true>;
            if (cudaError_t status = allow_shared<shared_kernel>(BYTES)) return status;
            if (cudaError_t status = cudaMemsetAsync(shape.shares.flags, 0, shape.shares.flag_bytes(), stream)) return status;
            KernelTimer timer("delta_reverse", stream);
            shared_kernel<<<shape.shares.places, WARPS * 32, BYTES, stream>>>(shape, x.q, x.k, x.dout, x.dfinal, saved, x.dstates, x.dbeta_parts, x.dv,
                                                                              x.dinitial, nullptr);
            return cudaGetLastError();
        }
    KernelTimer timer(LOCAL ? "delta_reverse_segments" : "delta_reverse", stream);
    kernel<<<dim3(unsigned(shape.segments.count(shape.layout)), shape.heads, shape.dv / (16 * WARPS)), WARPS * 32, BYTES, stream>>>(
        shape, x.q, x.k, x.dout, x.dfinal, saved, x.dstates, x.dbeta_parts, x.dv, x.dinitial, x.ends);
    return cudaGetLastError();
}

template <int D, int DV>
cudaError_t launch_gradient(const DeltaShape& shape, const DeltaGradients& x, const DeltaSaved& saved, cudaStream_t stream) {
    constexpr int BYTES = GradientShared<D, DV>::BYTES;
    constexpr auto* kernel = delta_gradient_kernel<D, DV>;
    if (cudaError_t status = allow_shared<kernel>(BYTES)) return status;
    KernelTimer timer("delta_gradient", stream);
    kernel<<<dim3(unsigned(shape.layout.slots()), shape.key_heads), GRADIENT_THREADS, BYTES, stream>>>(
        shape, x.q, x.k, x.dout, x.dv, saved, x.dstates, x.dbeta_parts, x.dq, x.dk, x.dg, x.dbeta);
    return cudaGetLastError();
}

template <int D>
cudaError_t launch_width(const DeltaShape& shape, const DeltaGradients& x, const DeltaSaved& saved, cudaStream_t stream) {
    cudaError_t status = shape.dv % 64 == 0 ? launch_reverse<D, 4>(shape, x, saved, stream) : launch_reverse<D, 2>(shape, x, saved, stream);
    if (status || shape.layout.slots() == 0) return status;
    if (shape.dv == 32) return launch_gradient<D, 32>(shape, x, saved, stream);
    if constexpr (D >= 64) return launch_delta_gradient_tensor(shape, x, saved, stream);
    else return shape.dv == 64 ? launch_gradient<D, 64>(shape, x, saved, stream) : launch_gradient<D, 128>(shape, x, saved, stream);
}
}  // namespace

cudaError_t read_reverse_fault(int* code) {
    if (cudaError_t status = cudaMemcpyFromSymbol(code, delta_reverse_fault, sizeof(int))) return status;
    const int zero = 0;
    return cudaMemcpyToSymbol(delta_reverse_fault, &zero, sizeof(int));
}

cudaError_t launch_delta_backward(const DeltaShape& shape, const DeltaGradients& x, const DeltaSaved& saved, cudaStream_t stream) {
    if (shape.d == 32) return launch_width<32>(shape, x, saved, stream);
    if (shape.d == 64) return launch_width<64>(shape, x, saved, stream);
    return launch_width<128>(shape, x, saved, stream);
}

}  // namespace dism
