// The trunk projection on int8 activations (a scale a token) and int8 weights (a scale a row): Y = epilogue(float(X W^T) sx sw).
//
// tcgen05.mma kind::i8 multiplies bytes at twice the rate of binary16 and adds them into exact 32-bit integers. Two things follow. No
// operand is converted on its way (the kernels of gemm_tc.cu widen an int8 weight first), so a k step is a load and four MMAs of K 32.
// And integer addition has no order: however k is cut, the sums, and with them the result's bits, are the same.
//
// Both kernels put the weights on the MMA's M side and the tokens on its N side, whose width is free in steps of 16 (pairs: 32): tokens are
// padded to whole tiles of that width, the last one too, and not to 128 or 256 rows.
//
//   gemm_s8_pair_kernel  CTA pairs, 256 weight rows by `bt` tokens to a tile, persistent, two accumulators in tensor memory (the epilogue of a
//                        tile runs behind the next tile's products).
//   gemm_s8_few_kernel   up to 256 tokens, where a few weight rows have a long k: 128 weight rows to a CTA, a tile's k cut over a cluster of up to
//                        eight CTAs, whose sums meet through distributed shared memory.
//
// What bounds them, and what they measured (launches back to back, weights from DRAM, clocks as they were):
//   - Full calls are bound by the tensor cores under the power cap: 4096 x 24576 x 4096 with SwiGLU 251 us in bursts (3.28 POP/s, where the
//     measured binary16 rate of the library product, doubled, is 3.31) and 270 to 280 over a quarter of a second.
//   - A few hundred tokens make one to five waves of tiles; a step takes about the 2 bt clocks of its MMAs (317 measured alone at bt 160; within
//     a launch 310 to 316 from one issue to the next, the last MMAs still queued at the end), and what is lost is the part of the last wave
//     without tiles and about 10,000 clocks a launch: 3000 until the launch before has ended, 1100 for the first boxes, 4100 for the last
//     tile's results (all pairs add theirs at once, to a Y that comes from DRAM then; leaving them lane by lane without the staging
//     boxes takes as long, and longer in binary16) and 1400 to leave. 900 x 2560 x 9728 added: 20.3 us (2.2 POP/s); 1337 x 6144 x 2560
//     16.9; 900 x 19456 x 2560 SwiGLU 36.
//   - Few tokens are bound by the launch (3.3 us with next to nothing to do) and then the reading of W: one token by 6144 x 2560 5.6 us, 2560 x 9728
//     7.4, 24576 x 4096 18.5 (15.4 at the memory's rate).
//   Requesting W ahead into the L2 changed nothing; nor did fewer commits.
#include "gemm_s8.hpp"

#include <atomic>
#include <cstdint>
#include <cstring>
#include <stdexcept>
#include <string>

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "gemm_device.cuh"
#include "gemm_few.hpp"
#include "ptx.cuh"

namespace sepal::b200 {

void count_launch();

namespace {

constexpr unsigned kBK = 128;                 // values of k to a step: one 128-byte swizzled row
constexpr unsigned kRows = 128;               // weight rows to a CTA
constexpr unsigned kWBytes = kRows * kBK;     // one box of W
constexpr unsigned kSmemMax = 232448;         // 227 KB, what one block may have

struct S8Params {
    void* y;
    unsigned long long ld_y;
    const float* sx;
    const float* sw;
    int* status;
    unsigned m, n;                            // tokens, weight rows
    unsigned k_iters, bt, stages, t_tiles, tiles, split;
    unsigned tmem_cols;
    unsigned epilogue, y_half, staged, vec_ok, early_w;
};

__device__ __forceinline__ float scaled(int sum, float sx, float sw) { return __fmul_rn(__fmul_rn(__int2float_rn(sum), sx), sw); }

// ---- CTA pairs ----------------------------------------------------------------------------------------------------------------------
//
//   warp 0      TMA producer: per step a [128 x 128] byte box of W and this CTA's half of the X tile, [bt / 2 x 128]
//   warp 1      MMA issuer (first CTA): four tcgen05.mma.cta_group::2 (M 256, N bt, K 32) to a step
//   warps 2..9  epilogue: two warps to a quarter of the accumulator's lanes, which take chunks of 32 tokens in turn. A lane is an output
//               column, its registers run along the tokens; a chunk leaves transposed through the warp's staging boxes and the TMA (a store,
//               or a reduce-add for the float32 residual update), or lane by lane where Y's rows are not whole 16-byte units.
constexpr unsigned kPairThreads = 320;
constexpr unsigned kMaxStages = 12;
constexpr unsigned kAccStride = 256;          // tensor-memory columns from one accumulator to the other
constexpr unsigned kEpilogueWarps = 8;
constexpr unsigned kBoxBytes = 2048;          // a staging box: 16 tokens x 32 float32, or 32 x 32 binary16; two to a warp
constexpr unsigned kPairBarriers = 2 * kMaxStages + 4;
constexpr unsigned kPairTail = kEpilogueWarps * 128 + kPairBarriers * 8 + 64;

// The issuing roles are run by a whole warp, every branch but the elected thread's own the same for all of it. Addresses and descriptors then
// stay in the warp's uniform registers, which the asynchronous instructions take their operands from; in a loop run by one thread (if
// lane == 0) each is moved there for every instruction: 468 clocks a step of four MMAs where the tensor cores need 2 bt.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "elect.sync _|p, 0xFFFFFFFF;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t"
        "}"
        : "=r"(one));
    return one != 0;
}
// wait_barrier by a whole warp: every branch is the same for all of it, so that the loops around it stay in uniform registers.
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile unsigned* abort_flag, int* status, int code) {
    if (__all_sync(0xFFFFFFFFu, ptx::mbar_try_wait(bar, parity))) return true;
    const long long t0 = clock64();
    for (unsigned spins = 1;; ++spins) {
        if (__all_sync(0xFFFFFFFFu, ptx::mbar_try_wait(bar, parity))) return true;
        if ((spins & 31u) == 0) {
            const bool late = clock64() - t0 > kWaitLimit;
            if (__any_sync(0xFFFFFFFFu, late || *abort_flag != 0)) {
                if (__any_sync(0xFFFFFFFFu, late) && threadIdx.x % 32 == 0) {
                    *abort_flag = 1;
                    atomicCAS(status, 0, code | (static_cast<int>(blockIdx.x) << 8));
                }
                __syncwarp();
                return false;
            }
        }
    }
}

// Both warps that share a chunk of the SwiGLU arrive with their own `ok`; true when both are.
__device__ __forceinline__ bool both_agree(uint32_t id, bool ok) {
    uint32_t r;
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.and.pred q, %2, 64, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t"
        "}"
        : "=r"(r)
        : "r"(ok ? 1u : 0u), "r"(id)
        : "memory");
    return r != 0;
}

template <int ROWS>
__device__ __forceinline__ void store_lane(const S8Params& p, unsigned token, unsigned col, unsigned n_out, const float (&v)[ROWS]) {
    if (col >= n_out) return;
    const bool add = p.epilogue == 1;
    if (p.y_half != 0) {
        __half* out = static_cast<__half*>(p.y) + static_cast<size_t>(token) * p.ld_y + col;
#pragma unroll
        for (unsigned j = 0; j < ROWS; ++j)
            if (token + j < p.m) out[j * p.ld_y] = __float2half_rn(add ? __fadd_rn(__half2float(out[j * p.ld_y]), v[j]) : v[j]);
    } else {
        float* out = static_cast<float*>(p.y) + static_cast<size_t>(token) * p.ld_y + col;
#pragma unroll
        for (unsigned j = 0; j < ROWS; ++j)
            if (token + j < p.m) out[j * p.ld_y] = add ? __fadd_rn(out[j * p.ld_y], v[j]) : v[j];
    }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
gemm_s8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_y,
                    const S8Params p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_addr(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw_addr);
    const unsigned bt = p.bt, x_box = bt / 2 * kBK, stage_bytes = kWBytes + x_box;
    const int stages = static_cast<int>(p.stages);
    // layout: ring | staging boxes | the warps' token scales | barriers
    const unsigned box_off = p.stages * stage_bytes;
    uint8_t* const tail = smem + box_off + kEpilogueWarps * 2 * kBoxBytes;
    const uint32_t bars = ptx::smem_addr(tail + kEpilogueWarps * 128);
    const auto full_bar = [&](int s) { return bars + 8u * s; };
    const auto empty_bar = [&](int s) { return bars + 8u * (kMaxStages + s); };
    const auto acc_full_bar = [&](int a) { return bars + 8u * (2 * kMaxStages + a); };
    const auto acc_empty_bar = [&](int a) { return bars + 8u * (2 * kMaxStages + 2 + a); };
    unsigned* const words = reinterpret_cast<unsigned*>(tail + kEpilogueWarps * 128 + kPairBarriers * 8);
    volatile unsigned* const abort_flag = words + 1;

    const unsigned warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;  // (the shuffle: known to be the same in the warp)
    const unsigned rank = ptx::cluster_ctarank();
    const unsigned pair = blockIdx.x / 2, pairs = gridDim.x / 2;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            ptx::mbar_init(full_bar(s), 1);   // the first CTA's producer announces the bytes of both CTAs
            ptx::mbar_init(empty_bar(s), 1);  // the commit of the pair's MMAs, delivered to both CTAs
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(acc_full_bar(a), 1);
            ptx::mbar_init(acc_empty_bar(a), 2 * kEpilogueWarps);  // the epilogue warps of both CTAs (used in the first CTA only)
        }
        words[1] = 0;
        ptx::fence_barrier_init();
        ptx::tma_prefetch_descriptor(&map_x);
        ptx::tma_prefetch_descriptor(&map_w);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair(ptx::smem_addr(words), 512);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();  // the partner's barriers exist before anything signals them
    ptx::tc_fence_after_sync();
    const uint32_t tmem_base = __shfl_sync(0xFFFFFFFFu, words[0], 0);
    ptx::grid_launch_dependents();
    // Static weights: the first tiles of W are requested before the kernel before this one has finished.
    const uint32_t full0 = ptx::map_to_cta(full_bar(0), 0);  // a step's bytes are counted in the first CTA
    const unsigned early = p.early_w != 0 ? min(p.stages, p.k_iters) : 0u;
    if (warp == 0 && early != 0) {
        const bool one = elect_one();
        const int row_w = static_cast<int>(pair / p.t_tiles * 256 + rank * kRows);
        for (unsigned i = 0; i < early; ++i) {
            if (one) {
                if (rank == 0) ptx::mbar_arrive_expect_tx(full_bar(i), 2 * stage_bytes);
                ptx::tma_load_2d_pair(base + i * stage_bytes, &map_w, full0 + 8u * i, static_cast<int>(i * kBK), row_w);
            }
        }
        __syncwarp();
    }
    ptx::grid_dependency_wait();

    // tile = weight tile * t_tiles + token tile, dealt round-robin: the pairs of a wave share few weight tiles and most of X, which the L2 holds
    if (warp == 0) {
        const bool one = elect_one();
        int stage = 0;
        unsigned phase = 0, issued = 0;
        bool ok = true;
        for (unsigned tile = pair; ok && tile < p.tiles; tile += pairs) {
            const int row_w = static_cast<int>(tile / p.t_tiles * 256 + rank * kRows);
            const int row_x = static_cast<int>(tile % p.t_tiles * bt + rank * (bt / 2));
            for (unsigned i = 0; i < p.k_iters; ++i, ++issued) {
                const bool begun = issued < early;
                if (!begun && !wait_warp(empty_bar(stage), phase ^ 1u, abort_flag, p.status, kStatusProducerEmpty)) {
                    ok = false;
                    break;
                }
                const uint32_t dst = base + stage * stage_bytes, bar = full_bar(stage), full_first = full0 + 8u * stage;
                if (one) {
                    if (!begun) {
                        if (rank == 0) ptx::mbar_arrive_expect_tx(bar, 2 * stage_bytes);
                        ptx::tma_load_2d_pair(dst, &map_w, full_first, static_cast<int>(i * kBK), row_w);
                    }
                    ptx::tma_load_2d_pair(dst + kWBytes, &map_x, full_first, static_cast<int>(i * kBK), row_x);
                }
                __syncwarp();
                if (++stage == stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        if (!ok) grace_for_copies_in_flight();
    } else if (warp == 1) {
        if (rank == 0) {
            const bool one = elect_one();
            const uint32_t idesc = ptx::instr_desc_s8_s32acc(256, bt);
            const uint64_t dw0 = ptx::smem_desc_k_major_sw128(base), dx0 = ptx::smem_desc_k_major_sw128(base + kWBytes);
            const uint32_t step16 = stage_bytes >> 4;
            int stage = 0, acc = 0;
            unsigned phase = 0, acc_phase = 0;
            bool ok = true;
            for (unsigned tile = pair; ok && tile < p.tiles; tile += pairs) {
                if (!wait_warp(acc_empty_bar(acc), acc_phase ^ 1u, abort_flag, p.status, kStatusMmaAccEmpty)) break;
                ptx::tc_fence_after_sync();
                const uint32_t d = tmem_base + static_cast<uint32_t>(acc) * kAccStride;
                for (unsigned i = 0; i < p.k_iters; ++i) {
                    if (!wait_warp(full_bar(stage), phase, abort_flag, p.status, kStatusMmaFull)) {
                        ok = false;
                        break;
                    }
                    ptx::tc_fence_after_sync();
                    const uint64_t dw = dw0 + stage * step16, dx = dx0 + stage * step16;
                    if (one) {
#pragma unroll
                        for (unsigned j = 0; j < 4; ++j) ptx::mma_i8_ss_pair(d, dw + 2 * j, dx + 2 * j, idesc, i + j);
                        ptx::mma_commit_pair(empty_bar(stage), 3);
                    }
                    __syncwarp();
                    if (++stage == stages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (ok && one) ptx::mma_commit_pair(acc_full_bar(acc), 3);
                __syncwarp();
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
        }
    } else {
        const unsigned worker = warp - 2, quarter = warp % 4, turn = worker / 4;
        uint8_t* const boxes = smem + box_off + worker * 2 * kBoxBytes;
        const uint32_t boxes_addr = base + box_off + worker * 2 * kBoxBytes;
        float* const my_sx = reinterpret_cast<float*>(tail + worker * 128);
        const bool gated = p.epilogue == 2, add = p.epilogue == 1;
        const unsigned n_out = gated ? p.n / 2 : p.n;
        const unsigned meet = 1 + (quarter & 1u) + 2 * turn;  // the barrier that warps q and q + 2 of a turn meet at
        // worker -> the worker with the other half of its chunk's rows (quarters q and q ^ 2 of the same turn)
        const float* const theirs = reinterpret_cast<const float*>(smem + box_off + (worker ^ 2u) * 2 * kBoxBytes);
        unsigned box = 0, acc_phase = 0;
        int acc = 0;
        for (unsigned tile = pair; tile < p.tiles; tile += pairs) {
            const unsigned row0 = tile / p.t_tiles * 256 + rank * kRows, t0 = tile % p.t_tiles * bt;
            const unsigned n = row0 + quarter * 32 + lane;
            // (plain loads: the kernel before this one, which may have left the scales, can still run when this one starts)
            const float sw = n < p.n ? p.sw[n] : 0.0f;
            float sx[4];
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) {
                const unsigned token = t0 + 64 * i + 32 * turn + lane;
                sx[i] = 64 * i + 32 * turn < bt && token < p.m ? p.sx[token] : 0.0f;
            }
            bool go = wait_barrier(acc_full_bar(acc), acc_phase, abort_flag, p.status, kStatusEpilogueAccFull);
            go = __all_sync(0xFFFFFFFFu, go) && *abort_flag == 0;
            go = gated ? both_agree(meet, go) : __all_sync(0xFFFFFFFFu, go) != 0;
            if (!go) break;
            ptx::tc_fence_after_sync();
            const uint32_t taddr = tmem_base + ((quarter * 32u) << 16) + static_cast<uint32_t>(acc) * kAccStride;
#pragma unroll
            for (unsigned i = 0; i < 4; ++i) {
                const unsigned c = 64 * i + 32 * turn;
                if (c >= bt || t0 + c >= p.m) break;
                uint32_t raw[32];
                ptx::tmem_ld_32x32(taddr + c, raw);
                __syncwarp();  // the scales of the chunk before have been read
                my_sx[lane] = sx[i];
                __syncwarp();
                ptx::tmem_ld_wait();
                float v[32];
#pragma unroll
                for (unsigned j = 0; j < 32; j += 4) {
                    const float4 s = *reinterpret_cast<const float4*>(my_sx + j);
                    v[j] = scaled(static_cast<int>(raw[j]), s.x, sw), v[j + 1] = scaled(static_cast<int>(raw[j + 1]), s.y, sw);
                    v[j + 2] = scaled(static_cast<int>(raw[j + 2]), s.z, sw), v[j + 3] = scaled(static_cast<int>(raw[j + 3]), s.w, sw);
                }
                if (gated) {
                    // The CTA's 128 rows are one packed block: gate rows on lanes 0..63, the up rows of the same columns on lanes 64..127. The
                    // gate's warp finishes the chunk's first 16 tokens, the up's the other 16; each hands the other what it lacks.
                    const bool gate = quarter < 2;
                    float* const mine = reinterpret_cast<float*>(boxes);
#pragma unroll
                    for (unsigned j = 0; j < 16; ++j) mine[j * 32 + lane] = v[gate ? 16 + j : j];
                    ptx::named_barrier_sync(meet, 64);
                    const unsigned first = t0 + c + (gate ? 0u : 16u), col0 = row0 / 2 + (quarter & 1u) * 32;
                    float r[16];
#pragma unroll
                    for (unsigned j = 0; j < 16; ++j) {
                        const float other = theirs[j * 32 + lane];
                        r[j] = gate ? swiglu(v[j], other) : swiglu(other, v[16 + j]);
                    }
                    ptx::named_barrier_sync(meet, 64);  // both have read: the boxes may be written again
                    if (p.staged == 0) {
                        store_lane(p, first, col0 + lane, n_out, r);
                    } else {
                        uint8_t* const stage = boxes + kBoxBytes + (p.y_half != 0 ? box * (kBoxBytes / 2) : 0u);
                        if (lane == 0) {  // binary16: two boxes of 1 KB in turn; float32: one of 2 KB
                            if (p.y_half != 0)
                                ptx::bulk_wait_group_read<1>();
                            else
                                ptx::bulk_wait_group_read<0>();
                        }
                        __syncwarp();
                        if (p.y_half != 0) {
#pragma unroll
                            for (unsigned j = 0; j < 16; ++j) reinterpret_cast<__half*>(stage)[j * 32 + lane] = __float2half_rn(r[j]);
                        } else {
#pragma unroll
                            for (unsigned j = 0; j < 16; ++j) reinterpret_cast<float*>(stage)[j * 32 + lane] = r[j];
                        }
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            if (col0 < n_out && first < p.m) ptx::tma_store_2d(&map_y, ptx::smem_addr(stage), static_cast<int>(col0), static_cast<int>(first));
                            ptx::bulk_commit_group();
                        }
                        box ^= 1u;
                    }
                } else if (p.staged == 0) {
                    store_lane(p, t0 + c, n, n_out, v);
                } else if (p.y_half != 0) {
                    if (lane == 0) ptx::bulk_wait_group_read<1>();  // the store before last has read its box
                    __syncwarp();
                    __half* const stage = reinterpret_cast<__half*>(boxes + box * kBoxBytes);
#pragma unroll
                    for (unsigned j = 0; j < 32; ++j) stage[j * 32 + lane] = __float2half_rn(v[j]);
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        if (n < p.n) ptx::tma_store_2d(&map_y, boxes_addr + box * kBoxBytes, static_cast<int>(n), static_cast<int>(t0 + c));
                        ptx::bulk_commit_group();
                    }
                    box ^= 1u;
                } else {
#pragma unroll
                    for (unsigned h = 0; h < 2; ++h) {
                        if (lane == 0) ptx::bulk_wait_group_read<1>();
                        __syncwarp();
                        float* const stage = reinterpret_cast<float*>(boxes + h * kBoxBytes);
#pragma unroll
                        for (unsigned j = 0; j < 16; ++j) stage[j * 32 + lane] = v[16 * h + j];
                        ptx::fence_proxy_async_smem();
                        __syncwarp();
                        if (lane == 0) {
                            const unsigned first = t0 + c + 16 * h;
                            if (n < p.n && first < p.m) {
                                if (add)
                                    ptx::tma_reduce_add_2d(&map_y, boxes_addr + h * kBoxBytes, static_cast<int>(n), static_cast<int>(first));
                                else
                                    ptx::tma_store_2d(&map_y, boxes_addr + h * kBoxBytes, static_cast<int>(n), static_cast<int>(first));
                            }
                            ptx::bulk_commit_group();
                        }
                    }
                }
            }
            ptx::tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster(ptx::map_to_cta(acc_empty_bar(acc), 0));
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
        if (p.staged != 0 && lane == 0) ptx::bulk_wait_group_read<0>();  // the boxes outlive the reads of them
        __syncwarp();
    }

    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync();  // neither CTA leaves while the other may still signal its barriers or read its shared memory
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc_pair(tmem_base, 512);
    }
}

// ---- few rows -----------------------------------------------------------------------------------------------------------------------
//
//   warp 0      TMA producer: per step a [128 x 128] byte box of W and the X box, [n_tok x 128]
//   warp 1      MMA issuer (M 128, N up to 256, K 32); a slot is committed back only where it is loaded again
//   warps 2..9  epilogue: the sums into shared memory, [token][row of W]; behind the cluster's barrier the parts of a token are added by the
//               CTA whose token it is (token mod split) and leave in rows of 128 consecutive columns.
//
// 2560 weight rows by k 9728 are ten tiles for 74 pairs: one token takes 12.3 us there and 7.4 here, cut in eight. The exchange costs 0.03 us a
// token (64 tokens 9.8 us, 128 tokens 11.5), so that the two are level at about 200 tokens, and at 16 to 64 with a shorter k or more rows.
constexpr unsigned kFewThreads = 320;
constexpr unsigned kFewBarriers = 2 * kMaxStages + 1;
constexpr unsigned kFewTail = kFewBarriers * 8 + 64;
constexpr unsigned kSmemHalf = 112 * 1024;    // two CTAs to an SM, with what the system takes of its 228 KB

// One token's four (SwiGLU: two) consecutive results of a lane.
template <int V>
__device__ __forceinline__ void store_results(const S8Params& p, unsigned token, unsigned col, unsigned n_out, const float (&v)[V]) {
    const bool add = p.epilogue == 1;
    const size_t at = static_cast<size_t>(token) * p.ld_y + col;
    if (p.vec_ok != 0 && col + V <= n_out) {
        if (p.y_half != 0) {
            __half2* out = reinterpret_cast<__half2*>(static_cast<__half*>(p.y) + at);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                float a = v[2 * i], b = v[2 * i + 1];
                if (add) {
                    const float2 old = __half22float2(out[i]);
                    a = __fadd_rn(old.x, a), b = __fadd_rn(old.y, b);
                }
                out[i] = __floats2half2_rn(a, b);
            }
        } else {
            float2* out = reinterpret_cast<float2*>(static_cast<float*>(p.y) + at);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                float2 r = make_float2(v[2 * i], v[2 * i + 1]);
                if (add) {
                    const float2 old = out[i];
                    r = make_float2(__fadd_rn(old.x, r.x), __fadd_rn(old.y, r.y));
                }
                out[i] = r;
            }
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if (col + i >= n_out) break;
        if (p.y_half != 0) {
            __half* out = static_cast<__half*>(p.y) + at + i;
            *out = __float2half_rn(add ? __fadd_rn(__half2float(*out), v[i]) : v[i]);
        } else {
            float* out = static_cast<float*>(p.y) + at + i;
            *out = add ? __fadd_rn(*out, v[i]) : v[i];
        }
    }
}

__global__ void __launch_bounds__(kFewThreads, 2)
gemm_s8_few_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const S8Params p) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = ptx::smem_addr(smem_raw);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* const smem = smem_raw + (base - raw_addr);
    const unsigned n_tok = p.bt, stage_bytes = kWBytes + n_tok * kBK;
    const int stages = static_cast<int>(p.stages);
    uint8_t* const tail = smem + p.stages * stage_bytes;  // layout: ring (a CTA's sums take its place at the end) | barriers
    const uint32_t bars = ptx::smem_addr(tail);
    const auto full_bar = [&](int s) { return bars + 8u * s; };
    const auto empty_bar = [&](int s) { return bars + 8u * (kMaxStages + s); };
    const uint32_t acc_bar = bars + 8u * (kFewBarriers - 1);
    unsigned* const words = reinterpret_cast<unsigned*>(tail + kFewBarriers * 8);
    volatile unsigned* const abort_flag = words + 1;

    const unsigned warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;
    const unsigned rank = blockIdx.x % p.split, row0 = blockIdx.x / p.split * kRows;
    const int k0 = static_cast<int>(p.k_iters * rank / p.split), k1 = static_cast<int>(p.k_iters * (rank + 1) / p.split);
    const int iters = k1 - k0;

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        ptx::mbar_init(acc_bar, 1);
        words[1] = 0;
        ptx::fence_barrier_init();
        ptx::tma_prefetch_descriptor(&map_x);
        ptx::tma_prefetch_descriptor(&map_w);
    }
    if (warp == 1) {
        ptx::tmem_alloc(ptx::smem_addr(words), p.tmem_cols);
        ptx::tmem_relinquish();
    }
    ptx::tc_fence_before_sync();
    __syncthreads();
    ptx::tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xFFFFFFFFu, words[0], 0);
    ptx::grid_launch_dependents();

    const auto load_w = [&](int i, int s) {
        ptx::mbar_arrive_expect_tx(full_bar(s), stage_bytes);
        ptx::tma_load_2d(base + s * stage_bytes, &map_w, full_bar(s), (k0 + i) * static_cast<int>(kBK), static_cast<int>(row0));
    };
    const int early = p.early_w != 0 ? min(stages, iters) : 0;
    if (warp == 0) {
        const bool one = elect_one();
        for (int i = 0; i < early; ++i) {
            if (one) load_w(i, i);
        }
        __syncwarp();
    }
    ptx::grid_dependency_wait();

    if (warp == 0) {
        const bool one = elect_one();
        int s = 0;
        unsigned phase = 1;
        for (int i = 0; i < iters; ++i) {
            if (i >= stages && !wait_warp(empty_bar(s), phase, abort_flag, p.status, kStatusProducerEmpty)) {
                grace_for_copies_in_flight();
                break;
            }
            if (one) {
                if (i >= early) load_w(i, s);
                ptx::tma_load_2d(base + s * stage_bytes + kWBytes, &map_x, full_bar(s), (k0 + i) * static_cast<int>(kBK), 0);
            }
            __syncwarp();
            if (++s == stages) s = 0, phase ^= 1u;
        }
    } else if (warp == 1) {
        const bool one = elect_one();
        const uint32_t idesc = ptx::instr_desc_s8_s32acc(kRows, n_tok);
        const uint64_t dw0 = ptx::smem_desc_k_major_sw128(base), dx0 = ptx::smem_desc_k_major_sw128(base + kWBytes);
        const uint32_t step16 = stage_bytes >> 4;
        int s = 0;
        unsigned phase = 0;
        bool ok = true;
        for (int i = 0; i < iters; ++i) {
            if (!wait_warp(full_bar(s), phase, abort_flag, p.status, kStatusMmaFull)) {
                ok = false;
                break;
            }
            ptx::tc_fence_after_sync();
            const uint64_t dw = dw0 + s * step16, dx = dx0 + s * step16;
            if (one) {
#pragma unroll
                for (unsigned j = 0; j < 4; ++j) ptx::mma_i8_ss(tmem, dw + 2 * j, dx + 2 * j, idesc, i + j);
                if (i + stages < iters) ptx::mma_commit(empty_bar(s));
            }
            __syncwarp();
            if (++s == stages) s = 0, phase ^= 1u;
        }
        if (ok && one) ptx::mma_commit(acc_bar);
        __syncwarp();
    } else {
        const unsigned quarter = warp % 4, turn = (warp - 2) / 4;
        const bool arrived = wait_barrier(acc_bar, 0, abort_flag, p.status, kStatusEpilogueAccFull);
        if (__all_sync(0xFFFFFFFFu, arrived)) {
            ptx::tc_fence_after_sync();
            unsigned* const mine = reinterpret_cast<unsigned*>(smem) + quarter * 32 + lane;  // the ring is idle once the last MMA has drained
            for (unsigned c = 16 * turn; c < p.m; c += 32) {
                uint32_t v[16];
                ptx::tmem_ld_32x16(tmem + ((quarter * 32u) << 16) + c, v);
                ptx::tmem_ld_wait();
#pragma unroll
                for (unsigned j = 0; j < 16; ++j) mine[(c + j) * kRows] = v[j];
            }
            ptx::tc_fence_before_sync();
        }
    }
    __syncwarp();
    ptx::cluster_sync();  // every part of the cluster's sums is in its CTA's shared memory
    if (warp >= 2 && *abort_flag == 0) {
        const unsigned worker = warp - 2;
        const bool gated = p.epilogue == 2;
        const unsigned n_out = gated ? p.n / 2 : p.n;
        // plain: lane l has columns 4 l .. 4 l + 3 of the tile; SwiGLU: gate rows 2 l, 2 l + 1 and the up rows 64 further on
        const unsigned at = gated ? 2 * lane : 4 * lane;
        const unsigned col = gated ? row0 / 2 + at : row0 + at;
        float sw[4];
#pragma unroll
        for (unsigned i = 0; i < 4; ++i) {
            const unsigned n = row0 + (gated ? at + i % 2 + (i / 2) * 64 : at + i);
            sw[i] = n < p.n ? p.sw[n] : 0.0f;
        }
        for (unsigned token = rank + p.split * worker; token < p.m; token += kEpilogueWarps * p.split) {
            const float sx = p.sx[token];
            const uint32_t here = base + token * (kRows * 4) + at * 4;
            int4 part[8];
#pragma unroll
            for (unsigned r = 0; r < 8; ++r) {
                part[r] = make_int4(0, 0, 0, 0);
                if (r < p.split) {
                    const uint32_t there = ptx::map_to_cta(here, r);
                    if (gated) {
                        const float2 g = ptx::ld_cluster_f32x2(there), u = ptx::ld_cluster_f32x2(there + 256);
                        part[r] = make_int4(__float_as_int(g.x), __float_as_int(g.y), __float_as_int(u.x), __float_as_int(u.y));
                    } else {
                        const float4 f = ptx::ld_cluster_f32x4(there);
                        part[r] = make_int4(__float_as_int(f.x), __float_as_int(f.y), __float_as_int(f.z), __float_as_int(f.w));
                    }
                }
            }
            int4 sum = part[0];
#pragma unroll
            for (unsigned r = 1; r < 8; ++r) sum.x += part[r].x, sum.y += part[r].y, sum.z += part[r].z, sum.w += part[r].w;
            const float v[4] = {scaled(sum.x, sx, sw[0]), scaled(sum.y, sx, sw[1]), scaled(sum.z, sx, sw[2]), scaled(sum.w, sx, sw[3])};
            if (gated) {
                const float r[2] = {swiglu(v[0], v[2]), swiglu(v[1], v[3])};
                store_results(p, token, col, n_out, r);
            } else {
                store_results(p, token, col, n_out, v);
            }
        }
    }
    __syncwarp();
    ptx::cluster_sync();  // nobody reads this CTA's part any more
    if (warp == 1) {
        ptx::tc_fence_after_sync();
        ptx::tmem_dealloc(tmem, p.tmem_cols);
    }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------

void configure(const Context& ctx) {
    static std::atomic<bool> configured[64] = {};  // per device; every writer sets the same attributes
    if (ctx.device < 64 && configured[ctx.device].load(std::memory_order_relaxed)) return;
    check(cudaFuncSetAttribute(gemm_s8_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax), "cudaFuncSetAttribute");
    check(cudaFuncSetAttribute(gemm_s8_few_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax), "cudaFuncSetAttribute");
    if (ctx.device < 64) configured[ctx.device].store(true, std::memory_order_relaxed);
}

CUtensorMap map_of_bytes(const Context& ctx, const std::int8_t* base, std::size_t rows, std::size_t cols, std::size_t ld, unsigned box_rows) {
    return make_tensor_map_2d(ctx, base, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, rows, cols, ld, box_rows, kBK, true);
}

void launch_pair(const Context& ctx, const std::int8_t* x, std::size_t ld_x, const std::int8_t* w, std::size_t ld_w, S8Params p, std::size_t k, unsigned bt,
                 cudaStream_t stream) {
    p.bt = bt;
    p.t_tiles = (p.m + bt - 1) / bt;
    p.tiles = p.t_tiles * ((p.n + 255) / 256);
    const unsigned fixed = 1024 + kEpilogueWarps * 2 * kBoxBytes + kPairTail, stage_bytes = kWBytes + bt / 2 * kBK;
    p.stages = (kSmemMax - fixed) / stage_bytes;
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    // A binary16 residual update is one float32 addition to the old value, rounded once, where the TMA's binary16 addition would round the product
    // first: read and written lane by lane, a column to a lane. That is what such a call costs on pairs: 900 x 2560 x 9728 62 us, 24 added to
    // float32, 22 stored in binary16. (The few-rows kernel adds along rows: 29 x 2560 x 9728 8.5 us, 8.7 to float32.) And a TMA store drops what lies past the matrix in units of 16 bytes
    // only: rows whose length is not a multiple of that would have their next columns overwritten.
    const std::size_t columns = p.epilogue == 2 ? p.n / 2 : p.n;
    p.staged = p.vec_ok != 0 && columns * (p.y_half != 0 ? 2 : 4) % 16 == 0 && !(p.epilogue == 1 && p.y_half != 0) ? 1u : 0u;
    CUtensorMap map_y;
    std::memset(&map_y, 0, sizeof map_y);
    if (p.staged != 0) {
        if (p.y_half != 0)
            map_y = make_tensor_map_2d(ctx, p.y, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, p.m, columns, p.ld_y, p.epilogue == 2 ? 16 : 32, 32, false);
        else
            map_y = make_tensor_map_2d(ctx, p.y, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 4, p.m, columns, p.ld_y, 16, 32, false);
    }
    const CUtensorMap map_x = map_of_bytes(ctx, x, p.m, k, ld_x, bt / 2), map_w = map_of_bytes(ctx, w, p.n, k, ld_w, kRows);
    configure(ctx);
    const unsigned pairs = p.tiles < static_cast<unsigned>(ctx.sm_count) / 2 ? p.tiles : static_cast<unsigned>(ctx.sm_count) / 2;
    launch_kernel(gemm_s8_pair_kernel, dim3(2 * pairs), dim3(kPairThreads), fixed + p.stages * stage_bytes, stream, "gemm_s8_pair_kernel launch", map_x, map_w, map_y, p);
    count_launch();
}

void launch_few(const Context& ctx, const std::int8_t* x, std::size_t ld_x, const std::int8_t* w, std::size_t ld_w, S8Params p, std::size_t k, FewSchedule sched,
                cudaStream_t stream) {
    p.bt = (p.m + 15) / 16 * 16;
    p.split = sched.split < p.k_iters ? sched.split : p.k_iters;
    p.tmem_cols = 32;
    while (p.tmem_cols < p.bt) p.tmem_cols *= 2;  // (up to 256 columns: two CTAs to an SM never wait for one another's)
    const unsigned stage_bytes = kWBytes + p.bt * kBK;
    p.stages = ((sched.slots == 2 ? kSmemHalf : kSmemMax) - 1024 - kFewTail) / stage_bytes;
    if (p.stages > kMaxStages) p.stages = kMaxStages;
    const CUtensorMap map_x = map_of_bytes(ctx, x, p.m, k, ld_x, p.bt), map_w = map_of_bytes(ctx, w, p.n, k, ld_w, kRows);
    configure(ctx);
    const unsigned tiles = (p.n + kRows - 1) / kRows;
    launch_cluster_kernel(gemm_s8_few_kernel, p.split, dim3(tiles * p.split), dim3(kFewThreads), 1024 + p.stages * stage_bytes + kFewTail, stream,
                          "gemm_s8_few_kernel launch", map_x, map_w, p);
    count_launch();
}

// The automatic choice: the kernel, and the pair kernel's tokens to a tile, by an estimate in microseconds fitted to every width and every split
// of k over thirteen projections (1024 to 24576 weight rows, k from 1024 to 12288) at 21 token counts from 1 to 4096 on 148 SMs: what it
// picks is on average 2 % slower than the best of them, on single shapes of a few microseconds up to 33 %. On six products outside that set (2560
// x 9216, 18432 x 2560, 12288 x 2048, 2048 x 6144, 5120 x 5120, 1500 x 2000) at seven counts up to 2048 also 2 %, at worst 18 (300 tokens by 1500
// x 2000; 10 elsewhere). The clock (1900 MHz) and the memory's rate are in it; a binary16 residual update's slower stores are not.
//   - A step of the pair kernel is 2 bt clocks of tensor cores, or 180 + 0.6 bt where the boxes' arrival bounds it (tiles under 128 tokens); a
//     wave of tiles has about 600 clocks of its own (first boxes, the last tile's epilogue).
//   - Cutting k over a cluster costs 0.028 us a token in the exchange of the sums: it wins where a few weight rows have a long k (2560 x 9728, one
//     token: 12.3 us on ten pairs, 7.4 cut in eight; level at about 200 tokens; 24576 x 4096: 18.5 on pairs from one token on).
//   - Neither reads the weights faster than the memory does, about 6.5 TB/s.
struct Choice {
    bool few = false;
    unsigned bt = 32;
    FewSchedule parts;
};
Choice choose(unsigned sm_count, std::size_t t, std::size_t n, std::size_t k) {
    const std::size_t iters = (k + kBK - 1) / kBK, pairs = sm_count / 2;
    const double reading = static_cast<double>(n) * static_cast<double>(k) / 6.5e6;
    Choice c;
    double best = 0.0;
    for (unsigned bt = 32; bt <= 256 && bt < t + 32; bt += 32) {
        const std::size_t tiles = (t + bt - 1) / bt * ((n + 255) / 256), waves = (tiles + pairs - 1) / pairs;
        const double step = 2.0 * bt > 180.0 + 0.6 * bt ? 2.0 * bt : 180.0 + 0.6 * bt;
        const double us = static_cast<double>(waves) * (static_cast<double>(iters) * step + 600.0) / 1900.0;
        if (best == 0.0 || us <= best) best = us, c.bt = bt;
    }
    if (t > kFewMaxRows) return c;
    // up to 32 tokens two CTAs to an SM, above one, whose ring is deeper (2560 x 9728, 64 tokens: 10.9 and 9.8 us)
    const FewSchedule parts = few_schedule(sm_count, t <= 32 ? t : 129, n, k, true);
    const std::size_t ctas = (n + kRows - 1) / kRows * parts.split, room = static_cast<std::size_t>(sm_count) * parts.slots;
    const double cut = 0.11 * static_cast<double>((ctas + room - 1) / room) * static_cast<double>((iters + parts.split - 1) / parts.split);
    if (3.2 + (cut > reading ? cut : reading) + 0.028 * static_cast<double>(t) < 3.6 + (best > reading ? best : reading)) {
        c.few = true;
        c.parts = parts;
    }
    return c;
}

}  // namespace

void launch_gemm_s8(Context& ctx, const std::int8_t* x, std::size_t ld_x, const float* sx, const std::int8_t* w, std::size_t ld_w, const float* sw, void* y,
                    std::size_t ld_y, bool y_half, std::size_t t, std::size_t n, std::size_t k, Epilogue epilogue, int config, cudaStream_t stream) {
    const bool gated = epilogue == Epilogue::SwiGLU;
    if (n == 0 || k == 0 || k > kS8MaxK || ld_x % 16 != 0 || ld_w % 16 != 0 || ld_x < k || ld_w < k || ld_y < (gated ? n / 2 : n) || (gated && n % 128 != 0))
        throw std::invalid_argument("launch_gemm_s8: unsupported shape [" + std::to_string(t) + " x " + std::to_string(k) + "] by [" + std::to_string(n) + " x " +
                                    std::to_string(k) + "] (K from 1 to 131071, the strides of X and W multiples of 16 that hold a row, that of Y one that "
                                    "holds a row, SwiGLU needs N a multiple of 128)");
    if (t > 0x7FFFFFFFu || n > 0x7FFFFFFFu) throw std::invalid_argument("launch_gemm_s8: dimension beyond 2^31");
    const bool few = config >= kFewConfig, pair = config >= 512 && !few;
    const int parts = few ? (config - kFewConfig) % 16 : 1, slots = few && config - kFewConfig >= 16 ? 1 : 2;
    if (config < -1 || (config >= 0 && config < 512) || (pair && (config - 512 < 32 || config - 512 > 256 || (config - 512) % 32 != 0)) ||
        (few && (config - kFewConfig >= 32 || parts < 1 || parts > 8)))
        throw std::invalid_argument("launch_gemm_s8: config is -1, 512 + w (w tokens to a tile: a multiple of 32 up to 256) or 1024 + s, 1024 + 16 + s (s parts "
                                    "of k, 1 to 8)");
    if (few && t > (slots == 2 ? 128u : kFewMaxRows))
        throw std::invalid_argument("launch_gemm_s8: the few-rows kernel takes up to 256 rows (two CTAs to an SM: 128)");
    if (t == 0) return;
    if (x == nullptr || w == nullptr || sx == nullptr || sw == nullptr || y == nullptr) throw std::invalid_argument("launch_gemm_s8: null pointer");
    if (reinterpret_cast<std::uintptr_t>(x) % 16 != 0 || reinterpret_cast<std::uintptr_t>(w) % 16 != 0)
        throw std::invalid_argument("launch_gemm_s8: X and W must be 16-byte aligned");
    if (reinterpret_cast<std::uintptr_t>(sx) % 4 != 0 || reinterpret_cast<std::uintptr_t>(sw) % 4 != 0 || reinterpret_cast<std::uintptr_t>(y) % (y_half ? 2 : 4) != 0)
        throw std::invalid_argument("launch_gemm_s8: a pointer is not aligned to its values");
    const std::size_t pair_tiles_at_most = (t + 31) / 32 * ((n + 255) / 256);
    if (pair_tiles_at_most > 0x7FFFFFFFu) throw std::invalid_argument("launch_gemm_s8: too many output tiles for one call");
    check(cudaSetDevice(ctx.device), "cudaSetDevice");
    S8Params p{};
    p.y = y;
    p.ld_y = ld_y;
    p.sx = sx;
    p.sw = sw;
    p.status = ctx.status;
    p.m = static_cast<unsigned>(t);
    p.n = static_cast<unsigned>(n);
    p.k_iters = static_cast<unsigned>((k + kBK - 1) / kBK);
    p.epilogue = static_cast<unsigned>(epilogue);
    p.y_half = y_half ? 1u : 0u;
    p.vec_ok = reinterpret_cast<std::uintptr_t>(y) % 16 == 0 && ld_y * (y_half ? 2 : 4) % 16 == 0 ? 1u : 0u;
    p.early_w = ctx.static_weights ? 1u : 0u;
    Choice c;
    if (config == -1) {
        c = choose(static_cast<unsigned>(ctx.sm_count), t, n, k);
    } else {
        c.few = few;
        c.bt = static_cast<unsigned>(config - 512);
        c.parts.split = static_cast<unsigned>(parts);
        c.parts.slots = static_cast<unsigned>(slots);
    }
    if (c.few)
        launch_few(ctx, x, ld_x, w, ld_w, p, k, c.parts, stream);
    else
        launch_pair(ctx, x, ld_x, w, ld_w, p, k, c.bt, stream);
}

}  // namespace sepal::b200
