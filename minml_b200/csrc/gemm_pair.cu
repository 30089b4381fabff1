/*
 * gemm_pair.cu -- fp16 matrix products on pairs of SMs, with the next step of the feed-forward and loss operators in the epilogue.
 *
 * One cluster of two CTAs computes 256 x 256 tiles with tcgen05.mma cta_group::2: each CTA holds 128 rows of A, half of the B tile and,
 * in tensor memory, the 128 accumulator rows of its own A half.  Against a 128 x 256 tile on one SM this halves the bytes of B that a
 * tile's multiplications need, which is what lets the copies into shared memory keep up with the tensor core.  Persistent: a
 * cluster walks over tiles (and, where a product is cut along K, over K ranges), two accumulator buffers let the epilogue of one tile
 * run under the multiplications of the next.
 *   warp 0      fetches this CTA's A and B boxes by TMA into a ring of stages of 64 K indices (128-byte rows, 128-byte swizzle)
 *   warp 1      in the even CTA: issues the multiplications; owns the tensor-memory allocation
 *   warps 4-11  epilogue: two warps per tensor-memory lane quarter, each half of the columns
 * An operand stored [K, rows] is fetched in boxes of 64 K indices x 64 rows and read as an MN-major operand.
 * K and row tails are zero-filled by TMA, results are clipped by their tensor maps.
 *
 * The tensor core cuts its fp32 sums where an fp32 addition would round: measured, 1.6e-8 of the sum for every 16 K indices, always toward
 * zero (4.2e-6 at K = 4096); where all terms have one sign 1e-7 (2.7e-5 at K = 4096, 1.7e-3 at 262 144).  A loss is kept in fp32, and where a
 * row is certain P - 1 is the difference of two numbers near 1, so both epilogues of logits add up accumulators of 1024 K indices each in
 * registers, in the same order: the gradient's logits are those that lse was made from, bit for bit.  Products that leave a plain result, among
 * them all weight gradients, whose K is the number of tokens, add up accumulators of 8192 (5.3e-5, a ninth of the rounding to fp16).  Only the
 * gated products, whose K is embed, take one accumulator for all of it.
 */
#include "common.cuh"
#include "tc.cuh"
#include "epilogue.cuh"
#include "gate.cuh"
#include "operands.cuh"
#include "gemm_pair.cuh"

#include <algorithm>
#include <cstring>
#include <mutex>

namespace mb200
{
	namespace
	{
		using namespace tc;
		using namespace epi;

		constexpr int BM = 128; // rows of A per CTA
		constexpr int BN = 256; // columns of a tile
		constexpr int BK = 64; // K indices per stage: 128 bytes
		constexpr int OPERAND_BYTES = 128 * 128; // one CTA's 128 rows (A) or columns (B) of a stage
		constexpr int STAGE_BYTES = 2 * OPERAND_BYTES;
		constexpr int EPI_WARPS = 8;
		constexpr int EPI_FIRST = 4; // first epilogue warp: registers are moved between groups of four warps
		constexpr int THREADS = (EPI_FIRST + EPI_WARPS) * 32;
		// of the 168 registers a thread starts with, what the first four warps give up is what the epilogue gets: 128 * 40 + 256 * 232 = 384 * 168
		constexpr int REGISTERS_FEW = 40, REGISTERS_MANY = 232;
		constexpr int HALF_BOX = 32 * 64, FLOAT_BOX = 32 * 128;
		constexpr int LOGITS_SEGMENT = 1024 / BK, RESULTS_SEGMENT = 8192 / BK; // K blocks per accumulator of a logit, and of a result rounded to fp16
		constexpr int ROW_GROUP = 8; // tiles of 256 rows that neighbouring clusters share their columns over

		enum Epilogue
		{
			STORE, // fp16 result
			SUMS, // fp32 sums, stored or added
			GATED,
			GATED_BACKWARD, // from a kept a and u
			GATED_RECOMPUTE, // the same, with a and u made again in the same tile
			STATISTICS,
			PROBABILITIES
		};

		constexpr int MAX_STAGES = 5;
		template<int EPI>
		struct Shape
		{
				// per epilogue warp: four 32 x 32 boxes of fp16 or two of fp32; GATED_RECOMPUTE: all six boxes of a tile
				static constexpr int staging_bytes = EPI == GATED_RECOMPUTE ? 6 * 2048 : 8192;
				static constexpr int stages = EPI == GATED_RECOMPUTE ? 4 : 5;
				// K blocks per accumulator; the two epilogues of logits have the same one and so the same logits, to the bit
				static constexpr int segment = EPI == STATISTICS || EPI == PROBABILITIES ? LOGITS_SEGMENT : EPI == STORE || EPI == SUMS ? RESULTS_SEGMENT : 1 << 30;
				static constexpr bool sums_segments = segment < 1 << 30;
				static constexpr bool moves_registers = EPI == GATED || EPI == GATED_RECOMPUTE || sums_segments; // they hold 128 accumulators a thread
				static constexpr int smem_bytes = stages * STAGE_BYTES + EPI_WARPS * staging_bytes + 1024;
				static_assert(stages <= MAX_STAGES && smem_bytes <= 227 * 1024, "the configuration exceeds the SM");
		};

		struct Params
		{
				int M, N, K; // N: columns of the result (GATED: of h)
				int a_mn, b_mn;
				int m_tiles, n_tiles, splits, blocks_per_split;
				int up_row; // GATED: row of w1 where the up half begins
				PairResult result; // STORE
				int direct; // STORE: element-wise stores, for results that TMA cannot address
				int accumulate; // SUMS
				int store_h; // GATED_RECOMPUTE
				float *kept; // a and u: written by GATED unless null, read by GATED_BACKWARD
				const int *targets;
				const float *row_weights, *lse;
				int first, vocab;
				float2 *parts;
				int groups;
				float *target_logit;
				int *status;
		};
		struct Barriers
		{
				uint64_t full[MAX_STAGES], empty[MAX_STAGES];
				uint64_t tmem_full[2], tmem_empty[2];
				uint64_t au_empty; // GATED_RECOMPUTE: a and u have been read
				uint32_t tmem_base;
				int abort_flag;
		};

		__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1)
		{
			asm volatile(
					"cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
					:: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1) : "memory");
		}
		__device__ __forceinline__ void tma_reduce_add_3d(const CUtensorMap *map, uint32_t src, int c0, int c1, int c2)
		{
			asm volatile(
					"cp.reduce.async.bulk.tensor.3d.global.shared::cta.add.bulk_group [%0, {%2, %3, %4}], [%1];"
					:: "l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(c0), "r"(c1), "r"(c2) : "memory");
		}
		__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, uint32_t src, int c0, int c1)
		{
			asm volatile(
					"cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
					:: "l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(c0), "r"(c1) : "memory");
		}

		/* The kept a and u: for every 32 rows the a of all columns, then the u; of each, for every four columns, the rows' 16-byte pieces one after the other.
		 * So a warp whose lanes are rows, as an epilogue's are, moves 512 contiguous bytes at a time.  This is the block of (row0, column), whose
		 * columns are multiples of four; the u lie rows * columns floats behind the a. */
		__device__ __forceinline__ float* kept_block(float *kept, const Params &p, int row0, int column)
		{
			return kept + static_cast<long long>(row0) * 2 * p.N + static_cast<long long>(column) * min(32, p.M - row0);
		}


		/* A warp's 32 x 32 boxes in shared memory: a lane owns one row.  fp16: 64-byte rows, 16-byte piece k at k ^ (row / 2 % 4) (64-byte
		 * swizzle); fp32: 128-byte rows, piece k at k ^ (row % 8) (128-byte swizzle). */
		__device__ __forceinline__ void write_half_box(uint32_t box, int lane, const float (&v)[32])
		{
#pragma unroll
			for (int k = 0; k < 4; k++)
				st_shared_v4(box + lane * 64 + ((k ^ ((lane >> 1) & 3)) * 16), pack_half8(v + 8 * k));
		}
		__device__ __forceinline__ void write_float_box(uint32_t box, int lane, const uint32_t (&v)[32])
		{
#pragma unroll
			for (int k = 0; k < 8; k++)
				st_shared_v4(box + lane * 128 + ((k ^ (lane & 7)) * 16), make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]));
		}
		__device__ __forceinline__ void load_chunk(uint32_t taddr, float (&v)[32])
		{
			uint32_t r[32];
			tmem_ld_32x32(taddr, r);
			tmem_wait_ld();
#pragma unroll
			for (int j = 0; j < 32; j++)
				v[j] = __uint_as_float(r[j]);
		}
		template<int EPI, int GATE>
		__global__ void __launch_bounds__(THREADS, 1) kernel_gemm_pair(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
				const __grid_constant__ CUtensorMap map_d, const __grid_constant__ CUtensorMap map_e, const __grid_constant__ CUtensorMap map_f,
				const __grid_constant__ CUtensorMap map_dy, const __grid_constant__ CUtensorMap map_w2, const Params p)
		{
			constexpr int STAGES = Shape<EPI>::stages;
			extern __shared__ uint8_t smem_raw[];
			__shared__ Barriers bars;
			const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
			const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
			const uint32_t rank = cluster_ctarank();
			const bool leader = rank == 0;

			const int tiles = p.m_tiles * p.n_tiles, units = tiles * p.splits;
			const int k_blocks = (p.K + BK - 1) / BK;
			const int first_unit = blockIdx.x / 2, unit_step = gridDim.x / 2;
			struct Unit
			{
					int m0, nt, kb0, kb1, split;
			};
			// Tiles in groups of ROW_GROUP row tiles, row tiles fastest: the clusters at work at one time share a few row and column tiles in L2.
			auto locate = [&](int unit) -> Unit
			{
				Unit u;
				u.split = unit / tiles;
				int rest = unit - u.split * tiles;
				const int group = rest / (ROW_GROUP * p.n_tiles);
				rest -= group * ROW_GROUP * p.n_tiles;
				const int rows = min(ROW_GROUP, p.m_tiles - group * ROW_GROUP);
				u.nt = rest / rows;
				u.m0 = ((group * ROW_GROUP + rest - u.nt * rows) * 2 + static_cast<int>(rank)) * BM;
				u.kb0 = u.split * p.blocks_per_split;
				u.kb1 = min(k_blocks, u.kb0 + p.blocks_per_split);
				return u;
			};
			constexpr int SEGMENT = Shape<EPI>::segment;

			if (threadIdx.x == 0)
			{
				for (int s = 0; s < STAGES; s++)
				{
					mbar_init(smem_u32(&bars.full[s]), 1);
					mbar_init(smem_u32(&bars.empty[s]), 1);
				}
				for (int a = 0; a < 2; a++)
				{
					mbar_init(smem_u32(&bars.tmem_full[a]), 1);
					mbar_init(smem_u32(&bars.tmem_empty[a]), 2 * EPI_WARPS);
				}
				mbar_init(smem_u32(&bars.au_empty), 2 * EPI_WARPS);
				bars.abort_flag = 0;
				fence_mbar_init();
			}
			if (warp == 1)
			{
				asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(&bars.tmem_base)), "r"(2 * BN) : "memory");
				asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
			}
			tcgen05_fence_before();
			cluster_sync(); // the peer's barriers exist before anything signals them
			tcgen05_fence_after();
			const uint32_t tmem_base = bars.tmem_base;
			volatile int *abort_flag = &bars.abort_flag;
			let_next_grid_start();
			wait_for_previous_grid();

			auto give_registers = [&]()
			{
				if (Shape<EPI>::moves_registers)
					asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(REGISTERS_FEW));
			};
			if (warp == 0)
			{ /* ------------------------------------------------ operands */
				give_registers();
				if (elect_one())
				{
					prefetch_tensormap(&map_a);
					prefetch_tensormap(&map_b);
					uint32_t it = 0;
					bool ok = true;
					for (int unit = first_unit; unit < units && ok; unit += unit_step)
					{
						const Unit u = locate(unit);
						const int n0 = EPI == GATED || EPI == GATED_RECOMPUTE ? u.nt * (BN / 2) + (leader ? 0 : p.up_row) : u.nt * BN + static_cast<int>(rank) * (BN / 2);
						if (EPI == GATED_RECOMPUTE)
							for (int kb = u.kb0; kb < u.kb1 && ok; kb++, it++)
							{ // dy and 64 columns of W2
								const int s = it % STAGES;
								if (!mbar_wait(smem_u32(&bars.empty[s]), ((it / STAGES) & 1u) ^ 1u, abort_flag))
								{
									ok = false;
									break;
								}
								const uint32_t full = smem_u32(&bars.full[s]);
								if (leader)
									mbar_arrive_expect_tx(full, 2 * (OPERAND_BYTES + OPERAND_BYTES / 2));
								const uint32_t full_leader = map_to_cta(full, 0);
								tma_load_2d_pair(smem_base + s * STAGE_BYTES, &map_dy, full_leader, kb * BK, u.m0);
								tma_load_2d_pair(smem_base + s * STAGE_BYTES + OPERAND_BYTES, &map_w2, full_leader, u.nt * (BN / 2) + static_cast<int>(rank) * 64, kb * BK);
							}
						for (int kb = u.kb0; kb < u.kb1 && ok; kb++, it++)
						{
							const int s = it % STAGES;
							if (!mbar_wait(smem_u32(&bars.empty[s]), ((it / STAGES) & 1u) ^ 1u, abort_flag))
							{
								ok = false;
								break;
							}
							const uint32_t full = smem_u32(&bars.full[s]);
							if (leader) // both CTAs' boxes are counted on the even one's barrier
								mbar_arrive_expect_tx(full, 2 * STAGE_BYTES);
							const uint32_t full_leader = map_to_cta(full, 0);
							const uint32_t a = smem_base + s * STAGE_BYTES, b = a + OPERAND_BYTES;
							if (p.a_mn)
							{
								tma_load_2d_pair(a, &map_a, full_leader, u.m0, kb * BK);
								tma_load_2d_pair(a + OPERAND_BYTES / 2, &map_a, full_leader, u.m0 + 64, kb * BK);
							}
							else
								tma_load_2d_pair(a, &map_a, full_leader, kb * BK, u.m0);
							if (p.b_mn)
							{
								tma_load_2d_pair(b, &map_b, full_leader, n0, kb * BK);
								tma_load_2d_pair(b + OPERAND_BYTES / 2, &map_b, full_leader, n0 + 64, kb * BK);
							}
							else
								tma_load_2d_pair(b, &map_b, full_leader, kb * BK, n0);
						}
					}
				}
				__syncwarp();
			}
			else if (warp == 1)
			{ /* ------------------------------------------- multiplications */
				give_registers();
				if (leader && elect_one())
				{
					const uint32_t idesc = make_idesc_f16_pair(BN) | (p.a_mn ? (1u << 15) : 0u) | (p.b_mn ? (1u << 16) : 0u);
					// descriptor step per instruction, in 16-byte units: 32 bytes along K, or 16 K indices of 128 bytes each
					const uint32_t step_a = p.a_mn ? 128 : 2, step_b = p.b_mn ? 128 : 2;
					uint32_t it = 0, buffers = 0;
					bool ok = true;
					for (int unit = first_unit; unit < units && ok; unit += unit_step)
					{
						const Unit u = locate(unit);
						if (EPI == GATED_RECOMPUTE)
						{ // dh into columns 256 + 128 i, two buffers; a and u, below, into columns 0 .. 255
							const uint32_t acc = buffers & 1u;
							if (!mbar_wait(smem_u32(&bars.tmem_empty[acc]), ((buffers >> 1) & 1u) ^ 1u, abort_flag))
								break;
							tcgen05_fence_after();
							const uint32_t idesc_dh = make_idesc_f16_pair(BN / 2) | (1u << 16);
							for (int kb = u.kb0; kb < u.kb1; kb++, it++)
							{
								const int s = it % STAGES;
								if (!mbar_wait(smem_u32(&bars.full[s]), (it / STAGES) & 1u, abort_flag))
								{
									ok = false;
									break;
								}
								tcgen05_fence_after();
								const uint32_t a = smem_base + s * STAGE_BYTES;
								const uint64_t desc_a = make_desc_k_sw128(a), desc_b = make_desc_mn_sw128(a + OPERAND_BYTES, OPERAND_BYTES / 2);
#pragma unroll
								for (int k = 0; k < 4; k++)
									mma_ss_pair<0>(tmem_base + BN + acc * (BN / 2), desc_a + 2 * k, desc_b + 128 * k, idesc_dh, kb > u.kb0 || k > 0 ? 1u : 0u);
								mma_commit_pair(smem_u32(&bars.empty[s]));
							}
							if (!ok || !mbar_wait(smem_u32(&bars.au_empty), (buffers & 1u) ^ 1u, abort_flag))
								break;
							tcgen05_fence_after();
						}
						for (int kb = u.kb0; kb < u.kb1 && ok;)
						{ // one accumulator buffer: a whole K range, or a segment of it
							const int end = min(u.kb1, kb + SEGMENT);
							const uint32_t acc = buffers & 1u;
							if (EPI != GATED_RECOMPUTE)
							{
								if (!mbar_wait(smem_u32(&bars.tmem_empty[acc]), ((buffers >> 1) & 1u) ^ 1u, abort_flag))
								{
									ok = false;
									break;
								}
								tcgen05_fence_after();
							}
							const uint32_t d = tmem_base + (EPI == GATED_RECOMPUTE ? 0 : acc * BN);
							uint32_t accumulate = 0;
							for (; kb < end; kb++, it++)
							{
								const int s = it % STAGES;
								if (!mbar_wait(smem_u32(&bars.full[s]), (it / STAGES) & 1u, abort_flag))
								{
									ok = false;
									break;
								}
								tcgen05_fence_after();
								const uint32_t a = smem_base + s * STAGE_BYTES, b = a + OPERAND_BYTES;
								const uint64_t desc_a = p.a_mn ? make_desc_mn_sw128(a, OPERAND_BYTES / 2) : make_desc_k_sw128(a);
								const uint64_t desc_b = p.b_mn ? make_desc_mn_sw128(b, OPERAND_BYTES / 2) : make_desc_k_sw128(b);
#pragma unroll
								for (int k = 0; k < 4; k++)
								{
									mma_ss_pair<0>(d, desc_a + step_a * k, desc_b + step_b * k, idesc, accumulate);
									accumulate = 1;
								}
								mma_commit_pair(smem_u32(&bars.empty[s])); // frees the stage in both CTAs
							}
							if (ok)
								mma_commit_pair(smem_u32(&bars.tmem_full[acc]));
							buffers++;
						}
					}
				}
				__syncwarp();
			}
			else if (warp < EPI_FIRST)
				give_registers();
			else
			{ /* ------------------------------------------------------------ epilogue */
				if (Shape<EPI>::moves_registers)
					asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(REGISTERS_MANY));
				const int e = warp - EPI_FIRST, q = warp % 4, half = e / 4;
				const uint32_t staging = smem_base + STAGES * STAGE_BYTES + e * Shape<EPI>::staging_bytes;
				const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
				uint32_t buffers = 0, boxes = 0;
				bool ok = true;
				auto wait_full = [&]() -> bool
				{
					if (!mbar_wait_warp(smem_u32(&bars.tmem_full[buffers & 1u]), (buffers >> 1) & 1u, abort_flag, 20u))
						return false;
					tcgen05_fence_after();
					return true;
				};
				auto release = [&]()
				{ // every load from this accumulator buffer has returned
					tcgen05_fence_before();
					__syncwarp();
					if (lane == 0)
						arrive_at_leader(smem_u32(&bars.tmem_empty[buffers & 1u]));
					buffers++;
				};
				auto publish = [&]()
				{ // plain stores to a box, before the copy engine reads it
					fence_proxy_async_smem();
					__syncwarp();
				};
				auto sum_segments = [&](const Unit &u, float (&v)[BN / 2]) -> bool
				{ // this lane's 128 columns of its row
					for (int kb = u.kb0; kb < u.kb1; kb += SEGMENT)
					{
						if (!wait_full())
							return false;
						const uint32_t taddr = lane_base + (buffers & 1u) * BN + half * (BN / 2);
#pragma unroll
						for (int c = 0; c < BN / 64; c++)
						{
							uint32_t r[32];
							tmem_ld_32x32(taddr + c * 32, r);
							tmem_wait_ld();
#pragma unroll
							for (int j = 0; j < 32; j++)
								v[c * 32 + j] = (kb == u.kb0 ? 0.0f : v[c * 32 + j]) + __uint_as_float(r[j]);
						}
						release();
					}
					return true;
				};
				for (int unit = first_unit; unit < units && ok; unit += unit_step)
				{
					const Unit u = locate(unit);
					const int row0 = u.m0 + q * 32, row = row0 + lane;
					const bool row_ok = row < p.M;

					if constexpr (EPI == STATISTICS)
					{
						float v[BN / 2];
						ok = sum_segments(u, v);
						if (!ok)
							break;
						const int n0 = u.nt * BN + half * (BN / 2), valid = p.N - n0;
						const int wanted = row_ok ? p.targets[row] : -1, at = wanted >= n0 ? wanted - n0 : -1;
						float top = -INFINITY, sum = 0.0f, target = 0.0f;
#pragma unroll
						for (int j = 0; j < BN / 2; j++)
						{
							if (j < valid)
								top = fmaxf(top, v[j]);
							if (j == at)
								target = v[j];
						}
						const float shift = top == -INFINITY ? 0.0f : top * LOG2E; // nothing but -inf: all terms are zero
#pragma unroll
						for (int j = 0; j < BN / 2; j++)
							sum += j < valid ? exp2_approx(fmaf(v[j], LOG2E, -shift)) : 0.0f;
						if (row_ok && valid > 0)
						{
							p.parts[static_cast<long long>(row) * p.groups + u.nt * 2 + half] = make_float2(top, sum);
							if (at >= 0 && at < min(BN / 2, valid))
								p.target_logit[row] = target;
						}
						continue;
					}

					if constexpr (EPI == PROBABILITIES)
					{
						// what the row needs, read under the multiplications
						int target = row_ok ? p.targets[row] : -1;
						const bool active = target >= 0 && target < p.vocab && (p.row_weights == nullptr || p.row_weights[row] != 0.0f);
						const float shift = row_ok ? fmaf(p.lse[row], -LOG2E, 15.0f) : 0.0f; // 2^15 exp(z - lse) = 2^(z log2 e + shift)
						target = active ? target - p.first : -1;
						float v[BN / 2];
						ok = sum_segments(u, v);
						if (!ok)
							break;
#pragma unroll
						for (int c = 0; c < BN / 64; c++)
						{
							const int n = u.nt * BN + half * (BN / 2) + c * 32;
							if (n >= p.N)
								break;
							float x[32];
#pragma unroll
							for (int j = 0; j < 32; j++)
							{
								const float e = exp2_approx(fmaf(v[c * 32 + j], LOG2E, shift)) - (target == n + j ? 32768.0f : 0.0f);
								x[j] = active ? e : 0.0f;
							}
							if (lane == 0)
								bulk_wait_group_read<3>();
							__syncwarp();
							const uint32_t box = staging + (boxes++ % 4) * HALF_BOX;
							write_half_box(box, lane, x);
							publish();
							if (lane == 0 && row0 < p.M)
							{
								tma_store_2d(&map_d, box, n, row0);
								bulk_commit_group();
							}
						}
						continue;
					}

					if constexpr (EPI == SUMS || EPI == STORE)
					{
						float scale = 1.0f;
						bool active = true; // read under the multiplications
						if (EPI == STORE)
						{
							scale = p.result.alpha * (p.result.alpha_device != nullptr ? *p.result.alpha_device : 1.0f);
							if (p.result.row_scale != nullptr)
								scale *= row_ok ? p.result.row_scale[row] : 0.0f;
							active = p.result.row_scale == nullptr || (row_ok && p.result.row_scale[row] != 0.0f);
						}
						float all[BN / 2];
						ok = sum_segments(u, all);
						if (!ok)
							break;
#pragma unroll
						for (int c = 0; c < BN / 64; c++)
						{
							const int n = u.nt * BN + half * (BN / 2) + c * 32;
							if (n >= p.N)
								break;
							if (EPI == SUMS)
							{
								if (lane == 0)
									bulk_wait_group_read<1>();
								__syncwarp();
								const uint32_t box = staging + (boxes++ % 2) * FLOAT_BOX;
								uint32_t raw[32];
#pragma unroll
								for (int j = 0; j < 32; j++)
									raw[j] = __float_as_uint(all[c * 32 + j]);
								write_float_box(box, lane, raw);
								publish();
								if (lane == 0 && row0 < p.M)
								{
									if (p.accumulate)
										tma_reduce_add_3d(&map_d, box, n, row0, u.split);
									else
										tma_store_3d(&map_d, box, n, row0, u.split);
									bulk_commit_group();
								}
								continue;
							}
							float v[32];
#pragma unroll
							for (int j = 0; j < 32; j++)
								v[j] = active ? all[c * 32 + j] * scale : 0.0f;
							__half *dst = p.result.d + static_cast<long long>(row) * p.result.ldd + n;
							if (p.result.beta != 0.0f && row_ok)
							{
								if (!p.direct && n + 32 <= p.N)
								{
#pragma unroll
									for (int k = 0; k < 4; k++)
										add_half8(v + 8 * k, reinterpret_cast<const uint4*>(dst)[k], p.result.beta);
								}
								else
								{
#pragma unroll
									for (int j = 0; j < 32; j++)
										if (n + j < p.N)
											v[j] += p.result.beta * __half2float(dst[j]);
								}
							}
							if (p.direct)
							{ // rows that TMA cannot address: through a box, so that a store instruction covers 64 bytes of one row instead of 2 bytes of 32
								write_half_box(staging, lane, v);
								__syncwarp();
								const int rows = min(32, p.M - row0);
								if (n + lane < p.N)
									for (int r = 0; r < rows; r++)
									{
										uint16_t bits;
										asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(staging + r * 64 + (((lane / 8) ^ ((r >> 1) & 3)) * 16) + lane % 8 * 2) : "memory");
										*reinterpret_cast<uint16_t*>(p.result.d + static_cast<long long>(row0 + r) * p.result.ldd + n + lane) = bits;
									}
								__syncwarp();
								continue;
							}
							if (lane == 0)
								bulk_wait_group_read<3>();
							__syncwarp();
							const uint32_t box = staging + (boxes++ % 4) * HALF_BOX;
							write_half_box(box, lane, v);
							publish();
							if (lane == 0 && row0 < p.M)
							{
								tma_store_2d(&map_d, box, n, row0);
								bulk_commit_group();
							}
						}
						continue;
					}

					if (!wait_full())
						break;
					const uint32_t taddr = lane_base + (buffers & 1u) * BN;

					if (EPI == GATED)
					{
						const int n0 = u.nt * (BN / 2) + half * 64;
						const uint32_t box = staging + (boxes++ % 2) * 2 * HALF_BOX; // h of 64 columns: two boxes, two such pairs take turns
						// this warp's accumulators into registers at once: the buffer goes back before the arithmetic
						uint32_t a[2][32], b[2][32];
#pragma unroll
						for (int c = 0; c < 2; c++)
						{
							tmem_ld_32x32(taddr + half * 64 + c * 32, a[c]);
							tmem_ld_32x32(taddr + BN / 2 + half * 64 + c * 32, b[c]);
						}
						tmem_wait_ld();
						release();
						uint32_t packed[2][16];
#pragma unroll
						for (int c = 0; c < 2; c++)
						{
							if (p.kept != nullptr && row_ok)
							{
								float *dst = kept_block(p.kept, p, row0, n0 + c * 32) + lane * 4;
								const int rows = min(32, p.M - row0);
#pragma unroll
								for (int k = 0; k < 8; k++)
									if (n0 + c * 32 + 4 * k < p.N)
									{
										*reinterpret_cast<uint4*>(dst + k * rows * 4) = make_uint4(a[c][4 * k], a[c][4 * k + 1], a[c][4 * k + 2], a[c][4 * k + 3]);
										*reinterpret_cast<uint4*>(dst + k * rows * 4 + rows * p.N) = make_uint4(b[c][4 * k], b[c][4 * k + 1], b[c][4 * k + 2], b[c][4 * k + 3]);
									}
							}
#pragma unroll
							for (int j = 0; j < 32; j += 2)
							{
								const Pair h = pair_mul(gate_value<GATE>(Pair { __uint_as_float(a[c][j]), __uint_as_float(a[c][j + 1]) }),
										Pair { __uint_as_float(b[c][j]), __uint_as_float(b[c][j + 1]) });
								packed[c][j / 2] = pack_half2(h.x, h.y);
							}
						}
						if (lane == 0)
							bulk_wait_group_read<1>();
						__syncwarp();
#pragma unroll
						for (int c = 0; c < 2; c++)
#pragma unroll
							for (int k = 0; k < 4; k++)
								st_shared_v4(box + c * HALF_BOX + lane * 64 + ((k ^ ((lane >> 1) & 3)) * 16),
										make_uint4(packed[c][4 * k], packed[c][4 * k + 1], packed[c][4 * k + 2], packed[c][4 * k + 3]));
						publish();
						if (lane == 0)
						{
							if (row0 < p.M)
							{
								if (n0 < p.N)
									tma_store_2d(&map_d, box, n0, row0);
								if (n0 + 32 < p.N)
									tma_store_2d(&map_d, box + HALF_BOX, n0 + 32, row0);
							}
							bulk_commit_group();
						}
						continue;
					}

					if constexpr (EPI == GATED_RECOMPUTE)
					{
						// a and u of this warp's 64 hidden columns into registers, so that the next tile's may be made under the arithmetic
						const int column = half * 64;
						const uint32_t au = lane_base + column, dh = lane_base + BN + (buffers & 1u) * (BN / 2) + column;
						uint32_t a[2][32], b[2][32];
						tmem_ld_32x32(au, a[0]);
						tmem_ld_32x32(au + BN / 2, b[0]);
						tmem_ld_32x32(au + 32, a[1]);
						tmem_ld_32x32(au + BN / 2 + 32, b[1]);
						tmem_wait_ld();
						tcgen05_fence_before();
						__syncwarp();
						if (lane == 0)
							arrive_at_leader(smem_u32(&bars.au_empty));
						if (lane == 0)
							bulk_wait_group_read<0>(); // the boxes of the tile before have left
						__syncwarp();
						const int n = u.nt * (BN / 2) + column;
#pragma unroll
						for (int c = 0; c < 2; c++)
						{
							float v[32];
							load_chunk(dh + c * 32, v);
							if (c == 1)
								release();
							// eight columns at a time: da, du and h of a row's 16-byte piece
#pragma unroll
							for (int k = 0; k < 4; k++)
							{
								float da[8], du[8], h[8];
#pragma unroll
								for (int j = 0; j < 8; j += 2)
								{
									const int i = 8 * k + j;
									const Pair g = { __uint_as_float(a[c][i]), __uint_as_float(a[c][i + 1]) }, up = { __uint_as_float(b[c][i]), __uint_as_float(b[c][i + 1]) }, d = { v[i], v[i + 1] };
									Pair value, derivative;
									gate_with_derivative<GATE>(g, value, derivative);
									const Pair x = pair_mul(d, pair_mul(up, derivative)), y = pair_mul(d, value), z = pair_mul(up, value);
									da[j] = x.x, da[j + 1] = x.y;
									du[j] = y.x, du[j + 1] = y.y;
									h[j] = z.x, h[j + 1] = z.y;
								}
								const uint32_t at = staging + c * 3 * HALF_BOX + lane * 64 + ((k ^ ((lane >> 1) & 3)) * 16);
								st_shared_v4(at, pack_half8(da));
								st_shared_v4(at + HALF_BOX, pack_half8(du));
								if (p.store_h)
									st_shared_v4(at + 2 * HALF_BOX, pack_half8(h));
							}
						}
						publish();
						if (lane == 0 && row0 < p.M)
						{
#pragma unroll
							for (int c = 0; c < 2; c++)
								if (n + c * 32 < p.N)
								{
									tma_store_2d(&map_d, staging + c * 3 * HALF_BOX, n + c * 32, row0);
									tma_store_2d(&map_e, staging + (c * 3 + 1) * HALF_BOX, n + c * 32, row0);
									if (p.store_h)
										tma_store_2d(&map_f, staging + (c * 3 + 2) * HALF_BOX, n + c * 32, row0);
								}
							bulk_commit_group();
						}
						continue;
					}

					if constexpr (EPI == GATED_BACKWARD)
					{
#pragma unroll 1
						for (int c = 0; c < BN / 64; c++)
						{
							const int n = u.nt * BN + half * (BN / 2) + c * 32;
							float v[32], a[32], b[32];
							const int rows = min(32, p.M - row0);
							const float *src = kept_block(p.kept, p, row0, n) + lane * 4;
#pragma unroll
							for (int k = 0; k < 8; k++)
							{
								const bool inside = row_ok && n + 4 * k < p.N;
								const float4 ta = inside ? *reinterpret_cast<const float4*>(src + k * rows * 4) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
								const float4 tb = inside ? *reinterpret_cast<const float4*>(src + k * rows * 4 + rows * p.N) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
								a[4 * k] = ta.x, a[4 * k + 1] = ta.y, a[4 * k + 2] = ta.z, a[4 * k + 3] = ta.w;
								b[4 * k] = tb.x, b[4 * k + 1] = tb.y, b[4 * k + 2] = tb.z, b[4 * k + 3] = tb.w;
							}
							load_chunk(taddr + half * (BN / 2) + c * 32, v);
							if (c == BN / 64 - 1)
								release();
							if (n >= p.N)
								continue;
							if (lane == 0)
								bulk_wait_group_read<0>();
							__syncwarp();
#pragma unroll
							for (int j = 0; j < 32; j += 2)
							{
								const Pair up = { b[j], b[j + 1] }, d = { v[j], v[j + 1] };
								Pair value, derivative;
								gate_with_derivative<GATE>(Pair { a[j], a[j + 1] }, value, derivative);
								const Pair x = pair_mul(d, pair_mul(up, derivative)), y = pair_mul(d, value), z = pair_mul(up, value);
								a[j] = x.x, a[j + 1] = x.y; // da
								v[j] = y.x, v[j + 1] = y.y; // du
								b[j] = z.x, b[j + 1] = z.y; // h
							}
							write_half_box(staging, lane, a);
							write_half_box(staging + HALF_BOX, lane, v);
							write_half_box(staging + 2 * HALF_BOX, lane, b);
							publish();
							if (lane == 0 && row0 < p.M)
							{
								tma_store_2d(&map_d, staging, n, row0);
								tma_store_2d(&map_e, staging + HALF_BOX, n, row0);
								tma_store_2d(&map_f, staging + 2 * HALF_BOX, n, row0);
								bulk_commit_group();
							}
						}
					}
				}
				if (lane == 0)
					bulk_wait_group_read<0>(); // shared memory stays until the last store has read it
				__syncwarp();
			}

			/* ---------------------------------------------------------------- teardown */
			tcgen05_fence_before();
			__syncthreads();
			if (bars.abort_flag != 0)
			{
				if (threadIdx.x == 0 && p.status != nullptr)
					atomicExch(p.status, 1);
				__nanosleep(1000000); // give copies that are still in flight time to land before the CTA retires
			}
			cluster_sync(); // neither CTA's shared or tensor memory goes while the other may still use it
			if (warp == 1)
			{
				tcgen05_fence_after();
				asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(tmem_base), "r"(2 * BN) : "memory");
			}
		}

		/* How many clusters of the kernel the device holds at once; 0 when clusters of this size cannot be placed.  Also opts the kernel in to its
		 * shared memory; both once per device. */
		template<int EPI, int GATE>
		int resident_clusters(mlContext_t ctx)
		{
			static int known[MAX_DEVICES] = { 0 }; // 0: not asked yet, -1: none
			static std::mutex mutex;
			std::lock_guard<std::mutex> lock(mutex);
			const int device = get(ctx)->device;
			if (device < 0 || device >= MAX_DEVICES)
				return 0;
			if (known[device] == 0)
			{
				use_stream(ctx);
				int n = 0;
				cudaLaunchConfig_t config = { };
				cudaLaunchAttribute attribute = { };
				attribute.id = cudaLaunchAttributeClusterDimension;
				attribute.val.clusterDim.x = 2;
				attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
				config.gridDim = dim3(2 * (get(ctx)->sm_count / 2));
				config.blockDim = dim3(THREADS);
				config.dynamicSmemBytes = Shape<EPI>::smem_bytes;
				config.attrs = &attribute;
				config.numAttrs = 1;
				if (cudaFuncSetAttribute(kernel_gemm_pair<EPI, GATE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<EPI>::smem_bytes) != cudaSuccess
						|| cudaOccupancyMaxActiveClusters(&n, kernel_gemm_pair<EPI, GATE>, &config) != cudaSuccess || n <= 0)
				{
					cudaGetLastError();
					n = -1;
				}
				known[device] = n;
			}
			return std::max(0, known[device]);
		}

		struct Maps
		{
				CUtensorMap a, b, d, e, f, dy, w2;
		};
		template<int EPI, int GATE>
		bool launch(mlContext_t ctx, const Maps &maps, Params p)
		{
			const int resident = resident_clusters<EPI, GATE>(ctx);
			if (resident == 0)
			{
				record_error(ctx, "gemm_pair: a cluster of two CTAs with %d bytes of shared memory each cannot be placed on this device", Shape<EPI>::smem_bytes);
				return false;
			}
			Context *c = get(ctx);
			p.status = c->dev_status;
			const int units = p.m_tiles * p.n_tiles * p.splits;
			cudaLaunchConfig_t config = { };
			cudaLaunchAttribute attributes[2] = { };
			attributes[0].id = cudaLaunchAttributeClusterDimension;
			attributes[0].val.clusterDim.x = 2;
			attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
			attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
			attributes[1].val.programmaticStreamSerializationAllowed = 1;
			config.gridDim = dim3(2 * std::min(units, resident));
			config.blockDim = dim3(THREADS);
			config.dynamicSmemBytes = Shape<EPI>::smem_bytes;
			config.stream = use_stream(ctx);
			config.attrs = attributes;
			config.numAttrs = 2;
			const cudaError_t status = cudaLaunchKernelEx(&config, kernel_gemm_pair<EPI, GATE>, maps.a, maps.b, maps.d, maps.e, maps.f, maps.dy, maps.w2, p);
			MB200_COUNT_LAUNCH();
			return check_cuda(ctx, status, "gemm_pair launch");
		}

		/* Boxes of an operand: 64 K indices of 128 rows (64 at a time when stored [K, rows]). */
		bool map_operand(mlContext_t ctx, CUtensorMap *map, const PairOperand &o, int rows, int K)
		{
			const uint64_t dims[2] = { static_cast<uint64_t>(o.mn ? rows : K), static_cast<uint64_t>(o.mn ? K : rows) };
			const uint64_t strides[1] = { static_cast<uint64_t>(o.ld) * 2 };
			const uint32_t box[2] = { 64, o.mn ? 64u : 128u };
			return encode_tensor_map(ctx, map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, o.data, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
		}
		bool map_halves(mlContext_t ctx, CUtensorMap *map, const void *d, int ld, int rows, int columns)
		{
			const uint64_t dims[2] = { static_cast<uint64_t>(columns), static_cast<uint64_t>(rows) };
			const uint64_t strides[1] = { static_cast<uint64_t>(ld) * 2 };
			const uint32_t box[2] = { 32, 32 };
			return encode_tensor_map(ctx, map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, d, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_64B);
		}
		/* Operand maps and tile counts; the result maps are filled with a copy where an epilogue has no use for them. */
		bool prepare(mlContext_t ctx, Maps &maps, Params &p, int M, int N, int K, const PairOperand &a, const PairOperand &b, int b_rows, int tile_columns, int splits)
		{
			std::memset(&p, 0, sizeof(p));
			if (!map_operand(ctx, &maps.a, a, M, K) || !map_operand(ctx, &maps.b, b, b_rows, K))
				return false;
			maps.d = maps.e = maps.f = maps.dy = maps.w2 = maps.a;
			p.M = M;
			p.N = N;
			p.K = K;
			p.a_mn = a.mn;
			p.b_mn = b.mn;
			p.m_tiles = (M + 2 * BM - 1) / (2 * BM);
			p.n_tiles = (N + tile_columns - 1) / tile_columns;
			const int k_blocks = (K + BK - 1) / BK;
			p.blocks_per_split = (k_blocks + splits - 1) / splits;
			p.splits = (k_blocks + p.blocks_per_split - 1) / p.blocks_per_split;
			if (static_cast<long long>(p.m_tiles) * p.n_tiles * p.splits > 0x3FFFFFFF)
			{
				record_error(ctx, "gemm_pair: %d x %d tiles are too many for one launch", p.m_tiles, p.n_tiles);
				return false;
			}
			return true;
		}

		/* One thread a group of VEC columns: the K ranges' sums in order, the factors, one rounding. */
		template<typename T, int VEC>
		__global__ void __launch_bounds__(256) kernel_finish_sums(T *d, int ldd, int M, const GridWalk walk, const float *sums, int pitch, int splits, float alpha,
				const float *alpha_device, const float *row_scale, float beta)
		{
			struct alignas(sizeof(T) * VEC) Out
			{
					T v[VEC];
			};
			wait_for_previous_grid();
			if (alpha_device != nullptr)
				alpha *= *alpha_device;
			const long long stride = static_cast<long long>(gridDim.x) * 256, range = static_cast<long long>(M) * pitch;
			for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < walk.total; i += stride)
			{
				long long m;
				int n;
				walk.place(i, m, n);
				n *= VEC;
				const float *src = sums + m * pitch + n;
				float v[VEC];
#pragma unroll
				for (int k = 0; k < VEC; k++)
					v[k] = 0.0f;
#pragma unroll 6
				for (int s = 0; s < splits; s++)
				{
					if (VEC == 4)
					{
						const float4 t = *reinterpret_cast<const float4*>(src + s * range);
						v[0] += t.x;
						v[1 % VEC] += t.y;
						v[2 % VEC] += t.z;
						v[3 % VEC] += t.w;
					}
					else
						v[0] += src[s * range];
				}
				const float c = row_scale != nullptr ? row_scale[m] : 1.0f;
				Out *dst = reinterpret_cast<Out*>(d + m * ldd + n);
				Out out;
				if (beta != 0.0f)
					out = *dst;
#pragma unroll
				for (int k = 0; k < VEC; k++)
				{
					const float x = c == 0.0f ? 0.0f : alpha * c * v[k];
					out.v[k] = from_float<T>(beta != 0.0f ? x + beta * to_float(out.v[k]) : x);
				}
				*dst = out;
			}
		}
	}

	template<typename T>
	bool finish_sums(mlContext_t ctx, T *d, int ldd, int M, int N, const float *sums, int pitch, int splits, float alpha, const float *alpha_device, const float *row_scale, float beta)
	{
		constexpr int VEC = 4;
		const bool wide = N % VEC == 0 && ldd % VEC == 0 && pitch % 4 == 0 && aligned_to(d, VEC * sizeof(T)) && aligned_to(sums, 16);
		const long long threads = static_cast<long long>(M) * (wide ? N / VEC : N);
		const int blocks = static_cast<int>(std::max<long long>(1, std::min<long long>((threads + 255) / 256, static_cast<long long>(get(ctx)->sm_count) * 8)));
		const cudaError_t status = launch_overlapped(wide ? kernel_finish_sums<T, VEC> : kernel_finish_sums<T, 1>, dim3(blocks), dim3(256), 0, use_stream(ctx), d, ldd, M, GridWalk(M, wide ? N / VEC : N), sums, pitch,
				splits, alpha, alpha_device, row_scale, beta);
		MB200_COUNT_LAUNCH();
		return check_cuda(ctx, status, "finish_sums");
	}
	template bool finish_sums<__half>(mlContext_t, __half*, int, int, int, const float*, int, int, float, const float*, const float*, float);
	template bool finish_sums<float>(mlContext_t, float*, int, int, int, const float*, int, int, float, const float*, const float*, float);

	/* A cut costs S partial results through memory and one more launch, and saves idle clusters in the last round of tiles.  The figures: a K block of
	 * a tile 0.28 us at full rate, 1.5 us for what a tile has before and after its K blocks, 8 bytes per partial sum at 5 TB/s, 4 us for the
	 * second kernel. */
	int pair_splits(mlContext_t ctx, int M, int N, int K)
	{
		const int clusters = std::max(1, resident_clusters<SUMS, 0>(ctx));
		const long long tiles = static_cast<long long>((M + 255) / 256) * ((N + 255) / 256);
		const int k_blocks = (K + BK - 1) / BK;
		if (tiles <= 0 || k_blocks <= 0)
			return 1;
		int best = 1;
		double best_time = 0.0;
		for (int s = 1; s <= 64 && (s == 1 || k_blocks / s >= 4); s++)
		{
			const int blocks = (k_blocks + s - 1) / s, splits = (k_blocks + blocks - 1) / blocks;
			if (splits != s)
				continue; // the same ranges as a smaller s
			const double rounds = static_cast<double>((tiles * s + clusters - 1) / clusters);
			const double partial_bytes = s == 1 ? 0.0 : 8.0 * s * M * N;
			if (partial_bytes > 2.0 * (size_t(512) << 20))
				break;
			const double time = rounds * (blocks * 0.28 + 1.5) + (s == 1 ? 0.0 : 4.0 + partial_bytes / 5.0e6);
			if (s == 1 || time < best_time)
			{
				best = s;
				best_time = time;
			}
		}
		return best;
	}
	namespace
	{
		int partial_pitch(int N)
		{
			return (N + 3) / 4 * 4;
		}
	}
	size_t pair_partial_elements(mlContext_t ctx, int M, int N, int K)
	{
		const int splits = pair_splits(ctx, M, N, K);
		return splits == 1 ? 0 : static_cast<size_t>(splits) * M * partial_pitch(N);
	}
	bool pair_product(mlContext_t ctx, int M, int N, int K, const PairOperand &a, const PairOperand &b, const PairResult &r, float *partials)
	{
		const int splits = pair_splits(ctx, M, N, K);
		if (splits > 1)
			return pair_product_sums(ctx, M, N, K, a, b, partials, partial_pitch(N), splits, false)
					&& finish_sums(ctx, r.d, r.ldd, M, N, partials, partial_pitch(N), splits, r.alpha, r.alpha_device, r.row_scale, r.beta);
		Maps maps;
		Params p;
		if (!prepare(ctx, maps, p, M, N, K, a, b, N, BN, 1))
			return false;
		p.result = r;
		p.direct = !aligned_to(r.d, 16) || r.ldd % 8 != 0;
		if (!p.direct && !map_halves(ctx, &maps.d, r.d, r.ldd, M, N))
			return false;
		return launch<STORE, 0>(ctx, maps, p);
	}
	bool pair_product_sums(mlContext_t ctx, int M, int N, int K, const PairOperand &a, const PairOperand &b, float *sums, int pitch, int splits, bool accumulate)
	{
		Maps maps;
		Params p;
		if (!prepare(ctx, maps, p, M, N, K, a, b, N, BN, splits))
			return false;
		p.accumulate = accumulate;
		const uint64_t dims[3] = { static_cast<uint64_t>(N), static_cast<uint64_t>(M), static_cast<uint64_t>(splits) };
		const uint64_t strides[2] = { static_cast<uint64_t>(pitch) * 4, static_cast<uint64_t>(pitch) * 4 * M };
		const uint32_t box[3] = { 32, 32, 1 };
		if (!encode_tensor_map(ctx, &maps.d, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 3, sums, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B))
			return false;
		return launch<SUMS, 0>(ctx, maps, p);
	}

	bool pair_gated(mlContext_t ctx, int tokens, int embed, int hidden, const PairOperand &x, const PairOperand &w1, int gate, __half *h, int ldh, float *kept)
	{
		Maps maps;
		Params p;
		if (!prepare(ctx, maps, p, tokens, hidden, embed, x, w1, 2 * hidden, BN / 2, 1) || !map_halves(ctx, &maps.d, h, ldh, tokens, hidden))
			return false;
		p.up_row = hidden;
		p.kept = kept;
		return with_gate(gate, [&](auto g)
		{
			return launch<GATED, decltype(g)::value>(ctx, maps, p);
		});
	}
	bool pair_gated_backward(mlContext_t ctx, int tokens, int embed, int hidden, const PairOperand &dy, const PairOperand &w2, int gate, const float *kept, __half *dau, __half *h)
	{
		Maps maps;
		Params p;
		if (!prepare(ctx, maps, p, tokens, hidden, embed, dy, w2, hidden, BN, 1) || !map_halves(ctx, &maps.d, dau, 2 * hidden, tokens, hidden)
				|| !map_halves(ctx, &maps.e, dau + hidden, 2 * hidden, tokens, hidden) || !map_halves(ctx, &maps.f, h, hidden, tokens, hidden))
			return false;
		p.kept = const_cast<float*>(kept);
		return with_gate(gate, [&](auto g)
		{
			return launch<GATED_BACKWARD, decltype(g)::value>(ctx, maps, p);
		});
	}

	bool pair_gated_recompute(mlContext_t ctx, int tokens, int embed, int hidden, const PairOperand &x, const PairOperand &w1, const PairOperand &dy, const PairOperand &w2, int gate, __half *dau,
			__half *h)
	{
		Maps maps;
		Params p;
		if (!prepare(ctx, maps, p, tokens, hidden, embed, x, w1, 2 * hidden, BN / 2, 1) || !map_operand(ctx, &maps.dy, dy, tokens, embed) || !map_operand(ctx, &maps.w2, w2, hidden, embed)
				|| !map_halves(ctx, &maps.d, dau, 2 * hidden, tokens, hidden) || !map_halves(ctx, &maps.e, dau + hidden, 2 * hidden, tokens, hidden)
				|| (h != nullptr && !map_halves(ctx, &maps.f, h, hidden, tokens, hidden)))
			return false;
		p.up_row = hidden;
		p.store_h = h != nullptr;
		return with_gate(gate, [&](auto g)
		{
			return launch<GATED_RECOMPUTE, decltype(g)::value>(ctx, maps, p);
		});
	}

	int pair_statistics_parts(int N)
	{
		return (N + BN / 2 - 1) / (BN / 2);
	}
	bool pair_statistics(mlContext_t ctx, int tokens, int N, int embed, const PairOperand &x, const PairOperand &w, const int *targets, float2 *parts, float *target_logit)
	{
		Maps maps;
		Params p;
		if (!prepare(ctx, maps, p, tokens, N, embed, x, w, N, BN, 1))
			return false;
		p.targets = targets;
		p.parts = parts;
		p.groups = pair_statistics_parts(N);
		p.target_logit = target_logit;
		return launch<STATISTICS, 0>(ctx, maps, p);
	}
	bool pair_probabilities(mlContext_t ctx, int tokens, int N, int embed, const PairOperand &x, const PairOperand &w, const int *targets, const float *row_weights, const float *lse, int first,
			int vocab, __half *probabilities, int ldp)
	{
		Maps maps;
		Params p;
		if (!prepare(ctx, maps, p, tokens, N, embed, x, w, N, BN, 1) || !map_halves(ctx, &maps.d, probabilities, ldp, tokens, N))
			return false;
		p.targets = targets;
		p.row_weights = row_weights;
		p.lse = lse;
		p.first = first;
		p.vocab = vocab;
		return launch<PROBABILITIES, 0>(ctx, maps, p);
	}
} /* namespace mb200 */
