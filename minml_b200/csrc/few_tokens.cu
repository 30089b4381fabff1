/*
 * few_tokens.cu -- products of a few rows x [T, K], T <= 64, with a weight matrix W [N, K]: bound by reading W once.
 *
 * The weights are the 128-row operand A of tcgen05.mma and the tokens its 16 .. 64 columns, so no multiplication is spent on padding
 * tokens to a tile.  What counts is bytes in flight and how few instructions ask for them: a ring of 190 KB in stages of up to 48 KB
 * (measured, one token x 2048 x 50021: 37 us; with half the ring 42 us; in stages of 16 KB made of 2 KB boxes 98 us).  Every CTA takes an equal
 * share of the weight rows in groups of 16; a tile is up to eight groups, one box, and the unused rows of the 128-row operand are whatever
 * shared memory holds there: they end in accumulator rows that nothing reads.  The gate and up rows of the same hidden units are two
 * operands whose accumulators lie in the same lanes, so the epilogue has both.  A CTA with few rows would be bound by its multiplications (about
 * 50 cycles each however few rows are real): then a cluster of 2, 4 or 8 CTAs takes each set of rows, one K range a CTA, and adds the
 * sums up through distributed shared memory in a fixed order.
 *   warp 0 TMA, warp 1 multiplications, warps 2-5 epilogue: a lane is a weight row, so results leave as 64 contiguous bytes a token.
 * Row statistics take an accumulator for every 1024 K indices and add them in fp32, because the tensor core cuts its sums (gemm_pair.cu); those of
 * a tile that do not fit a buffer of tensor memory (embed above 4096 for 64 tokens) come in several.
 * Measured, gated block of 4096 x 11008: 1 token 48 us (two launches, 270 MB: 5.6 TB/s), 64 tokens 57 us, where the paired kernel (gemm_pair.cu)
 * takes 75; 2048 x 8192: 16 tokens 23 us, 48 28 (paired: 35), 64 31 (36).  Logits' statistics, 2048 x 50021: 48 tokens 43 us (47), 64 47 (49).
 * Above 64 rows, which is what accumulators and epilogue are made for, the paired kernel takes 78 us for 65 and for 96 rows of 4096 x 11008.
 */
#include "common.cuh"
#include "tc.cuh"
#include "gate.cuh"
#include "operands.cuh"
#include "few_tokens.cuh"

#include <algorithm>
#include <cstring>
#include <mutex>

namespace mb200
{
	namespace
	{
		using namespace tc;

		enum Kind
		{
			GATED,
			PRODUCT,
			STATISTICS
		};
		constexpr int GROUP = 16; // weight rows
		constexpr int BOX_BYTES = GROUP * 128;
		constexpr int TILE_GROUPS = 128 / GROUP;
		constexpr int MAX_STAGES = 12;
		constexpr int RING_BYTES = 12 * 16384;
		constexpr int EXTRA_BYTES = 16384 + 1024; // behind the ring, because the last plane is read as 128 rows; alignment
		constexpr int SMEM_BYTES = RING_BYTES + EXTRA_BYTES;
		constexpr int STAGE_BYTES = 49152; // a stage takes several K blocks when they are smaller than this
		constexpr int THREADS = 6 * 32;
		constexpr int BUFFER_COLUMNS = 256;
		constexpr int SEGMENT_BLOCKS = 16; // of 64 K indices
		constexpr int MAX_CLUSTER = 8;

		struct Params
		{
				int tokens, columns; // columns: tokens rounded up to 16
				int N, groups; // result columns (GATED: of h) and their groups of 16
				int k_blocks;
				int cluster; // CTAs that share a set of rows
				int tiles, tile_groups; // tiles of every set, and the most groups one has
				int blocks_per_stage, stages, block_bytes; // a stage: blocks_per_stage x (planes x tile_groups boxes, then the tokens' rows)
				int segment_blocks, pass_segments; // K blocks of an accumulator, accumulators that a buffer holds (STATISTICS)
				int tmem_columns; // two buffers
				__half *out;
				int ldo;
				float beta;
				const int *targets;
				float2 *parts;
				int part_groups;
				float *target_logit;
				int *status;
		};
		struct Barriers
		{
				uint64_t full[MAX_STAGES], empty[MAX_STAGES];
				uint64_t tmem_full[2], tmem_empty[2];
				uint32_t tmem_base;
				int abort_flag;
		};
		__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1)
		{
			asm volatile(
					"cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
					:: "r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1) : "memory");
		}
		__device__ __forceinline__ float ld_shared_cluster_f32(uint32_t addr)
		{
			float v;
			asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
			return v;
		}

		__device__ __forceinline__ float warp_max(float v)
		{ // of all lanes, in every lane; a NaN gives way to a number
			float m;
			asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
			return m;
		}
		__device__ __forceinline__ float2 join(float2 a, float2 b)
		{ // (maximum, sum of exp(z - maximum)) of two sets; an empty one is (-inf, 0)
			const float m = fmaxf(a.x, b.x);
			return make_float2(m, (a.x == m ? a.y : a.y * exp2_approx((a.x - m) * LOG2E)) + (b.x == m ? b.y : b.y * exp2_approx((b.x - m) * LOG2E)));
		}

		template<int KIND, int GATE>
		__global__ void __launch_bounds__(THREADS, 1) kernel_few_tokens(const __grid_constant__ CUtensorMap map_w,
				const __grid_constant__ CUtensorMap map_w_less, const __grid_constant__ CUtensorMap map_x, const Params p)
		{
			constexpr int PLANES = KIND == GATED ? 2 : 1;
			constexpr bool AFTER_GATED = KIND == PRODUCT;
			extern __shared__ uint8_t smem_raw[];
			__shared__ Barriers bars;
			__shared__ float2 running[KIND == STATISTICS ? 4 : 1][KIND == STATISTICS ? FEW_TOKENS : 1];
			const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
			const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;

			// this CTA's rows and K range
			const int set = blockIdx.x / p.cluster, sets = gridDim.x / p.cluster, rank = blockIdx.x - set * p.cluster;
			const int g0 = static_cast<int>(static_cast<long long>(p.groups) * set / sets), g1 = static_cast<int>(static_cast<long long>(p.groups) * (set + 1) / sets);
			const int tiles = p.tiles;
			const int kb0 = p.k_blocks * rank / p.cluster, kb1 = p.k_blocks * (rank + 1) / p.cluster;
			auto first_group = [&](int tile)
			{
				return g0 + (g1 - g0) * tile / tiles;
			};
			const int stage_bytes = p.blocks_per_stage * p.block_bytes;
			const int plane_bytes = p.tile_groups * BOX_BYTES;

			if (threadIdx.x == 0)
			{
				for (int s = 0; s < p.stages; s++)
				{
					mbar_init(smem_u32(&bars.full[s]), 1);
					mbar_init(smem_u32(&bars.empty[s]), 1);
				}
				for (int b = 0; b < 2; b++)
				{
					mbar_init(smem_u32(&bars.tmem_full[b]), 1);
					mbar_init(smem_u32(&bars.tmem_empty[b]), 4);
				}
				bars.abort_flag = 0;
				fence_mbar_init();
			}
			if (KIND == STATISTICS)
				for (int i = threadIdx.x; i < 4 * FEW_TOKENS; i += THREADS)
					running[i / FEW_TOKENS][i % FEW_TOKENS] = make_float2(-INFINITY, 0.0f);
			if (warp == 1)
			{
				tmem_alloc(smem_u32(&bars.tmem_base), p.tmem_columns);
				tmem_relinquish();
			}
			tcgen05_fence_before();
			__syncthreads();
			tcgen05_fence_after();
			const uint32_t tmem_base = bars.tmem_base;
			volatile int *abort_flag = &bars.abort_flag;
			if (!AFTER_GATED)
			{ // the next launch may start (and fetch weights) once every CTA is here: all that ran before this launch is then done
				wait_for_previous_grid();
				let_next_grid_start();
			}
			else if (warp != 0)
				wait_for_previous_grid();

			if (warp == 0)
			{ /* ------------------------------------------------ weights and tokens */
				if (elect_one())
				{
					prefetch_tensormap(&map_w);
					prefetch_tensormap(&map_x);
					// a tile has tile_groups groups or one less: one box of weights a plane and K block either way
					int row = g0 * GROUP, groups = 0;
					auto weights = [&](int kb, int s)
					{
						const int blocks = min(p.blocks_per_stage, kb1 - kb);
						const uint32_t full = smem_u32(&bars.full[s]);
						const CUtensorMap *map = groups == p.tile_groups ? &map_w : &map_w_less;
						mbar_arrive_expect_tx(full, blocks * (PLANES * groups * BOX_BYTES + p.columns * 128));
						uint32_t dst = smem_base + s * stage_bytes;
						for (int j = 0; j < blocks; j++, dst += p.block_bytes)
						{
							tma_load_2d(dst, map, full, (kb + j) * 64, row);
							if (PLANES == 2)
								tma_load_2d(dst + plane_bytes, map, full, (kb + j) * 64, p.N + row);
						}
					};
					auto tokens = [&](int kb, int s)
					{
						const int blocks = min(p.blocks_per_stage, kb1 - kb);
						const uint32_t full = smem_u32(&bars.full[s]);
						uint32_t dst = smem_base + s * stage_bytes + PLANES * plane_bytes;
						for (int j = 0; j < blocks; j++, dst += p.block_bytes)
							tma_load_2d(dst, &map_x, full, (kb + j) * 64, 0);
					};
					int ahead = 0; // stages whose weights were asked for before the launch ahead was done
					groups = first_group(1) - g0;
					if (AFTER_GATED)
					{
						for (int kb = kb0; kb < kb1 && ahead < p.stages; kb += p.blocks_per_stage, ahead++)
							weights(kb, ahead);
						wait_for_previous_grid();
					}
					int s = 0;
					uint32_t parity = 1u;
					bool ok = true;
					for (int tile = 0; tile < tiles && ok; tile++)
					{
						row = first_group(tile) * GROUP;
						groups = first_group(tile + 1) - first_group(tile);
						for (int kb = kb0; kb < kb1; kb += p.blocks_per_stage)
						{
							if (ahead > 0)
								ahead--;
							else
							{
								if (!mbar_wait(smem_u32(&bars.empty[s]), parity, abort_flag))
								{
									ok = false;
									break;
								}
								weights(kb, s);
							}
							tokens(kb, s);
							if (++s == p.stages)
							{
								s = 0;
								parity ^= 1u;
							}
						}
					}
				}
				__syncwarp();
				wait_for_previous_grid(); // the lanes that asked for nothing
			}
			else if (warp == 1)
			{ /* ------------------------------------------- multiplications */
				if (elect_one())
				{
					const uint32_t idesc = make_idesc_f16(p.columns);
					int s = 0;
					uint32_t parity = 0u, buffers = 0;
					bool ok = true;
					for (int tile = 0; tile < tiles && ok; tile++, buffers++)
					{
						if (!mbar_wait(smem_u32(&bars.tmem_empty[buffers & 1u]), ((buffers >> 1) & 1u) ^ 1u, abort_flag))
							break;
						tcgen05_fence_after();
						uint32_t d = tmem_base + (buffers & 1u) * (p.tmem_columns / 2);
						int in_segment = 0, segments = 0;
						for (int kb = kb0; kb < kb1; kb += p.blocks_per_stage)
						{
							if (!mbar_wait(smem_u32(&bars.full[s]), parity, abort_flag))
							{
								ok = false;
								break;
							}
							tcgen05_fence_after();
							const int blocks = min(p.blocks_per_stage, kb1 - kb);
							uint32_t base = smem_base + s * stage_bytes;
							for (int j = 0; j < blocks; j++, base += p.block_bytes)
							{
								if (KIND == STATISTICS && in_segment == p.segment_blocks)
								{ // the next accumulator, in the other buffer when this one is full
									in_segment = 0;
									d += p.columns;
									if (++segments == p.pass_segments)
									{
										mma_commit(smem_u32(&bars.tmem_full[buffers & 1u]));
										buffers++;
										ok = mbar_wait(smem_u32(&bars.tmem_empty[buffers & 1u]), ((buffers >> 1) & 1u) ^ 1u, abort_flag);
										if (!ok)
											break;
										tcgen05_fence_after();
										d = tmem_base + (buffers & 1u) * (p.tmem_columns / 2);
										segments = 0;
									}
								}
								const uint64_t desc_x = make_desc_k_sw128(base + PLANES * plane_bytes);
								const uint32_t accumulate = in_segment > 0 ? 1u : 0u;
#pragma unroll
								for (int plane = 0; plane < PLANES; plane++)
								{
									const uint64_t desc_w = make_desc_k_sw128(base + plane * plane_bytes);
#pragma unroll
									for (int k = 0; k < 4; k++)
										mma_ss<0>(d + plane * p.columns, desc_w + 2 * k, desc_x + 2 * k, idesc, accumulate | (k > 0 ? 1u : 0u));
								}
								in_segment++;
							}
							if (!ok)
								break;
							mma_commit(smem_u32(&bars.empty[s]));
							if (++s == p.stages)
							{
								s = 0;
								parity ^= 1u;
							}
						}
						if (ok)
							mma_commit(smem_u32(&bars.tmem_full[buffers & 1u]));
					}
				}
				__syncwarp();
			}
			else
			{ /* ------------------------------------------------------------ epilogue */
				const int q = warp % 4;
				uint32_t buffers = 0;
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
						mbar_arrive(smem_u32(&bars.tmem_empty[buffers & 1u]));
					buffers++;
				};
				for (int tile = 0; tile < tiles; tile++)
				{
					const int n = first_group(tile) * GROUP + q * 32 + lane; // this lane's result column
					const bool valid = q * 32 + lane < (first_group(tile + 1) - first_group(tile)) * GROUP && n < p.N;
					const uint32_t lane_base = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
					if constexpr (KIND == STATISTICS)
					{
						float z[FEW_TOKENS]; // this lane's column for every token, added up in fp32
						bool ok = true;
						for (int left = (kb1 - kb0 + p.segment_blocks - 1) / p.segment_blocks; left > 0; left -= p.pass_segments)
						{
							const bool first = left + p.pass_segments > (kb1 - kb0 + p.segment_blocks - 1) / p.segment_blocks;
							ok = wait_full();
							if (!ok)
								break;
							const uint32_t taddr = lane_base + (buffers & 1u) * (p.tmem_columns / 2);
#pragma unroll
							for (int c = 0; c < FEW_TOKENS; c += 16)
								if (c < p.columns)
									for (int s = 0; s < min(left, p.pass_segments); s++)
									{
										uint32_t r[16];
										tmem_ld_32x16(taddr + s * p.columns + c, r);
										tmem_wait_ld();
#pragma unroll
										for (int j = 0; j < 16; j++)
											z[c + j] = (first && s == 0 ? 0.0f : z[c + j]) + __uint_as_float(r[j]);
									}
							release();
						}
						if (!ok)
							break;
#pragma unroll
						for (int c = 0; c < FEW_TOKENS; c += 16)
						{
							if (c >= p.columns)
								break;
							float v[16], sum[16];
#pragma unroll
							for (int j = 0; j < 16; j++)
							{ // exponentials against the warp's maximum for the token
								const float mine = valid ? z[c + j] : -INFINITY, top = warp_max(mine);
								sum[j] = !valid || mine == -INFINITY ? 0.0f : exp2_approx((mine - top) * LOG2E);
								if (valid && c + j < p.tokens && p.targets[c + j] == n)
									p.target_logit[c + j] = mine;
								v[j] = top;
							}
							// lane l ends with the sum (and takes the maximum) of token c + l % 16: each step halves the tokens a lane holds
#pragma unroll
							for (int step = 8; step >= 1; step /= 2)
							{
								const bool upper = (lane & step) != 0;
#pragma unroll
								for (int j = 0; j < step; j++)
								{
									const float mine = upper ? sum[j + step] : sum[j], other = upper ? sum[j] : sum[j + step];
									sum[j] = mine + __shfl_xor_sync(0xffffffffu, other, step);
									v[j] = upper ? v[j + step] : v[j];
								}
							}
							sum[0] += __shfl_xor_sync(0xffffffffu, sum[0], 16);
							if (lane < 16 && c + lane < p.tokens)
								running[q][c + lane] = join(running[q][c + lane], make_float2(v[0], sum[0]));
						}
						continue;
					}
					if (!wait_full())
						break;
					const uint32_t taddr = lane_base + (buffers & 1u) * (p.tmem_columns / 2);
					for (int c = 0; c < p.columns; c += 16)
					{
						uint32_t r[16], r2[16];
						tmem_ld_32x16(taddr + c, r);
						if (KIND == GATED)
							tmem_ld_32x16(taddr + p.columns + c, r2);
						tmem_wait_ld();
						float v[16];
#pragma unroll
						for (int j = 0; j < 16; j++)
							v[j] = __uint_as_float(r[j]);
						if (p.cluster > 1)
						{ // this CTA's sums of [plane][token][row], over the ring: every stage has been read when the accumulators are full
#pragma unroll
							for (int j = 0; j < 16; j++)
								if (c + j < p.tokens)
								{
									st_shared_f32(smem_base + ((c + j) * 128 + q * 32 + lane) * 4, v[j]);
									if (KIND == GATED)
										st_shared_f32(smem_base + ((p.tokens + c + j) * 128 + q * 32 + lane) * 4, __uint_as_float(r2[j]));
								}
							continue;
						}
						if (!valid)
							continue;
#pragma unroll
						for (int j = 0; j < 16; j++)
						{
							const int t = c + j;
							if (t >= p.tokens)
								break; // uniform
							__half *dst = p.out + static_cast<long long>(t) * p.ldo + n;
							if (KIND == GATED)
								*dst = __float2half_rn(gate_value<GATE, true>(v[j]) * __uint_as_float(r2[j]));
							else
								*dst = __float2half_rn(p.beta != 0.0f ? v[j] + p.beta * __half2float(*dst) : v[j]);
						}
					}
					release();
				}
			}

			tcgen05_fence_before();
			__syncthreads();
			if (bars.abort_flag != 0)
			{
				if (threadIdx.x == 0 && p.status != nullptr)
					atomicExch(p.status, 1);
				__nanosleep(1000000); // give copies that are still in flight time to land before the CTA retires
			}
			if (KIND != STATISTICS && p.cluster > 1)
			{ // (one tile) every CTA finishes a share of the tokens
				cluster_sync();
				const int row = threadIdx.x, n = g0 * GROUP + row;
				if (row < 128 && row < (g1 - g0) * GROUP && n < p.N)
				{
					uint32_t from[MAX_CLUSTER]; // this row's sums of token 0 in every CTA
#pragma unroll
					for (int k = 0; k < MAX_CLUSTER; k++)
						from[k] = map_to_cta(smem_base + row * 4, min(k, p.cluster - 1));
#pragma unroll 2
					for (int t = rank; t < p.tokens; t += p.cluster)
					{ // all loads of a token (from up to eight SMs) before the first addition
						float v[MAX_CLUSTER], u[KIND == GATED ? MAX_CLUSTER : 1];
#pragma unroll
						for (int k = 0; k < MAX_CLUSTER; k++)
							if (k < p.cluster)
							{
								v[k] = ld_shared_cluster_f32(from[k] + t * 512);
								if (KIND == GATED)
									u[KIND == GATED ? k : 0] = ld_shared_cluster_f32(from[k] + (p.tokens + t) * 512);
							}
#pragma unroll
						for (int k = 1; k < MAX_CLUSTER; k++)
							if (k < p.cluster)
							{
								v[0] += v[k];
								if (KIND == GATED)
									u[0] += u[KIND == GATED ? k : 0];
							}
						__half *dst = p.out + static_cast<long long>(t) * p.ldo + n;
						if (KIND == GATED)
							*dst = __float2half_rn(gate_value<GATE, true>(v[0]) * u[0]);
						else
							*dst = __float2half_rn(p.beta != 0.0f ? v[0] + p.beta * __half2float(*dst) : v[0]);
					}
				}
				cluster_sync(); // no CTA's shared memory goes while another reads it
			}
			if (KIND == STATISTICS)
				for (int t = threadIdx.x; t < p.tokens; t += THREADS)
				{
					float2 total = running[0][t];
					for (int k = 1; k < 4; k++)
						total = join(total, running[k][t]);
					p.parts[static_cast<long long>(t) * p.part_groups + blockIdx.x] = total;
				}
			if (warp == 1)
			{
				tcgen05_fence_after();
				tmem_dealloc(tmem_base, p.tmem_columns);
			}
		}

		/* CTAs that share a set of rows: enough that each has six boxes to multiply at a time, and a K range of eight blocks.  Measured, 64
		 * tokens x 4096 x 11008: 61 us with three boxes at least, 57 us with six; 1 token 48.8 and 48.0. */
		int cluster_size(int sm_count, int boxes, int k_blocks)
		{
			int size = 1;
			while (size < MAX_CLUSTER && static_cast<long long>(boxes) * size < 6ll * sm_count && k_blocks >= 16 * size)
				size *= 2;
			return size;
		}

		/* How many clusters of this size the device holds at once (0: none); also opts the kernel in to its shared memory.  Asked once per device. */
		template<int KIND, int GATE>
		int resident_clusters(mlContext_t ctx, int size)
		{
			static int known[MAX_DEVICES][MAX_CLUSTER + 1] = { }; // 0: not asked yet, -1: none
			static std::mutex mutex;
			std::lock_guard<std::mutex> lock(mutex);
			const int device = get(ctx)->device;
			if (device < 0 || device >= MAX_DEVICES)
				return 0;
			int &n = known[device][size];
			if (n == 0)
			{
				use_stream(ctx);
				cudaLaunchAttribute attribute = { };
				attribute.id = cudaLaunchAttributeClusterDimension;
				attribute.val.clusterDim.x = size;
				attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
				cudaLaunchConfig_t config = { };
				config.gridDim = dim3(get(ctx)->sm_count / size * size);
				config.blockDim = dim3(THREADS);
				config.dynamicSmemBytes = SMEM_BYTES;
				config.attrs = &attribute;
				config.numAttrs = 1;
				if (cudaFuncSetAttribute(kernel_few_tokens<KIND, GATE>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) != cudaSuccess
						|| cudaOccupancyMaxActiveClusters(&n, kernel_few_tokens<KIND, GATE>, &config) != cudaSuccess || n <= 0)
				{
					cudaGetLastError();
					n = -1;
				}
			}
			return std::max(0, n);
		}

		template<int KIND, int GATE>
		bool launch(mlContext_t ctx, const FewTokens &f, Params p)
		{
			Context *c = get(ctx);
			constexpr int PLANES = KIND == GATED ? 2 : 1;
			p.tokens = f.tokens;
			p.columns = round_up(f.tokens, 16);
			p.groups = (p.N + GROUP - 1) / GROUP;
			p.k_blocks = (f.embed + 63) / 64;
			p.status = c->dev_status;
			p.cluster = KIND == STATISTICS ? 1 : cluster_size(c->sm_count, p.groups * PLANES, p.k_blocks);
			int sets = resident_clusters<KIND, GATE>(ctx, p.cluster);
			// a cluster joins the sums of one tile only
			while (p.cluster > 1 && (sets == 0 || (p.groups + sets - 1) / sets > TILE_GROUPS))
			{
				p.cluster /= 2;
				sets = resident_clusters<KIND, GATE>(ctx, p.cluster);
			}
			if (sets == 0)
			{
				record_error(ctx, "few_tokens: a CTA with %d bytes of shared memory cannot be placed on this device", SMEM_BYTES);
				return false;
			}
			if (p.cluster == 1)
				sets = c->sm_count; // no CTA waits for another one: what does not fit at once runs later
			sets = std::min(sets, p.groups);
			const int most = (p.groups + sets - 1) / sets; // groups of a set; no set has fewer than most - 1
			p.tiles = (most + TILE_GROUPS - 1) / TILE_GROUPS;
			p.tile_groups = (most + p.tiles - 1) / p.tiles;
			p.block_bytes = PLANES * p.tile_groups * BOX_BYTES + p.columns * 128;
			p.blocks_per_stage = std::max(1, std::min(8, STAGE_BYTES / p.block_bytes));
			p.stages = std::min(MAX_STAGES, RING_BYTES / (p.blocks_per_stage * p.block_bytes));
			p.segment_blocks = 1 << 30;
			if (KIND == STATISTICS)
			{
				const int segments = (p.k_blocks + SEGMENT_BLOCKS - 1) / SEGMENT_BLOCKS;
				p.segment_blocks = (p.k_blocks + segments - 1) / segments;
				p.pass_segments = std::min(segments, BUFFER_COLUMNS / p.columns);
			}
			const int used = 2 * p.columns * (KIND == STATISTICS ? p.pass_segments : PLANES);
			for (p.tmem_columns = 32; p.tmem_columns < used;)
				p.tmem_columns *= 2;
			CUtensorMap map_w, map_w_less, map_x;
			const uint64_t dims_w[2] = { static_cast<uint64_t>(f.embed), static_cast<uint64_t>(p.N) * PLANES }, dims_x[2] = { static_cast<uint64_t>(f.embed), static_cast<uint64_t>(f.tokens) };
			const uint64_t strides_w[1] = { static_cast<uint64_t>(f.ldw) * 2 }, strides_x[1] = { static_cast<uint64_t>(f.ldx) * 2 };
			const uint32_t box_w[2] = { 64, static_cast<uint32_t>(p.tile_groups) * GROUP }, box_less[2] = { 64, static_cast<uint32_t>(std::max(1, p.tile_groups - 1)) * GROUP }, box_x[2] = { 64, static_cast<uint32_t>(p.columns) };
			if (!encode_tensor_map(ctx, &map_w, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, f.w, dims_w, strides_w, box_w, CU_TENSOR_MAP_SWIZZLE_128B)
					|| !encode_tensor_map(ctx, &map_w_less, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, f.w, dims_w, strides_w, box_less, CU_TENSOR_MAP_SWIZZLE_128B)
					|| !encode_tensor_map(ctx, &map_x, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, f.x, dims_x, strides_x, box_x, CU_TENSOR_MAP_SWIZZLE_128B))
				return false;
			cudaLaunchAttribute attributes[2] = { };
			attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
			attributes[0].val.programmaticStreamSerializationAllowed = 1;
			attributes[1].id = cudaLaunchAttributeClusterDimension;
			attributes[1].val.clusterDim.x = p.cluster;
			attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
			cudaLaunchConfig_t config = { };
			config.gridDim = dim3(sets * p.cluster);
			config.blockDim = dim3(THREADS);
			config.dynamicSmemBytes = SMEM_BYTES;
			config.stream = use_stream(ctx);
			config.attrs = attributes;
			config.numAttrs = 2;
			const cudaError_t status = cudaLaunchKernelEx(&config, kernel_few_tokens<KIND, GATE>, map_w, map_w_less, map_x, p);
			MB200_COUNT_LAUNCH();
			return check_cuda(ctx, status, "few_tokens launch");
		}
	}

	bool few_gated(mlContext_t ctx, const FewTokens &f, int hidden, int gate, __half *h, int ldh)
	{
		Params p;
		std::memset(&p, 0, sizeof(p));
		p.N = hidden;
		p.out = h;
		p.ldo = ldh;
		return with_gate(gate, [&](auto g)
		{
			return launch<GATED, decltype(g)::value>(ctx, f, p);
		});
	}
	bool few_product_after_gated(mlContext_t ctx, const FewTokens &f, int N, __half *y, int ldy, float beta)
	{
		Params p;
		std::memset(&p, 0, sizeof(p));
		p.N = N;
		p.out = y;
		p.ldo = ldy;
		p.beta = beta;
		return launch<PRODUCT, 0>(ctx, f, p);
	}
	int few_statistics_parts(mlContext_t ctx, int N)
	{ // one per CTA
		return std::min(get(ctx)->sm_count, (N + GROUP - 1) / GROUP);
	}
	bool few_statistics(mlContext_t ctx, const FewTokens &f, int N, const int *targets, float2 *parts, float *target_logit)
	{
		Params p;
		std::memset(&p, 0, sizeof(p));
		p.N = N;
		p.targets = targets;
		p.parts = parts;
		p.part_groups = few_statistics_parts(ctx, N);
		p.target_logit = target_logit;
		return launch<STATISTICS, 0>(ctx, f, p);
	}
} /* namespace mb200 */
