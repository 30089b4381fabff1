/*
 * layernorm_train.cu -- layer normalisation for training: the forward pass that keeps each row's mean and 1 / stddev, and the
 * backward pass with the reduction of the weight and bias gradients.  Same function as cuda_layernorm_forward (norm_attn.cu):
 *   s = x + ext;   m = mean(s);   r = 1 / sqrt(1e-6 + sum((s - m)^2) / (N - 1));   xh = (s - m) r;   y = gamma xh + beta
 * Differentiating, with g = gamma dy (the unbiased variance puts N - 1, not N, under the second sum):
 *   dx = r (g - sum(g) / N - xh sum(g xh) / (N - 1));     dgamma = sum over rows of dy xh;     dbeta = sum over rows of dy
 * and the gradient of ext is that of x.
 *
 * Both passes are bound by memory: forward reads s and writes y, backward reads s and dy and writes dx.  A row belongs to a team
 * of 32 .. 512 threads that holds it in registers (8 or 16 elements a thread, by the row's length), so it is read once: through a ring in
 * shared memory that bulk copies keep filled, or, where rows do not start on 16-byte boundaries, by loads one row ahead.
 * Backward, a thread owns the same columns in every row of its team, so the column sums of dgamma and dbeta stay in its fp32 registers
 * until the end.  Each block then writes one partial row of each, and a second kernel adds the blocks' rows in a fixed order: no
 * atomics, the same bits on every run.  All sums are fp32; y and dx are rounded once.
 */
#include "common.cuh"
#include "operands.cuh"
#include "pairs.cuh"
#include "tc.cuh"

#include <algorithm>
#include <mutex>

namespace mb200
{
	namespace
	{
		constexpr float EPSILON = 1.0e-6f; // inside the square root, as in cuda_layernorm_forward

		/* Sums a and b over the threads of a team of W: a warp by shuffles, several warps through `scratch` (two halves used in turn,
		 * so one barrier a call is enough: a thread that writes half h again has passed the barrier of the call in between). */
		template<int W>
		__device__ __forceinline__ void team_sum(float &a, float &b, float2 (*scratch)[16], uint32_t &turn)
		{
#pragma unroll
			for (int k = 16; k >= 1; k /= 2)
			{
				a += __shfl_xor_sync(0xffffffffu, a, k);
				b += __shfl_xor_sync(0xffffffffu, b, k);
			}
			if (W > 32)
			{
				const int half = turn & 1u;
				turn++;
				if (threadIdx.x % 32 == 0)
					scratch[half][threadIdx.x / 32] = make_float2(a, b);
				__syncthreads();
				a = b = 0.0f;
#pragma unroll
				for (int k = 0; k < W / 32; k++)
				{
					const float2 t = scratch[half][k];
					a += t.x;
					b += t.y;
				}
			}
		}

		template<typename T, int E>
		struct RowPart
		{ // a thread's share of one row, as loaded
				T v[E];
				template<int W>
				__device__ __forceinline__ void load(const T *row, int lane, int channels)
				{
#pragma unroll
					for (int k = 0; k < E; k++)
					{
						const int c = k * W + lane;
						v[k] = c < channels ? row[c] : from_float<T>(0.0f);
					}
				}
				__device__ __forceinline__ float get(int k) const
				{
					return to_float(v[k]);
				}
		};

		template<typename T, int W, int E>
		__global__ void __launch_bounds__(W == 32 ? 256 : W) kernel_layernorm_train(T *output, const T *input, const T *ext, const T *__restrict__ gamma,
				const T *__restrict__ beta, float2 *__restrict__ stats, long long rows, int channels)
		{
			__shared__ float2 scratch[2][16];
			uint32_t turn = 0;
			const int lane = threadIdx.x % W;
			const int teams_per_block = blockDim.x / W;
			const long long teams = static_cast<long long>(gridDim.x) * teams_per_block;
			for (long long r = static_cast<long long>(blockIdx.x) * teams_per_block + threadIdx.x / W; r < rows; r += teams)
			{
				RowPart<T, E> x, e;
				x.template load<W>(input + r * channels, lane, channels);
				if (ext != nullptr)
					e.template load<W>(ext + r * channels, lane, channels);
				float v[E];
				float sum = 0.0f, unused = 0.0f;
#pragma unroll
				for (int k = 0; k < E; k++)
				{
					v[k] = x.get(k) + (ext != nullptr ? e.get(k) : 0.0f);
					sum += v[k];
				}
				team_sum<W>(sum, unused, scratch, turn);
				const float mean = sum / static_cast<float>(channels);
				float var = 0.0f;
#pragma unroll
				for (int k = 0; k < E; k++)
				{
					const bool inside = k * W + lane < channels;
					v[k] -= mean;
					var += inside ? v[k] * v[k] : 0.0f;
				}
				team_sum<W>(var, unused, scratch, turn);
				const float inv_stddev = 1.0f / sqrtf(EPSILON + var / static_cast<float>(channels - 1));
				if (lane == 0)
					stats[r] = make_float2(mean, inv_stddev);
#pragma unroll
				for (int k = 0; k < E; k++)
				{
					const int c = k * W + lane;
					if (c < channels)
						output[r * channels + c] = from_float<T>((gamma != nullptr ? to_float(gamma[c]) : 1.0f) * v[k] * inv_stddev + (beta != nullptr ? to_float(beta[c]) : 0.0f));
				}
			}
		}

		/* partial: [2][gridDim.x][channels], the block's column sums of dy xh and of dy */
		template<typename T, int W, int E>
		__global__ void __launch_bounds__(W == 32 ? 256 : W) kernel_layernorm_backward(T *dx, const T *input, const T *ext, const T *dy,
				const T *__restrict__ gamma, const float2 *__restrict__ stats, float beta_dx, float *__restrict__ partial, long long rows, int channels)
		{
			__shared__ float2 scratch[2][16];
			__shared__ float columns[W == 32 ? 7 * 32 * E : 1]; // the other warps' column sums, when a block has eight one-warp teams
			uint32_t turn = 0;
			const int lane = threadIdx.x % W;
			const int teams_per_block = blockDim.x / W;
			const long long teams = static_cast<long long>(gridDim.x) * teams_per_block;
			const float inv_n = 1.0f / static_cast<float>(channels), inv_n1 = 1.0f / static_cast<float>(channels - 1);

			RowPart<T, E> g, x, e, d;
			if (gamma != nullptr)
				g.template load<W>(gamma, lane, channels);
			float sum_w[E], sum_b[E];
#pragma unroll
			for (int k = 0; k < E; k++)
				sum_w[k] = sum_b[k] = 0.0f;

			long long r = static_cast<long long>(blockIdx.x) * teams_per_block + threadIdx.x / W;
			float2 st = make_float2(0.0f, 0.0f);
			auto fetch = [&](long long row)
			{
				x.template load<W>(input + row * channels, lane, channels);
				d.template load<W>(dy + row * channels, lane, channels);
				if (ext != nullptr)
					e.template load<W>(ext + row * channels, lane, channels);
				st = stats[row];
			};
			if (r < rows)
				fetch(r);
			for (; r < rows; r += teams)
			{
				float xh[E], gy[E];
				float s1 = 0.0f, s2 = 0.0f;
				const float mean = st.x, inv_stddev = st.y;
#pragma unroll
				for (int k = 0; k < E; k++)
				{
					const bool inside = k * W + lane < channels;
					const float dv = d.get(k);
					xh[k] = inside ? (x.get(k) + (ext != nullptr ? e.get(k) : 0.0f) - mean) * inv_stddev : 0.0f;
					gy[k] = dv * (gamma != nullptr ? g.get(k) : 1.0f);
					s1 += gy[k];
					s2 += gy[k] * xh[k];
					sum_w[k] += dv * xh[k];
					sum_b[k] += dv;
				}
				if (r + teams < rows)
					fetch(r + teams);
				team_sum<W>(s1, s2, scratch, turn);
				s1 *= inv_n;
				s2 *= inv_n1;
#pragma unroll
				for (int k = 0; k < E; k++)
				{
					const int c = k * W + lane;
					if (c >= channels)
						continue;
					T *dst = dx + r * channels + c;
					const float v = inv_stddev * (gy[k] - s1 - xh[k] * s2);
					*dst = from_float<T>(beta_dx != 0.0f ? v + beta_dx * to_float(*dst) : v);
				}
			}

			let_next_grid_start();
			if (W == 32)
			{ // eight teams hold sums of the same columns: the first adds the others', one quantity after the other
				const int warp = threadIdx.x / 32;
#pragma unroll
				for (int what = 0; what < 2; what++)
				{
					__syncthreads();
					if (warp > 0)
					{
#pragma unroll
						for (int k = 0; k < E; k++)
							columns[((warp - 1) * E + k) * 32 + lane] = what == 0 ? sum_w[k] : sum_b[k];
					}
					__syncthreads();
					if (warp == 0)
					{
#pragma unroll
						for (int k = 0; k < E; k++)
						{
							float s = what == 0 ? sum_w[k] : sum_b[k];
#pragma unroll
							for (int t = 0; t < 7; t++)
								s += columns[(t * E + k) * 32 + lane];
							(what == 0 ? sum_w[k] : sum_b[k]) = s;
						}
					}
				}
				if (warp > 0)
					return;
			}
#pragma unroll
			for (int k = 0; k < E; k++)
			{
				const int c = k * W + lane;
				if (c < channels)
				{
					partial[static_cast<long long>(blockIdx.x) * channels + c] = sum_w[k];
					partial[(static_cast<long long>(gridDim.x) + blockIdx.x) * channels + c] = sum_b[k];
				}
			}
		}

		/* ---------------------------------------------------------------- rows through a ring in shared memory
		 * Rows of 16-byte multiples and more than 512 elements: a block is one team and has a ring of stages, a stage is one row of each operand, and the
		 * first thread asks for a row by bulk copies `stages` rows ahead, as soon as the team has taken the stage's last row into registers.  More bytes are in flight than
		 * registers could hold, and the arithmetic works on pairs of values: on fp16 rows these kernels run out of issue slots before memory.
		 * Measured, 8192 x 4096 fp16 with a summand: forward 47 -> 39 us, backward 99 -> 51 us (6.5 TB/s would be 31 and 41). */
		constexpr int RING_BYTES = 192 * 1024; // of an SM, shared by its blocks
		constexpr int MAX_STAGES = 8;
		struct RingBarriers
		{
				uint64_t full[MAX_STAGES];
				int abort_flag;
		};
		struct RingShape
		{
				int stages, row_bytes, operands; // operands of a stage: x, then dy (backward), then ext
		};
		struct Ring
		{
				RingBarriers &bars;
				const RingShape &shape;
				uint8_t *memory;
				int stage = 0;
				uint32_t parity = 0;
				const void *sources[3];
				__device__ __forceinline__ Ring(RingBarriers &barriers, const RingShape &ring_shape, uint8_t *ring_memory, const void *x, const void *dy, const void *ext) :
						bars(barriers),
						shape(ring_shape),
						memory(ring_memory),
						sources { x, dy, ext }
				{
					if (threadIdx.x == 0)
					{
						for (int k = 0; k < shape.stages; k++)
							tc::mbar_init(tc::smem_u32(&bars.full[k]), 1);
						bars.abort_flag = 0;
						tc::fence_mbar_init();
					}
					__syncthreads();
				}
				/* The first thread: row r into stage k. */
				__device__ __forceinline__ void ask(long long r, int k)
				{
					const uint32_t full = tc::smem_u32(&bars.full[k]);
					tc::mbar_arrive_expect_tx(full, shape.operands * shape.row_bytes);
					uint32_t dst = tc::smem_u32(memory) + k * shape.operands * shape.row_bytes;
#pragma unroll
					for (int i = 0; i < 3; i++)
						if (sources[i] != nullptr)
						{
							asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
									:: "r"(dst), "l"(reinterpret_cast<uint64_t>(sources[i]) + r * shape.row_bytes), "r"(shape.row_bytes), "r"(full) : "memory");
							dst += shape.row_bytes;
						}
				}
				__device__ __forceinline__ void start(long long r, long long step, long long rows)
				{
					if (threadIdx.x == 0)
						for (int k = 0; k < shape.stages && r < rows; k++, r += step)
							ask(r, k);
				}
				/* The oldest stage's row, or null when its copies did not arrive. */
				__device__ __forceinline__ const uint8_t* take()
				{
					return tc::mbar_wait_all_lanes(tc::smem_u32(&bars.full[stage]), parity, &bars.abort_flag) ? memory + stage * shape.operands * shape.row_bytes : nullptr;
				}
				/* After a barrier of the team past its last read of the stage: asks for row r in its place. */
				__device__ __forceinline__ void release(long long r, long long rows)
				{
					if (threadIdx.x == 0 && r < rows)
						ask(r, stage);
					if (++stage == shape.stages)
					{
						stage = 0;
						parity ^= 1u;
					}
				}
		};
		__device__ __forceinline__ void ring_report(RingBarriers &bars, int *status)
		{
			__syncthreads();
			if (bars.abort_flag != 0)
			{
				if (threadIdx.x == 0 && status != nullptr)
					atomicExch(status, 1);
				__nanosleep(1000000); // give copies that are still in flight time to land before the block retires
			}
		}

		/* A thread's share of a row, E elements in 16-byte pieces, handed out in pairs. */
		template<typename T, int W, int E>
		struct RowPairs
		{
				static constexpr int VEC = 16 / sizeof(T), N = E / VEC;
				uint4 p[N];
				__device__ __forceinline__ void load(const void *row, int lane, int channels)
				{
#pragma unroll
					for (int i = 0; i < N; i++)
					{
						const int c = (i * W + lane) * VEC;
						p[i] = c < channels ? *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(row) + c) : make_uint4(0, 0, 0, 0);
					}
				}
				__device__ __forceinline__ Pair get(int j) const
				{ // elements 2 j and 2 j + 1
					if constexpr (sizeof(T) == 2)
					{
						const uint4 &v = p[j / 4];
						const uint32_t w = j % 4 == 0 ? v.x : j % 4 == 1 ? v.y : j % 4 == 2 ? v.z : v.w;
						const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
						return Pair { f.x, f.y };
					}
					else
					{
						const uint4 &v = p[j / 2];
						return j % 2 == 0 ? Pair { __uint_as_float(v.x), __uint_as_float(v.y) } : Pair { __uint_as_float(v.z), __uint_as_float(v.w) };
					}
				}
				/* piece i from its pairs */
				static __device__ __forceinline__ uint4 pack(const Pair *v)
				{
					if constexpr (sizeof(T) == 2)
						return make_uint4(tc::pack_half2(v[0].x, v[0].y), tc::pack_half2(v[1].x, v[1].y), tc::pack_half2(v[2].x, v[2].y), tc::pack_half2(v[3].x, v[3].y));
					else
						return make_uint4(__float_as_uint(v[0].x), __float_as_uint(v[0].y), __float_as_uint(v[1].x), __float_as_uint(v[1].y));
				}
		};
		/* Sum over a team: one value, or two at once.  Two values take five shuffles, not ten: the first step leaves
		 * each half of the warp with one of them.  Several warps meet in `scratch`, two halves in turn (see team_sum). */
		struct alignas(16) RingScratch
		{
				float v[2][2][16];
		};
		template<int W>
		__device__ __forceinline__ void ring_sum(float &a, float &b, RingScratch &scratch, uint32_t &turn)
		{
			const int lane = threadIdx.x % 32;
			const bool upper = lane >= 16;
			float v = (upper ? b : a) + __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
#pragma unroll
			for (int k = 8; k >= 1; k /= 2)
				v += __shfl_xor_sync(0xffffffffu, v, k);
			const int half = turn & 1u;
			turn++;
			if (lane % 16 == 0)
				scratch.v[half][upper][threadIdx.x / 32] = v;
			__syncthreads();
			a = b = 0.0f;
#pragma unroll
			for (int k = 0; k < W / 32; k += 4)
			{
				const float4 ta = *reinterpret_cast<const float4*>(&scratch.v[half][0][k]), tb = *reinterpret_cast<const float4*>(&scratch.v[half][1][k]);
				a += (ta.x + ta.y) + (ta.z + ta.w);
				b += (tb.x + tb.y) + (tb.z + tb.w);
			}
		}
		template<int W>
		__device__ __forceinline__ float ring_sum(float a, RingScratch &scratch, uint32_t &turn)
		{
#pragma unroll
			for (int k = 16; k >= 1; k /= 2)
				a += __shfl_xor_sync(0xffffffffu, a, k);
			const int half = turn & 1u;
			turn++;
			if (threadIdx.x % 32 == 0)
				scratch.v[half][0][threadIdx.x / 32] = a;
			__syncthreads();
			a = 0.0f;
#pragma unroll
			for (int k = 0; k < W / 32; k += 4)
			{
				const float4 t = *reinterpret_cast<const float4*>(&scratch.v[half][0][k]);
				a += (t.x + t.y) + (t.z + t.w);
			}
			return a;
		}
		/* Blocks per SM: enough to fill it, few enough that their partial rows (backward) cost little and their registers fit. */
		template<int W>
		constexpr int ring_blocks()
		{
			return W == 128 ? 4 : W == 256 ? 2 : 1;
		}

		template<int W, int E, int VEC>
		__device__ __forceinline__ void write_partial(float *__restrict__ partial, const Pair (&sum_w)[E / 2], const Pair (&sum_b)[E / 2], int lane, int channels)
		{
#pragma unroll
			for (int i = 0; i < E / VEC; i++)
			{
				const int c = (i * W + lane) * VEC;
				if (c >= channels)
					continue;
				float *w_row = partial + static_cast<long long>(blockIdx.x) * channels + c, *b_row = partial + (static_cast<long long>(gridDim.x) + blockIdx.x) * channels + c;
#pragma unroll
				for (int j = 0; j < VEC / 2; j += 2)
				{
					const int k = i * VEC / 2 + j;
					*reinterpret_cast<float4*>(w_row + 2 * j) = make_float4(sum_w[k].x, sum_w[k].y, sum_w[k + 1].x, sum_w[k + 1].y);
					*reinterpret_cast<float4*>(b_row + 2 * j) = make_float4(sum_b[k].x, sum_b[k].y, sum_b[k + 1].x, sum_b[k + 1].y);
				}
			}
		}

		/* ---------------------------------------------------------------- rows of up to 512 elements, 16-byte multiples
		 * A row is one warp's, ROWS of them at a time: their loads are in flight together, and so are the shuffles of their sums, which is what a single
		 * short row would wait for.  Measured, 57 600 x 256 fp16: forward 20 us, backward 25 us (one row at a time: 22 and 40). */
		constexpr int ROW_WARPS = 8;
		__device__ __forceinline__ float warp_sum(float v)
		{
#pragma unroll
			for (int k = 16; k >= 1; k /= 2)
				v += __shfl_xor_sync(0xffffffffu, v, k);
			return v;
		}
		template<typename T, int E, int ROWS, bool HAS_EXT>
		__global__ void __launch_bounds__(ROW_WARPS * 32, E == 8 ? 3 : 2) kernel_layernorm_train_rows(T *output, const T *input, const T *ext, const T *__restrict__ gamma, const T *__restrict__ beta,
				float2 *__restrict__ stats, long long rows, int channels)
		{
			using Part = RowPairs<T, 32, E>;
			constexpr int VEC = Part::VEC, N = Part::N, PAIRS = E / 2;
			const int lane = threadIdx.x % 32;
			const float inv_n = 1.0f / static_cast<float>(channels), inv_n1 = 1.0f / static_cast<float>(channels - 1);
			const long long step = static_cast<long long>(gridDim.x) * ROW_WARPS;
			Part g, b;
			if (gamma != nullptr)
				g.load(gamma, lane, channels);
			if (beta != nullptr)
				b.load(beta, lane, channels);
			for (long long r0 = static_cast<long long>(blockIdx.x) * ROW_WARPS + threadIdx.x / 32; r0 < rows; r0 += step * ROWS)
			{
				Part x[ROWS], e[HAS_EXT ? ROWS : 1];
#pragma unroll
				for (int q = 0; q < ROWS; q++)
				{
					const long long r = r0 + q * step;
					x[q].load(input + r * channels, lane, r < rows ? channels : 0);
					if (HAS_EXT)
						e[HAS_EXT ? q : 0].load(ext + r * channels, lane, r < rows ? channels : 0);
				}
				Pair v[ROWS][PAIRS];
				float mean[ROWS], squares[ROWS];
#pragma unroll
				for (int q = 0; q < ROWS; q++)
				{
					Pair sum = pair_of(0.0f);
#pragma unroll
					for (int j = 0; j < PAIRS; j++)
					{
						v[q][j] = HAS_EXT ? pair_add(x[q].get(j), e[HAS_EXT ? q : 0].get(j)) : x[q].get(j);
						sum = pair_add(sum, v[q][j]);
					}
					mean[q] = sum.x + sum.y;
				}
#pragma unroll
				for (int q = 0; q < ROWS; q++)
					mean[q] = warp_sum(mean[q]) * inv_n;
#pragma unroll
				for (int q = 0; q < ROWS; q++)
				{
					Pair sum = pair_of(0.0f);
#pragma unroll
					for (int i = 0; i < N; i++)
						if ((i * 32 + lane) * VEC < channels)
						{
#pragma unroll
							for (int j = i * VEC / 2; j < (i + 1) * VEC / 2; j++)
							{
								v[q][j] = pair_add(v[q][j], pair_of(-mean[q]));
								sum = pair_fma(v[q][j], v[q][j], sum);
							}
						}
					squares[q] = sum.x + sum.y;
				}
#pragma unroll
				for (int q = 0; q < ROWS; q++)
					squares[q] = 1.0f / sqrtf(EPSILON + warp_sum(squares[q]) * inv_n1);
#pragma unroll
				for (int q = 0; q < ROWS; q++)
				{
					const long long r = r0 + q * step;
					if (r >= rows)
						break;
					if (lane == 0)
						stats[r] = make_float2(mean[q], squares[q]);
#pragma unroll
					for (int i = 0; i < N; i++)
					{
						const int c = (i * 32 + lane) * VEC;
						if (c >= channels)
							continue;
						Pair out[VEC / 2];
#pragma unroll
						for (int j = 0; j < VEC / 2; j++)
						{
							const int k = i * VEC / 2 + j;
							const Pair scaled = pair_mul(v[q][k], pair_of(squares[q]));
							out[j] = pair_fma(scaled, gamma != nullptr ? g.get(k) : pair_of(1.0f), beta != nullptr ? b.get(k) : pair_of(0.0f));
						}
						*reinterpret_cast<uint4*>(output + r * channels + c) = Part::pack(out);
					}
				}
			}
		}
		template<typename T, int E, int ROWS, bool HAS_EXT>
		__global__ void __launch_bounds__(ROW_WARPS * 32, 2) kernel_layernorm_backward_rows(T *dx, const T *input, const T *ext, const T *dy, const T *__restrict__ gamma,
				const float2 *__restrict__ stats, float beta_dx, float *__restrict__ partial, long long rows, int channels)
		{
			using Part = RowPairs<T, 32, E>;
			constexpr int VEC = Part::VEC, N = Part::N, PAIRS = E / 2;
			__shared__ Pair columns[2][ROW_WARPS - 1][PAIRS][32]; // the other warps' column sums
			const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
			const float inv_n = 1.0f / static_cast<float>(channels), inv_n1 = 1.0f / static_cast<float>(channels - 1);
			const long long step = static_cast<long long>(gridDim.x) * ROW_WARPS;
			Part g;
			if (gamma != nullptr)
				g.load(gamma, lane, channels);
			Pair sum_w[PAIRS], sum_b[PAIRS];
#pragma unroll
			for (int j = 0; j < PAIRS; j++)
				sum_w[j] = sum_b[j] = pair_of(0.0f);
			for (long long r0 = static_cast<long long>(blockIdx.x) * ROW_WARPS + warp; r0 < rows; r0 += step * ROWS)
			{
				Part x[ROWS], d[ROWS], e[HAS_EXT ? ROWS : 1];
				float2 st[ROWS];
#pragma unroll
				for (int q = 0; q < ROWS; q++)
				{
					const long long r = r0 + q * step;
					const int inside = r < rows ? channels : 0; // a row beyond the last: zeros everywhere
					x[q].load(input + r * channels, lane, inside);
					d[q].load(dy + r * channels, lane, inside);
					if (HAS_EXT)
						e[HAS_EXT ? q : 0].load(ext + r * channels, lane, inside);
					st[q] = r < rows ? stats[r] : make_float2(0.0f, 0.0f);
				}
				Pair xh[ROWS][PAIRS];
				float s1[ROWS], s2[ROWS];
#pragma unroll
				for (int q = 0; q < ROWS; q++)
				{
					Pair t1 = pair_of(0.0f), t2 = pair_of(0.0f);
#pragma unroll
					for (int j = 0; j < PAIRS; j++)
					{
						Pair v = x[q].get(j);
						if (HAS_EXT) // first, as in the forward pass: where x and ext cancel, their sum is exact and x - mean is not
							v = pair_add(v, e[HAS_EXT ? q : 0].get(j));
						v = pair_add(v, pair_of(-st[q].x)); // before the factor: a large mean must not cost the difference its digits
						const Pair dv = d[q].get(j), gy = gamma != nullptr ? pair_mul(dv, g.get(j)) : dv;
						xh[q][j] = pair_mul(v, pair_of(st[q].y));
						t1 = pair_add(t1, gy);
						t2 = pair_fma(gy, xh[q][j], t2);
						sum_w[j] = pair_fma(dv, xh[q][j], sum_w[j]);
						sum_b[j] = pair_add(sum_b[j], dv);
					}
					s1[q] = t1.x + t1.y;
					s2[q] = t2.x + t2.y;
				}
#pragma unroll
				for (int q = 0; q < ROWS; q++)
				{
					s1[q] = warp_sum(s1[q]);
					s2[q] = warp_sum(s2[q]);
				}
#pragma unroll
				for (int q = 0; q < ROWS; q++)
				{
					const long long r = r0 + q * step;
					if (r >= rows)
						break;
					const Pair less = pair_of(-s1[q] * inv_n * st[q].y), slope = pair_of(-s2[q] * inv_n1 * st[q].y);
#pragma unroll
					for (int i = 0; i < N; i++)
					{
						const int c = (i * 32 + lane) * VEC;
						if (c >= channels)
							continue;
						T *dst = dx + r * channels + c;
						Pair out[VEC / 2];
#pragma unroll
						for (int j = 0; j < VEC / 2; j++)
						{
							const int k = i * VEC / 2 + j;
							const Pair dv = d[q].get(k), gy = gamma != nullptr ? pair_mul(dv, g.get(k)) : dv;
							out[j] = pair_fma(gy, pair_of(st[q].y), pair_fma(xh[q][k], slope, less));
						}
						if (beta_dx != 0.0f)
						{
#pragma unroll
							for (int j = 0; j < VEC; j++)
								(j % 2 == 0 ? out[j / 2].x : out[j / 2].y) += beta_dx * to_float(dst[j]);
						}
						*reinterpret_cast<uint4*>(dst) = Part::pack(out);
					}
				}
			}
			let_next_grid_start();
			if (warp > 0)
			{
#pragma unroll
				for (int j = 0; j < PAIRS; j++)
				{
					columns[0][warp - 1][j][lane] = sum_w[j];
					columns[1][warp - 1][j][lane] = sum_b[j];
				}
			}
			__syncthreads();
			if (warp > 0)
				return;
#pragma unroll
			for (int j = 0; j < PAIRS; j++)
#pragma unroll
				for (int t = 0; t < ROW_WARPS - 1; t++)
				{
					sum_w[j] = pair_add(sum_w[j], columns[0][t][j][lane]);
					sum_b[j] = pair_add(sum_b[j], columns[1][t][j][lane]);
				}
			write_partial<32, E, VEC>(partial, sum_w, sum_b, lane, channels);
		}

		template<typename T, int W, int E>
		__global__ void __launch_bounds__(W, ring_blocks<W>()) kernel_layernorm_train_ring(T *output, const T *input, const T *ext, const T *__restrict__ gamma,
				const T *__restrict__ beta, float2 *__restrict__ stats, long long rows, int channels, const RingShape shape, int *status)
		{
			using Part = RowPairs<T, W, E>;
			constexpr int VEC = Part::VEC, N = Part::N, PAIRS = E / 2;
			extern __shared__ __align__(128) uint8_t ring_memory[];
			__shared__ RingBarriers bars;
			__shared__ RingScratch scratch;
			Ring ring(bars, shape, ring_memory, input, nullptr, ext);
			const int lane = threadIdx.x;
			const long long step = gridDim.x, first = blockIdx.x;
			ring.start(first, step, rows);
			{
				uint32_t turn = 0;
				Pair g[PAIRS], b[PAIRS];
				{
					Part raw;
					if (gamma != nullptr)
						raw.load(gamma, lane, channels);
#pragma unroll
					for (int j = 0; j < PAIRS; j++)
						g[j] = gamma != nullptr ? raw.get(j) : pair_of(1.0f);
					if (beta != nullptr)
						raw.load(beta, lane, channels);
#pragma unroll
					for (int j = 0; j < PAIRS; j++)
						b[j] = beta != nullptr ? raw.get(j) : pair_of(0.0f);
				}
				const float inv_n = 1.0f / static_cast<float>(channels), inv_n1 = 1.0f / static_cast<float>(channels - 1);
				for (long long r = first; r < rows; r += step)
				{
					const uint8_t *row = ring.take();
					if (row == nullptr)
						break;
					Pair v[PAIRS];
					Pair sum = pair_of(0.0f);
					Part x;
					x.load(row, lane, channels);
#pragma unroll
					for (int j = 0; j < PAIRS; j++)
						v[j] = x.get(j);
					if (ext != nullptr)
					{
						x.load(row + shape.row_bytes, lane, channels);
#pragma unroll
						for (int j = 0; j < PAIRS; j++)
							v[j] = pair_add(v[j], x.get(j));
					}
#pragma unroll
					for (int j = 0; j < PAIRS; j++)
						sum = pair_add(sum, v[j]);
					const float mean = ring_sum<W>(sum.x + sum.y, scratch, turn) * inv_n;
					ring.release(r + shape.stages * step, rows);
					Pair squares = pair_of(0.0f);
#pragma unroll
					for (int i = 0; i < N; i++)
						if ((i * W + lane) * VEC < channels)
						{
#pragma unroll
							for (int j = i * VEC / 2; j < (i + 1) * VEC / 2; j++)
							{
								v[j] = pair_add(v[j], pair_of(-mean));
								squares = pair_fma(v[j], v[j], squares);
							}
						}
					const float inv_stddev = 1.0f / sqrtf(EPSILON + ring_sum<W>(squares.x + squares.y, scratch, turn) * inv_n1);
					if (lane == 0)
						stats[r] = make_float2(mean, inv_stddev);
#pragma unroll
					for (int i = 0; i < N; i++)
					{
						const int c = (i * W + lane) * VEC;
						if (c >= channels)
							continue;
						Pair out[VEC / 2];
#pragma unroll
						for (int j = 0; j < VEC / 2; j++)
							out[j] = pair_fma(pair_mul(v[i * VEC / 2 + j], pair_of(inv_stddev)), g[i * VEC / 2 + j], b[i * VEC / 2 + j]);
						*reinterpret_cast<uint4*>(output + r * channels + c) = Part::pack(out);
					}
				}
			}
			ring_report(bars, status);
		}

		/* (Elements beyond the row come out of RowPairs as zeros in dy, so they add nothing to any of the four sums.) */
		template<typename T, int W, int E>
		__global__ void __launch_bounds__(W, ring_blocks<W>()) kernel_layernorm_backward_ring(T *dx, const T *input, const T *ext, const T *dy, const T *__restrict__ gamma,
				const float2 *__restrict__ stats, float beta_dx, float *__restrict__ partial, long long rows, int channels, const RingShape shape, int *status)
		{
			using Part = RowPairs<T, W, E>;
			constexpr int VEC = Part::VEC, N = Part::N, PAIRS = E / 2;
			extern __shared__ __align__(128) uint8_t ring_memory[];
			__shared__ RingBarriers bars;
			__shared__ RingScratch scratch;
			Ring ring(bars, shape, ring_memory, input, dy, ext);
			const int lane = threadIdx.x;
			const long long step = gridDim.x, first = blockIdx.x;
			ring.start(first, step, rows);
			Pair sum_w[PAIRS], sum_b[PAIRS];
#pragma unroll
			for (int j = 0; j < PAIRS; j++)
				sum_w[j] = sum_b[j] = pair_of(0.0f);
			{
				const float inv_n = 1.0f / static_cast<float>(channels), inv_n1 = 1.0f / static_cast<float>(channels - 1);
				uint32_t turn = 0;
				Part g;
				if (gamma != nullptr)
					g.load(gamma, lane, channels);
				float2 st = first < rows ? stats[first] : make_float2(0.0f, 0.0f);
				for (long long r = first; r < rows; r += step)
				{
					const float mean = st.x, inv_stddev = st.y;
					if (r + step < rows)
						st = stats[r + step];
					const uint8_t *row = ring.take();
					if (row == nullptr)
						break;
					Pair xh[PAIRS];
					Part x, d;
					Pair t1 = pair_of(0.0f), t2 = pair_of(0.0f);
					x.load(row, lane, channels);
					d.load(row + shape.row_bytes, lane, channels);
#pragma unroll
					for (int j = 0; j < PAIRS; j++)
						xh[j] = x.get(j);
					if (ext != nullptr)
					{ // first, as in the forward pass: where x and ext cancel, their sum is exact and x - mean is not
						x.load(row + 2 * shape.row_bytes, lane, channels);
#pragma unroll
						for (int j = 0; j < PAIRS; j++)
							xh[j] = pair_add(xh[j], x.get(j));
					}
#pragma unroll
					for (int j = 0; j < PAIRS; j++)
					{
						const Pair dv = d.get(j), gy = gamma != nullptr ? pair_mul(dv, g.get(j)) : dv;
						// the mean before the factor: a large one must not cost the difference its digits
						xh[j] = pair_mul(pair_add(xh[j], pair_of(-mean)), pair_of(inv_stddev));
						t1 = pair_add(t1, gy);
						t2 = pair_fma(gy, xh[j], t2);
						sum_w[j] = pair_fma(dv, xh[j], sum_w[j]);
						sum_b[j] = pair_add(sum_b[j], dv);
					}
					float s1 = t1.x + t1.y, s2 = t2.x + t2.y;
					ring_sum<W>(s1, s2, scratch, turn);
					ring.release(r + shape.stages * step, rows);
					const Pair less = pair_of(-s1 * inv_n * inv_stddev), slope = pair_of(-s2 * inv_n1 * inv_stddev);
#pragma unroll
					for (int i = 0; i < N; i++)
					{
						const int c = (i * W + lane) * VEC;
						if (c >= channels)
							continue;
						T *dst = dx + r * channels + c;
						Pair out[VEC / 2];
#pragma unroll
						for (int j = 0; j < VEC / 2; j++)
						{
							const int k = i * VEC / 2 + j;
							const Pair dv = d.get(k), gy = gamma != nullptr ? pair_mul(dv, g.get(k)) : dv;
							out[j] = pair_fma(gy, pair_of(inv_stddev), pair_fma(xh[k], slope, less));
						}
						if (beta_dx != 0.0f)
						{
#pragma unroll
							for (int j = 0; j < VEC; j++)
								(j % 2 == 0 ? out[j / 2].x : out[j / 2].y) += beta_dx * to_float(dst[j]);
						}
						*reinterpret_cast<uint4*>(dst) = Part::pack(out);
					}
				}
			}
			let_next_grid_start();
			ring_report(bars, status);
			write_partial<W, E, VEC>(partial, sum_w, sum_b, lane, channels);
		}

		/* Rows longer than a team's registers hold: one block a row, which is read again (from L2) by each pass over it. */
		constexpr int LONG_THREADS = 512;
		template<typename T>
		__global__ void __launch_bounds__(LONG_THREADS) kernel_layernorm_train_long(T *output, const T *input, const T *ext, const T *__restrict__ gamma,
				const T *__restrict__ beta, float2 *__restrict__ stats, long long rows, int channels)
		{
			__shared__ float2 scratch[2][16];
			uint32_t turn = 0;
			for (long long r = blockIdx.x; r < rows; r += gridDim.x)
			{
				const long long at = r * channels;
				auto value = [&](int c)
				{
					return to_float(input[at + c]) + (ext != nullptr ? to_float(ext[at + c]) : 0.0f);
				};
				float sum = 0.0f, var = 0.0f, unused = 0.0f;
				for (int c = threadIdx.x; c < channels; c += LONG_THREADS)
					sum += value(c);
				team_sum<LONG_THREADS>(sum, unused, scratch, turn);
				const float mean = sum / static_cast<float>(channels);
				for (int c = threadIdx.x; c < channels; c += LONG_THREADS)
					var += (value(c) - mean) * (value(c) - mean);
				team_sum<LONG_THREADS>(var, unused, scratch, turn);
				const float inv_stddev = 1.0f / sqrtf(EPSILON + var / static_cast<float>(channels - 1));
				if (threadIdx.x == 0)
					stats[r] = make_float2(mean, inv_stddev);
				for (int c = threadIdx.x; c < channels; c += LONG_THREADS)
					output[at + c] = from_float<T>((gamma != nullptr ? to_float(gamma[c]) : 1.0f) * (value(c) - mean) * inv_stddev + (beta != nullptr ? to_float(beta[c]) : 0.0f));
			}
		}
		template<typename T>
		__global__ void __launch_bounds__(LONG_THREADS) kernel_layernorm_backward_long(T *dx, const T *input, const T *ext, const T *dy, const T *__restrict__ gamma,
				const float2 *__restrict__ stats, float beta_dx, long long rows, int channels)
		{
			__shared__ float2 scratch[2][16];
			uint32_t turn = 0;
			for (long long r = blockIdx.x; r < rows; r += gridDim.x)
			{
				const long long at = r * channels;
				const float2 st = stats[r];
				auto normalised = [&](int c)
				{
					return (to_float(input[at + c]) + (ext != nullptr ? to_float(ext[at + c]) : 0.0f) - st.x) * st.y;
				};
				auto scaled = [&](int c)
				{
					return to_float(dy[at + c]) * (gamma != nullptr ? to_float(gamma[c]) : 1.0f);
				};
				float s1 = 0.0f, s2 = 0.0f;
				for (int c = threadIdx.x; c < channels; c += LONG_THREADS)
				{
					s1 += scaled(c);
					s2 += scaled(c) * normalised(c);
				}
				team_sum<LONG_THREADS>(s1, s2, scratch, turn);
				for (int c = threadIdx.x; c < channels; c += LONG_THREADS)
				{
					const float v = st.y * (scaled(c) - s1 / static_cast<float>(channels) - normalised(c) * (s2 / static_cast<float>(channels - 1)));
					dx[at + c] = from_float<T>(beta_dx != 0.0f ? v + beta_dx * to_float(dx[at + c]) : v);
				}
			}
		}
		/* The column sums for those rows, a thread a column; block y takes rows y, y + gridDim.y, ... (launched before the kernel above,
		 * which may overwrite dy or x). */
		template<typename T>
		__global__ void __launch_bounds__(256) kernel_layernorm_columns(float *__restrict__ partial, const T *__restrict__ input, const T *__restrict__ ext, const T *__restrict__ dy,
				const float2 *__restrict__ stats, long long rows, int channels)
		{
			const int c = blockIdx.x * 256 + threadIdx.x;
			if (c >= channels)
				return;
			float sum_w = 0.0f, sum_b = 0.0f;
			for (long long r = blockIdx.y; r < rows; r += gridDim.y)
			{
				const float2 st = stats[r];
				const float d = to_float(dy[r * channels + c]);
				sum_w += d * (to_float(input[r * channels + c]) + (ext != nullptr ? to_float(ext[r * channels + c]) : 0.0f) - st.x) * st.y;
				sum_b += d;
			}
			partial[static_cast<long long>(blockIdx.y) * channels + c] = sum_w;
			partial[(static_cast<long long>(gridDim.y) + blockIdx.y) * channels + c] = sum_b;
		}

		/* dw, db = the sum of the partial rows (+ beta * the old value).  A block takes 32 columns of one of the two; its 32 warps add
		 * every 32nd row and then each other's sums, always in the same order. */
		template<typename G>
		__global__ void __launch_bounds__(1024) kernel_layernorm_add_partials(G *dw, G *db, const float *partial, int blocks, int channels, float beta)
		{
			__shared__ float sums[32][33];
			G *out = blockIdx.y == 0 ? dw : db;
			const float *src = partial + static_cast<long long>(blockIdx.y) * blocks * channels;
			const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
			const int c = blockIdx.x * 32 + lane;
			wait_for_previous_grid();
			if (out == nullptr)
				return;
			float s = 0.0f;
			if (c < channels)
			{
#pragma unroll 8
				for (int b = warp; b < blocks; b += 32)
					s += src[static_cast<long long>(b) * channels + c];
			}
			sums[warp][lane] = s;
			__syncthreads();
			if (warp == 0 && c < channels)
			{
				s = 0.0f;
#pragma unroll
				for (int k = 0; k < 32; k++)
					s += sums[k][lane];
				out[c] = from_float<G>(beta != 0.0f ? s + beta * to_float(out[c]) : s);
			}
		}

		constexpr int LONGEST_TEAM_ROW = 512 * 16;
		int blocks_per_sm(int channels)
		{
			return channels <= 512 ? 2 : channels <= 2048 ? ring_blocks<128>() : channels <= 4096 ? ring_blocks<256>() : ring_blocks<512>();
		}
		int team_blocks(int sm_count, long long rows, int channels, int per_sm)
		{
			const int teams_per_block = channels <= 512 ? 8 : 1;
			return static_cast<int>(std::max<long long>(1, std::min<long long>((rows + teams_per_block - 1) / teams_per_block, static_cast<long long>(sm_count) * per_sm)));
		}
		int long_row_chunks(int sm_count, long long rows, int channels)
		{ // row groups of kernel_layernorm_columns: enough blocks to fill the device
			return static_cast<int>(std::max<long long>(1, std::min<long long>(rows, static_cast<long long>(sm_count) * 8 / ((channels + 255) / 256))));
		}

		template<typename T>
		struct Args
		{
				T *out;
				const T *x, *ext, *dy, *gamma, *beta;
				float2 *stats;
				float beta_dx;
				float *partial;
				long long rows;
				int channels, blocks;
				int *status;
		};
		/* The ring's kernels need their shared memory opted in to, once per device. */
		template<typename K>
		bool opt_in(K kernel, int device, bool (&done)[MAX_DEVICES])
		{
			static std::mutex mutex;
			std::lock_guard<std::mutex> lock(mutex);
			if (!done[device])
				done[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RING_BYTES) == cudaSuccess;
			return done[device];
		}
		template<typename T, bool WIDE, int W, int E>
		void launch_team(mlContext_t ctx, cudaStream_t stream, const Args<T> &a, bool backward)
		{
			if constexpr (WIDE && W == 32)
			{
				// as many rows at once as the registers hold
				constexpr int ROWS = 32 / E / (sizeof(T) == 4 ? 2 : 1), FEWER = ROWS > 1 ? ROWS / 2 : 1, BACKWARD_ROWS = E == 8 ? ROWS : 1;
				const int threads = ROW_WARPS * 32;
				if (backward && a.ext != nullptr)
					kernel_layernorm_backward_rows<T, E, (E == 8 ? FEWER : 1), true> <<<a.blocks, threads, 0, stream>>>(a.out, a.x, a.ext, a.dy, a.gamma, a.stats, a.beta_dx, a.partial, a.rows, a.channels);
				else if (backward)
					kernel_layernorm_backward_rows<T, E, BACKWARD_ROWS, false> <<<a.blocks, threads, 0, stream>>>(a.out, a.x, a.ext, a.dy, a.gamma, a.stats, a.beta_dx, a.partial, a.rows, a.channels);
				else if (a.ext != nullptr)
					kernel_layernorm_train_rows<T, E, FEWER, true> <<<a.blocks, threads, 0, stream>>>(a.out, a.x, a.ext, a.gamma, a.beta, a.stats, a.rows, a.channels);
				else
					kernel_layernorm_train_rows<T, E, ROWS, false> <<<a.blocks, threads, 0, stream>>>(a.out, a.x, a.ext, a.gamma, a.beta, a.stats, a.rows, a.channels);
			}
			else if constexpr (WIDE)
			{
				static bool forward_done[MAX_DEVICES] = { }, backward_done[MAX_DEVICES] = { };
				const int device = get(ctx)->device;
				RingShape shape;
				shape.row_bytes = a.channels * static_cast<int>(sizeof(T));
				shape.operands = (backward ? 2 : 1) + (a.ext != nullptr ? 1 : 0);
				const int stage_bytes = shape.operands * shape.row_bytes;
				const int share = RING_BYTES / blocks_per_sm(a.channels) / 1024 * 1024 - 2048; // beside the barriers
				const int rows_of_block = static_cast<int>(std::min<long long>(MAX_STAGES, (a.rows + a.blocks - 1) / a.blocks));
				shape.stages = std::min(rows_of_block, std::max(2, share / stage_bytes));
				static_assert(2 * 3 * W * E * sizeof(T) <= RING_BYTES, "two stages of the longest rows of this team fit");
				if (device < 0 || device >= MAX_DEVICES
						|| !(backward ? opt_in(kernel_layernorm_backward_ring<T, W, E>, device, backward_done) : opt_in(kernel_layernorm_train_ring<T, W, E>, device, forward_done)))
				{
					record_error(ctx, "layer norm: %d bytes of shared memory are not available", RING_BYTES);
					return;
				}
				if (backward)
					kernel_layernorm_backward_ring<T, W, E> <<<a.blocks, W, shape.stages * stage_bytes, stream>>>(a.out, a.x, a.ext, a.dy, a.gamma, a.stats, a.beta_dx, a.partial, a.rows,
							a.channels, shape, a.status);
				else
					kernel_layernorm_train_ring<T, W, E> <<<a.blocks, W, shape.stages * stage_bytes, stream>>>(a.out, a.x, a.ext, a.gamma, a.beta, a.stats, a.rows, a.channels, shape,
							a.status);
			}
			else if (backward)
				kernel_layernorm_backward<T, W, E> <<<a.blocks, W == 32 ? 256 : W, 0, stream>>>(a.out, a.x, a.ext, a.dy, a.gamma, a.stats, a.beta_dx, a.partial, a.rows, a.channels);
			else
				kernel_layernorm_train<T, W, E> <<<a.blocks, W == 32 ? 256 : W, 0, stream>>>(a.out, a.x, a.ext, a.gamma, a.beta, a.stats, a.rows, a.channels);
		}
		template<typename T, bool WIDE>
		void launch_by_length(mlContext_t ctx, cudaStream_t stream, const Args<T> &a, bool backward)
		{
			if (a.channels <= 32 * 8)
				launch_team<T, WIDE, 32, 8>(ctx, stream, a, backward);
			else if (a.channels <= 32 * 16)
				launch_team<T, WIDE, 32, 16>(ctx, stream, a, backward);
			else if (a.channels <= 128 * 8)
				launch_team<T, WIDE, 128, 8>(ctx, stream, a, backward);
			else if (a.channels <= 128 * 16)
				launch_team<T, WIDE, 128, 16>(ctx, stream, a, backward);
			else if (a.channels <= 256 * 16)
				launch_team<T, WIDE, 256, 16>(ctx, stream, a, backward);
			else
				launch_team<T, WIDE, 512, 16>(ctx, stream, a, backward);
		}
		/* Through the ring when every row starts on a 16-byte boundary, else element by element into registers */
		template<typename T>
		void launch_rows(mlContext_t ctx, cudaStream_t stream, Args<T> a, bool backward)
		{
			constexpr int VEC = 16 / sizeof(T);
			const void *pointers[] = { a.out, a.x, a.ext, a.dy, a.gamma, a.beta, a.partial };
			bool wide = a.channels % VEC == 0;
			for (const void *p : pointers)
				wide = wide && aligned_to(p, 16);
			if (!backward)
			{ // narrow accesses: as many rows in flight as the registers allow
				const int sms = get(ctx)->sm_count;
				a.blocks = team_blocks(sms, a.rows, a.channels, wide ? (a.channels <= 512 ? 3 : blocks_per_sm(a.channels)) : a.channels <= 512 ? 8 : a.channels <= 2048 ? 16 : a.channels <= 4096 ? 8 : 4);
			}
			if (wide)
				launch_by_length<T, true>(ctx, stream, a, backward);
			else
				launch_by_length<T, false>(ctx, stream, a, backward);
		}

		template<typename T>
		void run_forward(mlContext_t ctx, Args<T> a)
		{
			cudaStream_t stream = use_stream(ctx);
			const long long sms = get(ctx)->sm_count;
			if (a.channels > LONGEST_TEAM_ROW)
				kernel_layernorm_train_long<T> <<<static_cast<int>(std::min<long long>(a.rows, sms * 4)), LONG_THREADS, 0, stream>>>(a.out, a.x, a.ext, a.gamma, a.beta, a.stats, a.rows,
						a.channels);
			else
			{
				a.status = get(ctx)->dev_status;
				launch_rows(ctx, stream, a, false);
			}
			MB200_COUNT_LAUNCH();
			check_cuda(ctx, cudaGetLastError(), "mb200_layernorm_forward");
		}
		template<typename T>
		bool run_backward(mlContext_t ctx, Args<T> a)
		{
			cudaStream_t stream = use_stream(ctx);
			const int sms = get(ctx)->sm_count;
			if (a.channels > LONGEST_TEAM_ROW)
			{
				a.blocks = long_row_chunks(sms, a.rows, a.channels);
				kernel_layernorm_columns<T> <<<dim3((a.channels + 255) / 256, a.blocks), 256, 0, stream>>>(a.partial, a.x, a.ext, a.dy, a.stats, a.rows, a.channels);
				MB200_COUNT_LAUNCH();
				kernel_layernorm_backward_long<T> <<<static_cast<int>(std::min<long long>(a.rows, static_cast<long long>(sms) * 4)), LONG_THREADS, 0, stream>>>(a.out, a.x, a.ext, a.dy,
						a.gamma, a.stats, a.beta_dx, a.rows, a.channels);
			}
			else
			{
				a.status = get(ctx)->dev_status;
				launch_rows(ctx, stream, a, true);
			}
			MB200_COUNT_LAUNCH();
			return check_cuda(ctx, cudaGetLastError(), "mb200_layernorm_backward");
		}
		template<typename G>
		void add_partials(mlContext_t ctx, const mlTensor_t &dw, const mlTensor_t &db, const float *partial, int blocks, int channels, float beta)
		{
			const cudaError_t status = launch_overlapped(kernel_layernorm_add_partials<G>, dim3((channels + 31) / 32, 2), dim3(1024), 0, use_stream(ctx),
					reinterpret_cast<G*>(dw.data), reinterpret_cast<G*>(db.data), partial, blocks, channels, beta);
			MB200_COUNT_LAUNCH();
			check_cuda(ctx, status, "mb200_layernorm_backward: column sums");
		}
		int partial_rows(int sm_count, long long rows, int channels)
		{
			return channels > LONGEST_TEAM_ROW ? long_row_chunks(sm_count, rows, channels) : team_blocks(sm_count, rows, channels, blocks_per_sm(channels));
		}
	}
} /* namespace mb200 */

using namespace mb200;

extern "C"
{
	void mb200_layernorm_forward(mlContext_t context, const mlTensor_t x, const mlTensor_t ext, const mlTensor_t w, const mlTensor_t b, mlTensor_t y, mlTensor_t stats)
	{
		const char *who = "mb200_layernorm_forward";
		MB200_REQUIRE(context, context != nullptr, "%s: null context", who);
		if (!check_extents(context, who, "x", x))
			return;
		MB200_REQUIRE(context, x.dtype == DTYPE_FLOAT16 || x.dtype == DTYPE_FLOAT32, "%s: x is %s, fp16 or fp32 expected", who, dtype_name(x.dtype));
		const int channels = last_dim(x);
		MB200_REQUIRE(context, channels >= 2, "%s: the unbiased variance needs at least 2 channels", who);
		MB200_REQUIRE(context, channels <= MAX_EXTENT, "%s: rows of %d channels are too long", who, channels);
		const long long rows = volume(x) / channels;
		if (!check_operand(context, who, "x", x, x.dtype, rows, channels) || !check_operand(context, who, "y", y, x.dtype, rows, channels)
				|| !check_operand(context, who, "stats", stats, DTYPE_FLOAT32, rows, 2)
				|| (!is_empty_descriptor(ext) && !check_operand(context, who, "ext", ext, x.dtype, rows, channels))
				|| (!is_empty_descriptor(w) && !check_operand(context, who, "weights", w, x.dtype, channels))
				|| (!is_empty_descriptor(b) && !check_operand(context, who, "bias", b, x.dtype, channels)))
			return;
		if (rows == 0)
			return; // nothing to normalise
		MB200_REQUIRE(context, aligned_to(stats.data, 8), "%s: stats must be 8-byte aligned", who);
		if (!check_distinct(context, who, "y", y, "x", x, true) || !check_distinct(context, who, "y", y, "ext", ext, true) || !check_distinct(context, who, "y", y, "stats", stats)
				|| !check_distinct(context, who, "y", y, "weights", w) || !check_distinct(context, who, "y", y, "bias", b) || !check_distinct(context, who, "stats", stats, "x", x)
				|| !check_distinct(context, who, "stats", stats, "ext", ext) || !check_distinct(context, who, "stats", stats, "weights", w)
				|| !check_distinct(context, who, "stats", stats, "bias", b))
			return;
		// a row longer than a team's registers is read again while it is written
		MB200_REQUIRE(context, channels <= LONGEST_TEAM_ROW || (y.data != x.data && (ext.data == nullptr || y.data != ext.data)), "%s: rows of %d channels cannot be normalised in place", who,
				channels);
		flush_pending(context);
		auto run = [&](auto type)
		{
			using T = decltype(type);
			Args<T> a { };
			a.out = reinterpret_cast<T*>(y.data);
			a.x = reinterpret_cast<const T*>(x.data);
			a.ext = reinterpret_cast<const T*>(ext.data);
			a.gamma = reinterpret_cast<const T*>(w.data);
			a.beta = reinterpret_cast<const T*>(b.data);
			a.stats = reinterpret_cast<float2*>(stats.data);
			a.rows = rows;
			a.channels = channels;
			run_forward(context, a);
		};
		if (x.dtype == DTYPE_FLOAT16)
			run(__half());
		else
			run(0.0f);
	}

	size_t mb200_layernorm_backward_get_workspace_size(mlContext_t context, mlShape_t shape)
	{
		if (context == nullptr || shape.rank < 1 || shape.rank > 6 || last_dim(shape) < 2 || last_dim(shape) > MAX_EXTENT)
			return 0;
		const long long rows = volume_without_last_dim(shape);
		return rows <= 0 ? 0 : static_cast<size_t>(2) * partial_rows(get(context)->sm_count, rows, last_dim(shape)) * last_dim(shape) * sizeof(float);
	}
	void mb200_layernorm_backward(mlContext_t context, const mlTensor_t x, const mlTensor_t ext, const mlTensor_t dy, const mlTensor_t w, const mlTensor_t stats, float beta_dx,
			mlTensor_t dx, float beta_dw, mlTensor_t dw, mlTensor_t db, mlTensor_t workspace)
	{
		const char *who = "mb200_layernorm_backward";
		MB200_REQUIRE(context, context != nullptr, "%s: null context", who);
		if (!check_extents(context, who, "x", x))
			return;
		MB200_REQUIRE(context, x.dtype == DTYPE_FLOAT16 || x.dtype == DTYPE_FLOAT32, "%s: x is %s, fp16 or fp32 expected", who, dtype_name(x.dtype));
		const int channels = last_dim(x);
		MB200_REQUIRE(context, channels >= 2, "%s: the unbiased variance needs at least 2 channels", who);
		MB200_REQUIRE(context, channels <= MAX_EXTENT, "%s: rows of %d channels are too long", who, channels);
		const long long rows = volume(x) / channels;
		const mlDataType_t grad = !is_empty_descriptor(dw) ? dw.dtype : !is_empty_descriptor(db) ? db.dtype : DTYPE_FLOAT32;
		MB200_REQUIRE(context, grad == DTYPE_FLOAT32 || grad == x.dtype, "%s: the weight gradients are %s, fp32 or the type of x expected", who, dtype_name(grad));
		if (!check_operand(context, who, "x", x, x.dtype, rows, channels) || !check_operand(context, who, "dy", dy, x.dtype, rows, channels)
				|| !check_operand(context, who, "dx", dx, x.dtype, rows, channels) || !check_operand(context, who, "stats", stats, DTYPE_FLOAT32, rows, 2)
				|| (!is_empty_descriptor(ext) && !check_operand(context, who, "ext", ext, x.dtype, rows, channels))
				|| (!is_empty_descriptor(w) && !check_operand(context, who, "weights", w, x.dtype, channels))
				|| (!is_empty_descriptor(dw) && !check_operand(context, who, "dw", dw, grad, channels))
				|| (!is_empty_descriptor(db) && !check_operand(context, who, "db", db, grad, channels)))
			return;
		const size_t needed = mb200_layernorm_backward_get_workspace_size(context, shape_of(x));
		if (!check_workspace(context, who, workspace, needed))
			return;
		if (rows > 0)
		{
			MB200_REQUIRE(context, aligned_to(stats.data, 8), "%s: stats must be 8-byte aligned", who);
			const struct { const char *name; const mlTensor_t &t; } inputs[] = { { "x", x }, { "ext", ext }, { "dy", dy }, { "weights", w }, { "stats", stats } };
			const struct { const char *name; const mlTensor_t &t; } results[] = { { "dx", dx }, { "dw", dw }, { "db", db }, { "workspace", workspace } };
			for (int i = 0; i < 4; i++)
			{
				for (int k = 0; k < 5; k++)
					if (!check_distinct(context, who, results[i].name, results[i].t, inputs[k].name, inputs[k].t, i == 0 && k < 3))
						return;
				for (int k = 0; k < i; k++)
					if (!check_distinct(context, who, results[i].name, results[i].t, results[k].name, results[k].t))
						return;
			}
			MB200_REQUIRE(context, channels <= LONGEST_TEAM_ROW || (dx.data != x.data && dx.data != dy.data && (ext.data == nullptr || dx.data != ext.data)),
					"%s: rows of %d channels cannot be differentiated in place", who, channels);
		}
		flush_pending(context);
		const int blocks = rows > 0 ? partial_rows(get(context)->sm_count, rows, channels) : 0;
		auto run = [&](auto type) -> bool
		{
			using T = decltype(type);
			Args<T> a { };
			a.out = reinterpret_cast<T*>(dx.data);
			a.x = reinterpret_cast<const T*>(x.data);
			a.ext = reinterpret_cast<const T*>(ext.data);
			a.dy = reinterpret_cast<const T*>(dy.data);
			a.gamma = reinterpret_cast<const T*>(w.data);
			a.stats = reinterpret_cast<float2*>(stats.data);
			a.beta_dx = beta_dx;
			a.partial = reinterpret_cast<float*>(workspace.data);
			a.rows = rows;
			a.channels = channels;
			a.blocks = blocks;
			return run_backward(context, a);
		};
		if (rows > 0 && !(x.dtype == DTYPE_FLOAT16 ? run(__half()) : run(0.0f)))
			return;
		if (is_empty_descriptor(dw) && is_empty_descriptor(db))
			return;
		// no rows: the sums are zero, and what is left is beta * the old value
		if (grad == DTYPE_FLOAT16)
			add_partials<__half>(context, dw, db, reinterpret_cast<const float*>(workspace.data), blocks, channels, beta_dw);
		else
			add_partials<float>(context, dw, db, reinterpret_cast<const float*>(workspace.data), blocks, channels, beta_dw);
	}
}
