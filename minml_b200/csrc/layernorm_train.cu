/*
 * layernorm_train.cu -- layer normalisation for training: the forward pass that keeps each row's mean and 1 / stddev, and the
 * backward pass with the reduction of the weight and bias gradients.  Same function as cuda_layernorm_forward (norm_attn.cu):
 *   s = x + ext;   m = mean(s);   r = 1 / sqrt(1e-6 + sum((s - m)^2) / (N - 1));   xh = (s - m) r;   y = gamma xh + beta
 * Differentiating, with g = gamma dy (the unbiased variance puts N - 1, not N, under the second sum):
 *   dx = r (g - sum(g) / N - xh sum(g xh) / (N - 1));     dgamma = sum over rows of dy xh;     dbeta = sum over rows of dy
 * and the gradient of ext is that of x.
 *
 * Both passes are bound by memory: forward reads s and writes y, backward reads s and dy and writes dx.  A row belongs to a team
 * of 32 .. 512 threads that holds it in registers (8 or 16 elements a thread, by the row's length), so it is read once.
 * Backward, a team walks rows r, r + teams, ... with the next row's loads in flight under the current row's two sums; a thread
 * owns the same columns in every row, so the column sums of dgamma and dbeta stay in its fp32 registers until the end.  Each
 * block then writes one partial row of each, and a second kernel adds the blocks' rows in a fixed order: no atomics, the same
 * bits on every run.  All sums are fp32; y and dx are rounded once.
 */
#include "common.cuh"
#include "operands.cuh"

#include <algorithm>

namespace mb200
{
	namespace
	{
		constexpr float EPSILON = 1.0e-6f; // inside the square root, as in cuda_layernorm_forward

		template<typename T, int VEC>
		struct alignas(sizeof(T) * VEC) Pack
		{
				T v[VEC];
		};

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

		template<typename T, int VEC, int E>
		struct RowPart
		{ // a thread's share of one row, as loaded
				static constexpr int N = E / VEC;
				Pack<T, VEC> p[N];
				template<int W>
				__device__ __forceinline__ void load(const T *row, int lane, int channels)
				{
#pragma unroll
					for (int i = 0; i < N; i++)
					{
						const int c = (i * W + lane) * VEC;
						if (c < channels)
							p[i] = *reinterpret_cast<const Pack<T, VEC>*>(row + c);
						else
						{
#pragma unroll
							for (int k = 0; k < VEC; k++)
								p[i].v[k] = from_float<T>(0.0f);
						}
					}
				}
				__device__ __forceinline__ float get(int e) const
				{
					return to_float(p[e / VEC].v[e % VEC]);
				}
		};

		template<typename T, int VEC, int W, int E>
		__global__ void __launch_bounds__(W == 32 ? 256 : W) kernel_layernorm_train(T *output, const T *input, const T *ext, const T *__restrict__ gamma,
				const T *__restrict__ beta, float2 *__restrict__ stats, long long rows, int channels)
		{
			constexpr int N = E / VEC;
			__shared__ float2 scratch[2][16];
			uint32_t turn = 0;
			const int lane = threadIdx.x % W;
			const int teams_per_block = blockDim.x / W;
			const long long teams = static_cast<long long>(gridDim.x) * teams_per_block;
			for (long long r = static_cast<long long>(blockIdx.x) * teams_per_block + threadIdx.x / W; r < rows; r += teams)
			{
				RowPart<T, VEC, E> x, e;
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
					const bool inside = (k / VEC * W + lane) * VEC < channels;
					v[k] -= mean;
					var += inside ? v[k] * v[k] : 0.0f;
				}
				team_sum<W>(var, unused, scratch, turn);
				const float inv_stddev = 1.0f / sqrtf(EPSILON + var / static_cast<float>(channels - 1));
				if (lane == 0)
					stats[r] = make_float2(mean, inv_stddev);
#pragma unroll
				for (int i = 0; i < N; i++)
				{
					const int c = (i * W + lane) * VEC;
					if (c >= channels)
						continue;
					Pack<T, VEC> g, b, out;
					if (gamma != nullptr)
						g = *reinterpret_cast<const Pack<T, VEC>*>(gamma + c);
					if (beta != nullptr)
						b = *reinterpret_cast<const Pack<T, VEC>*>(beta + c);
#pragma unroll
					for (int k = 0; k < VEC; k++)
						out.v[k] = from_float<T>((gamma != nullptr ? to_float(g.v[k]) : 1.0f) * v[i * VEC + k] * inv_stddev + (beta != nullptr ? to_float(b.v[k]) : 0.0f));
					*reinterpret_cast<Pack<T, VEC>*>(output + r * channels + c) = out;
				}
			}
		}

		/* partial: [2][gridDim.x][channels], the block's column sums of dy xh and of dy */
		template<typename T, int VEC, int W, int E>
		__global__ void __launch_bounds__(W == 32 ? 256 : W) kernel_layernorm_backward(T *dx, const T *input, const T *ext, const T *dy,
				const T *__restrict__ gamma, const float2 *__restrict__ stats, float beta_dx, float *__restrict__ partial, long long rows, int channels)
		{
			constexpr int N = E / VEC;
			__shared__ float2 scratch[2][16];
			__shared__ float columns[W == 32 ? 7 * 32 * E : 1]; // the other warps' column sums, when a block has eight one-warp teams
			uint32_t turn = 0;
			const int lane = threadIdx.x % W;
			const int teams_per_block = blockDim.x / W;
			const long long teams = static_cast<long long>(gridDim.x) * teams_per_block;
			const float inv_n = 1.0f / static_cast<float>(channels), inv_n1 = 1.0f / static_cast<float>(channels - 1);

			RowPart<T, VEC, E> g, x, e, d;
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
					const bool inside = (k / VEC * W + lane) * VEC < channels;
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
				for (int i = 0; i < N; i++)
				{
					const int c = (i * W + lane) * VEC;
					if (c >= channels)
						continue;
					Pack<T, VEC> *dst = reinterpret_cast<Pack<T, VEC>*>(dx + r * channels + c);
					Pack<T, VEC> out;
					if (beta_dx != 0.0f)
						out = *dst;
#pragma unroll
					for (int k = 0; k < VEC; k++)
					{
						const float v = inv_stddev * (gy[i * VEC + k] - s1 - xh[i * VEC + k] * s2);
						out.v[k] = from_float<T>(beta_dx != 0.0f ? v + beta_dx * to_float(out.v[k]) : v);
					}
					*dst = out;
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
				const int c = (k / VEC * W + lane) * VEC + k % VEC;
				if (c < channels)
				{
					partial[static_cast<long long>(blockIdx.x) * channels + c] = sum_w[k];
					partial[(static_cast<long long>(gridDim.x) + blockIdx.x) * channels + c] = sum_b[k];
				}
			}
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
		__global__ void __launch_bounds__(1024) kernel_layernorm_add_partials(G *dw, G *db, const float *__restrict__ partial, int blocks, int channels, float beta)
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
		/* Blocks per SM that the backward kernel is launched with: partial rows are what it costs to have more. */
		int backward_blocks(int sm_count, long long rows, int channels)
		{
			const int teams_per_block = channels <= 512 ? 8 : 1;
			const int per_sm = channels <= 512 ? 2 : channels <= 2048 ? 4 : channels <= 4096 ? 2 : 1;
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
		};
		template<typename T, int VEC, int W, int E>
		void launch_team(cudaStream_t stream, const Args<T> &a, bool backward)
		{
			constexpr int threads = W == 32 ? 256 : W;
			if (backward)
				kernel_layernorm_backward<T, VEC, W, E> <<<a.blocks, threads, 0, stream>>>(a.out, a.x, a.ext, a.dy, a.gamma, a.stats, a.beta_dx, a.partial, a.rows, a.channels);
			else
				kernel_layernorm_train<T, VEC, W, E> <<<a.blocks, threads, 0, stream>>>(a.out, a.x, a.ext, a.gamma, a.beta, a.stats, a.rows, a.channels);
		}
		template<typename T, int VEC>
		void launch_by_length(cudaStream_t stream, const Args<T> &a, bool backward)
		{
			if (a.channels <= 32 * 8)
				launch_team<T, VEC, 32, 8>(stream, a, backward);
			else if (a.channels <= 32 * 16)
				launch_team<T, VEC, 32, 16>(stream, a, backward);
			else if (a.channels <= 128 * 8)
				launch_team<T, VEC, 128, 8>(stream, a, backward);
			else if (a.channels <= 128 * 16)
				launch_team<T, VEC, 128, 16>(stream, a, backward);
			else if (a.channels <= 256 * 16)
				launch_team<T, VEC, 256, 16>(stream, a, backward);
			else
				launch_team<T, VEC, 512, 16>(stream, a, backward);
		}
		/* 16-byte accesses when every row starts on a 16-byte boundary, else element by element */
		template<typename T>
		void launch_rows(cudaStream_t stream, const Args<T> &a, bool backward)
		{
			constexpr int VEC = 16 / sizeof(T);
			const void *pointers[] = { a.out, a.x, a.ext, a.dy, a.gamma, a.beta };
			bool wide = a.channels % VEC == 0;
			for (const void *p : pointers)
				wide = wide && aligned_to(p, 16);
			if (wide)
				launch_by_length<T, VEC>(stream, a, backward);
			else
				launch_by_length<T, 1>(stream, a, backward);
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
				const int teams_per_block = a.channels <= 512 ? 8 : 1;
				const long long per_sm = a.channels <= 512 ? 8 : a.channels <= 2048 ? 16 : a.channels <= 4096 ? 8 : 4;
				a.blocks = static_cast<int>(std::min<long long>((a.rows + teams_per_block - 1) / teams_per_block, sms * per_sm));
				launch_rows(stream, a, false);
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
				launch_rows(stream, a, true);
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
			return channels > LONGEST_TEAM_ROW ? long_row_chunks(sm_count, rows, channels) : backward_blocks(sm_count, rows, channels);
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
		if (context == nullptr || shape.rank < 1 || shape.rank > 6 || last_dim(shape) < 2)
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
