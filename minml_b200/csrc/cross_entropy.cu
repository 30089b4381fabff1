/*
 * cross_entropy.cu -- softmax cross entropy over a large vocabulary, straight from the hidden states, and its gradients.
 *
 * With logits z = x W^T, lse_t = log sum_v exp(z_tv):
 *   loss_t = lse_t - z_t,target        dx_t = alpha c_t sum_v P_tv W_v        dW_v = alpha sum_t c_t P_tv x_t        P_tv = exp(z_tv - lse_t) - [v = target_t]
 * c_t is the row's weight (1 without weights).  A row whose target is no index of the vocabulary, or whose weight is 0, takes no part: its
 * loss is 0 for the former, its gradient 0 for both, and whatever its x holds reaches nothing else.
 *
 * The [tokens, vocabulary] logits are never kept: the vocabulary is taken in pieces as wide as the caller's workspace allows, forward
 * keeps a running maximum and sum per row, backward computes each piece's logits again from lse.
 *
 * fp16 gradients: P reaches down to 1 / vocabulary, where fp16 has left its normal range, so it is rounded as 2^15 P (at most 32768;
 * relative precision down to 2^-29).  Row weights do not go into P, where small ones would cost dx its digits, but into dx's fp32
 * result and into a copy of x, as c_t / max |c| (exact where all weights are equal).
 *
 * fp16 runs on gemm_pair.cu (up to 64 rows forward: few_tokens.cu): forward is one product whose epilogue leaves (maximum, sum of
 * exponentials) for every row and group of columns, joined by a second kernel, and the whole vocabulary is one piece; backward makes 2^15 P of a piece in the epilogue of its logits and
 * multiplies it with W and x.  dx is added up over the pieces in fp32.  fp32 keeps one piece's logits.  An embed that is no multiple of 16
 * bytes is copied to padded rows first.  Forward, a few rows in fp32, or in fp16 with such an embed, go through few_rows.cu, which leaves the
 * same statistics as one product and copies nothing.
 */
#include "common.cuh"
#include "operands.cuh"
#include "gemm_pair.cuh"
#include "gemm_fp32.cuh"
#include "few_tokens.cuh"
#include "few_rows.cuh"

#include <algorithm>

namespace mb200
{
	namespace
	{
		constexpr float P_SCALE = 32768.0f; // fp16 only
		constexpr int MIN_PIECE = 256; // columns; the narrowest piece a workspace may force
		constexpr size_t PIECE_BYTES = size_t(256) << 20; // what get_workspace_size asks for

		struct Problem
		{
				mlDataType_t dtype;
				long long tokens;
				int embed, vocab;
		};
		struct Rows
		{ // what decides whether and how much a row takes part
				const int *targets;
				const float *weights; // may be null
				int vocab;
				__device__ __forceinline__ float weight(long long t) const
				{ // 0: no part
					const int target = targets[t];
					return target < 0 || target >= vocab ? 0.0f : weights == nullptr ? 1.0f : weights[t];
				}
		};

		__device__ __forceinline__ float2 merge(float2 a, float2 b)
		{ // (maximum, sum of exp(z - maximum)) of the union of two sets; an empty one is (-inf, 0)
			const float m = fmaxf(a.x, b.x);
			// equal maxima (both -inf among them) keep their sums as they are; a NaN sum stays
			const float sa = a.x == m ? a.y : a.y * expf(a.x - m), sb = b.x == m ? b.y : b.y * expf(b.x - m);
			return make_float2(m, sa + sb);
		}
		__device__ __forceinline__ float2 merge_warp(float2 a)
		{
#pragma unroll
			for (int k = 16; k >= 1; k /= 2)
				a = merge(a, make_float2(__shfl_xor_sync(0xffffffffu, a.x, k), __shfl_xor_sync(0xffffffffu, a.y, k)));
			return a;
		}
		__device__ __forceinline__ void finish_row(long long t, float2 total, const Rows &rows, const float *target_logit, float *loss, float *lse)
		{
			const float value = total.x + logf(total.y);
			if (lse != nullptr)
				lse[t] = value;
			const int target = rows.targets[t];
			loss[t] = target < 0 || target >= rows.vocab ? 0.0f : value - target_logit[t];
		}

		/* One block a row: joins the piece's columns [first, first + width) into the row's running maximum and sum. */
		__global__ void __launch_bounds__(256) kernel_piece_statistics(const float *z, int pitch, float2 *running, float *target_logit, Rows rows,
				long long tokens, int first, int width, bool last, float *loss, float *lse)
		{
			__shared__ float2 scratch[8];
			wait_for_previous_grid();
			for (long long t = blockIdx.x; t < tokens; t += gridDim.x)
			{
				const float *row = z + t * pitch;
				float2 mine = make_float2(-INFINITY, 0.0f);
				for (int c = threadIdx.x * 4; c < width; c += 256 * 4 * 4)
				{ // sixteen values at a time: their maximum, then their exponentials (rows are padded to a multiple of 64 floats)
					float4 v[4];
					float top = -INFINITY;
#pragma unroll
					for (int k = 0; k < 4; k++)
					{
						const int at = c + k * 1024;
						v[k] = at < width ? *reinterpret_cast<const float4*>(row + at) : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
						if (at + 1 >= width)
							v[k].y = -INFINITY;
						if (at + 2 >= width)
							v[k].z = -INFINITY;
						if (at + 3 >= width)
							v[k].w = -INFINITY;
						top = fmaxf(top, fmaxf(fmaxf(v[k].x, v[k].y), fmaxf(v[k].z, v[k].w))); // a NaN gives way to a number here and reaches the sum
					}
					const float shift = top == -INFINITY ? 0.0f : top;
					float sum = 0.0f;
#pragma unroll
					for (int k = 0; k < 4; k++)
						sum += (expf(v[k].x - shift) + expf(v[k].y - shift)) + (expf(v[k].z - shift) + expf(v[k].w - shift));
					mine = merge(mine, make_float2(top, sum));
				}
				mine = merge_warp(mine);
				if (threadIdx.x % 32 == 0)
					scratch[threadIdx.x / 32] = mine;
				__syncthreads();
				if (threadIdx.x == 0)
				{
					float2 total = first == 0 ? make_float2(-INFINITY, 0.0f) : running[t];
					for (int k = 0; k < 8; k++)
						total = merge(total, scratch[k]);
					const int target = rows.targets[t];
					if (target >= first && target - first < width)
						target_logit[t] = row[target - first];
					if (last)
						finish_row(t, total, rows, target_logit, loss, lse);
					else
						running[t] = total;
				}
				__syncthreads();
			}
		}

		/* z becomes alpha c_t (exp(z - lse) - [target]) for one piece, four columns a thread; rows that take no part are zero */
		__global__ void __launch_bounds__(256) kernel_piece_gradient(float *z, int pitch, const float *lse, Rows rows, const GridWalk walk, int first, float alpha)
		{
			wait_for_previous_grid();
			const long long stride = static_cast<long long>(gridDim.x) * 256;
			for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < walk.total; i += stride)
			{
				long long t;
				int c;
				walk.place(i, t, c);
				c *= 4;
				const float weight = rows.weight(t), l = lse[t], factor = alpha * weight;
				const int target = weight != 0.0f ? rows.targets[t] - first - c : -1; // (a row that takes no part may name any number)
				float4 *at = reinterpret_cast<float4*>(z + t * pitch + c);
				float4 v = *at;
				if (weight == 0.0f)
					v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
				else
					v = make_float4(factor * (expf(v.x - l) - (target == 0 ? 1.0f : 0.0f)), factor * (expf(v.y - l) - (target == 1 ? 1.0f : 0.0f)),
							factor * (expf(v.z - l) - (target == 2 ? 1.0f : 0.0f)), factor * (expf(v.w - l) - (target == 3 ? 1.0f : 0.0f)));
				*at = v;
			}
		}

		/* out[0] = the largest |weight| of the rows that take part */
		__global__ void __launch_bounds__(1024) kernel_largest_weight(float *__restrict__ out, Rows rows, long long tokens)
		{
			__shared__ float scratch[32];
			float m = 0.0f;
			for (long long t = threadIdx.x; t < tokens; t += 1024)
				m = fmaxf(m, fabsf(rows.weight(t)));
			for (int k = 16; k >= 1; k /= 2)
				m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
			if (threadIdx.x % 32 == 0)
				scratch[threadIdx.x / 32] = m;
			__syncthreads();
			if (threadIdx.x < 32)
			{
				m = scratch[threadIdx.x];
				for (int k = 16; k >= 1; k /= 2)
					m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, k));
				if (threadIdx.x == 0)
					out[0] = m;
			}
		}
		/* x, times c_t / max |c| where weights are `applied`; zero in the rows that take no part, whatever they hold */
		template<typename T>
		__global__ void __launch_bounds__(256) kernel_weighted_rows(T *__restrict__ out, const T *__restrict__ x, Rows rows, bool applied, const float *__restrict__ largest,
				long long tokens, int embed)
		{
			for (long long t = blockIdx.x; t < tokens; t += gridDim.x)
			{
				const float c = rows.weight(t), factor = c == 0.0f ? 0.0f : largest != nullptr ? c / largest[0] : applied ? c : 1.0f;
				for (int k = threadIdx.x; k < embed; k += 256)
					out[t * embed + k] = factor == 0.0f ? from_float<T>(0.0f) : from_float<T>(to_float(x[t * embed + k]) * factor);
			}
		}
		/* Joins the statistics of a row's groups, parts[t][group]: a block a row. */
		__global__ void __launch_bounds__(256) kernel_join_statistics(const float2 *parts, int groups, const float *target_logit, Rows rows,
				float *loss, float *lse)
		{
			__shared__ float2 scratch[8];
			const long long t = blockIdx.x;
			wait_for_previous_grid();
			float2 mine = make_float2(-INFINITY, 0.0f);
#pragma unroll 4
			for (int g = threadIdx.x; g < groups; g += 256)
				mine = merge(mine, parts[t * groups + g]);
			mine = merge_warp(mine);
			if (threadIdx.x % 32 == 0)
				scratch[threadIdx.x / 32] = mine;
			__syncthreads();
			if (threadIdx.x == 0)
			{
				float2 total = scratch[0];
				for (int k = 1; k < 8; k++)
					total = merge(total, scratch[k]);
				finish_row(t, total, rows, target_logit, loss, lse);
			}
		}

		int elementwise_blocks(mlContext_t ctx, long long elements)
		{
			return static_cast<int>(std::max<long long>(1, std::min<long long>((elements + 255) / 256, static_cast<long long>(get(ctx)->sm_count) * 8)));
		}
		int row_blocks(mlContext_t ctx, long long rows)
		{
			return static_cast<int>(std::max<long long>(1, std::min<long long>(rows, static_cast<long long>(get(ctx)->sm_count) * 8)));
		}

		/* Forward: rows are read in place by few_rows.cu; in fp16 only where the weights would be copied. */
		bool by_few_rows(const Problem &q)
		{
			return q.dtype == DTYPE_FLOAT32 ? q.tokens <= FEW_ROWS_FP32 : q.tokens <= FEW_ROWS_FP16 && q.embed % 8 != 0;
		}
		int statistics_groups(mlContext_t ctx, const Problem &q)
		{
			if (by_few_rows(q))
				return few_rows_statistics_parts(ctx, static_cast<int>(q.tokens), q.vocab, q.embed);
			return q.tokens <= FEW_TOKENS ? few_statistics_parts(ctx, q.vocab) : pair_statistics_parts(q.vocab);
		}
		bool in_pieces(const Problem &q, bool training)
		{ // the forward pass in fp16, or of a few rows, keeps 8 bytes for every row and 128 (or 4 to 64) columns and has no use for pieces
			return training || (q.dtype == DTYPE_FLOAT32 && !by_few_rows(q));
		}
		/* The workspace of one call with pieces of `piece` columns. */
		struct Plan
		{
				int embed; // padded to a pitch that TMA can address
				int piece, pitch; // columns of a piece of logits or probabilities, and its rows' pitch
				int dx_splits; // fp32 sums that dx is kept in until the last piece
				float2 *running = nullptr; // per row; not in pieces: per row and group of columns
				float *target_logit = nullptr, *z = nullptr, *dx_sums = nullptr, *partials = nullptr, *largest = nullptr;
				void *p = nullptr, *x = nullptr, *w = nullptr, *weighted_x = nullptr;
				size_t bytes = 0;
				Plan(mlContext_t ctx, const Problem &q, void *workspace, bool training, int columns)
				{
					Carver carve(workspace);
					const bool half = q.dtype == DTYPE_FLOAT16;
					const int es = size_of(q.dtype), tokens = static_cast<int>(q.tokens);
					embed = round_up(q.embed, 16 / es);
					piece = columns;
					pitch = round_up(columns, 64);
					dx_splits = half && training ? pair_splits(ctx, tokens, q.embed, piece) : 1;
					if (!training && by_few_rows(q))
					{
						target_logit = carve.take<float>(q.tokens);
						running = carve.take<float2>(q.tokens * statistics_groups(ctx, q));
						bytes = carve.used;
						return;
					}
					const size_t cells = static_cast<size_t>(q.tokens) * pitch, rows = static_cast<size_t>(q.tokens) * embed;
					if (embed != q.embed)
					{
						x = carve.take<uint8_t>(rows * es);
						w = carve.take<uint8_t>(static_cast<size_t>(q.vocab) * embed * es);
					}
					if (!training)
					{
						target_logit = carve.take<float>(q.tokens);
						running = carve.take<float2>(q.tokens * (half ? statistics_groups(ctx, q) : 1));
					}
					if (!half)
						z = carve.take<float>(cells);
					if (training)
					{
						largest = carve.take<float>(1);
						weighted_x = carve.take<uint8_t>(rows * es);
						p = half ? carve.take<uint8_t>(cells * es) : nullptr; // fp32: in place of the logits
						dx_sums = half ? carve.take<float>(rows * dx_splits) : nullptr;
					}
					// products that are cut along K: of a whole piece, and of the last, narrower one
					size_t partial = 0;
					for (int width : { piece, q.vocab - (q.vocab - 1) / piece * piece })
					{
						if (half && training)
							partial = std::max(partial, pair_partial_elements(ctx, width, q.embed, tokens));
						if (!half)
							partial = std::max(partial, float_partial_elements(ctx, tokens, width, q.embed));
						if (!half && training)
							partial = std::max( { partial, float_partial_elements(ctx, tokens, q.embed, width), float_partial_elements(ctx, width, q.embed, tokens) });
					}
					partials = carve.take<float>(partial);
					bytes = carve.used;
				}
		};
		/* Pieces of equal width, multiples of 256 columns, of at most about PIECE_BYTES. */
		int recommended_piece(const Problem &q, bool training)
		{
			if (!in_pieces(q, training))
				return q.vocab;
			const long long most = std::max<long long>(MIN_PIECE, static_cast<long long>(PIECE_BYTES / size_of(q.dtype)) / std::max<long long>(1, q.tokens));
			const long long pieces = (q.vocab + most - 1) / most;
			return static_cast<int>(std::min<long long>(q.vocab, round_up(static_cast<int>((q.vocab + pieces - 1) / pieces), 256)));
		}
		/* The widest piece up to the recommended one, a multiple of 64 columns or the whole vocabulary, whose scratch fits the workspace; 0 if
		 * none does. */
		int piece_that_fits(mlContext_t ctx, const Problem &q, bool training, size_t bytes)
		{
			const int best = recommended_piece(q, training);
			if (Plan(ctx, q, nullptr, training, best).bytes <= bytes)
				return best;
			for (int piece = best / 2 / 64 * 64; piece > MIN_PIECE; piece = piece * 3 / 4 / 64 * 64)
				if (Plan(ctx, q, nullptr, training, piece).bytes <= bytes)
					return piece;
			return Plan(ctx, q, nullptr, training, std::min(MIN_PIECE, best)).bytes <= bytes ? std::min(MIN_PIECE, best) : 0;
		}

		bool fits_indices(const Problem &q)
		{
			return q.tokens <= MAX_EXTENT && q.vocab <= MAX_EXTENT && q.embed <= MAX_EXTENT;
		}
		bool check_problem(mlContext_t ctx, const char *who, const mlTensor_t &x, const mlTensor_t &w, const mlTensor_t &targets, Problem &q)
		{
			if (!check_extents(ctx, who, "x", x) || !check_extents(ctx, who, "weights", w))
				return false;
			if (x.dtype != DTYPE_FLOAT16 && x.dtype != DTYPE_FLOAT32)
			{
				record_error(ctx, "%s: x is %s, fp16 or fp32 expected", who, dtype_name(x.dtype));
				return false;
			}
			if (w.rank != 2 || w.dim[0] == 0 || w.dim[1] == 0)
			{
				record_error(ctx, "%s: weights must be [vocabulary, embed]", who);
				return false;
			}
			q.dtype = x.dtype;
			q.vocab = w.dim[0];
			q.embed = w.dim[1];
			q.tokens = volume(x) / q.embed;
			if (!fits_indices(q))
			{
				record_error(ctx, "%s: %lld tokens, %d columns and an embed of %d are too many for one call", who, q.tokens, q.vocab, q.embed);
				return false;
			}
			return check_operand(ctx, who, "x", x, x.dtype, q.tokens, q.embed) && check_operand(ctx, who, "weights", w, x.dtype, q.vocab, q.embed)
					&& check_operand(ctx, who, "targets", targets, DTYPE_INT32, q.tokens);
		}
		/* Width of the pieces for this workspace; 0 (and an error) when it holds none. */
		int check_piece(mlContext_t ctx, const char *who, const Problem &q, bool training, const mlTensor_t &workspace)
		{
			if (!check_workspace(ctx, who, workspace, 1))
				return 0;
			const int piece = piece_that_fits(ctx, q, training, static_cast<size_t>(bytes_of(workspace)));
			if (piece == 0)
				record_error(ctx, "%s: the workspace has %lld bytes, %zu are needed", who, bytes_of(workspace),
						Plan(ctx, q, nullptr, training, std::min(MIN_PIECE, recommended_piece(q, training))).bytes);
			return piece;
		}
		template<typename T>
		struct Operands
		{
				const T *x, *w;
				Operands(mlContext_t ctx, const Problem &q, const Plan &plan, const mlTensor_t &x_, const mlTensor_t &w_) :
						x(reinterpret_cast<const T*>(x_.data)),
						w(reinterpret_cast<const T*>(w_.data))
				{
					if (plan.x != nullptr)
					{
						pack_rows<T>(ctx, reinterpret_cast<T*>(plan.x), plan.embed, q.tokens, x, q.tokens, q.embed);
						pack_rows<T>(ctx, reinterpret_cast<T*>(plan.w), plan.embed, q.vocab, w, q.vocab, q.embed);
						x = reinterpret_cast<const T*>(plan.x);
						w = reinterpret_cast<const T*>(plan.w);
					}
				}
		};
		bool check_alignment(mlContext_t ctx, const char *who, const char *name, const mlTensor_t &t, bool copied)
		{
			if (copied || aligned_to(t.data, 16))
				return true;
			record_error(ctx, "%s: %s must be 16-byte aligned", who, name);
			return false;
		}

		void join_statistics(mlContext_t ctx, const Problem &q, const Rows &rows, const Plan &plan, float *loss, float *lse)
		{
			const cudaError_t status = launch_overlapped(kernel_join_statistics, dim3(static_cast<int>(q.tokens)), dim3(256), 0, use_stream(ctx), plan.running, statistics_groups(ctx, q),
					plan.target_logit, rows, loss, lse);
			MB200_COUNT_LAUNCH();
			check_cuda(ctx, status, "mb200_softmax_cross_entropy_forward");
		}
		template<typename T>
		void forward_few_rows(mlContext_t ctx, const Problem &q, const Rows &rows, const Plan &plan, const mlTensor_t &x, const mlTensor_t &w, float *loss, float *lse)
		{
			const FewRows<T> operands { static_cast<int>(q.tokens), q.embed, reinterpret_cast<const T*>(x.data), reinterpret_cast<const T*>(w.data) };
			if (few_rows_statistics(ctx, operands, q.vocab, rows.targets, plan.running, plan.target_logit))
				join_statistics(ctx, q, rows, plan, loss, lse);
		}
		void forward_half(mlContext_t ctx, const Problem &q, const Rows &rows, const Plan &plan, const Operands<__half> &o, float *loss, float *lse)
		{
			const int tokens = static_cast<int>(q.tokens);
			const bool ok = tokens <= FEW_TOKENS
					? few_statistics(ctx, FewTokens { tokens, plan.embed, o.x, plan.embed, o.w, plan.embed }, q.vocab, rows.targets, plan.running, plan.target_logit)
					: pair_statistics(ctx, tokens, q.vocab, q.embed, PairOperand { o.x, plan.embed, false }, PairOperand { o.w, plan.embed, false }, rows.targets, plan.running,
							plan.target_logit);
			if (ok)
				join_statistics(ctx, q, rows, plan, loss, lse);
		}
		void forward_float(mlContext_t ctx, const Problem &q, const Rows &rows, const Plan &plan, const Operands<float> &o, float *loss, float *lse)
		{
			for (long long begin = 0; begin < q.vocab; begin += plan.piece)
			{
				const int first = static_cast<int>(begin), width = std::min(plan.piece, q.vocab - first);
				if (!float_product(ctx, static_cast<int>(q.tokens), width, q.embed, FloatOperand { o.x, plan.embed, false },
						FloatOperand { o.w + static_cast<size_t>(first) * plan.embed, plan.embed, false }, plan.z, plan.pitch, 0.0f, plan.partials))
					return;
				const cudaError_t status = launch_overlapped(kernel_piece_statistics, dim3(row_blocks(ctx, q.tokens)), dim3(256), 0, use_stream(ctx), plan.z, plan.pitch, plan.running,
						plan.target_logit, rows, q.tokens, first, width, first + width == q.vocab, loss, lse);
				MB200_COUNT_LAUNCH();
				if (!check_cuda(ctx, status, "mb200_softmax_cross_entropy_forward"))
					return;
			}
		}
		template<typename T>
		void backward(mlContext_t ctx, const Problem &q, const Rows &rows, const Plan &plan, const Operands<T> &o, const float *lse, float alpha, float beta_dx, T *dx, float beta_dw, T *dw)
		{
			cudaStream_t stream = use_stream(ctx);
			constexpr bool half = sizeof(T) == 2;
			const int tokens = static_cast<int>(q.tokens), D = q.embed, ld = plan.embed;
			// fp16: factors go into results and the copy of x (see above); fp32 has the range to take them all into P, and the copy only masks rows
			const float unscale = alpha / P_SCALE;
			const float *largest = half && rows.weights != nullptr ? plan.largest : nullptr;
			if (dw != nullptr)
			{
				if (largest != nullptr)
				{
					kernel_largest_weight<<<1, 1024, 0, stream>>>(plan.largest, rows, q.tokens);
					MB200_COUNT_LAUNCH();
				}
				kernel_weighted_rows<T> <<<row_blocks(ctx, q.tokens), 256, 0, stream>>>(reinterpret_cast<T*>(plan.weighted_x), o.x, rows, half, largest, q.tokens, ld);
				MB200_COUNT_LAUNCH();
				if (!check_cuda(ctx, cudaGetLastError(), "mb200_softmax_cross_entropy_backward: row weights"))
					return;
			}
			const T *weighted_x = reinterpret_cast<const T*>(plan.weighted_x);
			for (long long begin = 0; begin < q.vocab; begin += plan.piece)
			{
				const int first = static_cast<int>(begin), width = std::min(plan.piece, q.vocab - first);
				const T *w = o.w + static_cast<size_t>(first) * ld;
				if constexpr (half)
				{
					__half *p = reinterpret_cast<__half*>(plan.p);
					if (!pair_probabilities(ctx, tokens, width, D, PairOperand { o.x, ld, false }, PairOperand { w, ld, false }, rows.targets, rows.weights, lse, first, q.vocab, p, plan.pitch))
						return;
					if (dx != nullptr
							&& !pair_product_sums(ctx, tokens, D, width, PairOperand { p, plan.pitch, false }, PairOperand { w, ld, true }, plan.dx_sums, ld, plan.dx_splits, first > 0))
						return;
					if (dw != nullptr
							&& !pair_product(ctx, width, D, tokens, PairOperand { p, plan.pitch, true }, PairOperand { weighted_x, ld, true },
									PairResult { dw + static_cast<size_t>(first) * D, D, unscale, beta_dw, largest }, plan.partials))
						return;
				}
				else
				{
					if (!float_product(ctx, tokens, width, D, FloatOperand { o.x, ld, false }, FloatOperand { w, ld, false }, plan.z, plan.pitch, 0.0f, plan.partials))
						return;
					const cudaError_t status = launch_overlapped(kernel_piece_gradient, dim3(elementwise_blocks(ctx, q.tokens * ((width + 3) / 4))), dim3(256), 0, stream, plan.z, plan.pitch, lse,
							rows, GridWalk(q.tokens, (width + 3) / 4), first, alpha);
					MB200_COUNT_LAUNCH();
					if (!check_cuda(ctx, status, "mb200_softmax_cross_entropy_backward: probabilities"))
						return;
					if (dx != nullptr
							&& !float_product(ctx, tokens, D, width, FloatOperand { plan.z, plan.pitch, false }, FloatOperand { w, ld, true }, dx, D, first > 0 ? 1.0f : beta_dx, plan.partials))
						return;
					if (dw != nullptr
							&& !float_product(ctx, width, D, tokens, FloatOperand { plan.z, plan.pitch, true }, FloatOperand { weighted_x, ld, true }, dw + static_cast<size_t>(first) * D, D,
									beta_dw, plan.partials))
						return;
				}
			}
			if constexpr (half)
				if (dx != nullptr)
					finish_sums<T>(ctx, dx, D, tokens, D, plan.dx_sums, ld, plan.dx_splits, unscale, nullptr, rows.weights, beta_dx);
		}
	}
} /* namespace mb200 */

using namespace mb200;

extern "C"
{
	size_t mb200_softmax_cross_entropy_get_workspace_size(mlContext_t context, mlShape_t x_shape, mlShape_t w_shape, mlDataType_t dtype, bool training)
	{
		if (context == nullptr || x_shape.rank < 1 || x_shape.rank > 6 || w_shape.rank != 2 || w_shape.dim[0] <= 0 || w_shape.dim[1] <= 0 || last_dim(x_shape) != w_shape.dim[1])
			return 0;
		const Problem q { dtype, volume_without_last_dim(x_shape), w_shape.dim[1], w_shape.dim[0] };
		if (q.tokens <= 0 || !fits_indices(q) || (dtype != DTYPE_FLOAT16 && dtype != DTYPE_FLOAT32))
			return 0;
		// the forward call of a training step takes its scratch from the same workspace
		const size_t forward = Plan(context, q, nullptr, false, recommended_piece(q, false)).bytes;
		return training ? std::max(forward, Plan(context, q, nullptr, true, recommended_piece(q, true)).bytes) : forward;
	}

	void mb200_softmax_cross_entropy_forward(mlContext_t context, const mlTensor_t x, const mlTensor_t w, const mlTensor_t targets, mlTensor_t loss, mlTensor_t lse, mlTensor_t workspace)
	{
		const char *who = "mb200_softmax_cross_entropy_forward";
		MB200_REQUIRE(context, context != nullptr, "%s: null context", who);
		Problem q;
		if (!check_problem(context, who, x, w, targets, q) || !check_operand(context, who, "loss", loss, DTYPE_FLOAT32, q.tokens)
				|| (!is_empty_descriptor(lse) && !check_operand(context, who, "lse", lse, DTYPE_FLOAT32, q.tokens)))
			return;
		if (q.tokens == 0)
			return;
		const struct { const char *name; const mlTensor_t &t; } inputs[] = { { "x", x }, { "weights", w }, { "targets", targets } }, results[] = { { "loss", loss }, { "lse", lse }, {
				"workspace", workspace } };
		for (int i = 0; i < 3; i++)
		{
			for (const auto &in : inputs)
				if (!check_distinct(context, who, results[i].name, results[i].t, in.name, in.t))
					return;
			for (int k = 0; k < i; k++)
				if (!check_distinct(context, who, results[i].name, results[i].t, results[k].name, results[k].t))
					return;
		}
		const int piece = check_piece(context, who, q, false, workspace);
		if (piece == 0)
			return;
		const Plan plan(context, q, workspace.data, false, piece);
		if (!check_alignment(context, who, "x", x, plan.embed != q.embed) || !check_alignment(context, who, "weights", w, plan.embed != q.embed))
			return;
		flush_pending(context);
		const Rows rows { reinterpret_cast<const int*>(targets.data), nullptr, q.vocab };
		float *loss_data = reinterpret_cast<float*>(loss.data), *lse_data = reinterpret_cast<float*>(lse.data);
		if (by_few_rows(q) && q.dtype == DTYPE_FLOAT16)
			forward_few_rows<__half>(context, q, rows, plan, x, w, loss_data, lse_data);
		else if (by_few_rows(q))
			forward_few_rows<float>(context, q, rows, plan, x, w, loss_data, lse_data);
		else if (q.dtype == DTYPE_FLOAT16)
			forward_half(context, q, rows, plan, Operands<__half>(context, q, plan, x, w), loss_data, lse_data);
		else
			forward_float(context, q, rows, plan, Operands<float>(context, q, plan, x, w), loss_data, lse_data);
	}

	void mb200_softmax_cross_entropy_backward(mlContext_t context, const mlTensor_t x, const mlTensor_t w, const mlTensor_t targets, const mlTensor_t lse, float alpha,
			const mlTensor_t row_weights, float beta_dx, mlTensor_t dx, float beta_dw, mlTensor_t dw, mlTensor_t workspace)
	{
		const char *who = "mb200_softmax_cross_entropy_backward";
		MB200_REQUIRE(context, context != nullptr, "%s: null context", who);
		Problem q;
		if (!check_problem(context, who, x, w, targets, q) || !check_operand(context, who, "lse", lse, DTYPE_FLOAT32, q.tokens)
				|| (!is_empty_descriptor(row_weights) && !check_operand(context, who, "row_weights", row_weights, DTYPE_FLOAT32, q.tokens))
				|| (!is_empty_descriptor(dx) && !check_operand(context, who, "dx", dx, x.dtype, q.tokens, q.embed))
				|| (!is_empty_descriptor(dw) && !check_operand(context, who, "dw", dw, x.dtype, q.vocab, q.embed)))
			return;
		const struct { const char *name; const mlTensor_t &t; } inputs[] = { { "x", x }, { "weights", w }, { "targets", targets }, { "lse", lse }, { "row_weights", row_weights } }, results[] = {
				{ "dx", dx }, { "dw", dw }, { "workspace", workspace } };
		for (int i = 0; i < 3; i++)
		{
			for (const auto &in : inputs)
				if (!check_distinct(context, who, results[i].name, results[i].t, in.name, in.t))
					return;
			for (int k = 0; k < i; k++)
				if (!check_distinct(context, who, results[i].name, results[i].t, results[k].name, results[k].t))
					return;
		}
		flush_pending(context);
		if (q.tokens == 0)
		{ // the gradient of a sum of nothing
			if (!is_empty_descriptor(dw))
				cuda_scale_tensor(context, beta_dw, dw);
			return;
		}
		const int piece = check_piece(context, who, q, true, workspace);
		if (piece == 0)
			return;
		const Plan plan(context, q, workspace.data, true, piece);
		if (!check_alignment(context, who, "x", x, plan.x != nullptr) || !check_alignment(context, who, "weights", w, plan.x != nullptr))
			return;
		const Rows rows { reinterpret_cast<const int*>(targets.data), reinterpret_cast<const float*>(row_weights.data), q.vocab };
		const float *lse_data = reinterpret_cast<const float*>(lse.data);
		if (q.dtype == DTYPE_FLOAT16)
			backward<__half>(context, q, rows, plan, Operands<__half>(context, q, plan, x, w), lse_data, alpha, beta_dx, reinterpret_cast<__half*>(dx.data), beta_dw,
					reinterpret_cast<__half*>(dw.data));
		else
			backward<float>(context, q, rows, plan, Operands<float>(context, q, plan, x, w), lse_data, alpha, beta_dx, reinterpret_cast<float*>(dx.data), beta_dw,
					reinterpret_cast<float*>(dw.data));
	}
}
