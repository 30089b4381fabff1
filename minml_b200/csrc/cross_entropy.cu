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
 */
#include "common.cuh"
#include "operands.cuh"

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
		__global__ void __launch_bounds__(256) kernel_piece_statistics(const float *__restrict__ z, float2 *__restrict__ running, float *__restrict__ target_logit, Rows rows,
				long long tokens, int first, int width, bool last, float *__restrict__ loss, float *__restrict__ lse)
		{
			__shared__ float2 scratch[8];
			for (long long t = blockIdx.x; t < tokens; t += gridDim.x)
			{
				const float *row = z + t * width;
				float2 mine = make_float2(-INFINITY, 0.0f);
				for (int c = threadIdx.x; c < width; c += 256)
				{
					const float v = row[c];
					if (v > mine.x)
					{
						mine.y = mine.y * expf(mine.x - v) + 1.0f;
						mine.x = v;
					}
					else
						mine.y += mine.x == v && v == -INFINITY ? 0.0f : expf(v - mine.x); // a NaN reaches the sum
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

		/* p = scale (exp(z - lse) - [target]) for one piece; rows that take no part are zero */
		template<typename T>
		__global__ void __launch_bounds__(256) kernel_piece_gradient(T *__restrict__ p, const float *__restrict__ z, const float *__restrict__ lse, Rows rows, long long tokens,
				int first, int width, float scale)
		{
			const long long total = tokens * width, stride = static_cast<long long>(gridDim.x) * 256;
			for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total; i += stride)
			{
				const long long t = i / width;
				const int c = static_cast<int>(i - t * width);
				const float v = expf(z[i] - lse[t]) - (rows.targets[t] - first == c ? 1.0f : 0.0f);
				p[i] = from_float<T>(rows.weight(t) != 0.0f ? scale * v : 0.0f);
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
		/* x times c_t / max |c|; zero in the rows that take no part, whatever they hold */
		template<typename T>
		__global__ void __launch_bounds__(256) kernel_weighted_rows(T *__restrict__ out, const T *__restrict__ x, Rows rows, const float *__restrict__ largest, long long tokens,
				int embed)
		{
			for (long long t = blockIdx.x; t < tokens; t += gridDim.x)
			{
				const float c = rows.weight(t), factor = c == 0.0f ? 0.0f : largest == nullptr ? c : c / largest[0];
				for (int k = threadIdx.x; k < embed; k += 256)
					out[t * embed + k] = factor == 0.0f ? from_float<T>(0.0f) : from_float<T>(to_float(x[t * embed + k]) * factor);
			}
		}
		/* out = alpha * (largest) * (row weight) * sum + beta * out, the rounding of an fp32 sum to the gradient's type */
		template<typename T>
		__global__ void __launch_bounds__(256) kernel_finish_gradient(T *out, const float *__restrict__ sum, float alpha, const float *__restrict__ largest, const float *__restrict__ row_weights,
				float beta, long long elements, int columns)
		{
			const long long stride = static_cast<long long>(gridDim.x) * 256;
			const float factor = largest == nullptr ? alpha : alpha * largest[0];
			for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < elements; i += stride)
			{
				const float c = row_weights == nullptr ? 1.0f : row_weights[i / columns];
				const float v = c == 0.0f ? 0.0f : factor * c * sum[i]; // a sum of a row that takes no part is zero already
				out[i] = from_float<T>(beta != 0.0f ? v + beta * to_float(out[i]) : v);
			}
		}

		mlTensor_t matrix(const void *data, mlDataType_t dtype, long long rows, int columns)
		{
			return make_tensor(data, dtype, make_shape( { static_cast<int>(rows), columns }));
		}
		int elementwise_blocks(mlContext_t ctx, long long elements)
		{
			return static_cast<int>(std::max<long long>(1, std::min<long long>((elements + 255) / 256, static_cast<long long>(get(ctx)->sm_count) * 8)));
		}
		int row_blocks(mlContext_t ctx, long long rows)
		{
			return static_cast<int>(std::max<long long>(1, std::min<long long>(rows, static_cast<long long>(get(ctx)->sm_count) * 8)));
		}

		/* The workspace of one call with pieces of `piece` columns. */
		struct Scratch
		{
				float2 *running = nullptr;
				float *target_logit = nullptr, *z = nullptr, *dx_sum = nullptr, *dw_sum = nullptr, *largest = nullptr;
				void *p = nullptr, *x = nullptr;
				size_t bytes = 0;
				Scratch(const Problem &q, void *workspace, bool training, int piece)
				{
					Carver carve(workspace);
					const size_t es = size_of(q.dtype), cells = static_cast<size_t>(q.tokens) * piece, rows = static_cast<size_t>(q.tokens) * q.embed;
					running = carve.take<float2>(q.tokens);
					target_logit = carve.take<float>(q.tokens);
					z = carve.take<float>(cells);
					if (training)
					{
						largest = carve.take<float>(1);
						x = carve.take<uint8_t>(rows * es);
						dx_sum = carve.take<float>(rows);
						p = carve.take<uint8_t>(cells * es);
						dw_sum = carve.take<float>(static_cast<size_t>(piece) * q.embed);
					}
					bytes = carve.used;
				}
		};
		int recommended_piece(const Problem &q)
		{
			const long long columns = static_cast<long long>(PIECE_BYTES / 4) / std::max<long long>(1, q.tokens) / 64 * 64;
			return static_cast<int>(std::min<long long>(q.vocab, std::max<long long>(MIN_PIECE, columns)));
		}
		/* The widest piece, a multiple of 64 columns or the whole vocabulary, whose scratch fits the workspace; 0 if none does. */
		int piece_that_fits(const Problem &q, bool training, size_t bytes)
		{
			if (Scratch(q, nullptr, training, q.vocab).bytes <= bytes)
				return q.vocab;
			int low = std::min(MIN_PIECE, q.vocab), high = q.vocab; // low fits (checked), high does not
			if (Scratch(q, nullptr, training, low).bytes > bytes)
				return 0;
			while (high - low > 64)
			{
				const int middle = low + (high - low) / 2;
				(Scratch(q, nullptr, training, middle).bytes <= bytes ? low : high) = middle;
			}
			return std::max(std::min(MIN_PIECE, q.vocab), low / 64 * 64);
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
			if (q.tokens > 0x7FFFFFFFll)
			{
				record_error(ctx, "%s: %lld tokens are too many for one call", who, q.tokens);
				return false;
			}
			return check_operand(ctx, who, "x", x, x.dtype, q.tokens, q.embed) && check_operand(ctx, who, "weights", w, x.dtype, q.vocab, q.embed)
					&& check_operand(ctx, who, "targets", targets, DTYPE_INT32, q.tokens);
		}
		int check_piece(mlContext_t ctx, const char *who, const Problem &q, bool training, const mlTensor_t &workspace)
		{
			const size_t least = Scratch(q, nullptr, training, std::min(MIN_PIECE, q.vocab)).bytes;
			if (!check_workspace(ctx, who, workspace, least))
				return 0;
			return piece_that_fits(q, training, static_cast<size_t>(bytes_of(workspace)));
		}
		mlTensor_t piece_of(const mlTensor_t &w, int first, int width)
		{
			return matrix(reinterpret_cast<const uint8_t*>(w.data) + static_cast<size_t>(first) * w.dim[1] * size_of(w.dtype), w.dtype, width, w.dim[1]);
		}
		template<typename T>
		void backward_pieces(mlContext_t ctx, const Problem &q, const Rows &rows, const mlTensor_t &x, const mlTensor_t &w, const float *lse, float alpha, float beta_dx,
				const mlTensor_t &dx, float beta_dw, const mlTensor_t &dw, const Scratch &s, int piece)
		{
			cudaStream_t stream = use_stream(ctx);
			const float scale = q.dtype == DTYPE_FLOAT16 ? P_SCALE : 1.0f;
			const bool want_dx = !is_empty_descriptor(dx), want_dw = !is_empty_descriptor(dw);
			const float *largest = rows.weights == nullptr ? nullptr : s.largest;
			if (largest != nullptr)
			{
				kernel_largest_weight<<<1, 1024, 0, stream>>>(s.largest, rows, q.tokens);
				MB200_COUNT_LAUNCH();
			}
			if (want_dw)
			{
				kernel_weighted_rows<T> <<<row_blocks(ctx, q.tokens), 256, 0, stream>>>(reinterpret_cast<T*>(s.x), reinterpret_cast<const T*>(x.data), rows, largest, q.tokens, q.embed);
				MB200_COUNT_LAUNCH();
			}
			const mlTensor_t x2 = matrix(x.data, q.dtype, q.tokens, q.embed), dx_sum = matrix(s.dx_sum, DTYPE_FLOAT32, q.tokens, q.embed);
			for (int first = 0; first < q.vocab; first += piece)
			{
				const int width = std::min(piece, q.vocab - first);
				const mlTensor_t wp = piece_of(w, first, width), p = matrix(s.p, q.dtype, q.tokens, width);
				cuda_gemm_v2(ctx, 'n', 't', 1.0f, x2, wp, 0.0f, matrix(s.z, DTYPE_FLOAT32, q.tokens, width));
				kernel_piece_gradient<T> <<<elementwise_blocks(ctx, q.tokens * width), 256, 0, stream>>>(reinterpret_cast<T*>(s.p), s.z, lse, rows, q.tokens, first, width, scale);
				MB200_COUNT_LAUNCH();
				if (want_dx)
					cuda_gemm_v2(ctx, 'n', 'n', 1.0f, p, wp, first == 0 ? 0.0f : 1.0f, dx_sum);
				if (want_dw)
				{
					cuda_gemm_v2(ctx, 't', 'n', 1.0f, p, matrix(s.x, q.dtype, q.tokens, q.embed), 0.0f, matrix(s.dw_sum, DTYPE_FLOAT32, width, q.embed));
					const long long n = static_cast<long long>(width) * q.embed;
					kernel_finish_gradient<T> <<<elementwise_blocks(ctx, n), 256, 0, stream>>>(reinterpret_cast<T*>(dw.data) + static_cast<size_t>(first) * q.embed, s.dw_sum, alpha / scale,
							largest, nullptr, beta_dw, n, q.embed);
					MB200_COUNT_LAUNCH();
				}
			}
			if (want_dx)
			{
				const long long n = q.tokens * q.embed;
				kernel_finish_gradient<T> <<<elementwise_blocks(ctx, n), 256, 0, stream>>>(reinterpret_cast<T*>(dx.data), s.dx_sum, alpha / scale, nullptr, rows.weights, beta_dx, n, q.embed);
				MB200_COUNT_LAUNCH();
			}
			check_cuda(ctx, cudaGetLastError(), "mb200_softmax_cross_entropy_backward");
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
		return q.tokens <= 0 ? 0 : Scratch(q, nullptr, training, recommended_piece(q)).bytes;
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
		flush_pending(context);
		const Scratch s(q, workspace.data, false, piece);
		const Rows rows { reinterpret_cast<const int*>(targets.data), nullptr, q.vocab };
		const mlTensor_t x2 = matrix(x.data, q.dtype, q.tokens, q.embed);
		for (int first = 0; first < q.vocab; first += piece)
		{
			const int width = std::min(piece, q.vocab - first);
			cuda_gemm_v2(context, 'n', 't', 1.0f, x2, piece_of(w, first, width), 0.0f, matrix(s.z, DTYPE_FLOAT32, q.tokens, width));
			kernel_piece_statistics<<<row_blocks(context, q.tokens), 256, 0, use_stream(context)>>>(s.z, s.running, s.target_logit, rows, q.tokens, first, width,
					first + width == q.vocab, reinterpret_cast<float*>(loss.data), reinterpret_cast<float*>(lse.data));
			MB200_COUNT_LAUNCH();
		}
		check_cuda(context, cudaGetLastError(), who);
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
		const Scratch s(q, workspace.data, true, piece);
		const Rows rows { reinterpret_cast<const int*>(targets.data), reinterpret_cast<const float*>(row_weights.data), q.vocab };
		const float *lse_data = reinterpret_cast<const float*>(lse.data);
		if (q.dtype == DTYPE_FLOAT16)
			backward_pieces<__half>(context, q, rows, x, w, lse_data, alpha, beta_dx, dx, beta_dw, dw, s, piece);
		else
			backward_pieces<float>(context, q, rows, x, w, lse_data, alpha, beta_dx, dx, beta_dw, dw, s, piece);
	}
}
