/*
 * feed_forward.cu -- the gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) W2^T and its backward pass.
 *
 * W1 = [Wg; Wu] is one matrix [2 F, D] (gate rows first), W2 is [D, F], as a Dense layer stores its weights.  With a = x Wg^T,
 * u = x Wu^T, h = act(a) u and dh = dy W2:
 *   da = dh u act'(a);   du = dh act(a);   dx = [da du] W1;   dW1 = [da du]^T x;   dW2 = dy^T h
 * 6 T D F operations forward and 12 backward; a few tokens are bound by reading the 3 D F weights instead.
 *
 * fp16: two launches forward (gemm_pair.cu): the first product's tile holds 128 gate and the matching 128 up columns, so its epilogue
 * writes h alone; backward four, [da du] and h coming out of the product that makes dh.  h, da, du are rounded to fp16 once, a and u
 * reach the backward pass in fp32 (rounded to fp16 they would double its error).  fp32: five and eight launches, with the gate between.
 * Forward, a few tokens take two launches of few_tokens.cu (fp16) or of few_rows.cu (fp32, and fp16 rows of odd length, in place).  Elsewhere
 * extents that are no multiple of 16 bytes are copied to padded rows first: F with zero weights, whose h, da and du are zero.
 */
#include "common.cuh"
#include "operands.cuh"
#include "gate.cuh"
#include "gemm_pair.cuh"
#include "gemm_fp32.cuh"
#include "few_tokens.cuh"
#include "few_rows.cuh"

#include <algorithm>

namespace mb200
{
	namespace
	{
		/* The gate between two fp32 products.  Four hidden units a thread; a and u lie `up` floats apart in rows of 2 up (up is hidden, or hidden
		 * without its padding in a kept au, whose rows may start anywhere); the padding's a and u count as zero. */
		struct alignas(16) Four
		{
				float v[4];
		};
		__device__ __forceinline__ void load_pre_activations(Four &a, Four &u, const float *au, long long token, int column, int up)
		{
			const float *src = au + token * 2 * up + column;
			if (up % 4 == 0)
			{
				a = *reinterpret_cast<const Four*>(src);
				u = *reinterpret_cast<const Four*>(src + up);
				return;
			}
#pragma unroll
			for (int k = 0; k < 4; k++)
			{
				a.v[k] = column + k < up ? src[k] : 0.0f;
				u.v[k] = column + k < up ? src[up + k] : 0.0f;
			}
		}
		template<int GATE>
		__global__ void __launch_bounds__(256) kernel_gate(float *h, const float *au, const GridWalk walk, int hidden, int up)
		{
			let_next_grid_start();
			wait_for_previous_grid();
			const long long stride = static_cast<long long>(gridDim.x) * 256;
			for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < walk.total; i += stride)
			{
				long long t;
				int c;
				walk.place(i, t, c);
				c *= 4;
				Four a, u;
				load_pre_activations(a, u, au, t, c, up);
#pragma unroll
				for (int k = 0; k < 4; k++)
					u.v[k] *= gate_value<GATE, false>(a.v[k]);
				*reinterpret_cast<Four*>(h + t * hidden + c) = u;
			}
		}
		/* [da du] and h from dh [tokens, hidden] and the pre-activations */
		template<int GATE>
		__global__ void __launch_bounds__(256) kernel_gate_backward(float *dau, float *h, const float *dh, const float *au,
				const GridWalk walk, int hidden, int up)
		{
			let_next_grid_start();
			wait_for_previous_grid();
			const long long stride = static_cast<long long>(gridDim.x) * 256;
			for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < walk.total; i += stride)
			{
				long long t;
				int c;
				walk.place(i, t, c);
				c *= 4;
				Four a, u, d = *reinterpret_cast<const Four*>(dh + t * hidden + c);
				load_pre_activations(a, u, au, t, c, up);
#pragma unroll
				for (int k = 0; k < 4; k++)
				{
					float value, derivative;
					gate_with_derivative<GATE, false>(a.v[k], value, derivative);
					a.v[k] = d.v[k] * u.v[k] * derivative;
					d.v[k] *= value;
					u.v[k] *= value;
				}
				float *dst = dau + t * 2 * hidden + c;
				*reinterpret_cast<Four*>(dst) = a;
				*reinterpret_cast<Four*>(dst + hidden) = d;
				*reinterpret_cast<Four*>(h + t * hidden + c) = u;
			}
		}
		int elementwise_blocks(mlContext_t ctx, long long elements)
		{
			return static_cast<int>(std::max<long long>(1, std::min<long long>((elements + 255) / 256, static_cast<long long>(get(ctx)->sm_count) * 16)));
		}

		struct Problem
		{
				mlDataType_t dtype;
				long long tokens;
				int embed, hidden, gate;
		};
		/* Keeping a and u moves 16 bytes for every token and hidden unit, making them again costs 4 embed operations: about the same time at
		 * embed = 900 (6 TB/s against 1.4 PFLOP/s).  57 600 tokens x 256 x 1024, forward and backward: 614 us kept, 432 us made again.  Where they are made
		 * again, `saved` keeps h, so that the backward tile, bound by what it writes, does not write it a second time: 367 -> 352 us. */
		constexpr int RECOMPUTE_UP_TO = 1024;
		/* Pitches that TMA can address, and what a run needs of the workspace. */
		struct Plan
		{
				int embed, hidden; // padded
				bool pack_x, pack_w1, pack_w2;
				bool few_rows; // the forward pass goes by few_rows.cu, which reads all rows in place
				bool keeps, keeps_h; // what the forward pass leaves in `saved`: a and u, or h, or nothing
				void *x = nullptr, *w1 = nullptr, *w2 = nullptr, *dy = nullptr, *h = nullptr, *dau = nullptr;
				float *au = nullptr, *dh = nullptr, *partials = nullptr;
				size_t bytes = 0;
				Plan(mlContext_t ctx, const Problem &p, void *workspace, bool backward, bool saved, void *saved_data)
				{
					Carver carve(workspace);
					const int es = size_of(p.dtype), unit = 16 / es;
					const int tokens = static_cast<int>(p.tokens);
					embed = round_up(p.embed, unit);
					hidden = round_up(p.hidden, unit);
					pack_x = embed != p.embed;
					pack_w1 = pack_x || hidden != p.hidden;
					pack_w2 = hidden != p.hidden;
					keeps = saved && (p.dtype == DTYPE_FLOAT32 || (hidden == p.hidden && p.embed > RECOMPUTE_UP_TO));
					// in fp16 only where weights would be copied, and not where `saved` has the form that the tensor-core tile of the backward pass reads
					few_rows = !backward && (p.dtype == DTYPE_FLOAT32 ? p.tokens <= FEW_ROWS_FP32 : p.tokens <= FEW_ROWS_FP16 && pack_w1 && !saved);
					keeps_h = saved && !keeps && hidden <= 4 * p.hidden; // a quarter of the room of a and u, unless it is nearly all padding
					const size_t th = static_cast<size_t>(p.tokens) * hidden, te = static_cast<size_t>(p.tokens) * embed;
					if (few_rows)
					{
						h = carve.take<uint8_t>(th * es);
						bytes = carve.used;
						return;
					}
					if (pack_x)
						x = carve.take<uint8_t>(te * es);
					if (pack_w1)
						w1 = carve.take<uint8_t>(static_cast<size_t>(2) * hidden * embed * es);
					if (pack_w2)
						w2 = carve.take<uint8_t>(static_cast<size_t>(p.embed) * hidden * es);
					h = keeps_h ? saved_data : carve.take<uint8_t>(th * es);
					if (!keeps && p.dtype == DTYPE_FLOAT32)
						au = carve.take<float>(2 * th);
					auto cut = [&](int M, int N, int K)
					{
						return p.dtype == DTYPE_FLOAT16 ? pair_partial_elements(ctx, M, N, K) : float_partial_elements(ctx, M, N, K);
					};
					size_t partial = cut(tokens, p.embed, hidden); // y
					if (p.dtype == DTYPE_FLOAT32)
						partial = std::max( { partial, cut(tokens, 2 * hidden, p.embed), cut(tokens, p.hidden, p.embed) });
					if (backward)
					{
						if (pack_x)
							dy = carve.take<uint8_t>(te * es);
						dau = carve.take<uint8_t>(2 * th * es);
						if (p.dtype == DTYPE_FLOAT32)
						{
							dh = carve.take<float>(th);
							partial = std::max(partial, cut(tokens, hidden, p.embed));
						}
						partial = std::max( { partial, cut(tokens, p.embed, 2 * hidden), cut(2 * p.hidden, p.embed, tokens), cut(p.hidden, p.embed, tokens), cut(p.embed, p.hidden, tokens) });
					}
					partials = carve.take<float>(partial);
					bytes = carve.used;
				}
		};

		/* One pass over operands that TMA can address, in either type. */
		template<typename T>
		struct Run
		{
				mlContext_t ctx;
				const Problem &p;
				const Plan &plan;
				const T *x, *w1, *w2, *dy;
				int tokens;
				Run(mlContext_t context, const Problem &problem, const Plan &scratch, const mlTensor_t &x_, const mlTensor_t &w1_, const mlTensor_t &w2_, const mlTensor_t &dy_) :
						ctx(context),
						p(problem),
						plan(scratch),
						x(padded(x_, plan.x, plan.embed, p.tokens, p.tokens, p.embed, 1)),
						w1(padded(w1_, plan.w1, plan.embed, plan.hidden, p.hidden, p.embed, 2)),
						w2(padded(w2_, plan.w2, plan.hidden, p.embed, p.embed, p.hidden, 1)),
						dy(is_empty_descriptor(dy_) ? nullptr : padded(dy_, plan.dy, plan.embed, p.tokens, p.tokens, p.embed, 1)),
						tokens(static_cast<int>(p.tokens))
				{
				}
				const T* padded(const mlTensor_t &t, void *copy, int pitch, long long padded_rows, long long rows, int columns, int blocks)
				{
					if (copy == nullptr)
						return reinterpret_cast<const T*>(t.data);
					pack_rows<T>(ctx, reinterpret_cast<T*>(copy), pitch, padded_rows, reinterpret_cast<const T*>(t.data), rows, columns, blocks);
					return reinterpret_cast<const T*>(copy);
				}
				/* d [M, N] = a b^T + beta d */
				bool product(int M, int N, int K, const T *a, int lda, bool a_mn, const T *b, int ldb, bool b_mn, T *d, int ldd, float beta)
				{
					if constexpr (sizeof(T) == 2)
						return pair_product(ctx, M, N, K, PairOperand { a, lda, a_mn }, PairOperand { b, ldb, b_mn }, PairResult { d, ldd, 1.0f, beta }, plan.partials);
					else
						return float_product(ctx, M, N, K, FloatOperand { a, lda, a_mn }, FloatOperand { b, ldb, b_mn }, d, ldd, beta, plan.partials);
				}
				/* h, and a and u unless au is null (fp32 needs them) */
				bool gate(float *au)
				{
					if constexpr (sizeof(T) == 2)
						return pair_gated(ctx, tokens, p.embed, plan.hidden, PairOperand { x, plan.embed, false }, PairOperand { w1, plan.embed, false }, p.gate,
								reinterpret_cast<__half*>(plan.h), plan.hidden, au);
					else
					{
						// one product, or two where the rows of a kept au have no padding between a and u
						const int up = up_offset(), parts = up == plan.hidden ? 1 : 2;
						for (int i = 0; i < parts; i++)
							if (!product(tokens, 2 * up / parts, p.embed, x, plan.embed, false, w1 + static_cast<size_t>(i) * plan.hidden * plan.embed, plan.embed, false, au + i * up, 2 * up, 0.0f))
								return false;
						cudaError_t status = cudaSuccess;
						with_gate(p.gate, [&](auto gate)
						{
							status = launch_overlapped(kernel_gate<decltype(gate)::value>, dim3(elementwise_blocks(ctx, p.tokens * plan.hidden / 4)), dim3(256), 0, use_stream(ctx),
									reinterpret_cast<float*>(plan.h), au, GridWalk(p.tokens, plan.hidden / 4), plan.hidden, up);
						});
						MB200_COUNT_LAUNCH();
						return check_cuda(ctx, status, "gated feed-forward: gate");
					}
				}
				int up_offset() const
				{
					return plan.keeps ? p.hidden : plan.hidden;
				}
				bool gate_backward(const float *au)
				{
					if constexpr (sizeof(T) == 2)
						return au == nullptr
								? pair_gated_recompute(ctx, tokens, p.embed, plan.hidden, PairOperand { x, plan.embed, false }, PairOperand { w1, plan.embed, false },
										PairOperand { dy, plan.embed, false }, PairOperand { w2, plan.hidden, true }, p.gate, reinterpret_cast<__half*>(plan.dau),
										plan.keeps_h ? nullptr : reinterpret_cast<__half*>(plan.h))
								: pair_gated_backward(ctx, tokens, p.embed, plan.hidden, PairOperand { dy, plan.embed, false }, PairOperand { w2, plan.hidden, true }, p.gate, au,
								reinterpret_cast<__half*>(plan.dau), reinterpret_cast<__half*>(plan.h));
					else
					{
						if (!product(tokens, plan.hidden, p.embed, dy, plan.embed, false, w2, plan.hidden, true, plan.dh, plan.hidden, 0.0f))
							return false;
						cudaError_t status = cudaSuccess;
						with_gate(p.gate, [&](auto gate)
						{
							status = launch_overlapped(kernel_gate_backward<decltype(gate)::value>, dim3(elementwise_blocks(ctx, p.tokens * plan.hidden / 4)), dim3(256), 0, use_stream(ctx),
									reinterpret_cast<float*>(plan.dau), reinterpret_cast<float*>(plan.h), plan.dh, au, GridWalk(p.tokens, plan.hidden / 4), plan.hidden,
									up_offset());
						});
						MB200_COUNT_LAUNCH();
						return check_cuda(ctx, status, "gated feed-forward: gate backward");
					}
				}
				void forward(T *y, float beta, float *saved)
				{
					float *au = plan.keeps ? saved : plan.au;
					const T *h = reinterpret_cast<const T*>(plan.h);
					if constexpr (sizeof(T) == 2)
						if (tokens <= FEW_TOKENS && au == nullptr)
						{ // decoding: both launches stream their weights once
							if (few_gated(ctx, FewTokens { tokens, plan.embed, x, plan.embed, w1, plan.embed }, plan.hidden, p.gate, reinterpret_cast<__half*>(plan.h), plan.hidden))
								few_product_after_gated(ctx, FewTokens { tokens, plan.hidden, h, plan.hidden, w2, plan.hidden }, p.embed, y, p.embed, beta);
							return;
						}
					if (gate(au))
						product(tokens, p.embed, plan.hidden, h, plan.hidden, false, w2, plan.hidden, false, y, p.embed, beta);
				}
				void backward(const float *saved, float beta_dx, T *dx, float beta_dw, T *dw1, T *dw2)
				{
					const float *au = plan.keeps ? saved : plan.au;
					// without a kept a and u, fp16 makes them again inside gate_backward
					if ((!plan.keeps && sizeof(T) == 4 && !gate(plan.au)) || !gate_backward(au))
						return;
					const T *dau = reinterpret_cast<const T*>(plan.dau), *h = reinterpret_cast<const T*>(plan.h);
					const int F = plan.hidden;
					if (dx != nullptr && !product(tokens, p.embed, 2 * F, dau, 2 * F, false, w1, plan.embed, true, dx, p.embed, beta_dx))
						return;
					if (dw1 != nullptr)
					{ // one product, or two where padding separates the gate rows from the up rows
						const int parts = F == p.hidden ? 1 : 2;
						for (int i = 0; i < parts; i++)
							if (!product(2 * p.hidden / parts, p.embed, tokens, dau + i * F, 2 * F, true, x, plan.embed, true, dw1 + static_cast<size_t>(i) * p.hidden * p.embed, p.embed,
									beta_dw))
								return;
					}
					if (dw2 != nullptr)
						product(p.embed, p.hidden, tokens, dy, plan.embed, true, h, F, true, dw2, p.hidden, beta_dw);
				}
		};
		template<typename T>
		T* data_of(const mlTensor_t &t)
		{
			return reinterpret_cast<T*>(t.data);
		}
		/* The forward pass where plan.few_rows */
		template<typename T>
		void forward_few_rows(mlContext_t ctx, const Problem &p, const Plan &plan, const mlTensor_t &x, const mlTensor_t &w1, const mlTensor_t &w2, T *y, float beta, float *au)
		{
			T *h = reinterpret_cast<T*>(plan.h);
			const int tokens = static_cast<int>(p.tokens);
			if (few_rows_gated(ctx, FewRows<T> { tokens, p.embed, data_of<T>(x), data_of<T>(w1) }, p.hidden, p.gate, h, au))
				few_rows_product(ctx, FewRows<T> { tokens, p.hidden, h, data_of<T>(w2) }, p.embed, y, beta);
		}
		/* TMA reads operands whose rows need no padding from where they lie. */
		bool check_alignment(mlContext_t ctx, const char *who, const char *name, const mlTensor_t &t, bool copied)
		{
			if (copied || t.data == nullptr || aligned_to(t.data, 16))
				return true;
			record_error(ctx, "%s: %s must be 16-byte aligned", who, name);
			return false;
		}

		bool fits_indices(const Problem &p)
		{ // (of w1: two padded rows for every hidden unit)
			return p.tokens <= MAX_EXTENT / 2 && p.hidden <= MAX_EXTENT / 2 && p.embed <= MAX_EXTENT;
		}
		bool check_problem(mlContext_t ctx, const char *who, const mlTensor_t &x, const mlTensor_t &w1, const mlTensor_t &w2, int gate, Problem &p)
		{
			if (!check_extents(ctx, who, "x", x) || !check_extents(ctx, who, "w1", w1) || !check_extents(ctx, who, "w2", w2))
				return false;
			if (x.dtype != DTYPE_FLOAT16 && x.dtype != DTYPE_FLOAT32)
			{
				record_error(ctx, "%s: x is %s, fp16 or fp32 expected", who, dtype_name(x.dtype));
				return false;
			}
			if (gate < MB200_GATE_SIGMOID || gate > MB200_GATE_GELU)
			{
				record_error(ctx, "%s: unknown gate %d", who, gate);
				return false;
			}
			if (w1.rank != 2 || w2.rank != 2 || w1.dim[0] % 2 != 0 || w1.dim[0] == 0 || w1.dim[1] == 0 || w2.dim[0] != w1.dim[1] || w2.dim[1] != w1.dim[0] / 2)
			{
				record_error(ctx, "%s: w1 must be [2 hidden, embed] and w2 [embed, hidden]", who);
				return false;
			}
			p.dtype = x.dtype;
			p.embed = w1.dim[1];
			p.hidden = w1.dim[0] / 2;
			p.gate = gate;
			p.tokens = volume(x) / p.embed;
			if (!fits_indices(p))
			{
				record_error(ctx, "%s: %lld tokens, %d hidden units and an embed of %d are too many for one call", who, p.tokens, p.hidden, p.embed);
				return false;
			}
			return check_operand(ctx, who, "x", x, x.dtype, p.tokens, p.embed) && check_operand(ctx, who, "w1", w1, x.dtype, 2ll * p.hidden, p.embed)
					&& check_operand(ctx, who, "w2", w2, x.dtype, p.embed, p.hidden);
		}
	}
} /* namespace mb200 */

using namespace mb200;

extern "C"
{
	size_t mb200_gated_feed_forward_get_workspace_size(mlContext_t context, mlShape_t x_shape, mlShape_t w1_shape, mlDataType_t dtype, bool training, bool saved)
	{
		if (context == nullptr || x_shape.rank < 1 || x_shape.rank > 6 || w1_shape.rank != 2 || w1_shape.dim[0] <= 0 || w1_shape.dim[1] <= 0 || last_dim(x_shape) != w1_shape.dim[1])
			return 0;
		const Problem p { dtype, volume_without_last_dim(x_shape), w1_shape.dim[1], w1_shape.dim[0] / 2, MB200_GATE_SILU };
		if (p.tokens <= 0 || !fits_indices(p) || (dtype != DTYPE_FLOAT16 && dtype != DTYPE_FLOAT32))
			return 0;
		return std::max(Plan(context, p, nullptr, false, training && saved, nullptr).bytes, training ? Plan(context, p, nullptr, true, saved, nullptr).bytes : 0);
	}

	void mb200_gated_feed_forward_forward(mlContext_t context, const mlTensor_t x, const mlTensor_t w1, const mlTensor_t w2, float beta, mlTensor_t y, int gate, mlTensor_t saved,
			mlTensor_t workspace)
	{
		const char *who = "mb200_gated_feed_forward_forward";
		MB200_REQUIRE(context, context != nullptr, "%s: null context", who);
		Problem p;
		if (!check_problem(context, who, x, w1, w2, gate, p) || !check_operand(context, who, "y", y, x.dtype, p.tokens, p.embed))
			return;
		const bool keep = !is_empty_descriptor(saved);
		if (keep && !check_operand(context, who, "saved", saved, DTYPE_FLOAT32, p.tokens, 2ll * p.hidden))
			return;
		if (p.tokens == 0)
			return;
		const Plan plan(context, p, workspace.data, false, keep, saved.data);
		if (!check_workspace(context, who, workspace, plan.bytes) || !check_alignment(context, who, "x", x, plan.pack_x) || !check_alignment(context, who, "w1", w1, plan.pack_w1)
				|| !check_alignment(context, who, "w2", w2, plan.pack_w2) || !check_alignment(context, who, "saved", saved, !(plan.keeps && plan.hidden == p.hidden) && !plan.keeps_h))
			return;
		const struct { const char *name; const mlTensor_t &t; } inputs[] = { { "x", x }, { "w1", w1 }, { "w2", w2 } }, results[] = { { "y", y }, { "saved", saved }, { "workspace", workspace } };
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
		if (plan.few_rows && p.dtype == DTYPE_FLOAT16)
			forward_few_rows<__half>(context, p, plan, x, w1, w2, data_of<__half>(y), beta, nullptr);
		else if (plan.few_rows)
			forward_few_rows<float>(context, p, plan, x, w1, w2, data_of<float>(y), beta, data_of<float>(saved));
		else if (p.dtype == DTYPE_FLOAT16)
			Run<__half>(context, p, plan, x, w1, w2, no_tensor()).forward(data_of<__half>(y), beta, data_of<float>(saved));
		else
			Run<float>(context, p, plan, x, w1, w2, no_tensor()).forward(data_of<float>(y), beta, data_of<float>(saved));
	}

	void mb200_gated_feed_forward_backward(mlContext_t context, const mlTensor_t x, const mlTensor_t w1, const mlTensor_t w2, const mlTensor_t saved, const mlTensor_t dy, float beta_dx,
			mlTensor_t dx, float beta_dw, mlTensor_t dw1, mlTensor_t dw2, int gate, mlTensor_t workspace)
	{
		const char *who = "mb200_gated_feed_forward_backward";
		MB200_REQUIRE(context, context != nullptr, "%s: null context", who);
		Problem p;
		if (!check_problem(context, who, x, w1, w2, gate, p) || !check_operand(context, who, "dy", dy, x.dtype, p.tokens, p.embed))
			return;
		const bool kept = !is_empty_descriptor(saved), want_dx = !is_empty_descriptor(dx), want_dw1 = !is_empty_descriptor(dw1), want_dw2 = !is_empty_descriptor(dw2);
		if ((kept && !check_operand(context, who, "saved", saved, DTYPE_FLOAT32, p.tokens, 2ll * p.hidden))
				|| (want_dx && !check_operand(context, who, "dx", dx, x.dtype, p.tokens, p.embed))
				|| (want_dw1 && !check_operand(context, who, "dw1", dw1, x.dtype, 2ll * p.hidden, p.embed))
				|| (want_dw2 && !check_operand(context, who, "dw2", dw2, x.dtype, p.embed, p.hidden)))
			return;
		if (p.tokens == 0)
		{ // no tokens: the weight gradients are sums of nothing
			if (want_dw1)
				cuda_scale_tensor(context, beta_dw, dw1);
			if (want_dw2)
				cuda_scale_tensor(context, beta_dw, dw2);
			return;
		}
		const Plan plan(context, p, workspace.data, true, kept, saved.data);
		if (!check_workspace(context, who, workspace, plan.bytes) || !check_alignment(context, who, "x", x, plan.pack_x) || !check_alignment(context, who, "dy", dy, plan.pack_x)
				|| !check_alignment(context, who, "w1", w1, plan.pack_w1) || !check_alignment(context, who, "w2", w2, plan.pack_w2)
				|| !check_alignment(context, who, "saved", saved, !(plan.keeps && plan.hidden == p.hidden) && !plan.keeps_h))
			return;
		const struct { const char *name; const mlTensor_t &t; } inputs[] = { { "x", x }, { "w1", w1 }, { "w2", w2 }, { "saved", saved }, { "dy", dy } }, results[] = { { "dx", dx },
				{ "dw1", dw1 }, { "dw2", dw2 }, { "workspace", workspace } };
		for (int i = 0; i < 4; i++)
		{
			for (const auto &in : inputs)
				if (!check_distinct(context, who, results[i].name, results[i].t, in.name, in.t))
					return;
			for (int k = 0; k < i; k++)
				if (!check_distinct(context, who, results[i].name, results[i].t, results[k].name, results[k].t))
					return;
		}
		flush_pending(context);
		if (p.dtype == DTYPE_FLOAT16)
			Run<__half>(context, p, plan, x, w1, w2, dy).backward(data_of<float>(saved), beta_dx, data_of<__half>(dx), beta_dw, data_of<__half>(dw1), data_of<__half>(dw2));
		else
			Run<float>(context, p, plan, x, w1, w2, dy).backward(data_of<float>(saved), beta_dx, data_of<float>(dx), beta_dw, data_of<float>(dw1), data_of<float>(dw2));
	}
}
