/*
 * feed_forward.cu -- the gated feed-forward block y = (act(x Wg^T) * (x Wu^T)) W2^T and its backward pass.
 *
 * W1 = [Wg; Wu] is one matrix [2 F, D] (gate rows first), W2 is [D, F], as a Dense layer stores its weights.  With a = x Wg^T,
 * u = x Wu^T, h = act(a) u and dh = dy W2:
 *   da = dh u act'(a);   du = dh act(a);   dx = [da du] W1;   dW1 = [da du]^T x;   dW2 = dy^T h
 * 6 T D F operations forward and 12 backward; a few tokens are bound by reading the 3 D F weights instead.
 */
#include "common.cuh"
#include "operands.cuh"
#include "gate.cuh"

#include <algorithm>

namespace mb200
{
	namespace
	{
		/* h = act(a) u from the pre-activations au [tokens, 2 hidden], fp32 */
		template<typename T, int GATE>
		__global__ void __launch_bounds__(256) kernel_gate(T *__restrict__ h, const float *__restrict__ au, long long tokens, int hidden)
		{
			const long long total = tokens * hidden, stride = static_cast<long long>(gridDim.x) * 256;
			for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total; i += stride)
			{
				const long long t = i / hidden, at = t * 2 * hidden + (i - t * hidden);
				h[i] = from_float<T>(gate_value<GATE, false>(au[at]) * au[at + hidden]);
			}
		}
		/* [da du] and h from dh [tokens, hidden] and the pre-activations */
		template<typename T, int GATE>
		__global__ void __launch_bounds__(256) kernel_gate_backward(T *__restrict__ dau, T *__restrict__ h, const float *__restrict__ dh, const float *__restrict__ au,
				long long tokens, int hidden)
		{
			const long long total = tokens * hidden, stride = static_cast<long long>(gridDim.x) * 256;
			for (long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x; i < total; i += stride)
			{
				const long long t = i / hidden, at = t * 2 * hidden + (i - t * hidden);
				float value, derivative;
				gate_with_derivative<GATE, false>(au[at], value, derivative);
				const float u = au[at + hidden], d = dh[i];
				dau[at] = from_float<T>(d * u * derivative);
				dau[at + hidden] = from_float<T>(d * value);
				h[i] = from_float<T>(value * u);
			}
		}
		int elementwise_blocks(mlContext_t ctx, long long elements)
		{
			return static_cast<int>(std::max<long long>(1, std::min<long long>((elements + 255) / 256, static_cast<long long>(get(ctx)->sm_count) * 8)));
		}
		mlTensor_t matrix(const void *data, mlDataType_t dtype, long long rows, int columns)
		{
			return make_tensor(data, dtype, make_shape( { static_cast<int>(rows), columns }));
		}

		struct Problem
		{
				mlDataType_t dtype;
				long long tokens;
				int embed, hidden, gate;
		};
		/* What a run needs of the workspace, and where it lies. */
		struct Scratch
		{
				float *au = nullptr; // pre-activations, when the caller keeps none
				float *dh = nullptr;
				void *h = nullptr, *dau = nullptr;
				size_t bytes = 0;
				Scratch(const Problem &p, void *workspace, bool backward, bool own_au)
				{
					Carver carve(workspace);
					const size_t es = size_of(p.dtype), th = static_cast<size_t>(p.tokens) * p.hidden;
					h = carve.take<uint8_t>(th * es);
					if (own_au)
						au = carve.take<float>(2 * th);
					if (backward)
					{
						dau = carve.take<uint8_t>(2 * th * es);
						dh = carve.take<float>(th);
					}
					bytes = carve.used;
				}
		};

		template<typename T>
		void gate_forward(mlContext_t ctx, const Problem &p, void *h, const float *au)
		{
			const long long n = p.tokens * p.hidden;
			with_gate(p.gate, [&](auto gate)
			{
				kernel_gate<T, decltype(gate)::value> <<<elementwise_blocks(ctx, n), 256, 0, use_stream(ctx)>>>(reinterpret_cast<T*>(h), au, p.tokens, p.hidden);
			});
			MB200_COUNT_LAUNCH();
			check_cuda(ctx, cudaGetLastError(), "gated feed-forward: gate");
		}
		template<typename T>
		void gate_backward(mlContext_t ctx, const Problem &p, const Scratch &s, const float *au)
		{
			const long long n = p.tokens * p.hidden;
			with_gate(p.gate, [&](auto gate)
			{
				kernel_gate_backward<T, decltype(gate)::value> <<<elementwise_blocks(ctx, n), 256, 0, use_stream(ctx)>>>(reinterpret_cast<T*>(s.dau), reinterpret_cast<T*>(s.h), s.dh,
						au, p.tokens, p.hidden);
			});
			MB200_COUNT_LAUNCH();
			check_cuda(ctx, cudaGetLastError(), "gated feed-forward: gate backward");
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
			if (p.tokens > 0x7FFFFFFFll / 2)
			{
				record_error(ctx, "%s: %lld tokens are too many for one call", who, p.tokens);
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
		if (p.tokens <= 0)
			return 0;
		return Scratch(p, nullptr, training, !saved).bytes;
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
		const Scratch need(p, nullptr, false, !keep);
		if (!check_workspace(context, who, workspace, need.bytes))
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
		const Scratch s(p, workspace.data, false, !keep);
		float *au = keep ? reinterpret_cast<float*>(saved.data) : s.au;
		const mlTensor_t x2 = matrix(x.data, p.dtype, p.tokens, p.embed);
		cuda_gemm_v2(context, 'n', 't', 1.0f, x2, w1, 0.0f, matrix(au, DTYPE_FLOAT32, p.tokens, 2 * p.hidden));
		if (p.dtype == DTYPE_FLOAT16)
			gate_forward<__half>(context, p, s.h, au);
		else
			gate_forward<float>(context, p, s.h, au);
		cuda_gemm_v2(context, 'n', 't', 1.0f, matrix(s.h, p.dtype, p.tokens, p.hidden), w2, beta, matrix(y.data, p.dtype, p.tokens, p.embed));
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
		const Scratch need(p, nullptr, true, !kept);
		if (p.tokens > 0 && !check_workspace(context, who, workspace, need.bytes))
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
		if (p.tokens == 0)
		{ // no tokens: the weight gradients are sums of nothing
			if (want_dw1)
				cuda_scale_tensor(context, beta_dw, dw1);
			if (want_dw2)
				cuda_scale_tensor(context, beta_dw, dw2);
			return;
		}
		const Scratch s(p, workspace.data, true, !kept);
		const float *au = kept ? reinterpret_cast<const float*>(saved.data) : s.au;
		const mlTensor_t x2 = matrix(x.data, p.dtype, p.tokens, p.embed), dy2 = matrix(dy.data, p.dtype, p.tokens, p.embed);
		if (!kept)
			cuda_gemm_v2(context, 'n', 't', 1.0f, x2, w1, 0.0f, matrix(au, DTYPE_FLOAT32, p.tokens, 2 * p.hidden));
		cuda_gemm_v2(context, 'n', 'n', 1.0f, dy2, w2, 0.0f, matrix(s.dh, DTYPE_FLOAT32, p.tokens, p.hidden));
		if (p.dtype == DTYPE_FLOAT16)
			gate_backward<__half>(context, p, s, au);
		else
			gate_backward<float>(context, p, s, au);
		const mlTensor_t dau = matrix(s.dau, p.dtype, p.tokens, 2 * p.hidden);
		if (want_dx)
			cuda_gemm_v2(context, 'n', 'n', 1.0f, dau, w1, beta_dx, matrix(dx.data, p.dtype, p.tokens, p.embed));
		if (want_dw1)
			cuda_gemm_v2(context, 't', 'n', 1.0f, dau, x2, beta_dw, dw1);
		if (want_dw2)
			cuda_gemm_v2(context, 't', 'n', 1.0f, dy2, matrix(s.h, p.dtype, p.tokens, p.hidden), beta_dw, dw2);
	}
}
