/*
 * gate.cuh -- the activations of the gated feed-forward block and their derivatives, in fp32.
 *   sigmoid: s(g);   relu: max(g, 0), derivative 0 at 0;   silu: g s(g);   gelu: g Phi(g), Phi the normal distribution function
 * FAST takes the exponential from the hardware's base-2 one, relative error |g| * 2^-24 on top of two units in the last place: below
 * what is lost when the result is rounded to fp16, and not used for fp32 data.
 */
#pragma once

#include "common.cuh"

namespace mb200
{
	template<bool FAST>
	__device__ __forceinline__ float gate_exp(float x)
	{
		return FAST ? __expf(x) : expf(x);
	}
	template<bool FAST>
	__device__ __forceinline__ float gate_sigmoid(float g)
	{ // exp overflows to infinity for large negative g, which gives the right 0
		return FAST ? __fdividef(1.0f, 1.0f + __expf(-fmaxf(g, -80.0f))) : 1.0f / (1.0f + expf(-g));
	}
	template<int GATE, bool FAST>
	__device__ __forceinline__ void gate_with_derivative(float g, float &value, float &derivative)
	{
		if (GATE == MB200_GATE_RELU)
		{
			value = g < 0.0f ? 0.0f : g; // a NaN stays one
			derivative = g > 0.0f ? 1.0f : 0.0f;
		}
		else if (GATE == MB200_GATE_GELU)
		{
			const float phi = 0.5f + 0.5f * erff(g * 0.70710678f);
			value = g * phi;
			derivative = phi + 0.39894228f * g * gate_exp<FAST>(-0.5f * g * g);
		}
		else
		{
			const float s = gate_sigmoid<FAST>(g);
			value = GATE == MB200_GATE_SIGMOID ? s : g * s;
			derivative = GATE == MB200_GATE_SIGMOID ? s * (1.0f - s) : s * (1.0f + g * (1.0f - s));
		}
	}
	template<int GATE, bool FAST>
	__device__ __forceinline__ float gate_value(float g)
	{
		float value, derivative;
		gate_with_derivative<GATE, FAST>(g, value, derivative);
		return value;
	}
	/* Calls `f` with the gate as a compile-time constant. */
	template<int GATE>
	struct GateTag
	{
			static constexpr int value = GATE;
	};
	template<typename F>
	auto with_gate(int gate, F f)
	{
		switch (gate)
		{
			case MB200_GATE_SIGMOID:
				return f(GateTag<MB200_GATE_SIGMOID>());
			case MB200_GATE_RELU:
				return f(GateTag<MB200_GATE_RELU>());
			case MB200_GATE_GELU:
				return f(GateTag<MB200_GATE_GELU>());
			default:
				return f(GateTag<MB200_GATE_SILU>());
		}
	}
} /* namespace mb200 */
