/*
 * gate.cuh -- the activations of the gated feed-forward block and their derivatives, in fp32.
 *   sigmoid: s(g);   relu: max(g, 0), derivative 0 at 0;   silu: g s(g);   gelu: g Phi(g), Phi the normal distribution function
 * FAST takes the exponential from the hardware's base-2 one, relative error |g| * 2^-24 on top of two units in the last place: below
 * what is lost when the result is rounded to fp16, and not used for fp32 data.
 */
#pragma once

#include "common.cuh"
#include "pairs.cuh"

namespace mb200
{
	__device__ __forceinline__ float reciprocal_approx(float x)
	{
		float y;
		asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
		return y;
	}
	/* 1 / (1 + 2^(-g log2 e)) of two values with one reciprocal, 1 / a = b / (a b): the special-function unit is what an epilogue with this gate
	 * runs out of first (three instead of four of its instructions for two values).  The power is held at 2^60 so that the product stays
	 * finite, and a sigmoid that would be less than 2^-60 is 0 (2^-60 is not: g and u of 4e5 make 0.1 of it).  A NaN comes out as 2^-60. */
	__device__ __forceinline__ Pair sigmoid_fast(Pair g)
	{
		const Pair t = pair_mul(g, Pair { -1.44269504f, -1.44269504f });
		Pair e;
		asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(fminf(t.x, 60.0f)));
		asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(fminf(t.y, 60.0f)));
		e = pair_add(e, Pair { 1.0f, 1.0f });
		const float r = reciprocal_approx(e.x * e.y);
		const Pair s = pair_mul(Pair { r, r }, Pair { e.y, e.x });
		return Pair { t.x > 60.0f ? 0.0f : s.x, t.y > 60.0f ? 0.0f : s.y };
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
			derivative = phi + 0.39894228f * g * (FAST ? __expf(-0.5f * g * g) : expf(-0.5f * g * g));
		}
		else
		{ // exp overflows to infinity for large negative g, which gives the right 0
			const float s = FAST ? __fdividef(1.0f, 1.0f + __expf(-g)) : 1.0f / (1.0f + expf(-g));
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
	/* The FAST forms for two values at a time. */
	template<int GATE>
	__device__ __forceinline__ void gate_with_derivative(Pair g, Pair &value, Pair &derivative)
	{
		if (GATE == MB200_GATE_SILU || GATE == MB200_GATE_SIGMOID)
		{
			Pair s = sigmoid_fast(g);
			if (GATE == MB200_GATE_SIGMOID)
				s = Pair { g.x == g.x ? s.x : g.x, g.y == g.y ? s.y : g.y }; // (a NaN has passed sigmoid_fast as if it were large)
			const Pair rest = pair_fma(s, pair_of(-1.0f), pair_of(1.0f)); // 1 - s
			value = GATE == MB200_GATE_SIGMOID ? s : pair_mul(g, s);
			derivative = GATE == MB200_GATE_SIGMOID ? pair_mul(s, rest) : pair_fma(value, rest, s); // silu: s + g s (1 - s)
		}
		else
		{
			gate_with_derivative<GATE, true>(g.x, value.x, derivative.x);
			gate_with_derivative<GATE, true>(g.y, value.y, derivative.y);
		}
	}
	template<int GATE>
	__device__ __forceinline__ Pair gate_value(Pair g)
	{
		Pair value, derivative;
		gate_with_derivative<GATE>(g, value, derivative);
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
