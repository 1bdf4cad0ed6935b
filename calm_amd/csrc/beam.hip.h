// beam.hip.h -- the selection of a beam search: for every group of W hypotheses the W best of its W x vocabulary continuations.
//
// total(w, v) = score[w] + logit[w][v] - log sum exp logit[w][:], ordered by total (in 64 bits), ties to the lowest w * vocab + v.
// A finished hypothesis goes on in one way: (its end token, its score unchanged).  A beam whose log-sum-exp is not finite -- no finite
// logit, or a NaN or +inf among them -- or whose score is -inf has totals of -inf; among those the lowest index comes first, too.
//
// Reading the logits once bounds it.  k_beam_rows: a workgroup takes a chunk of one row into registers, finds its maximum, the sum of
// exponentials, and each wave its W best values (W rounds of a wave-wide maximum); four waves' lists become one.  k_beam_pick: one
// workgroup per group joins the chunks' sums and lists into every row's W best, then the rows into the group's.
//
// The sum decides the order of continuations of DIFFERENT beams, where 32 bits lose what matters: differences and the sum are 64 bits
// wide, the exponentials 32 (their errors, 2^-23 each, are not alike and average over the row).
#pragma once

namespace calm {

constexpr int BEAM_MAX = 32;
constexpr int BEAM_VPT = 32;              // values per thread
constexpr int BEAM_CHUNK = 256 * BEAM_VPT; // values per workgroup
constexpr float BEAM_NONE = -__builtin_inff();

struct BeamArgs {
	const void* logits;
	long row; // stride of a row of logits, in elements
	const float* score;
	const unsigned char* done;
	float* score_out;
	int *parent, *token;
	unsigned char* done_out;
	double* sums; // [row][chunk] x {maximum, sum}
	float* val;   // [row][chunk][W]
	int* idx;     // ... -1: no candidate
	int groups, beams, vocab, n_chunks, eos;
};

// better(value, index): larger value, then lower index
__device__ __forceinline__ bool beam_better(float v, int i, float w, int j) {
	return v > w || (v == w && i < j);
}
__device__ __forceinline__ bool beam_better(double v, int i, double w, int j) {
	return v > w || (v == w && i < j);
}

template <class T>
__device__ __forceinline__ void beam_wave_best(T& v, int& i) {
#pragma unroll
	for (int o = 32; o > 0; o >>= 1) {
		const T w = __shfl_xor(v, o);
		const int j = __shfl_xor(i, o);
		if (beam_better(w, j, v, i)) {
			v = w, i = j;
		}
	}
}

template <int DT>
__device__ __forceinline__ float beam_load(const void* p, size_t i) {
	if constexpr (DT == KV_F32) {
		return ((const float*)p)[i];
	} else if constexpr (DT == KV_F16) {
		return (float)((const _Float16*)p)[i];
	} else {
		return __builtin_bit_cast(float, (unsigned)((const unsigned short*)p)[i] << 16);
	}
}

// grid = (chunks, rows)
template <int DT>
__global__ __launch_bounds__(256) void k_beam_rows(BeamArgs a) {
	constexpr int VL = DT == KV_F32 ? 4 : 8; // values of a 16-byte load
	constexpr int NL = BEAM_VPT / VL;
	__shared__ float sm_v[4 * BEAM_MAX];
	__shared__ int sm_i[4 * BEAM_MAX];
	__shared__ float sm_m[4];
	__shared__ double sm_s[4];
	const int lane = lane_id(), wave = wave_id(), chunk = blockIdx.x, row = blockIdx.y, W = a.beams;
	const size_t part = (size_t)row * a.n_chunks + chunk;
	if (a.done && a.done[row]) { // the end token, then tokens that cannot come (-inf), the lowest first
		if (threadIdx.x < W) {
			const int i = (int)threadIdx.x;
			int tok = -1;
			if (chunk == 0) {
				tok = i == 0 ? a.eos : (i - 1 < a.eos ? i - 1 : i);
			}
			a.idx[part * W + i] = tok < a.vocab ? tok : -1;
			a.val[part * W + i] = i == 0 ? 0.f : BEAM_NONE;
		}
		if (threadIdx.x == 0) {
			a.sums[2 * part] = chunk == 0 ? 0. : (double)BEAM_NONE;
			a.sums[2 * part + 1] = chunk == 0 ? 1. : 0.;
		}
		return;
	}
	const size_t row0 = (size_t)row * (size_t)a.row;
	// 16-byte loads whatever the row's alignment: the row begins `mis` values behind a 16-byte boundary, and value i of the row is
	// value i + mis from there; loads that are not wholly inside the row go value by value
	constexpr int ES = DT == KV_F32 ? 4 : 2;
	const int mis = (int)((((size_t)a.logits + row0 * ES) & 15) / ES);
	float x[BEAM_VPT];
	const int base = chunk * BEAM_CHUNK - mis;
#pragma unroll
	for (int i = 0; i < NL; ++i) {
		const int at = base + (i * 256 + (int)threadIdx.x) * VL;
		if (at >= 0 && at + VL <= a.vocab) {
			const u32x4 w = *(const u32x4*)((const char*)a.logits + (row0 + (size_t)at) * ES);
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				const unsigned one = w[j];
				if constexpr (DT == KV_F32) {
					x[i * VL + j] = __builtin_bit_cast(float, one);
				} else {
					kv_two<DT>(one, x[i * VL + 2 * j], x[i * VL + 2 * j + 1]);
				}
			}
		} else {
#pragma unroll
			for (int j = 0; j < VL; ++j) {
				x[i * VL + j] = at + j >= 0 && at + j < a.vocab ? beam_load<DT>(a.logits, row0 + at + j) : BEAM_NONE;
			}
		}
	}
	float m = BEAM_NONE;
#pragma unroll
	for (int i = 0; i < BEAM_VPT; ++i) {
		m = fmaxf(m, x[i]);
	}
	m = wave_max_dpp(m);
	// sum of 2^((x - m) log2 e) relative to the wave's maximum
	double sum = 0.;
	const float ref = m == BEAM_NONE ? 0.f : m;
#pragma unroll
	for (int i = 0; i < BEAM_VPT; ++i) {
		const double t = ((double)x[i] - (double)ref) * 1.4426950408889634074;
		const double n = __builtin_rint(t);
		// (-inf: n = -inf, the difference NaN)
		const float f = x[i] == BEAM_NONE ? 0.f : ldexpf(kv_exp2((float)(t - n)), n < -200. ? -200 : (int)n);
		sum += (double)f;
	}
#pragma unroll
	for (int o = 32; o > 0; o >>= 1) {
		sum += __shfl_xor(sum, o);
	}
	if (lane == 0) {
		sm_m[wave] = m, sm_s[wave] = sum;
	}
	// the wave's W best: its lanes' best, W times; the lane that gave one looks for its next
	unsigned taken = 0;
	float bv;
	int bi;
	const auto rescan = [&]() {
		bv = BEAM_NONE, bi = 0x7fffffff;
#pragma unroll
		for (int i = 0; i < BEAM_VPT; ++i) {
			const int at = base + ((i / VL) * 256 + (int)threadIdx.x) * VL + i % VL;
			const bool ok = !((taken >> i) & 1) && at >= 0 && at < a.vocab && x[i] == x[i];
			if (ok && beam_better(x[i], at, bv, bi)) {
				bv = x[i], bi = at;
			}
		}
	};
	rescan();
	for (int k = 0; k < W; ++k) {
		float v = bv;
		int i = bi;
		beam_wave_best(v, i);
		if (lane == 0) {
			sm_v[wave * BEAM_MAX + k] = v, sm_i[wave * BEAM_MAX + k] = i == 0x7fffffff ? -1 : i;
		}
		if (i == bi && i != 0x7fffffff) {
			const int rel = i - base, q = rel / (256 * VL), r = rel % VL;
			taken |= 1u << (q * VL + r);
			rescan();
		}
	}
	__syncthreads();
	if (wave != 0) {
		return;
	}
	// four lists (each sorted) into one: lane l < 4 W holds candidate l
	float cv[2];
	int ci[2];
#pragma unroll
	for (int j = 0; j < 2; ++j) {
		const int c = lane + 64 * j;
		const bool ok = c < 4 * W;
		cv[j] = ok ? sm_v[(c / W) * BEAM_MAX + c % W] : BEAM_NONE;
		ci[j] = ok ? sm_i[(c / W) * BEAM_MAX + c % W] : -1;
		ci[j] = ci[j] < 0 ? 0x7fffffff : ci[j];
	}
	for (int k = 0; k < W; ++k) {
		const bool second = beam_better(cv[1], ci[1], cv[0], ci[0]);
		float v = second ? cv[1] : cv[0];
		int i = second ? ci[1] : ci[0];
		const int mine = i;
		beam_wave_best(v, i);
		if (lane == 0) {
			a.val[part * W + k] = v, a.idx[part * W + k] = i == 0x7fffffff ? -1 : i;
		}
		if (mine == i && i != 0x7fffffff) {
			if (second) {
				ci[1] = 0x7fffffff, cv[1] = BEAM_NONE;
			} else {
				ci[0] = 0x7fffffff, cv[0] = BEAM_NONE;
			}
		}
	}
	if (lane == 0) {
		const float M = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
		double s = 0.;
		for (int w = 0; w < 4; ++w) {
			if (sm_m[w] != BEAM_NONE) {
				s += sm_s[w] * exp((double)sm_m[w] - (double)M);
			} else {
				s += sm_s[w]; // 0, or NaN
			}
		}
		a.sums[2 * part] = (double)M, a.sums[2 * part + 1] = s;
	}
}

// grid = groups; one wave per row of the group at a time, then one wave for the group
__global__ __launch_bounds__(512) void k_beam_pick(BeamArgs a) {
	__shared__ double sm_t[BEAM_MAX * BEAM_MAX];
	__shared__ int sm_i[BEAM_MAX * BEAM_MAX];
	const int lane = lane_id(), wave = wave_id(), W = a.beams, g = blockIdx.x;
	for (int w = wave; w < W; w += 8) {
		const int row = g * W + w;
		const size_t part = (size_t)row * a.n_chunks;
		// log of the sum over the chunks, by the same order of additions for every row
		double M = (double)BEAM_NONE;
		for (int c = lane; c < a.n_chunks; c += 64) {
			const double m = a.sums[2 * (part + c)];
			M = m > M ? m : M;
		}
#pragma unroll
		for (int o = 32; o > 0; o >>= 1) {
			const double m = __shfl_xor(M, o);
			M = m > M ? m : M;
		}
		double s = 0.;
		for (int c = lane; c < a.n_chunks; c += 64) {
			const double m = a.sums[2 * (part + c)], x = a.sums[2 * (part + c) + 1];
			s += m == (double)BEAM_NONE ? x : x * exp(m - M);
		}
#pragma unroll
		for (int o = 32; o > 0; o >>= 1) {
			s += __shfl_xor(s, o);
		}
		const double lse = M + log(s), base = (double)a.score[row];
		const bool dead = !(lse - lse == 0.) || !(base > (double)BEAM_NONE); // not finite (NaN included)
		if (dead) {
			if (lane < W) {
				sm_t[w * W + lane] = (double)BEAM_NONE, sm_i[w * W + lane] = lane < a.vocab ? lane : -1;
			}
			continue;
		}
		// the W best of the chunks' lists: a lane walks the lists lane, lane + 64, ...; each list is sorted, so a lane's best is among
		// the heads of its lists
		const int nc = a.n_chunks * W;
		float last = __builtin_inff();
		int last_i = -1; // the one chosen before: the next is the best that is not better
		for (int k = 0; k < W; ++k) {
			float v = BEAM_NONE;
			int i = 0x7fffffff;
			for (int c = lane; c < nc; c += 64) {
				const float x = a.val[part * W + c];
				const int j = a.idx[part * W + c];
				if (j >= 0 && beam_better(last, last_i, x, j) && beam_better(x, j, v, i)) {
					v = x, i = j;
				}
			}
			beam_wave_best(v, i);
			last = v, last_i = i;
			if (lane == 0) {
				sm_t[w * W + k] = i == 0x7fffffff ? (double)BEAM_NONE : base + ((double)v - lse);
				sm_i[w * W + k] = i == 0x7fffffff ? -1 : i;
			}
		}
	}
	__syncthreads();
	if (wave != 0) {
		return;
	}
	double t[BEAM_MAX * BEAM_MAX / 64];
	int f[BEAM_MAX * BEAM_MAX / 64]; // index in the group's W x W list; ordered by (beam, token) below
#pragma unroll
	for (int j = 0; j < BEAM_MAX * BEAM_MAX / 64; ++j) {
		const int c = lane + 64 * j;
		const bool ok = c < W * W && sm_i[c] >= 0;
		t[j] = ok ? sm_t[c] : (double)BEAM_NONE;
		f[j] = ok ? c : -1;
	}
	const auto flat = [&](int c) { // (w, token) as one number that fits: w * vocab + token can pass 32 bits
		return c < 0 ? 0x7fffffffffffffffll : (long long)(c / W) * a.vocab + sm_i[c];
	};
	for (int k = 0; k < W; ++k) {
		double bt = (double)BEAM_NONE;
		int bc = -1;
#pragma unroll
		for (int j = 0; j < BEAM_MAX * BEAM_MAX / 64; ++j) {
			if (64 * j < W * W && f[j] >= 0 && (t[j] > bt || (t[j] == bt && flat(f[j]) < flat(bc)))) {
				bt = t[j], bc = f[j];
			}
		}
		long long bf = flat(bc);
#pragma unroll
		for (int o = 32; o > 0; o >>= 1) {
			const double ot = __shfl_xor(bt, o);
			const int oc = __shfl_xor(bc, o);
			const long long of = __shfl_xor(bf, o);
			if (ot > bt || (ot == bt && of < bf)) {
				bt = ot, bc = oc, bf = of;
			}
		}
#pragma unroll
		for (int j = 0; j < BEAM_MAX * BEAM_MAX / 64; ++j) {
			f[j] = f[j] == bc ? -1 : f[j];
		}
		if (lane == 0) {
			const int w = bc / W, tok = sm_i[bc], row = g * W + w;
			a.score_out[g * W + k] = (float)bt;
			a.parent[g * W + k] = w;
			a.token[g * W + k] = tok;
			a.done_out[g * W + k] = (a.done && a.done[row]) || (a.eos >= 0 && tok == a.eos) ? 1 : 0;
		}
	}
}

} // namespace calm
