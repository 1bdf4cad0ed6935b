// beam.hip.h -- the selection of a beam search: for every group of W hypotheses the W best of its W x vocabulary continuations.
//
// total(w, v) = score[w] + logit[w][v] - log sum exp logit[w][:], ordered by total (in 64 bits), ties to the lowest w * vocab + v.
// A finished hypothesis goes on in one way: (its end token, its score unchanged).  A beam whose log-sum-exp is not finite -- no finite
// logit, or a NaN or +inf among them -- or whose score is -inf has totals of -inf; among those the lowest index comes first, too.
//
// Reading the logits once bounds it.  k_beam_rows: a workgroup takes a chunk of one row into registers, finds its maximum, the sum of
// exponentials, and each wave its W best values (a bound that at least W reach, then an ordering of the few that do); four waves' lists
// become one.  k_beam_pick: one workgroup per group joins the chunks' sums and lists into every row's W best, then the rows into the group's.
//
// The sum decides the order of continuations of DIFFERENT beams, where 32 bits lose what matters: sums and totals are 64 bits wide from a
// lane's 32 values on.  The exponentials are 32 bits (2^-23 each; their errors are not alike and average over the row): all totals of a beam are off by
// one amount, below 2^-22 and 1e-8 as a rule, and candidates of two beams that are nearer to each other than that may come in either order.
// Rows that are equal, or differ by a constant, get equal sums (a value's place in them follows from its index alone), so equal totals stay equal.
#pragma once

namespace calm {

constexpr int BEAM_MAX = 32;
constexpr int BEAM_VPT = 32;              // values per thread
constexpr int BEAM_CHUNK = 256 * BEAM_VPT; // values per workgroup
constexpr int BEAM_HITS = 32;              // lanes of a wave that k_beam_rows looks through one by one
constexpr int BEAM_LIST = 128;             // candidates that a wave of k_beam_rows keeps
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

// sum over the wave's lanes, in every lane (register moves, as wave_sum63)
__device__ __forceinline__ double beam_wave_sum(double v) {
	const auto dpp = [](double x, auto ctrl, auto row_mask) {
		const unsigned long long b = __builtin_bit_cast(unsigned long long, x);
		const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, decltype(ctrl)::value, decltype(row_mask)::value, 0xf, true);
		const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), decltype(ctrl)::value, decltype(row_mask)::value, 0xf, true);
		return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
	};
	using F = std::integral_constant<int, 0xf>;
	v += dpp(v, std::integral_constant<int, 0xb1>(), F());
	v += dpp(v, std::integral_constant<int, 0x4e>(), F());
	v += dpp(v, std::integral_constant<int, 0x114>(), F());
	v += dpp(v, std::integral_constant<int, 0x118>(), F());
	v += dpp(v, std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>());
	v += dpp(v, std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>());
	const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
	const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)b, 63), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(b >> 32), 63);
	return __builtin_bit_cast(double, ((unsigned long long)hi << 32) | lo);
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

// e^d, d <= 0: the product with log2 e takes the constant's second half along, so that its own rounding (the same for every value) does not add up
__device__ __forceinline__ float beam_exp(float d) {
	return kv_exp2(__builtin_fmaf(d, 1.44269502e+00f, d * 1.92596299e-08f)); // (-inf: 0)
}

// the waves' maxima and sums as the chunk's (64-bit exponentials here would take a workgroup longer than all its values' take)
__device__ inline void beam_sums(const BeamArgs& a, size_t part, const float* m, const double* sum) {
	const float M = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
	double s = 0.;
	for (int w = 0; w < 4; ++w) {
		s += m[w] != BEAM_NONE ? sum[w] * (double)beam_exp(m[w] - M) : sum[w]; // (nothing: 0, or NaN)
	}
	a.sums[2 * part] = (double)M, a.sums[2 * part + 1] = s;
}

__device__ __forceinline__ unsigned beam_wave_max(unsigned v) { // over the wave's lanes, in every lane
	const auto dpp = [](unsigned x, auto ctrl, auto row_mask) { return (unsigned)__builtin_amdgcn_update_dpp((int)x, (int)x, decltype(ctrl)::value, decltype(row_mask)::value, 0xf, false); };
	using F = std::integral_constant<int, 0xf>;
	v = max(v, dpp(v, std::integral_constant<int, 0xb1>(), F()));
	v = max(v, dpp(v, std::integral_constant<int, 0x4e>(), F()));
	v = max(v, dpp(v, std::integral_constant<int, 0x141>(), F()));
	v = max(v, dpp(v, std::integral_constant<int, 0x140>(), F()));
	v = max(v, dpp(v, std::integral_constant<int, 0x142>(), std::integral_constant<int, 0xa>()));
	v = max(v, dpp(v, std::integral_constant<int, 0x143>(), std::integral_constant<int, 0xc>()));
	return (unsigned)__builtin_amdgcn_readlane((int)v, 63);
}
// a value (no NaN) and its index as one number, larger for the better one: the value's bits in order, then the index turned round
__device__ __forceinline__ unsigned long long beam_key(float v, int at) {
	const unsigned b = __builtin_bit_cast(unsigned, v + 0.f); // (-0 is 0)
	return ((unsigned long long)(b >> 31 ? ~b : b | 0x80000000u) << 32) | ~(unsigned)at;
}
__device__ __forceinline__ float beam_key_value(unsigned long long key) {
	const unsigned b = (unsigned)(key >> 32);
	return __builtin_bit_cast(float, b >> 31 ? b & 0x7fffffffu : ~b);
}

// Measured: 128 rows of 128256 fp32 logits 16.8 us = 3.9 TB/s, 80 rows of 32000 at 16 beams 10.9 us, 128 at 32 beams 18.6, 4 rows of 32000 at 4 beams 5.4.
// grid = (chunks, rows)
template <int DT>
__global__ __launch_bounds__(256) void k_beam_rows(BeamArgs a) {
	constexpr int VL = DT == KV_F32 ? 4 : 8; // values of a 16-byte load
	constexpr int NL = BEAM_VPT / VL;
	__shared__ float sm_v[4 * BEAM_MAX];
	__shared__ int sm_i[4 * BEAM_MAX];
	__shared__ float sm_m[4], sm_c[32];
	__shared__ unsigned long long sm_k[4 * BEAM_LIST];
	__shared__ int sm_n[4], sm_hl[4 * BEAM_HITS];
	__shared__ __attribute__((aligned(16))) float sm_h[4 * BEAM_HITS][BEAM_VPT + 4];
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
			a.val[part * W + i] = chunk == 0 && i == 0 ? 0.f : BEAM_NONE; // (k_beam_pick's bound takes values without a look at their tokens)
		}
		if (threadIdx.x == 0) {
			a.sums[2 * part] = chunk == 0 ? 0. : (double)BEAM_NONE;
			a.sums[2 * part + 1] = chunk == 0 ? 1. : 0.;
		}
		return;
	}
	const size_t row0 = (size_t)row * (size_t)a.row;
	// 16-byte loads, wherever the row begins (the memory unit takes them at any address): which thread holds which value must not follow the row's
	// alignment, or the sums of equal rows are added up in different orders and equal totals part.  Loads that are not wholly inside the row go
	// value by value
	constexpr int ES = DT == KV_F32 ? 4 : 2;
	typedef u32x4 any_u32x4 __attribute__((aligned(2)));
	float x[BEAM_VPT];
	const int base = chunk * BEAM_CHUNK;
	u32x4 raw[NL];
	const auto values = [&](int i) {
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			const unsigned one = raw[i][j];
			if constexpr (DT == KV_F32) {
				x[i * VL + j] = __builtin_bit_cast(float, one);
			} else {
				kv_two<DT>(one, x[i * VL + 2 * j], x[i * VL + 2 * j + 1]);
			}
		}
	};
	// (loads first, all of them, then what is made of them: a conversion beside its load is a wait for every one)
	if (base + BEAM_CHUNK <= a.vocab) {
#pragma unroll
		for (int i = 0; i < NL; ++i) {
			raw[i] = *(const any_u32x4*)((const char*)a.logits + (row0 + (size_t)(base + (i * 256 + (int)threadIdx.x) * VL)) * ES);
		}
#pragma unroll
		for (int i = 0; i < NL; ++i) {
			values(i);
		}
	} else {
#pragma unroll
		for (int i = 0; i < NL; ++i) {
			const int at = base + (i * 256 + (int)threadIdx.x) * VL;
			if (at + VL <= a.vocab) {
				raw[i] = *(const any_u32x4*)((const char*)a.logits + (row0 + (size_t)at) * ES);
			}
		}
#pragma unroll
		for (int i = 0; i < NL; ++i) {
			const int at = base + (i * 256 + (int)threadIdx.x) * VL;
			if (at + VL <= a.vocab) {
				values(i);
			} else {
#pragma unroll
				for (int j = 0; j < VL; ++j) {
					x[i * VL + j] = BEAM_NONE;
				}
				if (at < a.vocab) { // across the row's end
#pragma unroll
					for (int j = 0; j < VL; ++j) {
						const int k = at + j < a.vocab ? at + j : a.vocab - 1;
						const float one = beam_load<DT>(a.logits, row0 + k);
						x[i * VL + j] = k == at + j ? one : BEAM_NONE;
					}
				}
			}
		}
	}
	// this lane's largest value; the wave's
	float mine = BEAM_NONE;
#pragma unroll
	for (int i = 0; i < BEAM_VPT; ++i) {
		mine = fmaxf(mine, x[i]);
	}
	const float m = wave_max_dpp(mine);
	// sum of exponentials relative to the wave's maximum
	const float ref = m == BEAM_NONE ? 0.f : m;
	float part_sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
	for (int i = 0; i < BEAM_VPT; ++i) {
		part_sum[i & 3] += beam_exp(x[i] - ref);
	}
	const double sum = beam_wave_sum(((double)part_sum[0] + (double)part_sum[1]) + ((double)part_sum[2] + (double)part_sum[3]));
	if (lane == 0) {
		sm_m[wave] = m, sm_s[wave] = sum;
	}
	// The chunk's W best.  Its lanes are cut into groups, at least W of them; each group's largest value reaches the least of these, so at least W
	// values of the chunk reach that bound.  What does (three times W on average, unless many are equal) goes to a list in LDS, a
	// quarter a wave, as keys in order (beam_key), where a candidate's place is the number of larger ones.  Where a quarter would be longer than
	// BEAM_LIST -- equal values, the few values of a row's end -- rounds over all values find the best instead.  (One list with an atomic
	// counter: 7 us more for 16 x 8 beams over 128256.  Quarters of 64: one workgroup in 40 left for the rounds at 32 beams, and 4 x 32 over 32000
	// took 112 instead of 20 us.)
	float bound;
	{
		// (register moves across the lanes: through the LDS crossbar these few steps took as long as the logits)
		const auto dpp = [](float x, auto ctrl) {
			const int xi = __builtin_bit_cast(int, x);
			return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(xi, xi, decltype(ctrl)::value, 0xf, 0xf, false));
		};
		float v = mine;
		int size = 8; // lanes of a group; W <= 32 takes 8 groups a wave, 16: 4, 8: 2, 4: 1
		v = fmaxf(v, dpp(v, std::integral_constant<int, 0xb1>()));
		v = fmaxf(v, dpp(v, std::integral_constant<int, 0x4e>()));
		v = fmaxf(v, dpp(v, std::integral_constant<int, 0x141>()));
		if (W <= 16) {
			v = fmaxf(v, dpp(v, std::integral_constant<int, 0x140>())), size = 16;
		}
		if (W <= 8) {
			v = kv_max16(v), size = 32;
		}
		if (W <= 4) {
			v = kv_max32(v), size = 64;
		}
		if (lane % size == 0) {
			sm_c[wave * 8 + lane / size] = v;
		}
		__syncthreads();
		const float least = -wave_max_dpp((lane & 7) < 64 / size && lane < 32 ? -sm_c[lane] : -__builtin_inff());
		bound = least;
	}
	const auto place = [&](int i) { // the row's index of this lane's value i
		return base + ((i / VL) * 256 + (int)threadIdx.x) * VL + i % VL;
	};
	const auto inside = [&](int at) { return at < a.vocab; };
	int mine_n = 0; // of the wave's own quarter of the list
	const auto add = [&](bool in, float v, int at) {
		const unsigned long long who = __ballot(in);
		if (who) {
			const int k = mine_n + __builtin_popcountll(who & ((1ull << lane) - 1));
			if (in && k < BEAM_LIST) {
				sm_k[wave * BEAM_LIST + k] = beam_key(v, at);
			}
			mine_n += __builtin_popcountll(who);
		}
	};
	const unsigned long long hits = __ballot(mine >= bound);
	const int n_hits = __builtin_popcountll(hits);
	if (bound != BEAM_NONE && n_hits <= BEAM_HITS) {
		// few lanes hold such values: they put all of theirs into LDS, and the wave looks through two lanes' at a time (a ballot for each of the
		// 32 values of every lane: 6 us more for 16 x 8 beams over 128256)
		if (mine >= bound) {
			const int slot = wave * BEAM_HITS + __builtin_popcountll(hits & ((1ull << lane) - 1));
			sm_hl[slot] = (int)threadIdx.x;
#pragma unroll
			for (int i = 0; i < BEAM_VPT; i += 4) {
				*(kv_f32x4*)&sm_h[slot][i] = (kv_f32x4){x[i], x[i + 1], x[i + 2], x[i + 3]};
			}
		}
		__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
		__builtin_amdgcn_wave_barrier();
		for (int k = 0; k < n_hits; k += 2) {
			const int slot = wave * BEAM_HITS + k + (lane >> 5), i = lane & 31;
			const bool ok = k + (lane >> 5) < n_hits;
			const float v = ok ? sm_h[slot][i] : BEAM_NONE;
			add(v >= bound, v, ok ? base + ((i / VL) * 256 + sm_hl[slot]) * VL + i % VL : 0);
		}
	} else {
#pragma unroll
		for (int i = 0; i < BEAM_VPT; ++i) {
			bool in = x[i] >= bound; // (false for a NaN)
			if (bound == BEAM_NONE) {
				in = in && inside(place(i)); // (what lies outside the row is -inf, too)
			}
			add(in, x[i], place(i));
		}
	}
	if (lane == 0) {
		sm_n[wave] = mine_n;
	}
	__syncthreads();
	const int n0 = sm_n[0], n1 = sm_n[1], n2 = sm_n[2], n3 = sm_n[3], n = n0 + n1 + n2 + n3;
	if (n0 <= BEAM_LIST && n1 <= BEAM_LIST && n2 <= BEAM_LIST && n3 <= BEAM_LIST) {
		const int t = threadIdx.x;
		for (int c = lane; c < mine_n; c += 64) {
			const unsigned long long key = sm_k[wave * BEAM_LIST + c];
			int rank = 0;
#pragma unroll
			for (int w = 0; w < 4; ++w) {
				const int nw = w == 0 ? n0 : w == 1 ? n1 : w == 2 ? n2 : n3;
#pragma unroll 4
				for (int k = 0; k < nw; ++k) {
					rank += sm_k[w * BEAM_LIST + k] > key ? 1 : 0;
				}
			}
			if (rank < W) {
				a.val[part * W + rank] = beam_key_value(key), a.idx[part * W + rank] = (int)~(unsigned)key;
			}
		}
		if (t >= n && t < W) { // fewer than W values in all
			a.val[part * W + t] = BEAM_NONE, a.idx[part * W + t] = -1;
		}
		if (t == 0) {
			beam_sums(a, part, sm_m, sm_s);
		}
		return;
	}
	unsigned taken = 0;
	float bv;
	int bi;
	const auto rescan = [&]() {
		bv = BEAM_NONE, bi = 0x7fffffff;
#pragma unroll
		for (int i = 0; i < BEAM_VPT; ++i) {
			const int at = place(i);
			const bool ok = !((taken >> i) & 1) && inside(at) && x[i] == x[i];
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
	// four lists (each sorted) into one: a candidate's place is its place in its own list plus the better ones of the others
	for (int c = lane; c < 4 * W; c += 64) {
		const int w = c / W, k = c % W;
		const float v = sm_v[w * BEAM_MAX + k];
		const int at = sm_i[w * BEAM_MAX + k];
		int rank = k;
		for (int u = 1; u < 4; ++u) {
			const int q = ((w + u) & 3) * BEAM_MAX;
			for (int j = 0; j < W; ++j) {
				const int other = sm_i[q + j];
				rank += other >= 0 && beam_better(sm_v[q + j], other, v, at) ? 1 : 0;
			}
		}
		if (at >= 0 && rank < W) {
			a.val[part * W + rank] = v, a.idx[part * W + rank] = at;
		}
	}
	{ // fewer than W candidates: the places behind them are empty
		int n = 0;
		for (int c = lane; c < 4 * W; c += 64) {
			n += sm_i[(c / W) * BEAM_MAX + c % W] >= 0;
		}
#pragma unroll
		for (int o = 32; o > 0; o >>= 1) {
			n += __shfl_xor(n, o);
		}
		for (int k = n + lane; k < W; k += 64) {
			a.val[part * W + k] = BEAM_NONE, a.idx[part * W + k] = -1;
		}
	}
	if (lane == 0) {
		beam_sums(a, part, sm_m, sm_s);
	}
}

// grid = groups; a wave per row of the group (16 at a time), then the group's join
__global__ __launch_bounds__(1024) void k_beam_pick(BeamArgs a) {
	__shared__ double sm_t[BEAM_MAX * BEAM_MAX];
	__shared__ int sm_i[BEAM_MAX * BEAM_MAX], sm_r[16 * 16];
	__shared__ float sm_v[16][BEAM_MAX];
	__shared__ int sm_j[16][BEAM_MAX];
	const int lane = lane_id(), wave = wave_id(), W = a.beams, g = blockIdx.x, threads = blockDim.x;
	for (int c = threadIdx.x; c < 256; c += threads) {
		sm_r[c] = 0;
	}
	for (int w = wave; w < W; w += threads / 64) {
		const int row = g * W + w;
		const size_t part = (size_t)row * a.n_chunks;
		const int nc = a.n_chunks * W;
		float v_n;
		int at_n;
		const auto fetch = [&](int c) { // the next portion of candidates, a portion ahead
			const bool ok = c + lane < nc;
			v_n = ok ? a.val[part * W + c + lane] : BEAM_NONE;
			at_n = ok ? a.idx[part * W + c + lane] : -1;
		};
		fetch(0);
		// (at least W candidates reach the least of the chunks' values at place `deep`)
		float bound = -BEAM_NONE;
		const int deep = (W + a.n_chunks - 1) / a.n_chunks - 1;
		for (int c = lane; c < a.n_chunks; c += 64) {
			bound = fminf(bound, a.val[(part + c) * W + deep]);
		}
		bound = -wave_max_dpp(-bound);
		// log of the sum over the chunks, by the same order of additions for every row
		float top = BEAM_NONE; // (the maxima are fp32 numbers)
		for (int c = lane; c < a.n_chunks; c += 64) {
			top = fmaxf(top, (float)a.sums[2 * (part + c)]);
		}
		const double M = (double)wave_max_dpp(top);
		double s = 0.;
		for (int c = lane; c < a.n_chunks; c += 64) {
			const double m = a.sums[2 * (part + c)], x = a.sums[2 * (part + c) + 1];
			s += m == (double)BEAM_NONE ? x : x * (double)beam_exp((float)(m - M)); // (a difference of fp32 numbers)
		}
		s = beam_wave_sum(s);
		const double ls = log(s), base = (double)a.score[row];
		const bool dead = !(M + ls - (M + ls) == 0.) || !(base > (double)BEAM_NONE); // not finite (NaN included)
		if (dead) {
			if (lane < W) {
				sm_t[w * W + lane] = (double)BEAM_NONE, sm_i[w * W + lane] = lane < a.vocab ? lane : -1;
			}
			continue;
		}
		// the W best of the chunks' lists, in portions of 64 candidates: each joins the best so far (one a lane) by counting
		float bv = BEAM_NONE;
		int bi = -1;
		for (int c0 = 0; c0 < nc; c0 += 64) {
			const float v = v_n;
			const int at = at_n;
			fetch(c0 + 64);
			// only what beats the last of the best so far matters
			const float wv = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, bv), W - 1));
			const int wi = __builtin_amdgcn_readlane(bi, W - 1);
			const bool in = at >= 0 && v >= bound && (wi < 0 || beam_better(v, at, wv, wi));
			const unsigned long long who = __ballot(in);
			if (!who) {
				continue;
			}
			int rank_old = bi >= 0 ? lane : 64, rank_new = 0; // lanes [0, W) hold the best so far in order
			for (unsigned long long b = who; b; b &= b - 1) {
				const int l = __builtin_ctzll(b);
				const float x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
				const int j = __builtin_amdgcn_readlane(at, l);
				rank_old += beam_better(x, j, bv, bi) ? 1 : 0;
				rank_new += beam_better(x, j, v, at) ? 1 : 0;
			}
			for (int k = 0; k < W; ++k) {
				const float x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, bv), k));
				const int j = __builtin_amdgcn_readlane(bi, k);
				rank_new += j >= 0 && beam_better(x, j, v, at) ? 1 : 0;
			}
			if (bi >= 0 && lane < W && rank_old < W) {
				sm_v[wave][rank_old] = bv, sm_j[wave][rank_old] = bi;
			}
			if (in && rank_new < W) {
				sm_v[wave][rank_new] = v, sm_j[wave][rank_new] = at;
			}
			__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
			__builtin_amdgcn_wave_barrier();
			const int total = __builtin_popcountll(__ballot(bi >= 0)) + __builtin_popcountll(who);
			if (lane < W && lane < total) {
				bv = sm_v[wave][lane], bi = sm_j[wave][lane];
			}
			__builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
			__builtin_amdgcn_wave_barrier();
		}
		if (lane < W) {
			sm_t[w * W + lane] = bi < 0 ? (double)BEAM_NONE : base + (((double)bv - M) - ls); // (a constant on all of a row's logits leaves no trace)
			sm_i[w * W + lane] = bi;
		}
	}
	__syncthreads();
	// The rows' lists are in order.  Up to 16 rows: a candidate's place in the group is its place in its own list plus, for every other row, how many
	// of that row are better, found by halving, a thread per candidate and other row.  More: one wave, a row a lane, takes the best of their
	// heads W times.  Equal totals: the lower row first (its indices are lower), a row's own in its order.  Measured, the one and the other, this whole
	// kernel: 1 x 4 rows of 4 chunks 4.5 / 5.0 us, 16 x 8 rows of 16 9.7 / 11.4, 5 x 16 rows of 4 14.2 / 13.8, 4 x 32 rows of 4 157 / 37.
	if (W <= 16) {
		for (int it = threadIdx.x; it < W * W * W; it += threads) {
			const int c = it / W, u = it - c * W, w = c / W;
			if (sm_i[c] < 0) {
				continue;
			}
			const double t = sm_t[c];
			int lo = 0, hi = W; // entries [0, lo) are better, [hi, W) are not (empty places, at the end, never are)
			if (u == w) {
				lo = hi = c - w * W;
			}
			while (lo < hi) {
				const int mid = (lo + hi) >> 1;
				const double x = sm_t[u * W + mid];
				const bool better = sm_i[u * W + mid] >= 0 && (x > t || (x == t && u < w));
				lo = better ? mid + 1 : lo, hi = better ? hi : mid;
			}
			if (lo) {
				atomicAdd(&sm_r[c], lo);
			}
		}
		__syncthreads();
		for (int c = threadIdx.x; c < W * W; c += threads) {
			const int w = c / W, at = sm_i[c], rank = sm_r[c];
			if (at >= 0 && rank < W) {
				const int row = g * W + w, out = g * W + rank;
				a.score_out[out] = (float)sm_t[c];
				a.parent[out] = w;
				a.token[out] = at;
				a.done_out[out] = (a.done && a.done[row]) || (a.eos >= 0 && at == a.eos) ? 1 : 0;
			}
		}
		return;
	}
	if (wave != 0) {
		return;
	}
	int k = 0, at = lane < W ? sm_i[lane * W] : -1;
	double t = lane < W ? sm_t[lane * W] : 0.;
	for (int r = 0; r < W; ++r) {
		const unsigned long long b = __builtin_bit_cast(unsigned long long, t + 0.), key = at < 0 ? 0ull : b >> 63 ? ~b : b | 1ull << 63;
		const unsigned hi = (unsigned)(key >> 32), lo = (unsigned)key;
		const unsigned top = beam_wave_max(hi), low = beam_wave_max(hi == top ? lo : 0u);
		const unsigned long long who = __ballot(at >= 0 && hi == top && lo == low);
		if (who && lane == __builtin_ctzll(who)) {
			const int row = g * W + lane, out = g * W + r;
			a.score_out[out] = (float)t;
			a.parent[out] = lane;
			a.token[out] = at;
			a.done_out[out] = (a.done && a.done[row]) || (a.eos >= 0 && at == a.eos) ? 1 : 0;
			++k;
			at = k < W ? sm_i[lane * W + k] : -1;
			t = k < W ? sm_t[lane * W + k] : 0.;
		}
	}
}

} // namespace calm
