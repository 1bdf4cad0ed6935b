// paged.hip.h -- a cache of several sequences in pages of 8-bit codes, and the kernels that fill, read, share and move them.
//
// Layout (struct KvPool, include/calm_hip.h).  A page holds KV_PAGE = 64 tokens of one sequence for every layer and kv head:
//   K codes  [page][kv head][token 64][dim]                              int8, a token's dims contiguous
//   V codes  [page][kv head][quad 4][dim][block 4][token 4]               int8: quad g of a dim holds tokens 4 g .. 4 g + 3 of each of
//                                                                         the page's four blocks -- the 16 bytes one lane feeds to the
//                                                                         V operand of two (four) matrix instructions
//   scales   [page][kv head][block 4] for K and for V                     fp32 powers of two: a block is KV_BLOCK = 16 tokens of one head
// value = code * scale, codes in [-127, 127].  Powers of two make every step exact but the one rounding to a code: the division, the
// value read back, and the products of codes on the matrix cores (an int8 is exact in binary16).  Next to a free scale max / 127 they cost
// at most one bit of the eight (half a bit on average over a block's maximum); in return a block whose scale grows (a later token of the
// block is larger) is re-rounded by a shift, and results do not depend on how a division rounds.
// A block that met an infinity or a NaN has the scale NaN: every row that sees one of its tokens is NaN, no other row is.
#pragma once

namespace calm {

constexpr int KV_PAGE = 64, KV_BLOCK = 16;

// bits of KvPool::status, raised by the kernels and cleared by the host
enum { KV_BAD_PAGE = 1, KV_NO_PAGE = 2, KV_BAD_BATCH = 4, KV_BAD_PARENT = 8 };
enum { KV_F32 = 0, KV_F16 = 1, KV_BF16 = 2 };

typedef _Float16 kv_f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 kv_f16x8 __attribute__((ext_vector_type(8)));
typedef float kv_f32x4 __attribute__((ext_vector_type(4)));
typedef int kv_i32x4 __attribute__((ext_vector_type(4)));
typedef float kv_f32x16 __attribute__((ext_vector_type(16)));

// one layer of a pool
struct KvLayer {
	signed char *k, *v;
	float *ks, *vs;
	unsigned* status;
	int n_pages, n_kv_heads;
};
// the rows of a call: sequence s owns rows [cu[s], cu[s + 1]) of the packed row arrays, its last ones; lens[s] counts them in
struct KvRows {
	const int *cu, *lens, *table;
	int n_seqs, max_pages, n_rows, max_rows;
};

__device__ __forceinline__ void kv_flag(unsigned* status, unsigned bit) {
	atomicOr(status, bit);
}

// ---- types ----------------------------------------------------------------------------------------------------------------------------

// the two values of a word of a 16-bit type
template <int DT>
__device__ __forceinline__ void kv_two(unsigned w, float& a, float& b) {
	if constexpr (DT == KV_F16) {
		const kv_f16x2 h = __builtin_bit_cast(kv_f16x2, w);
		a = (float)h[0], b = (float)h[1];
	} else {
		a = __builtin_bit_cast(float, w << 16), b = __builtin_bit_cast(float, w & 0xffff0000u);
	}
}
// four values as they are stored
template <int DT>
struct KvQuad {
	typename std::conditional<DT == KV_F32, u32x4, u32x2>::type w;
	__device__ __forceinline__ void zero() {
		w = w ^ w;
	}
	__device__ __forceinline__ void load(const void* base, size_t at) {
		w = *(const decltype(w)*)((const char*)base + at * (DT == KV_F32 ? 4 : 2));
	}
	__device__ __forceinline__ void get(float (&v)[4]) const {
		if constexpr (DT == KV_F32) {
#pragma unroll
			for (int i = 0; i < 4; ++i) {
				const unsigned one = w[i];
				v[i] = __builtin_bit_cast(float, one);
			}
		} else {
			const unsigned a = w[0], b = w[1]; // (a bit_cast of a vector's element itself reads element 0)
			kv_two<DT>(a, v[0], v[1]);
			kv_two<DT>(b, v[2], v[3]);
		}
	}
};
template <int DT>
__device__ __forceinline__ void kv_load4(const void* base, size_t at, float (&v)[4]) {
	KvQuad<DT> q;
	q.load(base, at);
	q.get(v);
}
template <int DT>
__device__ __forceinline__ unsigned short kv_half(float x) { // to nearest even: half a step of the type
	if constexpr (DT == KV_F16) {
		return __builtin_bit_cast(unsigned short, (_Float16)x);
	} else {
		return __builtin_bit_cast(unsigned short, (__bf16)x);
	}
}
template <int DT>
__device__ __forceinline__ void kv_store4(void* base, size_t at, const float (&v)[4]) {
	if constexpr (DT == KV_F32) {
		*(kv_f32x4*)((float*)base + at) = (kv_f32x4){v[0], v[1], v[2], v[3]};
	} else {
		const u32x2 w = {kv_half<DT>(v[0]) | ((unsigned)kv_half<DT>(v[1]) << 16), kv_half<DT>(v[2]) | ((unsigned)kv_half<DT>(v[3]) << 16)};
		*(u32x2*)((unsigned short*)base + at) = w;
	}
}

// eight codes as binary16, exactly: a code's byte with its sign bit turned over is code + 128, under the exponent byte 0x64 it reads
// 1024 + (code + 128); five instructions for four codes
__device__ __forceinline__ kv_f16x8 kv_codes8(unsigned w0, unsigned w1) {
	const kv_f16x2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
	u32x4 r;
	w0 ^= 0x80808080u, w1 ^= 0x80808080u;
	r[0] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04010400u);
	r[1] = __builtin_amdgcn_perm(0x64646464u, w0, 0x04030402u);
	r[2] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04010400u);
	r[3] = __builtin_amdgcn_perm(0x64646464u, w1, 0x04030402u);
#pragma unroll
	for (int i = 0; i < 4; ++i) {
		const unsigned two = r[i];
		r[i] = __builtin_bit_cast(unsigned, __builtin_bit_cast(kv_f16x2, two) + off);
	}
	return __builtin_bit_cast(kv_f16x8, r);
}

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float kv_exp2i(int e) {
	return __builtin_bit_cast(float, (unsigned)(e + 127) << 23);
}
// least e >= -126 with a <= 127 * 2^e, from the bits of a >= 0 (finite)
__device__ __forceinline__ int kv_scale_exp(unsigned a) {
	const int e = (int)(a >> 23) - 127 - 6 + ((a & 0x7fffffu) > 0x7e0000u ? 1 : 0); // 127 / 64 = 1.984375 = 1 + 0x7e0000 / 2^23
	return e < -126 ? -126 : e;
}

// ---- append ---------------------------------------------------------------------------------------------------------------------------

struct KvAppendArgs {
	KvLayer p;
	KvRows r;
	const void *k, *v;
	long k_row, k_head, v_row, v_head; // strides in elements
};

// item number `target` of a list that gives sequence s count(s) items: its sequence, and which of the sequence's it is; false behind the
// end.  64 sequences at a time: counts across the lanes, their running sum, one ballot.
template <class F>
__device__ __forceinline__ bool kv_find(int n_seqs, int target, F count, int& seq, int& item) {
	const int lane = lane_id();
	for (int s0 = 0; s0 < n_seqs; s0 += 64) {
		const int mine = s0 + lane < n_seqs ? count(s0 + lane) : 0;
		int sum = mine;
#pragma unroll
		for (int o = 1; o < 64; o <<= 1) {
			const int up = __shfl_up(sum, o);
			sum += lane >= o ? up : 0;
		}
		const unsigned long long b = __ballot(sum > target);
		if (b) {
			const int l = __builtin_ctzll(b);
			seq = s0 + l;
			item = target - __builtin_amdgcn_readlane(sum - mine, l);
			return true;
		}
		target -= __builtin_amdgcn_readlane(sum, 63);
	}
	return false;
}

// does sequence s of a batch fit its bounds?
__device__ __forceinline__ bool kv_rows_fit(const KvRows& r, int s) {
	const int row0 = r.cu[s], n = r.cu[s + 1] - row0;
	return row0 >= 0 && n >= 0 && n <= r.max_rows && r.n_rows - row0 >= n;
}
// the rows of sequence s that count: inside the packed arrays, at positions >= 0
__device__ __forceinline__ void kv_rows_of(const KvRows& r, int s, int& row0, int& n, int& len) {
	row0 = r.cu[s], n = r.cu[s + 1] - row0, len = r.lens[s];
	if (row0 < 0 || n < 0 || r.n_rows - row0 < n) {
		n = 0;
	}
	len = len < 0 ? 0 : len;
}

// One workgroup quantises what a call adds to one page and kv head, wave w the page's block w: rows in (K's and V's at once), the largest
// magnitude of the block's new values, the scale, codes out.  Bytes bound it (a token's rows once in, a quarter or half of them out); a lane
// takes four tokens x four dims, so K goes out as a dword per token and V as a dword per dim without crossing lanes.  Where all four blocks
// get new tokens (a prompt's pages) V's dwords meet in LDS and go out as whole lines: four bytes every sixteen cost 5 of 48 us for the
// 15k tokens of six prompts, 8 heads of 128.  Measured: those 26.6 us, 86 MB = 3.2 TB/s (fp16 in), one fp32 token of 48 sequences 6.1 us (two round trips).
// grid = (pages touched at most, + 1, kv heads)
template <int D, int DT>
__global__ __launch_bounds__(256, DT == KV_F32 || D > 128 ? 1 : D == 96 ? 7 : 8) void k_kv_append(KvAppendArgs a) {
	constexpr int NI = (D + 63) / 64; // items (quad of tokens, four dims) per lane: 4 x D / 4 over 64 lanes
	__shared__ u32x4 sm_v[4 * D];     // [quad][dim] x the four blocks' dwords, turned by dim / 4 (lanes four dims apart would meet in four banks)
	const int lane = lane_id(), blk = wave_id(), h = blockIdx.y;
	int s, at;
	const KvRows& r = a.r;
	if (blockIdx.x == gridDim.x - 1) { // one workgroup more than there can be pages: it looks every sequence's bounds over
		for (int i = threadIdx.x; h == 0 && i < r.n_seqs; i += 256) {
			if (!kv_rows_fit(r, i)) {
				kv_flag(a.p.status, KV_BAD_BATCH);
			}
		}
		return;
	}
	const auto pages = [&](int i) {
		int row0, n, len;
		kv_rows_of(r, i, row0, n, len);
		n = n < len ? n : len;
		return n > 0 ? (len - 1) / KV_PAGE - (len - n) / KV_PAGE + 1 : 0;
	};
	if (!kv_find(r.n_seqs, (int)blockIdx.x, pages, s, at)) {
		return;
	}
	int row0, n, len;
	kv_rows_of(r, s, row0, n, len);
	if (n > len) { // rows before position 0
		row0 += n - len, n = len;
	}
	const int before = len - n;
	const int pg = before / KV_PAGE + at, p0 = pg * KV_PAGE;
	const int pid = pg < r.max_pages ? r.table[(size_t)s * r.max_pages + pg] : -1;
	if (pid < 0 || pid >= a.p.n_pages) {
		if (threadIdx.x == 0 && h == 0) {
			kv_flag(a.p.status, KV_BAD_PAGE);
		}
		return;
	}
	const bool all = before < p0 + KV_BLOCK && len > p0 + 3 * KV_BLOCK; // every block of the page gets new tokens
	const int b0 = p0 + blk * KV_BLOCK; // first position of the block
	const int lo = before > b0 ? before - b0 : 0, hi = len - b0 < KV_BLOCK ? len - b0 : KV_BLOCK; // its new tokens
	if (lo >= hi) {
		return; // (not where `all`)
	}
	const size_t page = (size_t)pid * a.p.n_kv_heads + h;
	signed char* const kp = a.p.k + page * (KV_PAGE * D) + blk * KV_BLOCK * D;
	unsigned* const vp = (unsigned*)(a.p.v + page * (KV_PAGE * D)) + blk; // + (quad * D + dim) * 4
	KvQuad<DT> x[2][NI][4]; // [K, V][item][token], four dims each
#pragma unroll
	for (int kv = 0; kv < 2; ++kv) {
		const long row = kv ? a.v_row : a.k_row;
		const size_t src0 = (size_t)(row0 + b0 + lo - before) * (size_t)row + (size_t)h * (size_t)(kv ? a.v_head : a.k_head);
#pragma unroll
		for (int i = 0; i < NI; ++i) {
			const int it = lane + 64 * i, g = it / (D / 4), d = it % (D / 4) * 4;
#pragma unroll
			for (int t = 0; t < 4; ++t) {
				x[kv][i][t].zero();
				if (it < D && 4 * g + t >= lo && 4 * g + t < hi) {
					x[kv][i][t].load(kv ? a.v : a.k, src0 + (size_t)(4 * g + t - lo) * (size_t)row + d);
				}
			}
		}
	}
#pragma unroll
	for (int kv = 0; kv < 2; ++kv) {
		float big = 0.f, odd = 0.f; // odd: NaN once an infinity or a NaN came by (fmaxf passes over a NaN)
#pragma unroll
		for (int i = 0; i < NI; ++i) {
#pragma unroll
			for (int t = 0; t < 4; ++t) {
				float y[4];
				x[kv][i][t].get(y);
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					big = fmaxf(big, fabsf(y[e]));
					odd = __builtin_fmaf(y[e], 0.f, odd);
				}
			}
		}
		const bool wild = __ballot(odd != 0.f) != 0;
		const unsigned top = __builtin_bit_cast(unsigned, wave_max_dpp(big));
		float* const sp = (kv ? a.p.vs : a.p.ks) + page * 4 + blk;
		const unsigned was = lo > 0 ? __builtin_bit_cast(unsigned, *sp) & 0x7fffffffu : 0;
		const bool poison = wild || was >= 0x7f800000u;
		int e = wild ? -126 : kv_scale_exp(top);
		const int e_was = was >= 0x00800000u && was < 0x7f800000u ? (int)(was >> 23) - 127 : -126;
		e = e > e_was ? e : e_was; // (no old tokens: e_was is the least there is)
		// A code is the low byte of 1.5 * 2^23 + x 2^-e: the product is exact, the one rounding of the sum is to a whole number, to even; e <= 122.
		// (A poisoned block's codes are 0: 0 * x would not be.)
		const float inv = poison ? 0.f : kv_exp2i(-e);
		const bool shift = lo > 0 && e > e_was;
		const float shrink = shift ? kv_exp2i(e_was - e < -126 ? -126 : e_was - e) : 1.f;
#pragma unroll
		for (int i = 0; i < NI; ++i) {
			const int it = lane + 64 * i, g = it / (D / 4), d = it % (D / 4) * 4;
			const bool changes = 4 * g < hi && (4 * g + 3 >= lo || shift);
			if (it >= D || (!changes && !(kv && all))) {
				continue; // nothing of this quad changes
			}
			unsigned code[4][4]; // [token][dim], in the low byte
#pragma unroll
			for (int t = 0; t < 4; ++t) {
				float y[4];
				x[kv][i][t].get(y);
#pragma unroll
				for (int c = 0; c < 4; ++c) {
					code[t][c] = __builtin_bit_cast(unsigned, __builtin_fmaf(poison ? 0.f : y[c], inv, 12582912.f));
				}
			}
			unsigned out[4]; // K: a token's four dims; V: a dim's four tokens
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				const unsigned c0 = kv ? code[0][j] : code[j][0], c1 = kv ? code[1][j] : code[j][1], c2 = kv ? code[2][j] : code[j][2], c3 = kv ? code[3][j] : code[j][3];
				out[j] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(c3, c2, 0x0c0c0400u), __builtin_amdgcn_perm(c1, c0, 0x0c0c0400u), 0x05040100u);
			}
			if (4 * g < lo) { // old tokens among them
#pragma unroll
				for (int j = 0; j < 4; ++j) {
					unsigned old = kv ? vp[(size_t)(g * D + d + j) * 4] : 4 * g + j < lo ? *(const unsigned*)(kp + (4 * g + j) * D + d) : 0;
					if (shift) {
						unsigned w = 0;
#pragma unroll
						for (int c = 0; c < 4; ++c) {
							w |= ((unsigned)(int)__builtin_rintf((float)(int)(signed char)(old >> (8 * c)) * shrink) & 0xffu) << (8 * c);
						}
						old = w;
					}
					const int olds = lo - 4 * g < 4 ? lo - 4 * g : 4; // V: this many of the dword's bytes
					const unsigned keep = kv ? (olds >= 4 ? ~0u : (1u << (8 * olds)) - 1) : 4 * g + j < lo ? ~0u : 0u;
					out[j] = (out[j] & ~keep) | (old & keep);
				}
			}
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				if (!kv) {
					if (4 * g + j < hi && (4 * g + j >= lo || shift)) {
						*(unsigned*)(kp + (4 * g + j) * D + d) = out[j];
					}
				} else if (all) {
					((unsigned*)sm_v)[(g * D + d + j) * 4 + ((blk + (d >> 2)) & 3)] = out[j];
				} else {
					vp[(size_t)(g * D + d + j) * 4] = out[j];
				}
			}
		}
		if (lane == 0) {
			*(unsigned*)sp = poison ? 0x7fc00000u : __builtin_bit_cast(unsigned, kv_exp2i(e));
		}
	}
	if (!all) {
		return;
	}
	__syncthreads();
	u32x4* const dst = (u32x4*)(a.p.v + page * (KV_PAGE * D));
	for (int it = threadIdx.x; it < 4 * D; it += 256) {
		const u32x4 w = sm_v[it];
		const int turn = (it % D) >> 2; // word (blk + turn) & 3 is block blk's
		const u32x4 y = turn & 1 ? (u32x4){w[1], w[2], w[3], w[0]} : w;
		dst[it] = turn & 2 ? (u32x4){y[2], y[3], y[0], y[1]} : y;
	}
}

// ---- read back ------------------------------------------------------------------------------------------------------------------------

struct KvReadArgs {
	KvLayer p;
	const int *table, *lens, *start;
	void *k, *v; // [seq][count][kv head][D]
	int n_seqs, max_pages, count;
};

// values of positions start[s] .. start[s] + count - 1 of every sequence, zeros outside [0, lens[s]); a wave per (sequence, cache block, kv head):
// bytes bound it.  Measured: 203 MB (six sequences of up to 4.1k tokens, fp32 out) 47.5 us = 4.3 TB/s; the last tokens of 48 sequences 7.9 us
// grid = (blocks, kv heads, seqs)
template <int D, int DT>
__global__ __launch_bounds__(64) void k_kv_read(KvReadArgs a) {
	const int lane = lane_id(), h = blockIdx.y, s = blockIdx.z, H = a.p.n_kv_heads;
	const int start = a.start[s];
	int len = a.lens[s];
	len = len < 0 ? 0 : len;
	const long b0 = ((long)(start >> 4) + blockIdx.x) * KV_BLOCK; // first position of the block (floor: start may be negative)
	const long first = b0 > start ? b0 : start, last = b0 + KV_BLOCK < (long)start + a.count ? b0 + KV_BLOCK : (long)start + a.count;
	if (first >= last) {
		return;
	}
	int pid = -1;
	if (b0 >= 0 && b0 < len) {
		pid = b0 / KV_PAGE < a.max_pages ? a.table[(size_t)s * a.max_pages + b0 / KV_PAGE] : -1;
		if (pid < 0 || pid >= a.p.n_pages) {
			if (lane == 0 && h == 0) {
				kv_flag(a.p.status, KV_BAD_PAGE);
			}
			pid = -2;
		}
	}
	const int blk = (int)((b0 >> 4) & 3);
	const size_t page = (size_t)(pid < 0 ? 0 : pid) * H + h;
	const float nan = __builtin_nanf("");
	const float ks = pid >= 0 ? a.p.ks[page * 4 + blk] : nan, vs = pid >= 0 ? a.p.vs[page * 4 + blk] : nan;
#pragma unroll
	for (int kv = 0; kv < 2; ++kv) {
		for (int it = lane; it < D; it += 64) {
			const int g = it / (D / 4), d = it % (D / 4) * 4;
			unsigned w[4];
#pragma unroll
			for (int j = 0; j < 4; ++j) {
				w[j] = 0;
				if (pid >= 0) {
					w[j] = kv ? ((const unsigned*)(a.p.v + page * (KV_PAGE * D)))[(size_t)(g * D + d + j) * 4 + blk]
					          : *(const unsigned*)(a.p.k + page * (KV_PAGE * D) + (blk * KV_BLOCK + 4 * g + j) * D + d);
				}
			}
#pragma unroll
			for (int t = 0; t < 4; ++t) {
				const long pos = b0 + 4 * g + t;
				if (pos < first || pos >= last) {
					continue;
				}
				float y[4];
#pragma unroll
				for (int c = 0; c < 4; ++c) {
					const int code = (int)(signed char)(w[kv ? c : t] >> (8 * (kv ? t : c)));
					y[c] = pos >= 0 && pos < len ? (float)code * (kv ? vs : ks) : 0.f;
				}
				kv_store4<DT>(kv ? a.v : a.k, (((size_t)s * a.count + (size_t)(pos - start)) * H + h) * D + d, y);
			}
		}
	}
}

// ---- attention ------------------------------------------------------------------------------------------------------------------------
//
// Row (t, head) of sequence s stands at position p = lens[s] - n + t and sees tokens j <= p with no window, or j > p - window, or
// j < sinks.  out = sum_j P_j V_j / sum_j P_j with P_j = 2^(x_j - m), x_j = (q . K_j) scale log2(e), m the running maximum.
// Both products run on the matrix cores, transposed: S^T = K q^T puts a query row into a lane's column, so maximum, sum and rescaling
// of a row are its lane's own (plus the other lanes of the same column), and the weights are already the operand layout that
// O^T = V^T P^T wants.  Numerics.  Codes are exact, as bytes and as binary16.  q is cut in two ways:
//   k_kv_decode  three signed digits of base 254 relative to the row's largest magnitude, d0 + d1 / 254 + d2 / 254^2: the scores are sums of byte
//                products in whole numbers, exact; what is left out of q is 6e-8 of its row's largest.  (Two digits for 16-bit rows, 1.6e-5, are
//                2 - 4 % faster on 64 sequences with heads of 64 -- 37.5 instead of 39 us -- and cost a row with an outlier channel more than its type does.)
//   k_kv_chunk   one binary16 after the row is scaled by a power of two to at most 1 (fp16 and bf16 rows lose nothing above 2^-14 of their largest
//                element), fp32 rows as the sum of two (22 bits); scores are fp32 sums.
// Scores are then fp32, times the block's K scale.  A weight goes into the second product with its block's V scale, relative to the largest such
// that the ROW met (KvRefs), as one binary16 for fp16 / bf16 outputs -- off by at most 2^-11, half a step -- and as the sum of two for fp32 (2^-22); sums
// are fp32.  Below 2^-20 of the largest a weight keeps an absolute 2^-31 of it.  fp16 outputs, whose own rounding the weights' comes up to, take the
// sum of the ROUNDED weights, so that they are averages of V's and a token that has all the weight is returned exactly: off by 2.6e-4 of their
// root mean square, 2.9e-4 with the sum of the unrounded (2.07e-4 is the output's own; for bf16 it is 1.66e-3, and nothing is gained) -- unless a block's V scale
// is so far below the reference (KV_NEAR) that its weights round to few bits or none, and the sum would lose what they weigh.

struct KvAttnArgs {
	KvLayer p;
	KvRows r;
	const void* q;
	void* out; // [row][head][D]
	long q_row, q_head;
	float* part; // [row x head][split][D + 4]: partial sums, then reference, sum of weights and reference of the sums (KvRefs)
	int n_heads, group, window, sinks, chunk, n_splits;
	float scale; // scale * log2(e)
};

// the pages that rows at positions p_min .. p_max see: [0, first tokens' pages) and [start, p_max / 64]
struct KvSpan {
	int ns, start, np;
	__device__ __forceinline__ KvSpan(int p_min, int p_max, int window, int sinks) {
		const int lo = window > 0 && p_min >= window ? p_min - window + 1 : 0;
		const int s = sinks < lo ? sinks : lo;
		ns = (s + KV_PAGE - 1) / KV_PAGE;
		start = lo / KV_PAGE;
		start = start < ns ? ns : start;
		np = p_max < 0 ? 0 : ns + (p_max / KV_PAGE >= start ? p_max / KV_PAGE - start + 1 : 0);
	}
	__device__ __forceinline__ int page(int i) const {
		return i < ns ? i : start + i - ns;
	}
};

// maximum with the lane 32 (16) away: a swap of register halves, no trip through the LDS crossbar
__device__ __forceinline__ float kv_max32(float v) {
	const unsigned b = __builtin_bit_cast(unsigned, v);
	const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
	const unsigned x = r[0], y = r[1];
	return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
__device__ __forceinline__ float kv_max16(float v) {
	const unsigned b = __builtin_bit_cast(unsigned, v);
	const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
	const unsigned x = r[0], y = r[1];
	return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
__device__ __forceinline__ float kv_exp2(float x) {
	return __builtin_amdgcn_exp2f(x); // one unit in the last place; below 2^-126 zero
}
// the power of two that brings a row with largest magnitude `top` to at most 1 (a row of zeros, or one with an infinity: 1 / a NaN product)
__device__ __forceinline__ int kv_row_exp(float top) {
	const unsigned b = __builtin_bit_cast(unsigned, top);
	int e = (int)(b >> 23) - 126;
	e = e < -126 ? -126 : e;
	return e > 126 ? 126 : e;
}

// A row's references, whole numbers both: m follows the scores x_j, m + g follows x_j + v_j (v_j: the exponent field of V's scale), each over the
// tokens that the row itself sees.  Sums of weights are relative to 2^m; what goes into the product with V's codes is y_j = 2^(x_j + v_j - m - g + KV_LIFT),
// so nothing that a row does not see, or gives no weight, takes bits from it, however large its V.  A block's share of the sum of weights is that of
// its y, times 2^k, k = g - KV_LIFT - v.  k is KV_REACH at most: beyond, V is 2^-53 of what the row's output is made of and takes part as if it were no
// smaller.  The references stay unless one is passed by 2^8 (weights up to 2^8 are no less exact, and sums are seldom rescaled), and then both follow, so
// that k is what V's scales make it: -7 for equal ones, and up to KV_NEAR where the rounded weights may stand for the weights (fp16).  y <= 2^15 is inside
// binary16; KV_LIFT moves its subnormals away.  Scores of 2^20 and more take their differences from m before anything small is added (kv_far_score).
constexpr float KV_LIFT = 7.f, KV_REACH = 60.f, KV_NEAR = -2.f;
// A row's tokens lie in several lanes.  Each keeps what it has met itself; the row's is put together (`join`: the maximum over its lanes) where a lane
// asks for a move, so that a page that moves nothing takes no trip across the lanes and one branch.
constexpr float KV_LOW = -3e38f, KV_NO_GAP = -1000.f; // no token seen yet
struct KvRefs {
	float m = KV_LOW, g = KV_NO_GAP;                       // the references
	float top = -__builtin_inff(), tv = -__builtin_inff(); // the largest x_j that the lane met, the largest x_j - m + v_j
	bool far = false;                                      // (of the wave) a score's last place is near a weight's size
	// the lane's largest score of a page, and its largest x_j - m + v_j
	__device__ __forceinline__ bool asks(float x, float v) {
		top = fmaxf(top, x);
		return top > m + 8.f || v > g + 8.f;
	}
	__device__ __forceinline__ float shift(bool to_top, float& l) {
		const float to = to_top ? ceilf(top) : m, d = m - to;
		m = to, g += d, l *= kv_exp2(d);
		return d;
	}
	// the references after a page in which some row's asked for it -> what multiplies the products' sums.  again(m): the page's largest x_j - m + v_j
	template <class J, class A>
	__device__ __forceinline__ float follow(float& l, J join, A again) {
		top = join(top);
		bool rose = top > m + 8.f;
		tv += shift(rose, l);
		tv = join(fmaxf(tv, again(m)));
		rose = rose || tv > g + 8.f;
		tv += shift(rose, l);
		const float gap = rose ? ceilf(tv) : g, by = kv_exp2(g - gap);
		g = gap;
		far = __ballot(m != KV_LOW && !(fabsf(m) < 1048576.f)) != 0;
		return by;
	}
};
// x - m with x the product as it was compared (not fused: in the last place of a large score there is room for more than a weight)
__device__ __forceinline__ float kv_far_score(float sc, float f, float m) {
#pragma clang fp contract(off)
	const float x = sc * f;
	return x - m;
}
// acc + the two binary16 numbers of a word
__device__ __forceinline__ float kv_add2(float acc, unsigned h2) {
	const kv_f16x2 one = {(_Float16)1.f, (_Float16)1.f};
	return __builtin_amdgcn_fdot2(__builtin_bit_cast(kv_f16x2, h2), one, acc, false);
}
// sum of y_j V_j over the sum of weights, with V's scale back in (g: finite)
__device__ __forceinline__ float kv_result(float y, float g) {
	return __builtin_amdgcn_ldexpf(y, (int)(g - 127.f - KV_LIFT));
}

// the result of a row, or its part of a split: a quad of dims
template <int D, int DT>
__device__ __forceinline__ void kv_put(const KvAttnArgs& a, bool direct, size_t row, int split, int d, const float (&o)[4]) {
	if (direct) {
		kv_store4<DT>(a.out, row * D + d, o);
	} else {
		float* const p = a.part + (row * a.n_splits + split) * (D + 4) + d;
		*(kv_f32x4*)p = (kv_f32x4){o[0], o[1], o[2], o[3]};
	}
}

// Few rows (one token of a sequence, or a few): the cache's bytes bound it.  A workgroup takes one sequence, one kv head, 16 rows (token x head
// of the group) and a range of pages, dealt to its NW waves a page at a time; a wave holds a page's codes in registers as the matrix
// operands they are (no conversion: that is what whole-number scores are for), asks for the next page's K behind the first product and for its
// V behind the second, so 8 - 16 KiB per wave are in flight throughout.  (Two sets of registers, a whole page ahead: slower.)  The waves' sums
// meet in LDS; ranges of one row meet in k_kv_merge.  Eight waves for heads up to 128: four, with twice the workgroups, lose 5 - 10 % to the
// waits at both ends of a workgroup (64 sequences of 91 - 8191, heads of 64, with two digits: 39.6 -> 36.2 us).
// Measured, one row a sequence: 24 x 13.9 - 16.4k tokens, 8 kv heads of 128: 136 us, 746 MB = 5.5 TB/s; 8 x 4093 (fp32): 17.2 us + 3.9 for the join, 67 MB = 3.2;
// 64 x 91 - 8191, 4 of 64: 39.6 us, 137 MB = 3.5 (the longest sequences' chain of pages is what remains); up to five rows of 16 x 6 - 9k under a window of
// 1024: 14.1 us, 35 MB = 2.5.
// grid = (splits, kv heads x tiles, seqs)
template <int D, int DT, int NW>
__global__ __launch_bounds__(64 * NW, D <= 128 ? 2 : 1) void k_kv_decode(KvAttnArgs a) {
	constexpr int ND = D / 16;  // dim tiles of O^T
	constexpr int KW = D / 16;  // dwords of a K row per lane
	constexpr bool HL = DT == KV_F32;
	extern __shared__ float kv_lds[]; // [wave][16 rows][D + 4]
	const int lane = lane_id(), wave = wave_id();
	const int col = lane & 15, g = lane >> 4;
	const int H = a.p.n_kv_heads, h = blockIdx.y % H, tile = blockIdx.y / H, s = blockIdx.z, split = blockIdx.x;
	int row0, n, len;
	kv_rows_of(a.r, s, row0, n, len);
	const int nrows = n * a.group, r0 = tile * 16;
	if (threadIdx.x == 0 && tile == 0 && h == 0 && split == 0 && !kv_rows_fit(a.r, s)) {
		kv_flag(a.p.status, KV_BAD_BATCH);
	}
	if (r0 >= nrows) {
		return;
	}
	const int rl = r0 + 15 < nrows - 1 ? r0 + 15 : nrows - 1;
	const int p_first = len - n + r0 / a.group, p_max = len - n + rl / a.group;
	const int p_min = p_first < 0 ? 0 : p_first; // (rows before position 0 see nothing; their distance to a window's end may pass 32 bits)
	const KvSpan sp(p_min, p_max, a.window, a.sinks);
	// ranges of a.chunk pages; the last takes what a sequence longer than the host's bound has beyond them
	const bool direct = sp.np <= a.chunk || a.n_splits == 1;
	const int i0 = split * a.chunk, i1 = split + 1 < a.n_splits && (split + 1) * a.chunk < sp.np ? (split + 1) * a.chunk : sp.np;
	const int rr = r0 + col;
	const bool live = rr < nrows;
	const int t = (live ? rr : r0) / a.group, hd = h * a.group + (live ? rr : r0) % a.group;
	const int pos = len - n + t, past = (pos < 0 ? 0 : pos) - a.window; // (the last position before the window)
	const size_t row = (size_t)(row0 + t) * a.n_heads + hd;
	if (i0 >= i1 && split > 0) {
		if (!direct && wave == 0 && g == 0) { // a range without pages: marked empty for k_kv_merge
			if (live) {
				float* const p = a.part + (row * a.n_splits + split) * (D + 4) + D;
				p[0] = KV_LOW, p[1] = 0.f, p[2] = KV_NO_GAP;
			}
		}
		return;
	}
	// page ids of this wave's next 64 pages, one per lane; the first pages' codes are asked for before q is looked at
	int ids = -1, ids0 = i0 + wave; // lane i: page ids0 + NW i
	const auto fetch_ids = [&](int first) {
		ids0 = first;
		const int i = first + NW * lane;
		ids = -1;
		if (i < i1) {
			const int pg = sp.page(i);
			ids = pg < a.r.max_pages ? a.r.table[(size_t)s * a.r.max_pages + pg] : -1;
			if (ids < 0 || ids >= a.p.n_pages) {
				kv_flag(a.p.status, KV_BAD_PAGE);
				ids = -1;
			}
		}
	};
	unsigned kr[4][KW];
	u32x4 vr[ND];
	kv_f32x4 ksc, vsc;
	const auto load_k = [&](int pid) {
		const size_t page = (size_t)(pid < 0 ? 0 : pid) * H + h;
		const signed char* const p = a.p.k + page * (KV_PAGE * D) + (size_t)col * D + g * (D / 4);
#pragma unroll
		for (int t = 0; t < 4; ++t) {
			if constexpr (D % 64 == 0) {
#pragma unroll
				for (int i = 0; i < KW / 4; ++i) {
					const u32x4 w = *(const u32x4*)(p + t * 16 * D + 16 * i);
					kr[t][4 * i] = w[0], kr[t][4 * i + 1] = w[1], kr[t][4 * i + 2] = w[2], kr[t][4 * i + 3] = w[3];
				}
			} else {
#pragma unroll
				for (int i = 0; i < KW / 2; ++i) {
					const u32x2 w = *(const u32x2*)(p + t * 16 * D + 8 * i);
					kr[t][2 * i] = w[0], kr[t][2 * i + 1] = w[1];
				}
			}
		}
		ksc = *(const kv_f32x4*)(a.p.ks + page * 4);
	};
	const auto load_v = [&](int pid) {
		const size_t page = (size_t)(pid < 0 ? 0 : pid) * H + h;
		const u32x4* const p = (const u32x4*)(a.p.v + page * (KV_PAGE * D)) + g * D + col;
#pragma unroll
		for (int d = 0; d < ND; ++d) {
			vr[d] = p[16 * d];
		}
		vsc = *(const kv_f32x4*)(a.p.vs + page * 4);
	};
	// fp32 rows are asked for ahead of the codes -- loads come back in order, and the three digits are made while the codes are on their way -- 16-bit
	// rows behind them (8 fp32 rows on 4093 tokens 17.8 instead of 19.0 us; up to five 16-bit rows under a window 14.0 instead of 13.7)
	KvQuad<DT> qw[D / 16];
	const size_t at = (row / a.n_heads) * (size_t)a.q_row + (row % a.n_heads) * (size_t)a.q_head + g * (D / 4);
	const auto load_q = [&]() {
#pragma unroll
		for (int i = 0; i < D / 16; ++i) {
			qw[i].load(a.q, at + 4 * i);
		}
	};
	if constexpr (HL) {
		load_q();
	}
	int pid = -1;
	if (i0 + wave < i1) {
		fetch_ids(i0 + wave);
		pid = __builtin_amdgcn_readlane(ids, 0);
		load_k(pid);
		load_v(pid);
	}
	__builtin_amdgcn_sched_barrier(0); // (the loads stay ahead of what follows)
	if constexpr (!HL) {
		load_q();
	}
	// q as three signed digits of eight bits, row / 2^e = (d0 + d1 / 254 + d2 / 254^2) / 127: lane (col, g) holds dims g D / 4 .. of its row
	constexpr int NQ = 3;
	unsigned qd[NQ][KW];
	float x[D / 4];
	unsigned big = 0;
#pragma unroll
	for (int i = 0; i < D / 16; ++i) {
		float y[4];
		qw[i].get(y);
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			x[4 * i + j] = y[j];
			const unsigned u = __builtin_bit_cast(unsigned, y[j]) & 0x7fffffffu;
			big = big > u ? big : u;
		}
	}
	const unsigned t1 = __shfl_xor(big, 16);
	big = big > t1 ? big : t1;
	const unsigned t2 = __shfl_xor(big, 32);
	big = big > t2 ? big : t2;
	const int e0 = kv_row_exp(__builtin_bit_cast(float, big)), e = e0 < -119 ? -119 : e0; // (2^119 * 127 is a number; smaller rows' scores are none)
	const float inv = kv_exp2i(-e) * 127.f;
	// (a row with an infinity or a NaN is NaN)
	const float qf = big >= 0x7f800000u ? __builtin_nanf("") : kv_exp2i(e) * a.scale * (1.f / 127.f);
#pragma unroll
	for (int i = 0; i < KW; ++i) {
		unsigned w[NQ];
#pragma unroll
		for (int n = 0; n < NQ; ++n) {
			w[n] = 0;
		}
#pragma unroll
		for (int j = 0; j < 4; ++j) {
			float y = big >= 0x7f800000u ? 0.f : x[4 * i + j] * inv;
#pragma unroll
			for (int n = 0; n < NQ; ++n) {
				const float r = __builtin_rintf(y);
				w[n] |= ((unsigned)(int)r & 0xffu) << (8 * j);
				y = (y - r) * 254.f;
			}
		}
#pragma unroll
		for (int n = 0; n < NQ; ++n) {
			qd[n][i] = w[n];
		}
	}
	kv_f32x4 o[ND];
	KvRefs ref;
	float l = 0.f;
#pragma unroll
	for (int d = 0; d < ND; ++d) {
		o[d] = (kv_f32x4){0.f, 0.f, 0.f, 0.f};
	}
	for (int i = i0 + wave; i < i1; i += NW) {
		const int pg = sp.page(i), j0 = pg * KV_PAGE;
		const bool bad = pid < 0;
		const bool more = i + NW < i1;
		if (more && i + NW >= ids0 + 64 * NW) {
			fetch_ids(i + NW);
		}
		const int next = more ? __builtin_amdgcn_readlane(ids, (i + NW - ids0) / NW) : -1;
		// S^T of the page: tile t = block t, this lane's tokens 4 g + e; whole numbers, exactly
		kv_f32x4 sc[4];
#pragma unroll
		for (int t = 0; t < 4; ++t) {
			kv_i32x4 acc[NQ];
#pragma unroll
			for (int n = 0; n < NQ; ++n) {
				acc[n] = (kv_i32x4){0, 0, 0, 0};
				if constexpr (D % 64 == 0) {
#pragma unroll
					for (int k = 0; k < D / 64; ++k) {
						const kv_i32x4 kf = {(int)kr[t][4 * k], (int)kr[t][4 * k + 1], (int)kr[t][4 * k + 2], (int)kr[t][4 * k + 3]};
						const kv_i32x4 qv = {(int)qd[n][4 * k], (int)qd[n][4 * k + 1], (int)qd[n][4 * k + 2], (int)qd[n][4 * k + 3]};
						acc[n] = __builtin_amdgcn_mfma_i32_16x16x64_i8(kf, qv, acc[n], 0, 0, 0);
					}
				} else {
#pragma unroll
					for (int k = 0; k < D / 32; ++k) {
						const long kf = (long)(((unsigned long)kr[t][2 * k + 1] << 32) | kr[t][2 * k]);
						const long qv = (long)(((unsigned long)qd[n][2 * k + 1] << 32) | qd[n][2 * k]);
						acc[n] = __builtin_amdgcn_mfma_i32_16x16x32_i8(kf, qv, acc[n], 0, 0, 0);
					}
				}
			}
#pragma unroll
			for (int e = 0; e < 4; ++e) {
				// (|sums| < 2^23: the lower two in one whole number below 2^31)
				sc[t][e] = __builtin_fmaf((float)(__mul24(acc[1][e], 254) + acc[2][e]), 1.f / (254.f * 254.f), (float)acc[0][e]);
			}
		}
		// a missing page, and a block whose V scale is no number, are NaN through K, for the rows that see them
		float kscale[4], lv[4];
#pragma unroll
		for (int t = 0; t < 4; ++t) {
			const float one = vsc[t];
			kscale[t] = bad ? __builtin_nanf("") : __builtin_fmaf(one, 0.f, ksc[t]);
			lv[t] = (float)((__builtin_bit_cast(unsigned, one) >> 23) & 0xffu);
		}
		if (more) {
			load_k(next);
		}
		// every token of the page seen by every row of the tile?
		const bool whole = j0 + KV_PAGE - 1 <= p_min && (a.window <= 0 || j0 > p_max - a.window || j0 + KV_PAGE <= a.sinks);
		float least = 255.f; // the smallest V scale that this lane's tokens have (behind the row's mask a scale may be anything)
		float xb[4], top = -__builtin_inff();
#pragma unroll
		for (int t = 0; t < 4; ++t) {
			const float f = kscale[t] * qf;
			float x = -__builtin_inff();
			if (!whole) {
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					const int j = j0 + 16 * t + 4 * g + e;
					const bool seen = j <= pos && (a.window <= 0 || j > past || j < a.sinks);
					sc[t][e] = seen ? sc[t][e] * f : -__builtin_inff();
					x = fmaxf(x, sc[t][e]);
				}
				kscale[t] = 1.f;
			} else {
				const float hi = fmaxf(fmaxf(sc[t][0], sc[t][1]), fmaxf(sc[t][2], sc[t][3])) * f;
				const float lo = fminf(fminf(sc[t][0], sc[t][1]), fminf(sc[t][2], sc[t][3])) * f;
				x = fmaxf(hi, lo); // (a negative factor turns them round)
				kscale[t] = f;
			}
			xb[t] = x;
			top = fmaxf(top, x);
			least = fminf(least, x > -__builtin_inff() ? lv[t] : 255.f);
		}
		const auto join = [](float x) { return kv_max32(kv_max16(x)); };
		const auto largest = [&](float m) {
			return fmaxf(fmaxf((xb[0] - m) + lv[0], (xb[1] - m) + lv[1]), fmaxf((xb[2] - m) + lv[2], (xb[3] - m) + lv[3]));
		};
		const float tv = largest(ref.m);
		bool far = false;
		if (__ballot(ref.asks(top, tv)) || ref.far) {
			const float by = ref.follow(l, join, largest);
#pragma unroll
			for (int d = 0; d < ND; ++d) {
				o[d] *= by;
			}
			if (ref.far) {
				far = true;
#pragma unroll
				for (int t = 0; t < 4; ++t) {
#pragma unroll
					for (int e = 0; e < 4; ++e) {
						sc[t][e] = kv_far_score(sc[t][e], kscale[t], ref.m);
					}
					kscale[t] = 1.f;
				}
			}
		} else {
			ref.tv = fmaxf(ref.tv, tv);
		}
		const float rm = far ? 0.f : ref.m, gap = ref.g - KV_LIFT;
		kv_f16x8 pf[2], pl[HL ? 2 : 1];
		const auto weigh = [&](auto rounded) {
#pragma unroll
			for (int t = 0; t < 4; ++t) {
				const float k = fminf(gap - lv[t], KV_REACH), from = -(rm + k);
				float sum = 0.f;
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					const float y = kv_exp2(__builtin_fmaf(sc[t][e], kscale[t], from));
					sum += rounded ? 0.f : y;
					pf[t >> 1][4 * (t & 1) + e] = (_Float16)y;
					if constexpr (HL) {
						pl[t >> 1][4 * (t & 1) + e] = (_Float16)(y - (float)pf[t >> 1][4 * (t & 1) + e]);
					}
				}
				if constexpr (rounded) {
					const u32x4 w = __builtin_bit_cast(u32x4, pf[t >> 1]);
					sum = kv_add2(kv_add2(0.f, w[2 * (t & 1)]), w[2 * (t & 1) + 1]);
				}
				l = __builtin_fmaf(sum, kv_exp2(k), l);
			}
		};
		if (DT == KV_F16 && !__ballot(gap > least + KV_NEAR)) {
			weigh(std::integral_constant<bool, DT == KV_F16>());
		} else {
			weigh(std::false_type());
		}
#pragma unroll
		for (int d = 0; d < ND; ++d) {
#pragma unroll
			for (int u = 0; u < 2; ++u) {
				const kv_f16x8 vf = kv_codes8(vr[d][2 * u], vr[d][2 * u + 1]);
				o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[u], o[d], 0, 0, 0);
				if constexpr (HL) {
					o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl[u], o[d], 0, 0, 0);
				}
			}
		}
		if (more) {
			load_v(next);
		}
		pid = next;
	}
	// the waves' sums
	float* const mine = kv_lds + wave * (16 * (D + 4));
	l += __shfl_xor(l, 16);
	l += __shfl_xor(l, 32);
	float* const p = mine + (col) * (D + 4);
#pragma unroll
	for (int d = 0; d < ND; ++d) {
		*(kv_f32x4*)(p + 16 * d + 4 * g) = o[d];
	}
	if (g == 0) {
		p[D] = ref.m, p[D + 1] = l, p[D + 2] = ref.g;
	}
	__syncthreads();
	// a thread per (row, quad of dims)
	for (int it = threadIdx.x; it < 16 * (D / 4); it += 64 * NW) {
		const int rr = it / (D / 4), d = it % (D / 4) * 4;
		if (r0 + rr >= nrows) {
			break;
		}
		const float* const p = kv_lds + rr * (D + 4);
		constexpr int W = 16 * (D + 4);
		float M = KV_LOW, G = KV_NO_GAP, gw[NW];
#pragma unroll
		for (int w = 0; w < NW; ++w) {
			M = fmaxf(M, p[w * W + D]);
		}
#pragma unroll
		for (int w = 0; w < NW; ++w) { // the waves' second references, from M
			gw[w] = (p[w * W + D] - M) + p[w * W + D + 2];
			G = fmaxf(G, gw[w]);
		}
		float L = 0.f, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
		for (int w = 0; w < NW; ++w) {
			const float fo = kv_exp2(gw[w] - G);
			L += kv_exp2(p[w * W + D] - M) * p[w * W + D + 1];
			const kv_f32x4 x = *(const kv_f32x4*)(p + w * W + d);
#pragma unroll
			for (int e = 0; e < 4; ++e) {
				y[e] += fo * x[e];
			}
		}
		const int t = (r0 + rr) / a.group;
		const size_t at = (size_t)(row0 + t) * a.n_heads + h * a.group + (r0 + rr) % a.group;
		// (no token seen: zeros.  Tokens seen, and every score beyond fp32 below: NaN; k_kv_merge knows by a sum of -0)
		const bool blind = L == 0.f && len - n + t < 0;
		if (direct) {
			const float f = L == 0.f ? (blind ? 0.f : __builtin_nanf("")) : 1.f / L;
#pragma unroll
			for (int e = 0; e < 4; ++e) {
				y[e] = kv_result(y[e] * f, G);
			}
		}
		kv_put<D, DT>(a, direct, at, split, d, y);
		if (d == 0 && a.n_splits > 1) {
			float* const pm = a.part + (at * a.n_splits + split) * (D + 4) + D;
			pm[0] = M, pm[1] = direct ? -1.f : L == 0.f && !blind ? -0.f : L, pm[2] = G; // (no sum of weights is negative: the row is written already)
		}
	}
}

// the ranges of a row put together; a wave per row, the ranges' maxima across its lanes (n_splits <= 64).  Measured: 256 rows of 128 in four
// ranges 3.9 us, the launch and two round trips
template <int D, int DT>
__global__ __launch_bounds__(256) void k_kv_merge(KvAttnArgs a) {
	const int lane = lane_id();
	const size_t row = (size_t)blockIdx.x * 4 + wave_id();
	const int first = a.r.cu[0] < 0 ? 0 : a.r.cu[0], end = a.r.cu[a.r.n_seqs], last = end < a.r.n_rows ? end : a.r.n_rows;
	if (row >= (size_t)(last < 0 ? 0 : last) * a.n_heads || row < (size_t)first * a.n_heads) {
		return; // rows behind the last sequence stay as they are
	}
	const float* const p = a.part + row * a.n_splits * (D + 4);
	float m = KV_LOW, g = KV_NO_GAP, l = 0.f;
	if (lane < a.n_splits) {
		m = p[(size_t)lane * (D + 4) + D], l = p[(size_t)lane * (D + 4) + D + 1], g = p[(size_t)lane * (D + 4) + D + 2];
	}
	const int l0 = __builtin_amdgcn_readlane(__builtin_bit_cast(int, l), 0); // (the first range's)
	if (__builtin_bit_cast(float, l0) < 0.f) {
		return; // one range: written by its workgroup
	}
	const bool empty = m == KV_LOW && l == 0.f;
	const float M = wave_max_dpp(m);
	g += m - M; // (from M)
	const float G = wave_max_dpp(g);
	const float L = wave_sum(empty ? 0.f : kv_exp2(m - M) * l), w = kv_exp2(g - G);
	const unsigned long long some = __ballot(!empty);
	constexpr int N = (D + 255) / 256;
	const int d = lane * 4;
	float y[4] = {0.f, 0.f, 0.f, 0.f};
	static_assert(N == 1, "a quad of dims per lane");
	for (int i = 0; i < a.n_splits; ++i) {
		if ((some >> i) & 1) {
			const float f = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i));
			if (d < D) {
				const kv_f32x4 x = *(const kv_f32x4*)(p + (size_t)i * (D + 4) + d);
#pragma unroll
				for (int e = 0; e < 4; ++e) {
					y[e] += f * x[e];
				}
			}
		}
	}
	if (d < D) {
		const float f = L == 0.f ? (l0 < 0 ? __builtin_nanf("") : 0.f) : 1.f / L; // (-0: tokens seen, no score in range)
#pragma unroll
		for (int e = 0; e < 4; ++e) {
			y[e] = kv_result(y[e] * f, G);
		}
		kv_store4<DT>(a.out, row * D + d, y);
	}
}

// Many rows (a prompt chunk).  A workgroup takes 128 rows (32 per wave) of one sequence and kv head and walks
// the pages they see; a page's codes become binary16 ONCE per workgroup on their way into LDS (two buffers: the next page's loads are in
// flight while a page is computed), laid out so that every operand is one 16-byte read of consecutive lanes.
// Measured: 2049 rows of 32 heads (8 kv heads of 128) on 4099 tokens 169 - 174 us = 600 TFLOP/s; five ragged chunks of up to 1021 rows of 32 heads
// (4 kv heads of 64) behind a window of 2048 77 us.  What bounds it is the chain of pages of the heaviest tiles (65, 49 on average; 2.6 us each): of the first
// shape's 395k cycles the matrix unit is busy 100k and vector instructions issue 158k, with 1.31 of two possible waves on a SIMD on average -- light
// tiles end early, nothing follows them -- and a wave issues 46 % of its time, waits to issue 30 and for memory, LDS and barriers 24.  (Under the
// window: 203k cycles, 25k and 73k, 1.07 waves.)  Tried and slower: PV of a page with QK of
// the next in one phase, the other phase's waves beside it behind barriers (eight waves of 256 rows: 199 us; four waves: 181), products of
// neighbouring pages interleaved within a wave (257 us), light tiles behind heavy ones on a CU (187).
// grid = row tiles x seqs x splits x kv heads
template <int D>
struct KvChunk {
	static constexpr int KROW = 65;                // 16-byte units between two (k-step, half) columns of K: 64 tokens and one of padding
	static constexpr int KU = D / 8 * KROW, VU = 8 * D; // units of a page's K and V
	// two workgroups to a CU, never three: where there are no more than two for each, three on one CU leave others idle (five ragged chunks of up to
	// 1021 rows, heads of 64: 90 instead of 75 us)
	static constexpr size_t LDS = (size_t)2 * (KU + VU) * 16 < 56 * 1024 ? 56 * 1024 : (size_t)2 * (KU + VU) * 16;
};

// n operands' LDS reads, KV_AHEAD of them ahead, each feeding m matrix instructions
constexpr int KV_AHEAD = 6;
#define KV_FEED(n, m)                                              \
	do {                                                           \
		__builtin_amdgcn_sched_group_barrier(0x100, KV_AHEAD, 0);  \
		_Pragma("unroll") for (int mix_ = 0; mix_ < (n); ++mix_) { \
			__builtin_amdgcn_sched_group_barrier(0x008, m, 0);     \
			__builtin_amdgcn_sched_group_barrier(0x100, 1, 0);     \
		}                                                          \
	} while (0)

template <int D, int DT>
__global__ __launch_bounds__(256, D > 128 || (DT == KV_F32 && D > 64) ? 1 : 2) void k_kv_chunk(KvAttnArgs a) {
	constexpr int KS = D / 16, ND = D / 32;
	constexpr bool HL = DT == KV_F32;
	constexpr int NK = (4 * D + 255) / 256, NV = (2 * D + 255) / 256; // staging items per thread
	constexpr int KROW = KvChunk<D>::KROW, KU = KvChunk<D>::KU, VU = KvChunk<D>::VU;
	extern __shared__ u32x4 kv_st[];
	const int tid = threadIdx.x, lane = lane_id(), wave = wave_id();
	const int col = lane & 31, hh = lane >> 5;
	const int H = a.p.n_kv_heads;
	int r0, h, s, split;
	{
		// Workgroups in the order of their work, kv heads fastest: the tiles at a prompt's end see most pages and start first, and with the
		// usual eight kv heads a head's pages meet in one XCD's L2 (tiles fastest: 125 instead of 79 us for ragged chunks under a window)
		int i = (int)blockIdx.x;
		h = i % H, i /= H;
		split = i % a.n_splits, i /= a.n_splits;
		s = i % a.r.n_seqs, i /= a.r.n_seqs;
		r0 = ((int)gridDim.x / (H * a.n_splits * a.r.n_seqs) - 1 - i) * 128;
	}
	int row0, n, len;
	kv_rows_of(a.r, s, row0, n, len);
	const int nrows = n * a.group;
	if (tid == 0 && r0 == 0 && h == 0 && split == 0 && !kv_rows_fit(a.r, s)) {
		kv_flag(a.p.status, KV_BAD_BATCH);
	}
	if (r0 >= nrows) {
		return;
	}
	const int rl = r0 + 127 < nrows - 1 ? r0 + 127 : nrows - 1;
	const int p_first = len - n + r0 / a.group, p_max = len - n + rl / a.group;
	const int p_min = p_first < 0 ? 0 : p_first; // (rows before position 0 see nothing; their distance to a window's end may pass 32 bits)
	const KvSpan sp(p_min, p_max, a.window, a.sinks);
	// ranges of a.chunk pages; the last takes what a sequence longer than the host's bound has beyond them
	const bool direct = sp.np <= a.chunk || a.n_splits == 1;
	const int i0 = split * a.chunk, i1 = split + 1 < a.n_splits && (split + 1) * a.chunk < sp.np ? (split + 1) * a.chunk : sp.np;
	// this wave's rows
	const int rr = r0 + 32 * wave + col;
	const bool live = rr < nrows;
	const int t = (live ? rr : nrows - 1) / a.group, hd = h * a.group + (live ? rr : nrows - 1) % a.group;
	const int pos = len - n + t, past = (pos < 0 ? 0 : pos) - a.window; // (the last position before the window)
	const auto row_of = [&](int r) {
		return (size_t)(row0 + r / a.group) * a.n_heads + h * a.group + r % a.group;
	};
	const int wl = r0 + 32 * wave + 31 < nrows - 1 ? r0 + 32 * wave + 31 : nrows - 1;
	const bool any = r0 + 32 * wave < nrows;
	const int w_first = len - n + (any ? r0 + 32 * wave : 0) / a.group, w_min = w_first < 0 ? 0 : w_first, w_max = any ? len - n + wl / a.group : -1;
	if (i0 >= i1 && split > 0) {
		if (!direct && live && hh == 0) {
			float* const p = a.part + (row_of(rr) * a.n_splits + split) * (D + 4) + D;
			p[0] = KV_LOW, p[1] = 0.f, p[2] = KV_NO_GAP;
		}
		return;
	}
	kv_f16x8 qh[KS], ql[HL ? KS : 1];
	float qf;
	{
		const size_t at = (size_t)(row0 + t) * (size_t)a.q_row + (size_t)hd * (size_t)a.q_head + hh * 8;
		// (the row is read twice: its largest magnitude first -- half a row of fp32 in registers beside everything else would not fit)
		float top = 0.f, odd = 0.f; // odd: NaN once an infinity or a NaN came by (fmaxf passes over a NaN)
#pragma unroll 4
		for (int i = 0; i < 2 * KS; ++i) {
			float y[4];
			kv_load4<DT>(a.q, at + 16 * (i >> 1) + 4 * (i & 1), y);
#pragma unroll
			for (int c = 0; c < 4; ++c) {
				top = fmaxf(top, fabsf(y[c]));
				odd = __builtin_fmaf(y[c], 0.f, odd);
			}
		}
		top = kv_max32(top);
		odd += __shfl_xor(odd, 32);
		const int e = kv_row_exp(top);
		const float inv = kv_exp2i(-e);
		qf = kv_exp2i(e) * fabsf(a.scale) + odd; // (a row with an infinity or a NaN is NaN)
		const float sign = a.scale < 0.f ? -inv : inv;
#pragma unroll
		for (int i = 0; i < KS; ++i) {
#pragma unroll
			for (int j = 0; j < 2; ++j) {
				float y[4];
				kv_load4<DT>(a.q, at + 16 * i + 4 * j, y);
#pragma unroll
				for (int c = 0; c < 4; ++c) {
					y[c] *= sign;
					qh[i][4 * j + c] = (_Float16)y[c];
					if constexpr (HL) {
						ql[i][4 * j + c] = (_Float16)(y[c] - (float)qh[i][4 * j + c]);
					}
				}
			}
		}
	}
	KvRefs ref;
	float l = 0.f;
	kv_f32x16 o[ND], zero;
#pragma unroll
	for (int e = 0; e < 16; ++e) {
		zero[e] = 0.f;
	}
#pragma unroll
	for (int d = 0; d < ND; ++d) {
		o[d] = zero;
	}
	// page ids, 64 at a time across the lanes: a look-up per page would put two dependent round trips to memory into every step
	int ids = -1, ids0 = i0;
	const auto fetch_ids = [&](int first) {
		ids0 = first;
		const int i = first + lane;
		ids = -1;
		if (i < i1) {
			const int pg = sp.page(i);
			ids = pg < a.r.max_pages ? a.r.table[(size_t)s * a.r.max_pages + pg] : -1;
			if (ids < 0 || ids >= a.p.n_pages) {
				kv_flag(a.p.status, KV_BAD_PAGE);
				ids = -1;
			}
		}
	};
	u32x4 kr[NK], vr[NV][2];
	kv_f32x4 ksc_n, vsc_n; // the next page's scales
	const auto load = [&](int pid) {
		const size_t page = (size_t)(pid < 0 ? 0 : pid) * H + h;
		const u32x4* const kp = (const u32x4*)(a.p.k + page * (KV_PAGE * D));
		const u32x4* const vp = (const u32x4*)(a.p.v + page * (KV_PAGE * D));
#pragma unroll
		for (int i = 0; i < NK; ++i) {
			const int it = tid + 256 * i; // 16 dims of a token: unit it of the page
			if (4 * D % 256 == 0 || it < 4 * D) {
				kr[i] = kp[it];
			}
		}
#pragma unroll
		for (int i = 0; i < NV; ++i) {
			const int it = tid + 256 * i; // (half, dim): quads half and half + 2
			if (2 * D % 256 == 0 || it < 2 * D) {
				vr[i][0] = vp[it], vr[i][1] = vp[it + 2 * D];
			}
		}
		ksc_n = *(const kv_f32x4*)(a.p.ks + page * 4), vsc_n = *(const kv_f32x4*)(a.p.vs + page * 4);
	};
	const auto stage = [&](int buf) {
		u32x4* const kl = kv_st + buf * (KU + VU);
		u32x4* const vl = kl + KU;
#pragma unroll
		for (int i = 0; i < NK; ++i) {
			const int it = tid + 256 * i, key = it / (D / 16), st = it % (D / 16);
			if (4 * D % 256 == 0 || it < 4 * D) {
				kl[(2 * st) * KROW + key] = __builtin_bit_cast(u32x4, kv_codes8(kr[i][0], kr[i][1]));
				kl[(2 * st + 1) * KROW + key] = __builtin_bit_cast(u32x4, kv_codes8(kr[i][2], kr[i][3]));
			}
		}
#pragma unroll
		for (int i = 0; i < NV; ++i) {
			const int it = tid + 256 * i, half = it / D, d = it % D;
			if (2 * D % 256 == 0 || it < 2 * D) {
#pragma unroll
				for (int b = 0; b < 4; ++b) {
					vl[(2 * b + half) * D + d] = __builtin_bit_cast(u32x4, kv_codes8(vr[i][0][b], vr[i][1][b]));
				}
			}
		}
	};
	int pid = -1;
	if (i0 < i1) {
		fetch_ids(i0);
		pid = __builtin_amdgcn_readlane(ids, 0);
		load(pid);
		stage(0);
	}
	__syncthreads();
	for (int i = i0; i < i1; ++i) {
		const int buf = (i - i0) & 1;
		const bool more = i + 1 < i1;
		// the page's scales, one of everything for the wave: their bits, in scalar registers
		int kb[4], vb[4];
#pragma unroll
		for (int b = 0; b < 4; ++b) {
			const float x = ksc_n[b], y = vsc_n[b];
			kb[b] = __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)), vb[b] = __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, y));
		}
		int next = -1;
		if (more) {
			if (i + 1 >= ids0 + 64) {
				fetch_ids(i + 1);
			}
			next = __builtin_amdgcn_readlane(ids, i + 1 - ids0);
			load(next);
		}
		const int j0 = sp.page(i) * KV_PAGE;
		const bool some = j0 <= w_max && (a.window <= 0 || j0 + KV_PAGE - 1 > w_min - a.window || j0 < a.sinks);
		if (some) {
			const bool whole = j0 + KV_PAGE - 1 <= w_min && (a.window <= 0 || j0 > w_max - a.window || j0 + KV_PAGE <= a.sinks);
			// The operands' LDS reads run KV_AHEAD ahead of the matrix instructions, and the scheduler is held to it (left to itself it keeps two in
			// flight: 190 instead of 187 us for 2049 rows on 4099 tokens); the scores go first where two waves want to issue (187 -> 183 us)
			const u32x4* const kl = kv_st + buf * (KU + VU) + hh * KROW + col;
			const u32x4* const vl = kv_st + buf * (KU + VU) + KU + hh * D + col;
			kv_f32x16 sc[2];
			__builtin_amdgcn_s_setprio(1);
			__builtin_amdgcn_sched_barrier(0);
#pragma unroll
			for (int k = 0; k < KS; ++k) {
#pragma unroll
				for (int b = 0; b < 2; ++b) {
					const kv_f16x8 kf = __builtin_bit_cast(kv_f16x8, kl[2 * k * KROW + 32 * b]);
					sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh[k], k ? sc[b] : zero, 0, 0, 0);
					if constexpr (HL) {
						sc[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[k], sc[b], 0, 0, 0);
					}
				}
			}
			KV_FEED(2 * KS, HL ? 2 : 1);
			__builtin_amdgcn_sched_barrier(0);
			__builtin_amdgcn_s_setprio(0);
			kv_f16x8 pf[4], pl[HL ? 4 : 1];
			// (a block whose V scale is no number, and a missing page, are NaN through K, for the rows that see them)
			int lv[4]; // exponents of V's scales
#pragma unroll
			for (int b = 0; b < 4; ++b) {
				const bool number = pid >= 0 && (unsigned)vb[b] < 0x7f800000u;
				kb[b] = number ? kb[b] : 0x7fc00000;
				lv[b] = number ? vb[b] >> 23 : 0;
			}
			float f[4];
#pragma unroll
			for (int b = 0; b < 4; ++b) {
				const int k = kb[b];
				f[b] = __builtin_bit_cast(float, k) * qf; // (not negative)
			}
			if (!whole) {
#pragma unroll
				for (int b = 0; b < 4; ++b) {
#pragma unroll
					for (int e = 8 * (b & 1); e < 8 * (b & 1) + 8; ++e) {
						const int j = j0 + 32 * (b >> 1) + 8 * (e >> 2) + 4 * hh + (e & 3);
						const bool seen = (j <= pos) & ((a.window <= 0) | (j > past) | (j < a.sinks));
						sc[b >> 1][e] = seen ? sc[b >> 1][e] * f[b] : -__builtin_inff();
					}
					f[b] = 1.f;
				}
			}
			int least = 255; // (as in k_kv_decode)
			float xb[4], top = -__builtin_inff();
#pragma unroll
			for (int b = 0; b < 4; ++b) {
				float t = -__builtin_inff();
#pragma unroll
				for (int e = 0; e < 8; ++e) {
					t = fmaxf(t, sc[b >> 1][8 * (b & 1) + e]);
				}
				xb[b] = t * f[b];
				top = fmaxf(top, xb[b]);
				least = min(least, xb[b] > -__builtin_inff() ? lv[b] : 255);
			}
			const auto join = [](float x) { return kv_max32(x); };
			const auto largest = [&](float m) {
				return fmaxf(fmaxf((xb[0] - m) + (float)lv[0], (xb[1] - m) + (float)lv[1]), fmaxf((xb[2] - m) + (float)lv[2], (xb[3] - m) + (float)lv[3]));
			};
			const float tv = largest(ref.m);
			bool far = false;
			if (__ballot(ref.asks(top, tv)) || ref.far) {
				const float by = ref.follow(l, join, largest);
#pragma unroll
				for (int d = 0; d < ND; ++d) {
					o[d] *= by;
				}
				if (ref.far) {
					far = true;
#pragma unroll
					for (int b = 0; b < 4; ++b) {
#pragma unroll
						for (int e = 8 * (b & 1); e < 8 * (b & 1) + 8; ++e) {
							sc[b >> 1][e] = kv_far_score(sc[b >> 1][e], f[b], ref.m);
						}
						f[b] = 1.f;
					}
				}
			} else {
				ref.tv = fmaxf(ref.tv, tv);
			}
			const float rm = far ? 0.f : ref.m;
			const int gap = (int)(ref.g - KV_LIFT);
			const auto weigh = [&](auto rounded) {
#pragma unroll
				for (int b = 0; b < 4; ++b) {
					const int k = min(gap - lv[b], (int)KV_REACH);
					const float from = -(rm + (float)k);
					float sum = 0.f;
#pragma unroll
					for (int e = 0; e < 8; ++e) {
						const float y = kv_exp2(__builtin_fmaf(sc[b >> 1][8 * (b & 1) + e], f[b], from));
						sum += rounded ? 0.f : y;
						pf[b][e] = (_Float16)y;
						if constexpr (HL) {
							pl[b][e] = (_Float16)(y - (float)pf[b][e]);
						}
					}
					if constexpr (rounded) {
						const u32x4 w = __builtin_bit_cast(u32x4, pf[b]);
						sum = kv_add2(kv_add2(kv_add2(kv_add2(0.f, w[0]), w[1]), w[2]), w[3]);
					}
					l = __builtin_fmaf(sum, kv_exp2i(max(k, -126)), l);
				}
			};
			if (DT == KV_F16 && !__ballot(gap > least + (int)KV_NEAR)) {
				weigh(std::integral_constant<bool, DT == KV_F16>());
			} else {
				weigh(std::false_type());
			}
			__builtin_amdgcn_sched_barrier(0);
#pragma unroll
			for (int b = 0; b < 4; ++b) {
#pragma unroll
				for (int d = 0; d < ND; ++d) {
					const kv_f16x8 vf = __builtin_bit_cast(kv_f16x8, vl[2 * b * D + 32 * d]);
					o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pf[b], o[d], 0, 0, 0);
					if constexpr (HL) {
						o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pl[b], o[d], 0, 0, 0);
					}
				}
			}
			KV_FEED(4 * ND, HL ? 2 : 1);
			__builtin_amdgcn_sched_barrier(0);
		}
		if (more) {
			stage(buf ^ 1);
		}
		__syncthreads();
		pid = next;
	}
	l += __shfl_xor(l, 32);
	int again = rr; // (looked up anew: kept through the loop, the row would cost two registers)
	asm volatile("" : "+v"(again));
	if (again >= nrows) {
		return;
	}
	const size_t row = row_of(again);
	const bool blind = l == 0.f && len - n + again / a.group < 0;
	const float f = l == 0.f ? (blind ? 0.f : __builtin_nanf("")) : 1.f / l;
#pragma unroll
	for (int d = 0; d < ND; ++d) {
#pragma unroll
		for (int q = 0; q < 4; ++q) {
			float y[4];
#pragma unroll
			for (int e = 0; e < 4; ++e) {
				y[e] = direct ? kv_result(o[d][4 * q + e] * f, ref.g) : o[d][4 * q + e];
			}
			kv_put<D, DT>(a, direct, row, split, 32 * d + 8 * q + 4 * hh, y);
		}
	}
	if (hh == 0 && a.n_splits > 1) {
		float* const p = a.part + (row * a.n_splits + split) * (D + 4) + D;
		p[0] = ref.m, p[1] = direct ? -1.f : l == 0.f && !blind ? -0.f : l, p[2] = ref.g; // (as above)
	}
}

// ---- the pages themselves ---------------------------------------------------------------------------------------------------------------
//
// A table row lists a sequence's pages (-1: none), refs[p] counts the rows that list page p; a page with a count of 0 is free, and the
// lowest free pages are taken first.  Full pages may be shared; a page that new tokens go into, and pages behind it, belong to one row.
// The bookkeeping is a few thousand integers: ONE workgroup does it (a grid-wide hand-off costs more than it spreads), with integer
// atomics only, so results do not depend on their order; the page bytes move in a launch of their own.

constexpr int KV_BOOK = 1024;     // threads of the bookkeeping workgroup
constexpr int KV_MAX_ROWS = 2048; // rows of a table the bookkeeping holds in LDS

// exclusive sum of one int per thread over the workgroup, and the total; `sm`: 17 ints
__device__ __forceinline__ int kv_block_scan(int v, int* sm, int& total) {
	const int lane = lane_id(), wave = threadIdx.x >> 6;
	int sum = v;
#pragma unroll
	for (int o = 1; o < 64; o <<= 1) {
		const int up = __shfl_up(sum, o);
		sum += lane >= o ? up : 0;
	}
	__syncthreads(); // (sm of the call before has been read)
	if (lane == 63) {
		sm[wave] = sum;
	}
	__syncthreads();
	int before = 0, all = 0;
#pragma unroll
	for (int w = 0; w < KV_BOOK / 64; ++w) {
		const int x = sm[w];
		before += w < wave ? x : 0;
		all += x;
	}
	total = all;
	return before + sum - v;
}

// list[k] <- the k-th free page (refs == 0) in ascending order, k < want; returns how many there are (at most want).  refs written by this
// workgroup before: barrier and fence are the caller's.  LOCAL: refs is in LDS
template <bool LOCAL>
__device__ __forceinline__ int kv_free_pages(const int* refs, int n_pages, int want, int* list, int* sm) {
	int have = 0;
	for (int p0 = 0; p0 < n_pages && have < want; p0 += KV_BOOK * 8) {
		unsigned mask = 0;
		const int mine = p0 + (int)threadIdx.x * 8;
#pragma unroll
		for (int j = 0; j < 8; ++j) {
			if (mine + j < n_pages && (LOCAL ? refs[mine + j] : __hip_atomic_load(refs + mine + j, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) == 0) {
				mask |= 1u << j;
			}
		}
		int total;
		int at = have + kv_block_scan(__builtin_popcount(mask), sm, total);
		while (mask) {
			const int j = __builtin_ctz(mask);
			mask &= mask - 1;
			if (at < want) {
				list[at] = mine + j;
			}
			++at;
		}
		have += total;
	}
	__syncthreads();
	return have < want ? have : want;
}

struct KvForkArgs {
	const int *table, *lens, *refs, *parents;
	int *table_out, *refs_out, *copy; // copy: [rows] x {from, to}, to = -1: none
	unsigned* status;
	int n_rows, max_pages, n_pages;
};

// (its time is round trips to memory, one behind another: parents and lengths are kept in LDS, and what does not depend on the new counts --
// the shared part of the new table, who needs a page -- is done beside them.  LOCAL: the counts are in LDS too, as many as fit, and go out
// once: 11.8 -> 4.8 us for 48 rows of 19 pages.)
constexpr int KV_FORK_LOCAL = 24576, KV_COMPACT_LOCAL = 12288; // pages whose bookkeeping LDS holds

template <bool LOCAL>
__global__ __launch_bounds__(KV_BOOK) void k_kv_fork(KvForkArgs a) {
	__shared__ int first[KV_MAX_ROWS], count[KV_MAX_ROWS], list[KV_MAX_ROWS], par[KV_MAX_ROWS], len[KV_MAX_ROWS], sm[KV_BOOK / 64];
	extern __shared__ int kv_refs[];
	const int tid = threadIdx.x, n = a.n_rows, mp = a.max_pages;
	int* const refs = LOCAL ? kv_refs : a.refs_out;
	for (int i = tid; i < n; i += KV_BOOK) {
		const int p = a.parents[i], l = a.lens[i];
		first[i] = n, count[i] = 0;
		par[i] = p >= 0 && p < n ? p : -1, len[i] = l < 0 ? 0 : l;
		if (par[i] < 0) {
			kv_flag(a.status, KV_BAD_PARENT);
		}
	}
	for (int p = tid; p < a.n_pages; p += KV_BOOK) {
		refs[p] = a.refs[p];
	}
	__syncthreads();
	for (int i = tid; i < n; i += KV_BOOK) {
		if (par[i] >= 0) {
			atomicMin(&first[par[i]], i);
			atomicAdd(&count[par[i]], 1);
		}
	}
	if (!LOCAL) {
		__threadfence();
	}
	__syncthreads();
	for (int k = tid; k < n * mp; k += KV_BOOK) {
		// counts: a full page of row r is listed by count[r] rows from now on, a page of its own by one of them at most
		const int r = k / mp, c = k - r * mp;
		const int d = (c < len[r] / KV_PAGE ? count[r] : (count[r] > 0 ? 1 : 0)) - 1;
		const int old = d ? a.table[k] : -1;
		// the new row: all of its parent's for a first child, the full pages for the others
		int p = -1;
		if (par[r] >= 0 && (first[par[r]] == r || c < len[par[r]] / KV_PAGE)) {
			p = a.table[par[r] * mp + c];
		}
		a.table_out[k] = p;
		if (old >= 0) {
			if (old < a.n_pages) {
				atomicAdd(&refs[old], d);
			} else {
				kv_flag(a.status, KV_BAD_PAGE);
			}
		}
	}
	// rows that need a page of their own: not the first child, the parent's last page not full
	int want = 0;
	for (int i0 = 0; i0 < n; i0 += KV_BOOK) {
		const int i = i0 + tid;
		int from = -1;
		if (i < n && par[i] >= 0 && first[par[i]] != i) {
			const int l = len[par[i]], c = l / KV_PAGE;
			from = l % KV_PAGE && c < mp ? a.table[par[i] * mp + c] : -1;
			from = from < a.n_pages ? from : -1;
		}
		int total;
		const int at = want + kv_block_scan(from >= 0, sm, total);
		if (i < n) {
			a.copy[2 * i] = from;
			count[i] = from >= 0 ? at : -1; // (every thread is through with count: the scan's barriers)
		}
		want += total;
	}
	if (!LOCAL) {
		__threadfence();
	}
	__syncthreads();
	const int have = kv_free_pages<LOCAL>(refs, a.n_pages, want, list, sm);
	if (have < want && tid == 0) {
		kv_flag(a.status, KV_NO_PAGE);
	}
	for (int i = tid; i < n; i += KV_BOOK) {
		const int at = count[i];
		int to = -1;
		if (at >= 0 && at < have) {
			to = list[at];
			a.table_out[i * mp + len[par[i]] / KV_PAGE] = to;
			refs[to] = 1;
		}
		a.copy[2 * i + 1] = to;
	}
	if constexpr (LOCAL) {
		__syncthreads();
		for (int p = tid; p < a.n_pages; p += KV_BOOK) {
			a.refs_out[p] = refs[p];
		}
	}
}

struct KvReserveArgs {
	int *table, *refs;
	const int *lens, *lens_new;
	unsigned* status;
	int n_rows, max_pages, n_pages;
	// reserve: the pool, for the pages that are copied (as in KvCopyArgs)
	signed char *k, *v;
	float *ks, *vs;
	size_t page;
	int scales, n_layers;
};

// pages for the tokens [lens[r], lens_new[r]) of every row: rows in order, a row's pages in order, the lowest free page each.  A row that was cut back
// lists pages that other rows list, too (refs > 1), and is about to write there: it gives them up for pages of its own.  The one that its tokens end in
// takes the old one's bytes with it, or, with no page free, the row loses the entry; it counts as free from the next call on, so nothing is copied over before
// it has been read.  This workgroup copies the bytes itself: a list for other workgroups would take a workspace, and such rows are few.  Who gives up
// what is settled by the counts at the beginning, so it does not depend on the rows' order.  Measured: a token for each of 48 rows of 33 pages 3.0 us, 500
// rows 3.4, with nothing to copy; k_kv_trim of the same rows 2.1 and 1.9.
__global__ __launch_bounds__(KV_BOOK) void k_kv_reserve(KvReserveArgs a) {
	__shared__ int list[KV_MAX_ROWS], from[KV_MAX_ROWS], into[KV_MAX_ROWS], sm[KV_BOOK / 64], n_own, n_left;
	const int tid = threadIdx.x, n = a.n_rows, mp = a.max_pages;
	if (tid == 0) {
		n_own = 0, n_left = 0;
	}
	// entries [c0, c1) of row i are to be pages of its own; cut: the first of them holds tokens already
	const auto range = [&](int i, int& c0, int& c1, bool& cut) {
		const int len = a.lens[i] < 0 ? 0 : a.lens[i], to = a.lens_new[i] < 0 ? 0 : a.lens_new[i];
		c0 = len / KV_PAGE, c1 = to > len ? (to - 1) / KV_PAGE + 1 : c0, cut = len % KV_PAGE;
		c1 = c1 > mp ? mp : c1;
		return to > len && (to - 1) / KV_PAGE >= mp;
	};
	__syncthreads();
	for (int i = tid; i < n; i += KV_BOOK) {
		int c0, c1;
		bool cut;
		if (range(i, c0, c1, cut)) {
			kv_flag(a.status, KV_NO_PAGE);
		}
		list[i] = -1; // (until pages are looked for: the page that the row's tokens end in, if others list it)
		for (int c = c0; c < c1; ++c) {
			int* const entry = a.table + (size_t)i * mp + c;
			const int p = *entry;
			if (p >= 0 && p < a.n_pages && a.refs[p] > 1) {
				if (c == c0 && cut) {
					list[i] = p;
				} else { // (below: after every row has looked at the counts)
					*entry = -2 - p;
					n_left = 1;
				}
			} else if (p < 0) {
				*entry = -1;
			}
		}
	}
	__syncthreads();
	int mine[KV_MAX_ROWS / KV_BOOK]; // list[] of this thread's rows
#pragma unroll
	for (int k = 0; k < KV_MAX_ROWS / KV_BOOK; ++k) {
		mine[k] = k * KV_BOOK + tid < n ? list[k * KV_BOOK + tid] : -1;
	}
	if (n_left) {
		for (int i = tid; i < n; i += KV_BOOK) {
			int c0, c1;
			bool cut;
			range(i, c0, c1, cut);
			for (int c = c0; c < c1; ++c) {
				int* const entry = a.table + (size_t)i * mp + c;
				if (*entry < -1) {
					atomicSub(&a.refs[-2 - *entry], 1);
					*entry = -1;
				}
			}
		}
		__threadfence();
	}
	__syncthreads();
	// a row at a time per thread; a call adds few pages to a row (a prompt: its pages)
#pragma unroll
	for (int k = 0; k < KV_MAX_ROWS / KV_BOOK; ++k) {
		if (k * KV_BOOK >= n) {
			break;
		}
		const int i = k * KV_BOOK + tid;
		int c0 = 0, c1 = 0, shared = mine[k];
		if (i < n) {
			bool cut;
			range(i, c0, c1, cut);
			if (c0 < c1 && cut && a.table[(size_t)i * mp + c0] < 0) { // the row's last tokens are lost: a new page would pass its bytes off as them
				kv_flag(a.status, KV_BAD_PAGE);
				++c0;
			}
		}
		int need = shared >= 0;
		for (int c = c0; c < c1; ++c) {
			need += a.table[(size_t)i * mp + c] < 0;
		}
		int total;
		int at = kv_block_scan(need, sm, total);
		// in portions of what `list` holds
		for (int done = 0; done < total; done += KV_MAX_ROWS) {
			const int want = total - done < KV_MAX_ROWS ? total - done : KV_MAX_ROWS;
			const int have = kv_free_pages<false>(a.refs, a.n_pages, want, list, sm);
			if (have < want && tid == 0) {
				kv_flag(a.status, KV_NO_PAGE);
			}
			while (c0 < c1 && at < done + want) {
				int* const entry = a.table + (size_t)i * mp + c0;
				if (shared >= 0 || *entry < 0) {
					const int p = at - done < have ? list[at - done] : -1;
					if (p >= 0) {
						__hip_atomic_store(a.refs + p, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
					}
					if (shared >= 0) {
						const int own = atomicAdd(&n_own, 1);
						from[own] = shared, into[own] = p;
						shared = -1;
					}
					*entry = p;
					++at;
				}
				++c0;
			}
			__threadfence();
			__syncthreads();
		}
	}
	__syncthreads(); // (no row has needed a page: n_own)
	for (int k = tid; k < n_own; k += KV_BOOK) {
		atomicSub(&a.refs[from[k]], 1);
	}
	for (int k = 0; k < n_own; ++k) {
		for (int l = 0; into[k] >= 0 && l < a.n_layers; ++l) {
			const size_t src = (size_t)l * a.n_pages + from[k], dst = (size_t)l * a.n_pages + into[k];
			const u32x4* const ks = (const u32x4*)(a.k + src * a.page);
			const u32x4* const vs = (const u32x4*)(a.v + src * a.page);
			u32x4* const kd = (u32x4*)(a.k + dst * a.page);
			u32x4* const vd = (u32x4*)(a.v + dst * a.page);
			for (int b = tid; b < (int)(a.page / 16); b += KV_BOOK) {
				const u32x4 x = ks[b], y = vs[b];
				kd[b] = x, vd[b] = y;
			}
			for (int b = tid; b < a.scales; b += KV_BOOK) {
				a.ks[dst * a.scales + b] = a.ks[src * a.scales + b], a.vs[dst * a.scales + b] = a.vs[src * a.scales + b];
			}
		}
	}
}

// pages that no later token of their row sees: behind its tokens (lens[r] = 0: the whole row), or, under a window, before it and not
// among the first tokens
__global__ __launch_bounds__(256) void k_kv_trim(KvReserveArgs a, int window, int sinks) {
	const int k = blockIdx.x * 256 + threadIdx.x, mp = a.max_pages;
	if (k >= a.n_rows * mp) {
		return;
	}
	const int r = k / mp, c = k - r * mp;
	const int len = a.lens[r] < 0 ? 0 : a.lens[r];
	const bool behind = c * KV_PAGE >= len;
	const bool before = window > 0 && len >= window && c * KV_PAGE + KV_PAGE - 1 <= len - window && c * KV_PAGE >= sinks;
	const int p = behind || before ? a.table[k] : -1;
	if (p >= 0) {
		a.table[k] = -1;
		if (p < a.n_pages) {
			atomicSub(&a.refs[p], 1);
		} else {
			kv_flag(a.status, KV_BAD_PAGE);
		}
	}
}

struct KvCompactArgs {
	const int *table, *refs;
	int *table_out, *refs_out, *n_live, *map, *copy; // map: [pages], copy: [pages / 2] x {from, to}
	unsigned* status;
	int n_rows, max_pages, n_pages;
};

// live pages at or beyond n_live (their number) move into the free ones below it, both in ascending order.  LOCAL: counts and map are in LDS,
// and the table's first entries are asked for at the start (12.5 -> 5.1 us for 900 pages)
template <bool LOCAL>
__global__ __launch_bounds__(KV_BOOK) void k_kv_compact(KvCompactArgs a) {
	__shared__ int sm[KV_BOOK / 64];
	extern __shared__ int kv_book[]; // [pages] counts, [pages] map, [pages / 2] x {from, to}
	const int tid = threadIdx.x, n = a.n_pages, cells = a.n_rows * a.max_pages;
	int* const map = LOCAL ? kv_book + n : a.map;
	int* const copy = LOCAL ? kv_book + 2 * n : a.copy;
	const int early = LOCAL && tid < cells ? a.table[tid] : -1;
	const auto refs = [&](int p) {
		return LOCAL ? kv_book[p] : a.refs[p];
	};
	int live = 0;
	for (int p0 = 0; p0 < n; p0 += KV_BOOK) {
		const int p = p0 + tid, r = p < n ? a.refs[p] : 0;
		if (LOCAL && p < n) {
			kv_book[p] = r;
		}
		int total;
		kv_block_scan(r > 0, sm, total);
		live += total;
	}
	if (tid == 0) {
		*a.n_live = live;
	}
	int holes = 0, movers = 0;
	for (int p0 = 0; p0 < n; p0 += KV_BOOK) {
		const int p = p0 + tid, ref = p < n ? refs(p) : 0; // (LOCAL: this thread's own)
		int nh, nm;
		const bool hole = p < live && ref <= 0, mover = p < n && p >= live && ref > 0;
		const int h = holes + kv_block_scan(hole, sm, nh), m = movers + kv_block_scan(mover, sm, nm);
		if (hole) {
			copy[2 * h + 1] = p;
		}
		if (mover) {
			copy[2 * m] = p;
		}
		if (p < n) {
			map[p] = p;
			a.refs_out[p] = p < live ? ref : 0;
		}
		holes += nh, movers += nm;
	}
	if (!LOCAL) {
		__threadfence();
	}
	__syncthreads();
	for (int i = tid; i < n / 2; i += KV_BOOK) {
		int from = -1, to = -1;
		if (i < movers) {
			from = copy[2 * i], to = copy[2 * i + 1];
			map[from] = to;
			a.refs_out[to] = refs(from);
		}
		if (LOCAL) {
			a.copy[2 * i] = from;
		}
		if (LOCAL || to < 0) {
			a.copy[2 * i + 1] = to;
		}
	}
	if (!LOCAL) {
		__threadfence();
	}
	__syncthreads();
	for (int k = tid; k < cells; k += KV_BOOK) {
		const int p = LOCAL && k == tid ? early : a.table[k];
		int q = p;
		if (p >= n) {
			kv_flag(a.status, KV_BAD_PAGE);
		} else if (p >= 0) {
			q = map[p];
		}
		a.table_out[k] = q;
	}
}

struct KvCopyArgs {
	signed char *k, *v;
	float *ks, *vs;
	const int* copy;
	size_t page, pages; // bytes of a page's codes (K or V) of one layer; pages of a layer
	int scales;         // floats of a page's scales of one layer
};

// the bytes of the pages that move.  Measured: 315 MB (150 pages, 8 layers of 8 heads of 128) 66 us = 4.8 TB/s, 76 MB 17.8 us = 4.3
// grid = (copies at most, pieces of a page, layers): piece = 16 KiB of K and of V
constexpr int KV_PIECE = 16384;
__global__ __launch_bounds__(256) void k_kv_copy(KvCopyArgs a) {
	const int from = a.copy[2 * blockIdx.x], to = a.copy[2 * blockIdx.x + 1];
	if (to < 0) {
		return;
	}
	const size_t l0 = blockIdx.z * a.pages;
	const size_t src = (l0 + from) * a.page, dst = (l0 + to) * a.page;
	const size_t b0 = (size_t)blockIdx.y * KV_PIECE + threadIdx.x * 16;
	u32x4 x[2][KV_PIECE / 4096];
#pragma unroll
	for (int i = 0; i < KV_PIECE / 4096; ++i) {
		const size_t b = b0 + 4096 * i;
		if (b < a.page) {
			x[0][i] = *(const u32x4*)(a.k + src + b), x[1][i] = *(const u32x4*)(a.v + src + b);
		}
	}
#pragma unroll
	for (int i = 0; i < KV_PIECE / 4096; ++i) {
		const size_t b = b0 + 4096 * i;
		if (b < a.page) {
			*(u32x4*)(a.k + dst + b) = x[0][i], *(u32x4*)(a.v + dst + b) = x[1][i];
		}
	}
	if (blockIdx.y == 0) {
		for (int i = threadIdx.x; i < a.scales; i += 256) {
			a.ks[(l0 + to) * a.scales + i] = a.ks[(l0 + from) * a.scales + i];
			a.vs[(l0 + to) * a.scales + i] = a.vs[(l0 + from) * a.scales + i];
		}
	}
}

} // namespace calm
