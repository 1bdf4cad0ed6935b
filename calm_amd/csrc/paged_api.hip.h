// paged_api.hip.h -- the C entries of the paged cache and of the beam selection (include/calm_hip.h): argument checks and launches.
//
// These entries work on memory and streams of the caller's (no model, no init_hip): they launch on the current device, allocate nothing,
// never synchronise, and report a refused call by their return value instead of aborting -- nothing has been launched then.
#pragma once

namespace {

thread_local char g_kv_error[256] = "";

int kv_fail(const char* what, const char* why) {
	snprintf(g_kv_error, sizeof(g_kv_error), "%s: %s", what, why);
	return -1;
}
int kv_launched(const char* what) {
	const hipError_t e = hipGetLastError();
	return e == hipSuccess ? 0 : kv_fail(what, hipGetErrorString(e));
}
#define KV_CHECK(cond, why)              \
	do {                                 \
		if (!(cond))                     \
			return kv_fail(__func__, why); \
	} while (0)

// compute units of the current device (asked once per device: the value never changes)
int kv_cus() {
	static std::atomic<int> known[64];
	int dev = 0;
	if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
		return 256;
	}
	int n = known[dev].load(std::memory_order_relaxed);
	if (!n) {
		n = 256;
		(void)hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev);
		known[dev].store(n, std::memory_order_relaxed);
	}
	return n;
}
// a kernel that wants more than 64 KiB of LDS has to say so, once per device
int kv_lds(const void* kernel, size_t bytes, const char* what) {
	if (bytes <= 64 * 1024) {
		return 0;
	}
	static std::mutex lock;
	static std::map<const void*, unsigned long long> told; // a bit per device
	int dev = 0;
	if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
		return kv_fail(what, "no current device");
	}
	std::lock_guard<std::mutex> hold(lock);
	unsigned long long& seen = told[kernel];
	if (!((seen >> dev) & 1)) {
		if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess) {
			(void)hipGetLastError();
			return kv_fail(what, "the device does not give a workgroup the LDS that this head size needs");
		}
		seen |= 1ull << dev;
	}
	return 0;
}

bool kv_aligned(const void* p, size_t to) {
	return ((size_t)p & (to - 1)) == 0;
}
const char* kv_pool_fault(const struct KvPool* p) {
	if (!p || !p->k || !p->v || !p->k_scale || !p->v_scale || !p->status) {
		return "a pool pointer is missing";
	}
	if (p->n_layers < 1 || p->n_layers > 65535 || p->n_pages < 1 || p->n_pages > 1 << 30 || p->n_kv_heads < 1 || p->n_kv_heads > 1024) {
		return "the pool has no layers, pages or heads, or more than 65535 layers, 2^30 pages or 1024 heads";
	}
	if (p->head_dim != 64 && p->head_dim != 96 && p->head_dim != 128 && p->head_dim != 256) {
		return "head sizes 64, 96, 128 and 256";
	}
	if (!kv_aligned(p->k, 16) || !kv_aligned(p->v, 16) || !kv_aligned(p->k_scale, 16) || !kv_aligned(p->v_scale, 16)) {
		return "pool arrays begin at 16-byte boundaries";
	}
	return nullptr;
}
const char* kv_batch_fault(const struct KvBatch* b) {
	if (!b || !b->table || !b->lens || !b->starts) {
		return "a batch pointer is missing";
	}
	if (b->n_seqs < 1 || b->n_seqs > 65535 || b->max_pages < 1 || b->n_rows < 0 || b->max_rows < 0 || b->max_len < 0) {
		return "a batch has 1 to 65535 sequences, at least one page column and no negative counts";
	}
	if ((long long)b->n_seqs * b->max_pages > 1 << 30) {
		return "a table of more than 2^30 entries";
	}
	return nullptr;
}
KvLayer kv_layer(const struct KvPool* p, int layer) {
	const size_t codes = (size_t)p->n_pages * p->n_kv_heads * KV_PAGE * p->head_dim, scales = (size_t)p->n_pages * p->n_kv_heads * 4;
	KvLayer l;
	l.k = p->k + layer * codes, l.v = p->v + layer * codes;
	l.ks = p->k_scale + layer * scales, l.vs = p->v_scale + layer * scales;
	l.status = p->status, l.n_pages = p->n_pages, l.n_kv_heads = p->n_kv_heads;
	return l;
}
KvRows kv_rows(const struct KvBatch* b) {
	return KvRows{b->starts, b->lens, b->table, b->n_seqs, b->max_pages, b->n_rows, b->max_rows};
}

// f(head size, type) with both as compile-time constants
template <class F>
int kv_dispatch(int head_dim, int type, F f) {
	const auto by_type = [&](auto D) {
		switch (type) {
		case KV_F32:
			return f(D, std::integral_constant<int, KV_F32>());
		case KV_F16:
			return f(D, std::integral_constant<int, KV_F16>());
		default:
			return f(D, std::integral_constant<int, KV_BF16>());
		}
	};
	switch (head_dim) {
	case 64:
		return by_type(std::integral_constant<int, 64>());
	case 96:
		return by_type(std::integral_constant<int, 96>());
	case 128:
		return by_type(std::integral_constant<int, 128>());
	default:
		return by_type(std::integral_constant<int, 256>());
	}
}

// How attention is cut: rows per workgroup, and the pages a workgroup walks.
struct KvCut {
	bool chunked;           // k_kv_chunk (128 rows a workgroup), else k_kv_decode (16)
	int nw, tiles, n_splits, chunk;
};
KvCut kv_cut(const struct KvPool* p, const struct KvBatch* b, int n_heads, int type, int window, int sinks) {
	KvCut c;
	const int group = n_heads / p->n_kv_heads, cus = kv_cus();
	const long long rows = (long long)(b->max_rows < 1 ? 1 : b->max_rows) * group; // rows of a sequence and kv head
	const long long base = (long long)b->n_seqs * p->n_kv_heads;
	// pages that a tile of `per` rows sees at most
	const auto pages = [&](int per) {
		long long seen = ((long long)b->max_len + KV_PAGE - 1) / KV_PAGE;
		if (window > 0) {
			const long long span = ((long long)window + per / group + 2 * KV_PAGE) / KV_PAGE + 1 + ((long long)sinks + KV_PAGE - 1) / KV_PAGE;
			seen = span < seen ? span : seen;
		}
		return seen < 1 ? 1 : seen;
	};
	// 16 rows a workgroup and whole-number scores, or 128 rows that share the conversion of a page's codes.  Measured, 16 / 128, us, 8 kv heads of 128, bf16: 32
	// sequences of 2048 with 32 rows a head 36 / 41, 36 rows 52 / 49, 64 rows 68 / 51, 128 rows 130 / 65; 8 of 4096 with 32 rows 23 / 28, 64 rows 29 / 34, 96 rows
	// 54 / 38; heads of 64 cross at about 50 rows, fp32 rows at 90, and one sequence alone beyond 128.
	// (fp32 rows of 256: both halves of q and the sums do not fit a wave's registers)
	c.chunked = rows > 32 && !(p->head_dim == 256 && type == KV_F32);
	if (c.chunked) { // two workgroups per CU, at least 8 pages each (the join moves every row's partial sums through memory)
		c.nw = 4, c.tiles = (int)((rows + 127) / 128);
		const long long wgs = base * c.tiles, seen = pages(128);
		long long splits = (2ll * cus + wgs - 1) / wgs;
		splits = splits < 1 ? 1 : splits > 64 ? 64 : splits;
		const long long chunk = (seen + splits - 1) / splits;
		c.chunk = (int)(chunk < 8 ? 8 : chunk);
		c.n_splits = (int)((seen + c.chunk - 1) / c.chunk);
		return c;
	}
	// What a cut into n ranges costs, in steps of a workgroup (a page for each of its waves, about 2 us): workgroups run in rounds of one
	// to a CU (their registers fill it), a round begins with look-ups and first loads (2 steps), and ranges are joined by a second launch.
	// Measured, n = 1 / 2 / 4 / 8, in us: 8 sequences of 4093, 8 kv heads of 128 (64 workgroups uncut) 30.3 / 23.2 / 20.5 / 28.5; 64 of 91 - 8191, 4 kv
	// heads of 64 (256) 39.3 / 46.2 / 54.1 / 68.9; 24 of 13.9 - 16.4k (192) 136 / 157 / 144 / 151; 16 under a window of 1024 (256) 14.3 / 27.7 / 30.4 / 30.6.
	const int nw = p->head_dim <= 128 ? 8 : 4;
	c.nw = nw, c.tiles = (int)((rows + 15) / 16);
	const long long wgs = base * c.tiles, seen = pages(16);
	double best = 0;
	for (long long n = 1; n <= 64 && (n == 1 || (n - 1) * nw < seen); ++n) {
		const double rounds = ceil((double)(wgs * n) / cus);
		const long long chunk = ((seen + n - 1) / n + nw - 1) / nw * nw; // whole steps
		const double cost = rounds * ((double)(chunk / nw) + 2.0) + (n > 1 ? 2.0 + 0.2 * (double)n : 0.0);
		if (n == 1 || cost < 0.97 * best) {
			best = cost;
			c.chunk = (int)chunk;
			c.n_splits = (int)((seen + chunk - 1) / chunk);
		}
	}
	return c;
}
size_t kv_cut_bytes(const KvCut& c, const struct KvPool* p, const struct KvBatch* b, int n_heads) {
	return c.n_splits > 1 ? (size_t)b->n_rows * n_heads * c.n_splits * (p->head_dim + 4) * sizeof(float) : 0;
}
const char* kv_attend_fault(const struct KvPool* p, const struct KvBatch* b, int n_heads, int window, int sinks) {
	if (n_heads < 1 || n_heads % p->n_kv_heads || n_heads / p->n_kv_heads > 1024) {
		return "query heads are a multiple (at most 1024 times) of the pool's kv heads";
	}
	if (window < 0 || sinks < 0) {
		return "a negative window or count of first tokens";
	}
	if ((long long)b->max_rows * n_heads > 0x7fffff00ll || (long long)b->n_rows * n_heads > 0x7fffff00ll) {
		return "more than 2^31 rows times heads";
	}
	return nullptr;
}

int kv_copy_pages(const struct KvPool* p, const int* copy, int n, hipStream_t stream, const char* what) {
	KvCopyArgs a;
	a.k = p->k, a.v = p->v, a.ks = p->k_scale, a.vs = p->v_scale, a.copy = copy;
	a.page = (size_t)p->n_kv_heads * KV_PAGE * p->head_dim, a.pages = p->n_pages, a.scales = p->n_kv_heads * 4;
	hipLaunchKernelGGL(k_kv_copy, dim3(n, (unsigned)((a.page + KV_PIECE - 1) / KV_PIECE), p->n_layers), dim3(256), 0, stream, a);
	return kv_launched(what);
}

} // namespace

extern "C" const char* calm_hip_error(void) {
	return g_kv_error;
}

extern "C" void* calm_hip_stream(void) {
	init_hip();
	return g_stream;
}

extern "C" int kv_append_hip(const struct KvPool* pool, const struct KvBatch* batch, int layer, const void* k, const void* v, int type, long k_row, long k_head, long v_row,
                             long v_head, void* stream) {
	const char* fault = kv_pool_fault(pool);
	fault = fault ? fault : kv_batch_fault(batch);
	KV_CHECK(!fault, fault);
	KV_CHECK(layer >= 0 && layer < pool->n_layers, "no such layer");
	KV_CHECK(type >= KV_F32 && type <= KV_BF16, "types 0 (fp32), 1 (fp16), 2 (bf16)");
	if (batch->n_rows == 0) {
		return 0;
	}
	KV_CHECK(k && v, "rows are missing");
	const size_t unit = type == KV_F32 ? 16 : 8;
	KV_CHECK(kv_aligned(k, unit) && kv_aligned(v, unit) && k_row % 4 == 0 && k_head % 4 == 0 && v_row % 4 == 0 && v_head % 4 == 0,
	         "rows and heads begin at multiples of four elements");
	KvAppendArgs a;
	a.p = kv_layer(pool, layer), a.r = kv_rows(batch);
	a.k = k, a.v = v, a.k_row = k_row, a.k_head = k_head, a.v_row = v_row, a.v_head = v_head;
	// pages touched: a sequence of n rows touches min(n, n / 64 + 2) of them at most
	const long long most = (long long)batch->n_rows / KV_PAGE + 2ll * batch->n_seqs;
	const unsigned pages = (unsigned)(most < batch->n_rows ? most : batch->n_rows);
	return kv_dispatch(pool->head_dim, type, [&](auto D, auto T) {
		hipLaunchKernelGGL((k_kv_append<decltype(D)::value, decltype(T)::value>), dim3(pages + 1, pool->n_kv_heads), dim3(256), 0, (hipStream_t)stream, a);
		return kv_launched("kv_append_hip");
	});
}

extern "C" int kv_read_hip(const struct KvPool* pool, int layer, const int* table, const int* lens, const int* start, int n_seqs, int max_pages, int count, void* k, void* v, int type,
                           void* stream) {
	const char* fault = kv_pool_fault(pool);
	KV_CHECK(!fault, fault);
	KV_CHECK(layer >= 0 && layer < pool->n_layers, "no such layer");
	KV_CHECK(type >= KV_F32 && type <= KV_BF16, "types 0 (fp32), 1 (fp16), 2 (bf16)");
	KV_CHECK(table && lens && start, "table, lengths or starts are missing");
	KV_CHECK(n_seqs >= 1 && n_seqs <= 65535 && max_pages >= 1 && count >= 0, "1 to 65535 sequences, at least one page column, no negative count");
	KV_CHECK(count <= 0x7fffff00, "too many tokens");
	if (count == 0) {
		return 0;
	}
	KV_CHECK(k && v && kv_aligned(k, type == KV_F32 ? 16 : 8) && kv_aligned(v, type == KV_F32 ? 16 : 8), "outputs are missing or not aligned to four elements");
	KvReadArgs a;
	a.p = kv_layer(pool, layer), a.table = table, a.lens = lens, a.start = start, a.k = k, a.v = v;
	a.n_seqs = n_seqs, a.max_pages = max_pages, a.count = count;
	return kv_dispatch(pool->head_dim, type, [&](auto D, auto T) {
		hipLaunchKernelGGL((k_kv_read<decltype(D)::value, decltype(T)::value>), dim3((count + 15) / 16 + 1, pool->n_kv_heads, n_seqs), dim3(64), 0, (hipStream_t)stream, a);
		return kv_launched("kv_read_hip");
	});
}

extern "C" long long kv_attend_workspace_hip(const struct KvPool* pool, const struct KvBatch* batch, int type, int n_heads, int window, int sinks) {
	const char* fault = kv_pool_fault(pool);
	fault = fault ? fault : kv_batch_fault(batch);
	fault = fault ? fault : kv_attend_fault(pool, batch, n_heads, window, sinks);
	KV_CHECK(!fault, fault);
	KV_CHECK(type >= KV_F32 && type <= KV_BF16, "types 0 (fp32), 1 (fp16), 2 (bf16)");
	return (long long)kv_cut_bytes(kv_cut(pool, batch, n_heads, type, window, sinks), pool, batch, n_heads);
}

extern "C" int kv_attend_hip(const struct KvPool* pool, const struct KvBatch* batch, int layer, const void* q, void* out, int type, int n_heads, long q_row, long q_head, float scale,
                             int window, int sinks, void* workspace, size_t workspace_size, void* stream) {
	const char* fault = kv_pool_fault(pool);
	fault = fault ? fault : kv_batch_fault(batch);
	fault = fault ? fault : kv_attend_fault(pool, batch, n_heads, window, sinks);
	KV_CHECK(!fault, fault);
	KV_CHECK(layer >= 0 && layer < pool->n_layers, "no such layer");
	KV_CHECK(type >= KV_F32 && type <= KV_BF16, "types 0 (fp32), 1 (fp16), 2 (bf16)");
	KV_CHECK(scale - scale == 0.f, "the scale is not a finite number");
	if (batch->n_rows == 0) {
		return 0;
	}
	KV_CHECK(q && out, "query rows or output are missing");
	const size_t unit = type == KV_F32 ? 16 : 8;
	KV_CHECK(kv_aligned(q, unit) && kv_aligned(out, unit) && q_row % 4 == 0 && q_head % 4 == 0, "rows and heads begin at multiples of four elements");
	const KvCut c = kv_cut(pool, batch, n_heads, type, window, sinks);
	const size_t need = kv_cut_bytes(c, pool, batch, n_heads);
	KV_CHECK(need == 0 || (workspace && workspace_size >= need && kv_aligned(workspace, 16)), "the workspace is missing, too small (kv_attend_workspace_hip) or not 16-byte aligned");
	{ // (a row of out may be written while another workgroup still reads that row of q)
		const long rows = batch->n_rows, item = type == KV_F32 ? 4 : 2, dr = (rows - 1) * q_row, dh = (n_heads - 1) * q_head;
		const char* const q0 = (const char*)q + item * ((dr < 0 ? dr : 0) + (dh < 0 ? dh : 0));
		const char* const q1 = (const char*)q + item * ((dr > 0 ? dr : 0) + (dh > 0 ? dh : 0) + pool->head_dim);
		KV_CHECK((const char*)out + item * rows * n_heads * pool->head_dim <= q0 || (const char*)out >= q1, "the output overlaps the query rows");
	}
	KvAttnArgs a;
	a.p = kv_layer(pool, layer), a.r = kv_rows(batch);
	a.q = q, a.out = out, a.q_row = q_row, a.q_head = q_head, a.part = (float*)workspace;
	a.n_heads = n_heads, a.group = n_heads / pool->n_kv_heads, a.window = window, a.sinks = sinks;
	a.chunk = c.chunk, a.n_splits = c.n_splits, a.scale = scale * 1.4426950408889634f;
	const int H = pool->n_kv_heads;
	KV_CHECK(c.chunked ? (long long)batch->n_seqs * c.n_splits * H * c.tiles <= 0x7fffffffll : (long long)H * c.tiles <= 65535, "too many sequences for rows this many and contexts this long");
	return kv_dispatch(pool->head_dim, type, [&](auto Dc, auto Tc) {
		constexpr int D = decltype(Dc)::value, T = decltype(Tc)::value;
		const hipStream_t st = (hipStream_t)stream;
		if (c.chunked) {
			if constexpr (D < 256 || T != KV_F32) {
				auto kern = k_kv_chunk<D, T>;
				constexpr size_t lds = KvChunk<D>::LDS;
				if (kv_lds((const void*)kern, lds, "kv_attend_hip")) {
					return -1;
				}
				hipLaunchKernelGGL(kern, dim3((unsigned)c.tiles * H * batch->n_seqs * c.n_splits), dim3(256), lds, st, a);
			}
		} else {
			constexpr int NW = D <= 128 ? 8 : 4;
			auto kern = k_kv_decode<D, T, NW>;
			constexpr size_t lds = (size_t)NW * 16 * (D + 4) * sizeof(float);
			if (kv_lds((const void*)kern, lds, "kv_attend_hip")) {
				return -1;
			}
			hipLaunchKernelGGL(kern, dim3(c.n_splits, H * c.tiles, batch->n_seqs), dim3(64 * NW), lds, st, a);
		}
		if (c.n_splits > 1) {
			hipLaunchKernelGGL((k_kv_merge<D, T>), dim3(((unsigned)batch->n_rows * n_heads + 3) / 4), dim3(256), 0, st, a);
		}
		return kv_launched("kv_attend_hip");
	});
}

static const char* kv_table_fault(const struct KvPool* pool, const int* table, const int* lens, const int* refs, int n_rows, int max_pages) {
	const char* fault = kv_pool_fault(pool);
	if (fault) {
		return fault;
	}
	if (!table || !refs || !lens) {
		return "table, lengths or counts are missing";
	}
	if (n_rows < 1 || n_rows > KV_MAX_ROWS || max_pages < 1 || (long long)n_rows * max_pages > 1 << 30) {
		return "1 to 2048 table rows, at least one page column, at most 2^30 entries";
	}
	return nullptr;
}

extern "C" int kv_reserve_hip(const struct KvPool* pool, int* table, int* refs, const int* lens, const int* lens_new, int n_rows, int max_pages, void* stream) {
	const char* fault = kv_table_fault(pool, table, lens, refs, n_rows, max_pages);
	KV_CHECK(!fault, fault);
	KV_CHECK(lens_new, "new lengths are missing");
	const size_t page = (size_t)pool->n_kv_heads * KV_PAGE * pool->head_dim;
	const KvReserveArgs a = {table, refs, lens, lens_new, pool->status, n_rows, max_pages, pool->n_pages, pool->k, pool->v, pool->k_scale, pool->v_scale, page,
	                         pool->n_kv_heads * 4, pool->n_layers};
	hipLaunchKernelGGL(k_kv_reserve, dim3(1), dim3(KV_BOOK), 0, (hipStream_t)stream, a);
	return kv_launched("kv_reserve_hip");
}

extern "C" int kv_trim_hip(const struct KvPool* pool, int* table, int* refs, const int* lens, int n_rows, int max_pages, int window, int sinks, void* stream) {
	const char* fault = kv_table_fault(pool, table, lens, refs, n_rows, max_pages);
	KV_CHECK(!fault, fault);
	KV_CHECK(window >= 0 && sinks >= 0, "a negative window or count of first tokens");
	const KvReserveArgs a = {table, refs, lens, nullptr, pool->status, n_rows, max_pages, pool->n_pages, nullptr, nullptr, nullptr, nullptr, 0, 0, 0};
	hipLaunchKernelGGL(k_kv_trim, dim3((unsigned)(((long long)n_rows * max_pages + 255) / 256)), dim3(256), 0, (hipStream_t)stream, a, window, sinks);
	return kv_launched("kv_trim_hip");
}

extern "C" int kv_fork_hip(const struct KvPool* pool, const int* table, const int* lens, const int* refs, const int* parents, int n_rows, int max_pages, int* table_out, int* refs_out,
                           void* workspace, size_t workspace_size, void* stream) {
	const char* fault = kv_table_fault(pool, table, lens, refs, n_rows, max_pages);
	KV_CHECK(!fault, fault);
	KV_CHECK(parents && table_out && refs_out, "parents or outputs are missing");
	KV_CHECK(table_out != table, "the new table is written beside the old one");
	KV_CHECK(workspace && workspace_size >= (size_t)n_rows * 2 * sizeof(int) && kv_aligned(workspace, 4), "the workspace is missing or smaller than 8 bytes a row");
	const KvForkArgs a = {table, lens, refs, parents, table_out, refs_out, (int*)workspace, pool->status, n_rows, max_pages, pool->n_pages};
	if (pool->n_pages <= KV_FORK_LOCAL) {
		if (kv_lds((const void*)k_kv_fork<true>, KV_FORK_LOCAL * sizeof(int), "kv_fork_hip")) {
			return -1;
		}
		hipLaunchKernelGGL(k_kv_fork<true>, dim3(1), dim3(KV_BOOK), (size_t)pool->n_pages * sizeof(int), (hipStream_t)stream, a);
	} else {
		hipLaunchKernelGGL(k_kv_fork<false>, dim3(1), dim3(KV_BOOK), 0, (hipStream_t)stream, a);
	}
	const int rc = kv_launched("kv_fork_hip");
	return rc ? rc : kv_copy_pages(pool, a.copy, n_rows, (hipStream_t)stream, "kv_fork_hip");
}

extern "C" int kv_compact_hip(const struct KvPool* pool, const int* table, const int* refs, int n_rows, int max_pages, int* table_out, int* refs_out, int* n_live, void* workspace,
                              size_t workspace_size, void* stream) {
	const char* fault = kv_table_fault(pool, table, refs, refs, n_rows, max_pages);
	KV_CHECK(!fault, fault);
	KV_CHECK(table_out && refs_out && n_live, "an output is missing");
	KV_CHECK(refs_out != refs, "the new counts are written beside the old ones");
	KV_CHECK(workspace && workspace_size >= (size_t)pool->n_pages * 2 * sizeof(int) && kv_aligned(workspace, 4), "the workspace is missing or smaller than 8 bytes a page");
	int* const map = (int*)workspace;
	const KvCompactArgs a = {table, refs, table_out, refs_out, n_live, map, map + pool->n_pages, pool->status, n_rows, max_pages, pool->n_pages};
	if (pool->n_pages <= KV_COMPACT_LOCAL) {
		if (kv_lds((const void*)k_kv_compact<true>, 3 * KV_COMPACT_LOCAL * sizeof(int), "kv_compact_hip")) {
			return -1;
		}
		hipLaunchKernelGGL(k_kv_compact<true>, dim3(1), dim3(KV_BOOK), (size_t)pool->n_pages * 3 * sizeof(int), (hipStream_t)stream, a);
	} else {
		hipLaunchKernelGGL(k_kv_compact<false>, dim3(1), dim3(KV_BOOK), 0, (hipStream_t)stream, a);
	}
	const int rc = kv_launched("kv_compact_hip");
	return rc || pool->n_pages < 2 ? rc : kv_copy_pages(pool, a.copy, pool->n_pages / 2, (hipStream_t)stream, "kv_compact_hip");
}

static int beam_chunks(int vocab) {
	return (vocab + BEAM_CHUNK - 1) / BEAM_CHUNK;
}

extern "C" long long beam_workspace_hip(int groups, int beams, int vocab) {
	KV_CHECK(groups >= 1 && beams >= 1 && beams <= BEAM_MAX && vocab >= 1 && vocab <= 1 << 30 && (long long)groups * beams <= 65535,
	         "1 to 32 beams, 1 to 2^30 tokens, at most 65535 rows");
	return (long long)groups * beams * beam_chunks(vocab) * (2ll * sizeof(double) + beams * (sizeof(float) + sizeof(int)));
}

extern "C" int beam_select_hip(const void* logits, int type, long row, int groups, int beams, int vocab, const float* scores, const unsigned char* done, int eos, float* scores_out,
                               int* parents, int* tokens, unsigned char* done_out, void* workspace, size_t workspace_size, void* stream) {
	const long long need = beam_workspace_hip(groups, beams, vocab);
	KV_CHECK(need > 0, "1 to 32 beams, 1 to 2^30 tokens, at most 65535 rows");
	KV_CHECK(type >= KV_F32 && type <= KV_BF16, "types 0 (fp32), 1 (fp16), 2 (bf16)");
	KV_CHECK(logits && scores && scores_out && parents && tokens && done_out, "a pointer is missing");
	KV_CHECK(kv_aligned(logits, type == KV_F32 ? 4 : 2), "logits are not aligned to their type");
	KV_CHECK(row >= vocab || row == 0, "rows of logits overlap"); // (0: every beam the same row)
	KV_CHECK(eos < vocab, "the end token is outside the vocabulary");
	KV_CHECK(workspace && (long long)workspace_size >= need && kv_aligned(workspace, 8), "the workspace is missing, too small (beam_workspace_hip) or not 8-byte aligned");
	KV_CHECK(scores_out != scores && done_out != done, "outputs are written beside the inputs");
	BeamArgs a;
	const size_t rows = (size_t)groups * beams;
	a.logits = logits, a.row = row, a.score = scores, a.done = eos < 0 ? nullptr : done;
	a.score_out = scores_out, a.parent = parents, a.token = tokens, a.done_out = done_out;
	a.groups = groups, a.beams = beams, a.vocab = vocab, a.n_chunks = beam_chunks(vocab), a.eos = eos;
	a.sums = (double*)workspace;
	a.val = (float*)(a.sums + 2 * rows * a.n_chunks);
	a.idx = (int*)(a.val + rows * a.n_chunks * beams);
	const dim3 grid(a.n_chunks, (unsigned)rows);
	const hipStream_t st = (hipStream_t)stream;
	if (type == KV_F32) {
		hipLaunchKernelGGL(k_beam_rows<KV_F32>, grid, dim3(256), 0, st, a);
	} else if (type == KV_F16) {
		hipLaunchKernelGGL(k_beam_rows<KV_F16>, grid, dim3(256), 0, st, a);
	} else {
		hipLaunchKernelGGL(k_beam_rows<KV_BF16>, grid, dim3(256), 0, st, a);
	}
	hipLaunchKernelGGL(k_beam_pick, dim3(groups), dim3(64 * (beams < 16 ? beams : 16)), 0, st, a);
	return kv_launched("beam_select_hip");
}
