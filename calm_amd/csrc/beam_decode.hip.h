// beam_decode.hip.h -- decode_beam_hip: a beam search of a prepared model on the device.
//
// W hypotheses share one stream of the weights per step: the layers run as a prompt chunk of W tokens (infer_hip.hip: prefill_chunk with a
// BatchStep) at one position, their K / V rows go into a paged 8-bit cache (kv_append_hip) and their attention reads it (kv_attend_hip), the
// W best continuations are chosen (beam_select_hip) and the cache's rows follow them (kv_fork_hip): the prompt's pages are held once, a
// hypothesis costs the pages behind its own fork.  Everything of a step is queued on the backend's stream; the host looks only at the end,
// and every 32 steps whether all hypotheses are finished.
#pragma once

namespace {

struct BeamBuffers {
	int pages = 0, cols = 0, steps = 0, beams = 0; // what the memory below is for, at most
	struct KvPool pool;
	std::vector<void*> owned;
	int *ints = nullptr;              // lengths of every step, row starts, tables, counts (beam_ints)
	int *tok = nullptr, *par = nullptr; // [step][W]
	float *score[2], *att = nullptr, *logits = nullptr;
	unsigned char* done[2];
	__half *k = nullptr, *v = nullptr; // [kv head][W][head_dim]
	__half* wide = nullptr;            // an fp8 cache's layer as binary16, K and V
	char* work = nullptr;
	size_t work_bytes = 0;
};

void beam_free(BeamBuffers* b) {
	if (b) {
		for (void* p : b->owned) {
			HIP_CHECK(hipFree(p));
		}
		delete b;
	}
}

} // namespace

namespace calm {

// attention rows (fp32) as the fragment-major hi + lo matrix the output projection reads; eight values a thread
// grid = (ceil(n / 2048), rows)
__global__ __launch_bounds__(256) void k_beam_pack(const float* att, void* out, int n) {
	const int k = (blockIdx.x * 256 + threadIdx.x) * 8, t = blockIdx.y;
	if (k < n) {
		float v[8];
#pragma unroll
		for (int i = 0; i < 8; ++i) {
			v[i] = att[(size_t)t * n + k + i];
		}
		pf_store8(out, t, k, pf_steps(n), v);
	}
}

// rows [0, n) of an e5m2 cache layer [head][seq_len][dim] as binary16 [head][n][dim], exactly; four values a thread
// grid = (ceil(n * dim / 1024), heads, K and V)
__global__ __launch_bounds__(256) void k_beam_widen(const unsigned char* k, const unsigned char* v, unsigned short* out, int n, int seq_len, int dim) {
	const size_t i = ((size_t)blockIdx.x * 256 + threadIdx.x) * 4, per = (size_t)n * dim;
	if (i < per) {
		const unsigned w = *(const unsigned*)((blockIdx.z ? v : k) + (size_t)blockIdx.y * seq_len * dim + i);
		u32x2 r = {((w & 0xffu) << 8) | ((w & 0xff00u) << 16), ((w & 0xff0000u) >> 8) | (w & 0xff000000u)};
		*(u32x2*)(out + (blockIdx.z * (size_t)gridDim.y + blockIdx.y) * per + i) = r;
	}
}

} // namespace calm

extern "C" int decode_beam_hip(struct Transformer* t, int token, int pos, int n_steps, const struct BeamOptions* opt, int* out_tokens, float* out_scores) {
	Ctx* c = ctx_of(t);
	const struct Weights* w = &t->weights;
	KV_CHECK(opt && out_tokens && out_scores, "options or outputs are missing");
	const int W = opt->n_beams;
	KV_CHECK(W >= 1 && W <= BEAM_MAX, "1 to 32 beams");
	KV_CHECK(token >= 0 && token < c->vocab && opt->eos < c->vocab, "a token outside the vocabulary");
	KV_CHECK(n_steps >= 1 && pos >= 0 && pos < c->seq_len && n_steps <= c->seq_len - pos, "the steps do not fit the context window behind pos");
	KV_CHECK(opt->window >= 0 && opt->sinks >= 0, "a negative window or count of first tokens");
	KV_CHECK(c->head_dim == 64 || c->head_dim == 96 || c->head_dim == 128 || c->head_dim == 256, "head sizes 64, 96, 128 and 256");
	KV_CHECK(c->n_experts == 0 || c->n_active <= PF_MAX_ACTIVE, "more active experts than the batched layers handle");
	KV_CHECK(w->token_embedding_table && w->wcls && w->rms_final_weight, "the model lacks its embedding or its classifier");
	pf_alloc(c);
	const int L = c->n_layers, H = c->n_kv_heads, D = c->head_dim;
	const int mp = (pos + n_steps + KV_PAGE - 1) / KV_PAGE;
	// the prompt once; a hypothesis owns what lies behind its fork: the page that was not full then, the steps' pages
	const int pages = (pos + KV_PAGE - 1) / KV_PAGE + W * (n_steps / KV_PAGE + 2);
	BeamBuffers* b = c->beam;
	if (!b || b->pages < pages || b->cols < mp || b->steps < n_steps || b->beams < W) {
		HIP_CHECK(hipStreamSynchronize(g_stream));
		beam_free(b);
		b = c->beam = new BeamBuffers;
		b->pages = pages, b->cols = mp, b->steps = n_steps, b->beams = W;
		const auto mem = [&](size_t bytes) {
			void* p = dev_alloc(bytes);
			b->owned.push_back(p);
			return p;
		};
		const size_t codes = (size_t)L * pages * H * KV_PAGE * D, scales = (size_t)L * pages * H * 4 * sizeof(float);
		b->pool.k = (signed char*)mem(codes), b->pool.v = (signed char*)mem(codes);
		b->pool.k_scale = (float*)mem(scales), b->pool.v_scale = (float*)mem(scales);
		b->pool.status = (unsigned*)mem(sizeof(unsigned));
		b->ints = (int*)mem(((size_t)(n_steps + 4) * W + 2 * (W + 1) + 2 * (size_t)W * mp + pages) * sizeof(int));
		b->tok = (int*)mem((size_t)(n_steps + 1) * W * sizeof(int)), b->par = (int*)mem((size_t)(n_steps + 1) * W * sizeof(int));
		for (int i = 0; i < 2; ++i) {
			b->score[i] = (float*)mem(W * sizeof(float)), b->done[i] = (unsigned char*)mem(W);
		}
		b->att = (float*)mem((size_t)W * c->q_dim * sizeof(float)), b->logits = (float*)mem((size_t)W * c->vocab * sizeof(float));
		b->k = (__half*)mem((size_t)W * c->kv_dim * sizeof(__half)), b->v = (__half*)mem((size_t)W * c->kv_dim * sizeof(__half));
	}
	struct KvPool pool = b->pool;
	pool.n_layers = L, pool.n_pages = b->pages, pool.n_kv_heads = H, pool.head_dim = D;
	// lengths of step i: row i + 3 (row 0: zeros; row 1: the prompt in row 0 of the table; row 2 + i: pos + i everywhere)
	const auto lens = [&](int row) { return b->ints + (size_t)row * W; };
	int* const starts = lens(n_steps + 3);
	int* const starts0 = starts + W + 1;
	int* table[2] = {starts0 + W + 1, starts0 + W + 1 + (size_t)W * mp};
	int* const refs = table[1] + (size_t)W * mp;
	std::vector<int> up((size_t)(refs - b->ints) + b->pages, 0);
	const auto host = [&](const int* p) { return up.data() + (p - b->ints); };
	host(lens(1))[0] = pos;
	for (int i = 0; i <= n_steps; ++i) {
		for (int k = 0; k < W; ++k) {
			host(lens(2 + i))[k] = pos + i;
		}
	}
	for (int k = 0; k <= W; ++k) {
		host(starts)[k] = k, host(starts0)[k] = k ? pos : 0;
	}
	std::fill(host(table[0]), host(refs), -1);
	dev_copy_sync(b->ints, up.data(), up.size() * sizeof(int), hipMemcpyHostToDevice);
	std::vector<float> first(W, -INFINITY);
	first[0] = 0.f; // every hypothesis is the prompt: one of them counts
	dev_copy_sync(b->score[0], first.data(), W * sizeof(float), hipMemcpyHostToDevice);
	const std::vector<int> toks(W, token);
	dev_copy_sync(b->tok, toks.data(), W * sizeof(int), hipMemcpyHostToDevice);
	dev_zero(b->par, W * sizeof(int)); // parents of the first fork: row 0
	dev_zero(b->done[0], W);
	dev_zero(pool.status, sizeof(unsigned));
	// an activation beyond binary16's range raises this call's word (prefill.hip.h)
	memset(c->pf_flag, 0, PF_FLAG_WORDS * sizeof(unsigned));
	HIP_CHECK(hipMemcpyToSymbolAsync(HIP_SYMBOL(calm_pf_range_ptr), &c->pf_flag_ptr[0], sizeof(unsigned*), 0, hipMemcpyHostToDevice, g_stream));
	dev_zero(c->pf_tile_count, PF_SPLIT_TILES * sizeof(unsigned));
	struct KvBatch rows = {table[0], lens(3), starts, W, mp, W, 1, pos + n_steps};
	const long long att_work = kv_attend_workspace_hip(&pool, &rows, KV_F32, c->n_heads, opt->window, opt->sinks), sel_work = beam_workspace_hip(1, W, c->vocab);
	if (att_work < 0 || sel_work < 0) {
		return -1;
	}
	const size_t work = std::max((size_t)std::max(att_work, sel_work), (size_t)W * 2 * sizeof(int));
	if (work > b->work_bytes) {
		b->work = (char*)dev_alloc(work); // (an earlier, smaller one stays in `owned` until the buffers are replaced)
		b->owned.push_back(b->work);
		b->work_bytes = work;
	}
	// the prompt's rows out of the model's own cache
	if (pos > 0) {
		if (kv_reserve_hip(&pool, table[0], refs, lens(0), lens(1), W, mp, g_stream)) {
			return -1;
		}
		const struct KvBatch prompt = {table[0], lens(1), starts0, W, mp, pos, pos, pos};
		int bad = 0;
		for (int l = 0; l < L && !bad; ++l) {
			const char* const kc = (const char*)c->kc + (size_t)l * c->kv_layer_bytes;
			const char* const vc = (const char*)c->vc + (size_t)l * c->kv_layer_bytes;
			const void *k = kc, *v = vc;
			long head = (long)c->seq_len * D;
			if (c->kvbits == 8) {
				const size_t per = (size_t)pos * c->kv_dim;
				if (l == 0) {
					b->wide = (__half*)dev_alloc(2 * per * sizeof(__half));
				}
				hipLaunchKernelGGL(k_beam_widen, dim3((unsigned)(((size_t)pos * D + 1023) / 1024), H, 2), dim3(256), 0, g_stream, (const unsigned char*)kc, (const unsigned char*)vc,
				                   (unsigned short*)b->wide, pos, c->seq_len, D);
				k = b->wide, v = b->wide + per, head = (long)pos * D;
			}
			bad = kv_append_hip(&pool, &prompt, l, k, v, KV_F16, D, head, D, head, g_stream);
		}
		if (c->kvbits == 8) {
			HIP_CHECK(hipStreamSynchronize(g_stream));
			HIP_CHECK(hipFree(b->wide));
			b->wide = nullptr;
		}
		if (bad || kv_fork_hip(&pool, table[0], lens(1), refs, b->par, W, mp, table[1], refs, b->work, b->work_bytes, g_stream)) {
			return -1;
		}
		std::swap(table[0], table[1]);
	}
	int steps = 0, rc = 0;
	BatchStep st;
	st.k = b->k, st.v = b->v, st.logits = b->logits;
	st.attend = [&](int l) {
		const long head = (long)W * D;
		rc |= kv_append_hip(&pool, &rows, l, b->k, b->v, KV_F16, D, head, D, head, g_stream);
		rc |= kv_attend_hip(&pool, &rows, l, c->pf_q, b->att, KV_F32, c->n_heads, c->q_dim, D, 1.f / sqrtf((float)D), opt->window, opt->sinks, b->work, b->work_bytes, g_stream);
		hipLaunchKernelGGL(k_beam_pack, dim3((c->q_dim + 2047) / 2048, W), dim3(256), 0, g_stream, b->att, c->pf_att, c->q_dim);
	};
	for (; steps < n_steps && !rc; ++steps) {
		const int i = steps;
		rows.table = table[0], rows.lens = lens(3 + i);
		rc |= kv_reserve_hip(&pool, table[0], refs, lens(2 + i), lens(3 + i), W, mp, g_stream);
		st.tokens = b->tok + (size_t)i * W;
		switch (c->dbits) {
		case 16:
			prefill_chunk<16, 16>(c, W, pos + i, false, true, &st);
			break;
		case 8:
			prefill_chunk<8, 16>(c, W, pos + i, false, true, &st);
			break;
		default:
			prefill_chunk<4, 16>(c, W, pos + i, false, true, &st);
		}
		int* const par = b->par + (size_t)(i + 1) * W;
		rc |= beam_select_hip(b->logits, KV_F32, c->vocab, 1, W, c->vocab, b->score[i & 1], b->done[i & 1], opt->eos, b->score[(i + 1) & 1], par, b->tok + (size_t)(i + 1) * W,
		                      b->done[(i + 1) & 1], b->work, b->work_bytes, g_stream);
		rc |= kv_fork_hip(&pool, table[0], lens(3 + i), refs, par, W, mp, table[1], refs, b->work, b->work_bytes, g_stream);
		std::swap(table[0], table[1]);
		if (opt->window > 0) {
			rc |= kv_trim_hip(&pool, table[0], refs, lens(3 + i), W, mp, opt->window, opt->sinks, g_stream);
		}
		if (opt->eos >= 0 && i % 32 == 31) {
			unsigned char d[BEAM_MAX];
			dev_copy_sync(d, b->done[(i + 1) & 1], W, hipMemcpyDeviceToHost);
			if (std::all_of(d, d + W, [](unsigned char x) { return x != 0; })) {
				++steps;
				break;
			}
		}
	}
	if (rc) {
		return -1;
	}
	std::vector<int> tok((size_t)(steps + 1) * W), par((size_t)(steps + 1) * W);
	unsigned status = 0;
	dev_copy_sync(tok.data(), b->tok, tok.size() * sizeof(int), hipMemcpyDeviceToHost);
	dev_copy_sync(par.data(), b->par, par.size() * sizeof(int), hipMemcpyDeviceToHost);
	dev_copy_sync(out_scores, b->score[steps & 1], W * sizeof(float), hipMemcpyDeviceToHost);
	dev_copy_sync(&status, pool.status, sizeof(status), hipMemcpyDeviceToHost);
	KV_CHECK(status == 0, "the cache's pages do not add up");
	KV_CHECK(c->pf_flag[0] == 0, "an activation left the range of binary16 (beyond 65504, or NaN): the batched layers cannot carry it");
	for (int k = 0; k < W; ++k) {
		int at = k;
		for (int i = n_steps - 1; i >= 0; --i) {
			if (i >= steps) {
				out_tokens[(size_t)k * n_steps + i] = opt->eos; // all were finished
			} else {
				out_tokens[(size_t)k * n_steps + i] = tok[(size_t)(i + 1) * W + at];
				at = par[(size_t)(i + 1) * W + at];
			}
		}
	}
	return 0;
}
