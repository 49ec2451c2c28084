// attn_weights_tc.cuh -- the attention weight of many keys a CTA on tcgen05 (16-bit caches).
//
// S^T = K Q^T: 128 keys are the product's M, the query rows (up to 256) its N, so that a key's scores lie in
// one TMEM lane and its weight is one thread's sum over columns, with nothing to exchange. Units, shares and
// tiles as in tree_attn.cuh. Warps:
//   0-3  a key per thread: sum over the rows' columns of exp(scale s - lse); what the key had, and the result,
//        are one coalesced access each
//   4    MMA issue, into one of two TMEM score buffers (one for more than 128 rows of 128 dimensions)
//   5-8  fetching: the tile's keys through the page table into the operand layout (four stages), by TMA boxes
//        where the pages suit them (k_tree_attn_tc), and at a unit's beginning its q
// What bounds it: HBM while the rows are few (a tile's 32 KB take 1425 cycles of the measured rate), then the sums, some 20
// cycles a row and tile: 32 rows take as long as 1 (16 sequences of up to 16001 positions, us: 70 and 69; 64 rows 92, 120 rows 144, 256
// rows 271). Measured: windows of 32 tokens (64 rows) over those 93 us, 3.6 TB/s, pages of 24 like pages of 64. The exponent is taken
// from the difference (weight_of): s log2 e - lse log2 e, one product less, is off by 2e-4 of a weight with scores of 3200. Scores of
// 128 dimensions in one sum, whose last bits the tensor core drops, had 1.6 times the error of the form here; they took as
// long up to 128 rows and 252 us for 256. Every wait is bounded (tc.cuh).
#pragma once

#include "tree_attn_tc.cuh"

namespace tgc {

struct TwBars {
	uint64_t kfull[4], kfree[4], s_full[2], s_free[2], rows_full, done;
	uint32_t tmem;
	int abort;
	long long scan[16];
	float less[2][256];              // -lse, by the unit's parity
	unsigned long long mask[2][256]; // the drafted tokens a row counts for
};

constexpr int TW_ROWS = 256;

template <int DP> struct TwTile {
	static constexpr int TK = 128, NW = 9, THREADS = 32 * NW, NST = 4, CH = DP / 8;
	static constexpr int KB = 128 * DP * 2, K = TW_ROWS * DP * 2, BARS = K + NST * KB, SMEM = BARS + (int)sizeof(TwBars);
	static_assert(SMEM <= 232448, "shared memory of a CTA");
};

template <class T, int DP>
__global__ void __launch_bounds__(288, 1) k_attn_weights_tc(const WeightArgs p, const __grid_constant__ CUtensorMap kmap)
{
	using W = TwTile<DP>;
	constexpr int TK = W::TK, CH = W::CH, NST = W::NST, RI = 32 / CH;
	extern __shared__ __align__(1024) uint8_t ta_raw[];
	uint8_t *sm = ta_raw;
	TwBars *B = (TwBars *)(sm + W::BARS);
	const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
	if (smem_u32(sm) & 1023) { // the operand tiles need 1024-byte alignment
		if (tid == 0) p.c.report(PG_WAIT);
		return;
	}
	if (tid == 0) {
		for (int i = 0; i < NST; i++) mbar_init(&B->kfull[i], 128), mbar_init(&B->kfree[i], 1);
		for (int i = 0; i < 2; i++) mbar_init(&B->s_full[i], 1), mbar_init(&B->s_free[i], 4);
		mbar_init(&B->rows_full, 4), mbar_init(&B->done, 1);
		B->abort = 0;
		fence_barrier_init();
	}
	const int rows = p.d.tokens * p.d.group, cols = (rows + 31) & ~31, chunks = p.c.dim / 8;
	// a score of 128 dimensions is two sums of 64, `high` columns apart, added in f32 (see add4: a weight is an f32 output); where
	// they fill TMEM there is one buffer
	const int high = cols <= TW_ROWS / 2 ? TW_ROWS / 2 : TW_ROWS, bufs = DP > 64 && high == TW_ROWS ? 1 : 2;
	AttnCursor c;
	long long left_, pos, share;
	if (!attn_share<TK, W::NW>(p, B->scan, 1, c, left_, pos, share)) return; // the whole CTA
	const int left = (int)left_;
	if (warp == 4) tmem_alloc(&B->tmem, 512);
	tc_fence_before();
	__syncthreads();
	tc_fence_after();
	const uint32_t tmem = B->tmem;

	if (warp > 4) {
		// ---------------- fetching: rows part * 32 + lane of every tile ----------------
		const int part = warp - 5, ch = lane % CH;
		const uint32_t s0 = smem_u32(sm), x0 = (uint32_t)((ch & 7) ^ (lane / CH)) << 4;
		const uint32_t dk = s0 + W::K + (uint32_t)((ch >> 3) * 16384 + (part * 32 + lane / CH) * 128);
		const uint32_t dq = s0 + (uint32_t)((ch >> 3) * (TW_ROWS * 128) + (lane / CH) * 128);
		const bool piece = ch < chunks;
		int entry = 0, in_page = -1, last = -1;
		// by TMA, lane i has box i / (DP / 64) of its warp's 32 keys, and 64 of the dimensions; keys past the end are not looked at
		constexpr int ND = DP / 64;
		const int boxes = p.box.rows ? 32 / p.box.rows : 0;
		auto look = [&]() { // the table's entry of this lane's key or box
			const bool drafted = c.tile >= c.ctx, box = boxes && !drafted;
			const int x = (drafted ? 0 : c.tile * TK) + part * 32 + (box ? lane / ND * p.box.rows : lane);
			in_page = -1;
			if (drafted) {
				if (x < p.d.drafted(c.b)) in_page = x;
			} else if (x < c.n && !(box && lane >= boxes * ND)) {
				const int page = x / p.c.page;
				in_page = x - page * p.c.page;
				entry = p.c.table[(long long)c.b * p.c.cols + page];
			}
		};
		look();
		for (int j = 0; j < left; j++) {
			const bool drafted = c.tile >= c.ctx, begin = j == 0 || c.tile == 0, box = boxes && !drafted;
			const int sh = drafted ? 4 : p.c.shift, st = j % NST, kvh = c.h, page = entry;
			const char *base = (drafted ? p.d.k + (long long)c.b * p.d.kv_seq + c.h * p.d.kv_head : p.c.k + c.h * p.c.head_b) + ch * 16;
			const char *qb = p.d.q + (long long)c.b * p.d.q_seq + (long long)c.h * p.d.group * p.d.q_head + ch * 16;
			const uint32_t at = in_page < 0 ? PG_NONE : box ? (uint32_t)((unsigned)entry < (unsigned)p.c.pages ? in_page : (p.c.report(PG_PAGE), -1)) : drafted ? (uint32_t)(in_page * p.d.kv_tok >> 4) : p.c.at(entry, in_page);
			if (j + 1 < left) {
				cursor_next<TK>(p, c, 1);
				look();
			}
			if (j >= NST && !ta_wait(B, &B->kfree[st], (j / NST - 1) & 1, p.c)) break;
			last = j;
			if (box) {
				if (lane == 0) ta_expect(&B->kfull[st], 32 * DP * 2);
				__syncwarp();
				if (lane < boxes * ND) {
					const int r = at == PG_NONE ? 0 : (int)at, g = at == PG_NONE ? -1 : page; // -1: zeros
					ta_box(s0 + W::K + st * W::KB + lane % ND * 16384 + (part * 32 + lane / ND * p.box.rows) * 128, &kmap, &B->kfull[st], lane % ND * 64,
					       p.box.swap ? kvh : r, p.box.swap ? r : kvh, g);
				}
			} else
#pragma unroll 8
			for (int y = 0; y < CH; y++) {
				const uint32_t o = __shfl_sync(~0u, at, y * RI + lane / CH);
				const bool have = o != PG_NONE && piece;
				cp16(dk + st * W::KB + y * RI * 128 + (x0 ^ ((y * RI & 7) << 4)), base + ((unsigned long long)(have ? o : 0) << sh), have);
			}
			if (begin) { // the unit's q, once the last product of the unit before is done; past the rows zeros
				if (j > 0 && !ta_wait(B, &B->kfree[(j - 1) % NST], (j - 1) / NST & 1, p.c)) break;
				for (int r0 = part * 32; r0 < cols; r0 += 128) {
					const int r = r0 + lane, t = r / p.d.group;
					const uint32_t mine = r < rows ? (uint32_t)(((long long)t * p.d.q_tok + (long long)(r - t * p.d.group) * p.d.q_head) >> 4) : PG_NONE;
#pragma unroll 4
					for (int y = 0; y < CH; y++) {
						const uint32_t o = __shfl_sync(~0u, mine, y * RI + lane / CH);
						const bool have = o != PG_NONE && piece;
						cp16(dq + (r0 + y * RI) * 128 + (x0 ^ ((y * RI & 7) << 4)), qb + ((unsigned long long)(have ? o : 0) << 4), have);
					}
				}
			}
			cp_arrive(&B->kfull[st]);
		}
		cp_commit();
		cp_wait<0>();
		// boxes still on their way land before the CTA's shared memory is released
		for (int j = last > NST - 1 ? last - NST + 1 : 0; j <= last; j++) mbar_wait(&B->kfull[j % NST], j / NST & 1, nullptr, 0);
	} else if (warp == 4) {
		// ---------------- MMA issue ----------------
		if (lane == 0) {
			const uint32_t id = (1u << 4) | (std::is_same<T, __half>::value ? 0u : (1u << 7) | (1u << 10)) | ((uint32_t)(128 >> 4) << 24) | ((uint32_t)(cols >> 3) << 17);
			const uint32_t base = smem_u32(sm);
			for (int j = 0; j < left; j++) {
				if (j >= bufs && !ta_poll(B, &B->s_free[(j - bufs) & 1], ((j - bufs) >> 1) & 1, p.c)) break;
				if (!ta_poll(B, &B->kfull[j % NST], j / NST & 1, p.c)) break;
				fence_async_smem();
				tc_fence_after();
				const uint32_t k = base + W::K + j % NST * W::KB;
#pragma unroll
				for (int kk = 0; kk < DP / 16; kk++)
					tc_mma_f16(tmem + j % bufs * TW_ROWS + (kk >> 2) * high, sw128_kmajor_desc(k + (kk >> 2) * 16384 + (kk & 3) * 32),
						   sw128_kmajor_desc(base + (kk >> 2) * (TW_ROWS * 128) + (kk & 3) * 32), id, (kk & 3) > 0);
				tc_commit(&B->s_full[j & 1]);
				tc_commit(&B->kfree[j % NST]);
			}
			// every MMA issued has completed before TMEM is released (also after an abort)
			tc_commit(&B->done);
			mbar_wait(&B->done, 0, p.c.status + PG_WAIT, 1);
		}
		__syncwarp();
	} else {
		// ---------------- a key per thread ----------------
		const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
		int unit = -1;
		for (int j = 0; j < left; j++, cursor_next<TK>(p, c, 1)) {
			if (j == 0 || c.tile == 0) { // a unit's rows: their lse, and whom they count for
				unit++;
				const int cnt = p.d.drafted(c.b);
				const unsigned long long sel = p.select ? p.select[c.b] : ~0ull;
				for (int r = tid; r < cols; r += 128) {
					const int t = r / p.d.group;
					const bool on = r < rows && t < cnt && (sel >> t & 1);
					const float lse = on ? p.lse[((long long)c.b * p.d.tokens + t) * p.d.nq + c.h * p.d.group + r - t * p.d.group] : -INFINITY;
					B->less[unit & 1][r] = -lse;
					B->mask[unit & 1][r] = lse == -INFINITY ? 0 : p.d.sees(c.b, t, cnt);
				}
				mbar_arrive_warp(&B->rows_full);
				if (!ta_wait(B, &B->rows_full, unit & 1, p.c)) break;
			}
			const bool drafted = c.tile >= c.ctx;
			const int key = (drafted ? 0 : c.tile * TK) + tid, end = drafted ? p.d.drafted(c.b) : c.n;
			const long long head = (long long)c.b * p.c.nkv + c.h;
			const float had = !drafted && p.acc && key < end ? p.acc[c.b * p.acc_seq + c.h * p.acc_head + key] : 0;
			if (!ta_wait(B, &B->s_full[j & 1], (j >> 1) & 1, p.c)) break;
			tc_fence_after();
			float w[4] = {0, 0, 0, 0};
			for (int x = 0; x < cols; x += 32) {
				float v[32];
				tmem_ld32(lanes + j % bufs * TW_ROWS + x, v);
				if constexpr (DP > 64) {
					float u[32];
					tmem_ld32(lanes + j % bufs * TW_ROWS + high + x, u);
#pragma unroll
					for (int e = 0; e < 32; e += 2) {
						const float2 y = add2(make_float2(v[e], v[e + 1]), make_float2(u[e], u[e + 1]));
						v[e] = y.x, v[e + 1] = y.y;
					}
				}
				const float *less = &B->less[unit & 1][x];
				if (drafted) {
					const unsigned long long *mask = &B->mask[unit & 1][x];
#pragma unroll
					for (int e = 0; e < 32; e++) w[e & 3] += tid < 64 && mask[e] >> (tid & 63) & 1 ? weight_of(v[e], p.d.scale, -less[e]) : 0;
				} else {
#pragma unroll
					for (int e = 0; e < 32; e += 2) { // weight_of, two at a time
						const float2 l = *(const float2 *)(less + e), d = fma2(make_float2(v[e], v[e + 1]), make_float2(p.d.scale, p.d.scale), l);
						const float2 y = mul2(d, make_float2(1.4426950408889634f, 1.4426950408889634f));
						w[e & 3] += l.x != INFINITY ? ex2(y.x) : 0, w[e + 1 & 3] += l.y != INFINITY ? ex2(y.y) : 0;
					}
				}
			}
			tc_fence_before();
			mbar_arrive_warp(&B->s_free[j & 1]);
			const float sum = (w[0] + w[1]) + (w[2] + w[3]);
			if (drafted) {
				if (key < p.d.tokens) p.fresh[head * p.d.tokens + key] = key < end ? sum : 0;
				for (long long x = (long long)c.n + tid; x < p.c.max_len; x += 128) p.acc_out[head * p.c.max_len + x] = 0; // nothing is past the cache's end
			} else if (key < end) p.acc_out[head * p.c.max_len + key] = had + sum;
		}
	}
	tc_fence_before();
	__syncthreads();
	if (warp == 4) {
		tc_fence_after();
		tmem_dealloc(tmem, 512);
	}
}

} // namespace tgc
