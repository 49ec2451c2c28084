// paged.cuh -- what the kernels over a paged key/value cache share: its device view, the
// address of a row, the status word, element types and the host's checks of a description.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <array>
#include <atomic>

#include "common.cuh"

namespace tgc {

// What a paged-cache kernel can meet in device data, or a wait of its own that gave up: each has a word of its own in mapped host
// memory, set by a plain store (no read-modify-write over the bus) and cleared by the next call.
enum : int { PG_LEN, PG_PAGE, PG_PATH, PG_ROOM, PG_WAIT, PG_WORDS };

constexpr uint32_t PG_NONE = 0xffffffffu;

// A pool in bytes: positions are table lookups, so every offset is 64-bit.
struct PgCache {
	char *k, *v;
	const int *table, *len;
	long long page_b, head_b, pos_b; // strides in bytes
	int page, pages, cols, max_len, nkv, dim;
	int shift;                       // rows lie at multiples of 2^shift bytes (at least 16)
	int *status;                     // PG_WORDS words, written only on an error

	__device__ __forceinline__ void report(int what) const { *(volatile int *)(status + what) = 1; }
	__device__ __forceinline__ int length(int b) const
	{
		const int n = len[b];
		if (n < 0 || n > max_len) report(PG_LEN);
		return n < 0 ? 0 : n > max_len ? max_len : n;
	}
	// byte offset of a sequence's row (head 0) at position p, -1 where the page number is not one
	__device__ __forceinline__ long long row(const int *tab, int p) const
	{
		const int c = p / page;
		const uint32_t o = at(tab[c], p - c * page);
		return o == PG_NONE ? -1 : (long long)((unsigned long long)o << shift);
	}
	// the same in units of 2^shift bytes for row r of page number g, which the host has checked to fit 32 bits
	// in the whole pool, PG_NONE for none: half a register pair's price where lanes pass addresses on
	__device__ __forceinline__ uint32_t at(int g, int r) const
	{
		if ((unsigned)g >= (unsigned)pages) {
			report(PG_PAGE);
			return PG_NONE;
		}
		return (uint32_t)(((long long)g * page_b + (long long)r * pos_b) >> shift);
	}
};

struct PgDrafts {
	const char *q, *k, *v;
	long long q_seq, q_tok, q_head, kv_seq, kv_tok, kv_head; // bytes
	const unsigned long long *mask;
	const int *count;
	int tokens, nq, group;
	float scale;

	__device__ __forceinline__ int drafted(int b) const
	{
		const int n = count ? count[b] : tokens;
		return n < 0 ? 0 : n > tokens ? tokens : n;
	}
	// the drafted tokens that token t attends to, those past the count taken out
	__device__ __forceinline__ unsigned long long sees(int b, int t, int n) const
	{
		const unsigned long long live = n >= 64 ? ~0ull : (1ull << n) - 1;
		return (mask ? mask[(long long)b * tokens + t] : (2ull << t) - 1) & live;
	}
};

template <class T> struct PgElem;
template <> struct PgElem<float> {
	static __device__ __forceinline__ float get(float x) { return x; }
	static __device__ __forceinline__ float put(float x) { return x; }
	// whether a word of elements holds an infinity or a NaN
	static __device__ __forceinline__ bool odd(uint32_t w) { return (w & 0x7f800000u) == 0x7f800000u; }
};
template <> struct PgElem<__half> {
	static __device__ __forceinline__ float get(__half x) { return __half2float(x); }
	static __device__ __forceinline__ __half put(float x) { return __float2half_rn(x); }
	static __device__ __forceinline__ bool odd(uint32_t w) { return (w & 0x7c00u) == 0x7c00u || (w & 0x7c000000u) == 0x7c000000u; }
};
template <> struct PgElem<__nv_bfloat16> {
	static __device__ __forceinline__ float get(__nv_bfloat16 x) { return __bfloat162float(x); }
	static __device__ __forceinline__ __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
	static __device__ __forceinline__ bool odd(uint32_t w) { return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u; }
};

// Dynamic shared memory of a kernel, allowed once per device: `done` is the kernel's own set of devices.
template <class K> static inline int pg_smem(K kernel, int bytes, int dev, std::atomic<unsigned long long> &done)
{
	if (done.load(std::memory_order_acquire) >> dev & 1) return TG_CUDA_OK;
	TGC_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
	done.fetch_or(1ull << dev, std::memory_order_release);
	return TG_CUDA_OK;
}

// paged.cu: checks a description and fills the device view. `who` opens the error text.
int pg_cache(const char *who, const tg_cuda_kv *desc, PgCache *out);
enum { PG_USE_Q = 1, PG_USE_K = 2, PG_USE_V = 4 };
int pg_drafts(const char *who, const tg_cuda_kv *c, const tg_cuda_drafts *desc, int use, int most, PgDrafts *out);
// EINVAL where rows of `row` elements that a call writes overlap: they would be written in any order. They lie apart where each
// dimension's stride spans all of the dimensions of smaller strides.
int pg_apart(const char *who, const char *what, int row, std::array<long long, 3> stride, std::array<int, 3> n);
// The device's number and SM count, and the address of its status word; EDEVICE when a kernel
// of an earlier call reported something.
int pg_device(const char *who, int *sms, int **status);
int pg_sms(const char *who, int *dev, int *sms); // the current device and its SM count alone
// A TMA map of a pool of 16-bit elements, for boxes of 64 dimensions x as many rows of a page as `rows` and the page
// allow, 128-byte swizzle. Coordinates: dimension, then row and head (head and row with `swap`: TMA wants
// ascending strides), then page. False where the pages or strides do not suit boxes of whole 8-row atoms.
struct PgBox {
	int rows, swap;
};
bool pg_map(CUtensorMap *m, const PgCache &c, const void *pool, bool f16, int rows, PgBox *box);
static inline int pg_size(int type) { return type == TG_CUDA_F32 ? 4 : 2; }

} // namespace tgc
