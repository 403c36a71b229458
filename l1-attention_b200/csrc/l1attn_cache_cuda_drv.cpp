// pybind module l1attn_cache_cuda_drv: the 8-bit cache on torch tensors -- checks, allocation, device and stream; the arithmetic is
// behind the C ABI (l1attn_cache_*).
#include <c10/util/Optional.h>
#include "drv_common.h"

namespace {

using Maybe = c10::optional<torch::Tensor>;

// a cache's four tensors, of one layer or (layers) of several behind one another
l1attn_cache cache_of(const std::vector<torch::Tensor> &c, bool layers)
{
	const char *const names[] = {"k_codes", "v_codes", "k_scale", "v_scale"};
	TORCH_CHECK(c.size() == 4, "a cache is four tensors");
	for (int i = 0; i < 4; i++) {
		TORCH_CHECK(c[i].is_cuda(), names[i], " must be a CUDA tensor");
		TORCH_CHECK(c[i].scalar_type() == (i < 2 ? torch::kInt8 : torch::kFloat32) && c[i].is_contiguous() && c[i].device() == c[0].device(), names[i],
			    " must be a contiguous ", i < 2 ? "int8" : "float32", " tensor on the cache's device");
	}
	const int64_t d = c[0].dim();
	TORCH_CHECK((d == 4 || (layers && d == 5)) && c[1].dim() == d && c[0].sizes().slice(0, d - 1) == c[1].sizes().slice(0, d - 1) &&
			    c[2].sizes() == c[0].sizes().slice(0, d - 2) && c[3].sizes() == c[2].sizes(),
		    "a cache is k_codes [n_pages, hk, page, w], v_codes [n_pages, hk, page, wv], k_scale and v_scale [n_pages, hk]");
	const int64_t page = c[0].size(d - 2), pages = c[0].size(d - 4);
	TORCH_CHECK(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "page must be one of (16, 32, 64, 128, 256)");
	TORCH_CHECK(c[0].size(d - 1) >= 1 && c[0].size(d - 1) <= 256 && c[1].size(d - 1) >= 1 && c[1].size(d - 1) <= 256 && c[0].size(d - 3) >= 1,
		    "widths must be 1 to 256, and heads 1 or more");
	TORCH_CHECK(reinterpret_cast<uintptr_t>(c[0].data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(c[1].data_ptr()) % 16 == 0,
		    "k_codes and v_codes must be aligned to 16 bytes");
	TORCH_CHECK(pages <= INT32_MAX && c[0].size(d - 3) <= 65535, "pages must fit int32, heads 16 bits");
	l1attn_cache r = {};
	r.k_codes = c[0].data_ptr<int8_t>();
	r.v_codes = c[1].data_ptr<int8_t>();
	r.k_scale = c[2].data_ptr<float>();
	r.v_scale = c[3].data_ptr<float>();
	r.n_pages = int(pages);
	r.page = int(page);
	r.n_kv_heads = int(c[0].size(d - 3));
	r.width = int(c[0].size(d - 1));
	r.v_width = int(c[1].size(d - 1));
	return r;
}

int32_t *ints(const torch::Tensor &t, const char *name, const torch::Tensor &like)
{
	TORCH_CHECK(t.is_cuda() && t.scalar_type() == torch::kInt32 && t.device() == like.device() && t.is_contiguous(), name,
		    " must be a contiguous int32 tensor on the cache's device");
	return t.data_ptr<int32_t>();
}

int32_t *status_of(const Maybe &status, const torch::Tensor &like)
{
	if (!status.has_value() || !status->defined())
		return nullptr;
	int32_t *const p = ints(*status, "status", like);
	TORCH_CHECK(status->numel() >= 1, "status must be [1]");
	return p;
}

l1attn_cache places(const std::vector<torch::Tensor> &c, const torch::Tensor &table, const torch::Tensor &start, const torch::Tensor &cu, const Maybe &status)
{
	l1attn_cache r = cache_of(c, false);
	r.table = ints(table, "table", c[0]);
	r.start = ints(start, "start", c[0]);
	r.cu = ints(cu, "cu", c[0]);
	r.status = status_of(status, c[0]);
	TORCH_CHECK(table.dim() == 2 && start.dim() == 1 && start.size(0) == table.size(0) && cu.dim() == 1 && cu.size(0) == table.size(0) + 1,
		    "table must be [n_seqs, max_pages], start [n_seqs], cu [n_seqs + 1], status [1]");
	TORCH_CHECK(table.size(0) < INT32_MAX && table.size(1) * r.page <= 1 << 30, "max_pages * page must be 2^30 at most");
	r.n_seqs = int(table.size(0));
	r.max_pages = int(table.size(1));
	return r;
}

// rows of tokens; heads < 0: any
torch::Tensor tokens(const torch::Tensor &t, const char *name, const torch::Tensor &like, int64_t heads, int64_t width)
{
	TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, " must be a CUDA tensor on the cache's device");
	const auto type = t.scalar_type();
	TORCH_CHECK(type == torch::kFloat32 || type == torch::kFloat16 || type == torch::kBFloat16, name, " must be float32, float16 or bfloat16");
	TORCH_CHECK(t.dim() == 3 && t.size(2) == width && (heads < 0 || t.size(1) == heads) && t.size(0) <= INT32_MAX, name, " must be [rows, ", heads < 0 ? "heads" : std::to_string(heads),
		    ", ", std::to_string(width), "]");
	l1b_no_tangent(t, name);
	return t.stride(2) == 1 || width == 1 ? t : t.contiguous();
}

void append(torch::Tensor k, torch::Tensor v, std::vector<torch::Tensor> cache, torch::Tensor table, torch::Tensor start, torch::Tensor cu, Maybe status)
{
	const l1attn_cache c = places(cache, table, start, cu, status);
	k = tokens(k, "k", cache[0], c.n_kv_heads, c.width);
	v = tokens(v, "v", cache[0], c.n_kv_heads, c.v_width);
	TORCH_CHECK(k.scalar_type() == v.scalar_type() && k.size(0) == v.size(0), "k and v must share dtype and rows");
	const c10::cuda::CUDAGuard guard(k.device());
	const int64_t strides[] = {k.stride(0), k.stride(1), v.stride(0), v.stride(1)};
	l1b_status(l1attn_cache_append(&c, k.data_ptr(), v.data_ptr(), strides, int(k.size(0)), l1b_dtype(k, "append", true), l1b_stream()), "l1attn_cache_append");
}

std::vector<torch::Tensor> gather(std::vector<torch::Tensor> cache, torch::Tensor table, torch::Tensor start, torch::Tensor cu, int64_t rows, torch::ScalarType type, Maybe k_out,
				  Maybe v_out, Maybe status)
{
	const l1attn_cache c = places(cache, table, start, cu, status);
	TORCH_CHECK(type == torch::kFloat32 || type == torch::kFloat16 || type == torch::kBFloat16, "dtype must be float32, float16 or bfloat16");
	TORCH_CHECK(rows >= 0 && rows <= INT32_MAX, "rows must fit int32");
	const c10::cuda::CUDAGuard guard(cache[0].device());
	const auto options = cache[2].options().dtype(type).requires_grad(false);
	std::vector<torch::Tensor> out;
	for (int i = 0; i < 2; i++) {
		const Maybe &given = i ? v_out : k_out;
		const std::vector<int64_t> shape = {rows, c.n_kv_heads, i ? c.v_width : c.width};
		if (given.has_value()) {
			TORCH_CHECK(given->sizes() == at::IntArrayRef(shape) && given->scalar_type() == type && given->device() == cache[0].device() && given->is_contiguous(),
				    "out must be contiguous ", type, " tensors of the right shapes on the cache's device");
			out.push_back(*given);
		} else
			out.push_back(torch::empty(shape, options));
	}
	l1b_status(l1attn_cache_gather(&c, out[0].data_ptr(), out[1].data_ptr(), int(rows), l1b_dtype(out[0], "gather", true), l1b_stream()), "l1attn_cache_gather");
	return out;
}

torch::Tensor attend(torch::Tensor q, std::vector<torch::Tensor> cache, torch::Tensor table, torch::Tensor start, torch::Tensor cu, int mode, int64_t window, double softcap,
		     Maybe slopes, int64_t max_len, Maybe given, Maybe status)
{
	const l1attn_cache c = places(cache, table, start, cu, status);
	q = tokens(q, "q", cache[0], -1, c.width);
	const int64_t h = q.size(1);
	TORCH_CHECK(h >= 1 && h % c.n_kv_heads == 0 && q.size(0) * h <= INT32_MAX, "the heads of q must be a multiple of the cache's");
	torch::Tensor sl;
	if (slopes.has_value() && slopes->defined()) {
		TORCH_CHECK(slopes->scalar_type() == torch::kFloat32 && slopes->dim() == 1 && slopes->size(0) == h && slopes->device() == q.device(),
			    "slopes must be a float32 tensor of shape ", l1b_shape({h}), " on the device of q");
		TORCH_CHECK(!(at::GradMode::is_enabled() && slopes->requires_grad()), "slopes is a constant: it must not require a gradient");
		l1b_no_tangent(*slopes, "slopes");
		sl = slopes->contiguous();
	}
	const c10::cuda::CUDAGuard guard(q.device());
	torch::Tensor vo;
	if (given.has_value()) {
		vo = *given;
		TORCH_CHECK(vo.dim() == 3 && vo.size(0) == q.size(0) && vo.size(1) == h && vo.size(2) == c.v_width && vo.scalar_type() == q.scalar_type() && vo.device() == q.device() &&
				    vo.is_contiguous(),
			    "out must be a contiguous tensor [rows, heads, v_width] of the type of q on its device");
		// (rows of q are read while others are written)
		const char *const q0 = static_cast<const char *>(q.data_ptr()), *const v0 = static_cast<const char *>(vo.data_ptr());
		const int64_t q_span = q.numel() ? ((q.size(0) - 1) * q.stride(0) + (h - 1) * q.stride(1) + c.width) * q.element_size() : 0;
		TORCH_CHECK(v0 + vo.nbytes() <= q0 || q0 + q_span <= v0 || !vo.numel() || !q_span, "out must not overlap q");
	} else
		vo = torch::empty({q.size(0), h, c.v_width}, q.options().requires_grad(false));
	const int rows = int(q.size(0)), type = l1b_dtype(q, "attend", true);
	const int64_t room = int64_t(c.max_pages) * c.page;
	const int longest = int(max_len < 0 || max_len > room ? room : max_len);
	const size_t bytes = l1attn_cache_attend_bytes(&c, rows, int(h), longest, type);
	const auto work = bytes ? torch::empty({int64_t(bytes)}, q.options().dtype(torch::kUInt8).requires_grad(false)) : torch::Tensor();
	const l1attn_mask mask = {1, int(window), mode, float(softcap), sl.defined() ? sl.data_ptr<float>() : nullptr, nullptr, nullptr};
	const int64_t strides[] = {q.stride(0), q.stride(1)};
	l1b_status(l1attn_cache_attend(&c, q.data_ptr(), strides, vo.data_ptr(), bytes ? work.data_ptr() : nullptr, rows, int(h), longest, &mask, type, l1b_stream()),
		   "l1attn_cache_attend");
	return vo;
}

void copy_pages(std::vector<torch::Tensor> cache, torch::Tensor src, torch::Tensor dst, Maybe status)
{
	l1attn_cache c = cache_of(cache, true);
	c.status = status_of(status, cache[0]);
	const int32_t *const s = ints(src, "src", cache[0]), *const d = ints(dst, "dst", cache[0]);
	TORCH_CHECK(src.dim() == 1 && src.sizes() == dst.sizes() && src.size(0) <= INT32_MAX, "src and dst must be contiguous int32 tensors of one length on the cache's device");
	const int64_t layers = cache[0].dim() == 5 ? cache[0].size(0) : 1;
	TORCH_CHECK(layers <= 32767, "too many layers");
	const c10::cuda::CUDAGuard guard(cache[0].device());
	l1b_status(l1attn_cache_copy_pages(&c, int(layers), s, d, int(src.size(0)), l1b_stream()), "l1attn_cache_copy_pages");
}

} // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
	m.def("append", &append, "quantise tokens into pages (CUDA, sm_100a)");
	m.def("gather", &gather, "read sequences back (CUDA, sm_100a)");
	m.def("attend", &attend, "L1 attention to a paged 8-bit cache (CUDA, sm_100a)");
	m.def("copy_pages", &copy_pages, "copy pages (CUDA, sm_100a)");
}
