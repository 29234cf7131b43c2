// kh_paged.hip - the paged cache's operators on the host side: checks, the C
// entries, the launches of a plan, and their meaning on the CPU.
#include <algorithm>
#include <cmath>
#include <exception>
#include <limits>
#include <vector>

#include "kh_paged.hpp"

namespace kh {

int abi_fail(int code, const std::string &msg);   // kh_plan.hip: sets kh_last_error
hipError_t launch_append(const kh_cache_append_op &a, hipStream_t stream);
void host_append(const kh_cache_append_op &a);
hipError_t launch_copy(const kh_pool *pools, int n_pools, const int32_t *source, const int32_t *target, int n,
                       hipStream_t stream);

namespace {

bool type_ok(int t) { return t == KH_TYPE_F32 || t == KH_TYPE_BF16 || t == KH_TYPE_F16; }

bool page_size_ok(int n) { return n >= 16 && n <= 1024 && (n & (n - 1)) == 0; }

// Rows of `bytes`-byte elements that start at multiples of 16 bytes.
bool aligned_strides(std::initializer_list<int64_t> strides, int bytes) {
  for (int64_t s : strides)
    if (s * bytes % 16) return false;
  return true;
}

}  // namespace

bool check_paged(const kh_paged &p, std::string &err, bool &unsupported) {
  unsupported = false;
  if (p.variant != KH_PAGED_ATTENTION && p.variant != KH_PAGED_SELECT) {
    err = "unknown paged operator";
    return false;
  }
  if (p.batch < 0 || p.draft < 0 || p.heads < 1 || p.kv_heads < 1 || p.dim < 1 || p.pages < 1 || p.width < 0 || p.top < 0) {
    err = "bad sizes";
    return false;
  }
  if (p.heads % p.kv_heads) {
    err = "heads must be a multiple of kv_heads";
    return false;
  }
  if (!type_ok(p.cache_type) || !type_ok(p.act_type)) {
    err = "unknown element type";
    return false;
  }
  unsupported = true;
  if (p.dim % 8 || p.dim > 256) {
    err = "head dimension " + std::to_string(p.dim) + " (multiples of 8 up to 256 have kernels)";
    return false;
  }
  if (!page_size_ok(p.page_size)) {
    err = "page size " + std::to_string(p.page_size) + " (powers of two from 16 to 1024 have kernels)";
    return false;
  }
  if (p.draft > kMaxDraft) {
    err = std::to_string(p.draft) + " new tokens of a sequence (at most " + std::to_string(kMaxDraft) + ")";
    return false;
  }
  if (p.batch > kMaxBatch) {
    err = std::to_string(p.batch) + " sequences (at most " + std::to_string(kMaxBatch) + ")";
    return false;
  }
  if (p.variant == KH_PAGED_ATTENTION && p.act_type != KH_TYPE_F32 && p.act_type != p.cache_type) {
    err = "activations are fp32 or of the cache's type";
    return false;
  }
  const int64_t most = std::numeric_limits<int32_t>::max();
  const int64_t keys = (int64_t)p.width * p.page_size;
  // (a length and a tile's keys are added in 32 bits)
  if (keys > most - std::max(kPagedTile, kWideTile) || (keys / 32 + 9) * std::max(p.batch, 1) > most || (int64_t)p.top * p.page_size > most ||
      (int64_t)p.batch * p.draft * p.heads > most / 2 || p.top > (1 << 20)) {
    err = "more keys or query rows than 32-bit counts hold";
    return false;
  }
  if (p.pages >= 1 << 27) {
    err = "a pool of 2^27 pages or more";
    return false;
  }
  // (every query row of a token in a block of its own at the worst)
  const int64_t tiles = (std::max(keys, p.top ? (int64_t)p.top * p.page_size : 0) / 32 + 10) * std::max(p.batch, 1);
  if (p.variant == KH_PAGED_ATTENTION && tiles * p.kv_heads > most / (((int64_t)p.draft * (p.heads / p.kv_heads) + 15) / 16 + p.draft)) {
    err = "more keys and query rows than 32-bit counts hold";
    return false;
  }
  if (p.variant == KH_PAGED_ATTENTION && paged_threads(p) > (int64_t)std::numeric_limits<uint32_t>::max()) {
    err = "more sequences, heads and tokens than one launch has room for (2^32 work items)";
    return false;
  }
  if (p.variant == KH_PAGED_ATTENTION && (p.kp_t > most / 8 / p.page_size - p.dim || p.vp_t > most / 8 / p.page_size - p.dim)) {
    err = "the pages' token stride is too large";
    return false;
  }
  if (p.variant == KH_PAGED_ATTENTION && (p.k_n > most / 512 || p.v_n > most / 512)) {
    err = "the new tokens' stride is too large";
    return false;
  }
  if (p.variant == KH_PAGED_SELECT &&
      ((int64_t)p.batch * p.kv_heads > 65535 || (p.width + 63) / 64 > (1 << 24))) {
    err = "more than 65535 (sequence, kv head) pairs";
    return false;
  }
  unsupported = false;
  const int ab = type_bytes(p.act_type), cb = type_bytes(p.cache_type);
  if (!aligned_strides({p.q_s, p.q_n, p.q_h}, ab)) {
    err = "q: rows must start at multiples of 16 bytes";
    return false;
  }
  if (p.variant == KH_PAGED_SELECT) {
    if (!aligned_strides({p.m_p, p.m_h}, 4)) {
      err = "k_means: rows must start at multiples of 16 bytes";
      return false;
    }
    return true;
  }
  // (row offsets inside a tile are unsigned 32-bit counts)
  if (p.kp_t < 0 || p.vp_t < 0) {
    err = "negative token stride of the pages";
    return false;
  }
  if (p.k_n < 0 || p.v_n < 0) {
    err = "negative token stride of the new tokens";
    return false;
  }
  if (!aligned_strides({p.k_s, p.k_n, p.k_h, p.v_s, p.v_n, p.v_h, p.o_s, p.o_n, p.o_h}, ab)) {
    err = "k, v, out: rows must start at multiples of 16 bytes";
    return false;
  }
  if (!aligned_strides({p.kp_p, p.kp_h, p.kp_t, p.vp_p, p.vp_h, p.vp_t}, cb)) {
    err = "pages: rows must start at multiples of 16 bytes";
    return false;
  }
  return true;
}

bool check_paged_pointers(const kh_paged &p, std::string &err) {
  auto row = [&](const void *x, const char *what) {
    if (x != nullptr && (uintptr_t)x % 16 == 0) return true;
    err = std::string(what) + (x ? ": not 16-byte aligned" : ": null pointer");
    return false;
  };
  auto word = [&](const void *x, const char *what) {
    if (x != nullptr && (uintptr_t)x % 4 == 0) return true;
    err = std::string(what) + (x ? ": not 4-byte aligned" : ": null pointer");
    return false;
  };
  if (p.batch == 0 || p.draft == 0) return true;
  if (!row(p.q, "q") || !word(p.lengths, "lengths") || (p.width > 0 && !word(p.table, "table"))) return false;
  if (p.variant == KH_PAGED_SELECT)
    return p.top == 0 || ((p.width == 0 || row(p.k_means, "k_means")) && word(p.selected, "selected"));
  return row(p.k, "k") && row(p.v, "v") && row(p.k_pages, "k_pages") && row(p.v_pages, "v_pages") && row(p.out, "out") &&
         (p.parents == nullptr || word(p.parents, "parents")) && (p.top == 0 || word(p.selected, "selected"));
}

// -- as launches of a plan ---------------------------------------------------------

kh_paged paged_of_launch(const kh_launch &L) {
  kh_paged p = {};
  p.variant = L.variant;
  p.batch = (int)L.shape[0];
  p.draft = (int)L.shape[1];
  p.heads = (int)L.shape[2];
  p.kv_heads = (int)L.shape[3];
  p.dim = (int)L.shape[4];
  p.page_size = (int)L.shape[5];
  p.pages = (int)L.gemm[0];
  p.width = (int)L.gemm[1];
  p.top = (int)L.gemm[2];
  p.cache_type = L.cfg[0];
  p.act_type = L.cfg[1];
  p.one_pass = L.cfg[2];
  p.scale = L.fparams[0];
  auto strides = [&](int j, std::initializer_list<int64_t *> to) {
    int i = 0;
    for (int64_t *s : to) *s = L.refs[j].strides[i++];
  };
  strides(0, {&p.q_s, &p.q_n, &p.q_h});
  if (L.variant == KH_PAGED_SELECT) {
    strides(1, {&p.m_p, &p.m_h});
    strides(2, {&p.table_s});
    strides(4, {&p.sel_s, &p.sel_n, &p.sel_h});
    return p;
  }
  strides(1, {&p.k_s, &p.k_n, &p.k_h});
  strides(2, {&p.v_s, &p.v_n, &p.v_h});
  strides(3, {&p.kp_p, &p.kp_h, &p.kp_t});
  strides(4, {&p.vp_p, &p.vp_h, &p.vp_t});
  strides(5, {&p.table_s});
  strides(7, {&p.o_s, &p.o_n, &p.o_h});
  if (L.cfg[3]) strides(L.cfg[3], {&p.parents_s});
  if (L.cfg[4]) strides(L.cfg[4], {&p.sel_s, &p.sel_n, &p.sel_h});
  return p;
}

void patch_paged(kh_paged &p, const kh_launch &L, float *const *ptrs) {
  auto ints = [&](int j) { return reinterpret_cast<int32_t *>(ptrs[j]); };
  p.q = ptrs[0];
  if (L.variant == KH_PAGED_SELECT) {
    p.k_means = ptrs[1];
    p.table = ints(2);
    p.lengths = ints(3);
    p.selected = ints(4);
    return;
  }
  p.k = ptrs[1];
  p.v = ptrs[2];
  p.k_pages = ptrs[3];
  p.v_pages = ptrs[4];
  p.table = ints(5);
  p.lengths = ints(6);
  p.out = ptrs[7];
  p.parents = L.cfg[3] ? ints(L.cfg[3]) : nullptr;
  p.selected = L.cfg[4] ? ints(L.cfg[4]) : nullptr;
}

int paged_ref_bytes(const kh_launch &L, int j) {
  if (L.variant == KH_PAGED_SELECT) return j == 0 ? type_bytes(L.cfg[1]) : 4;
  if (j == 3 || j == 4) return type_bytes(L.cfg[0]);
  return j <= 2 || j == 7 ? type_bytes(L.cfg[1]) : 4;
}

namespace {

size_t workspace_floats(const kh_paged &p) {
  if (p.batch == 0 || p.draft == 0) return 0;
  return p.variant == KH_PAGED_SELECT ? select_workspace_floats(p) : paged_workspace_floats(p);
}

class PagedOp : public Op {
 public:
  explicit PagedOp(const kh_launch &L) : launch_(L), p_(paged_of_launch(L)) {}
  hipError_t launch(float *const *ptrs, float *partials, hipStream_t stream) override {
    kh_paged p = p_;
    patch_paged(p, launch_, ptrs);
    std::string err;
    if (!check_paged_pointers(p, err)) return hipErrorInvalidValue;
    return p.variant == KH_PAGED_SELECT ? launch_select(p, partials, stream) : launch_paged(p, partials, stream);
  }
  size_t partial_floats() const override { return workspace_floats(p_); }

 private:
  kh_launch launch_;
  kh_paged p_;
};

}  // namespace

std::unique_ptr<Op> make_paged(const kh_launch &L, std::string &err, bool &unsupported) {
  const bool select = L.variant == KH_PAGED_SELECT;
  for (int i = 0; i < 6; ++i)
    if (L.shape[i] < 0 || L.shape[i] > std::numeric_limits<int32_t>::max()) err = "bad sizes";
  for (int i = 0; i < 3; ++i)
    if (L.gemm[i] < 0 || L.gemm[i] > std::numeric_limits<int32_t>::max()) err = "bad sizes";
  const int refs = select ? 5 : 8;
  if (!select && L.variant != KH_PAGED_ATTENTION) err = "unknown paged operator";
  else if (L.n_refs < refs) err = "missing operands";
  if (!select)
    for (int i = 3; i <= 4; ++i)
      if (L.cfg[i] != 0 && (L.cfg[i] < refs || L.cfg[i] >= L.n_refs)) err = "an optional operand's index is out of range";
  if (!select && err.empty() && (L.gemm[2] > 0) != (L.cfg[4] != 0)) err = "picked pages need their operand and their number";
  if (!err.empty()) return nullptr;
  if (!check_paged(paged_of_launch(L), err, unsupported)) return nullptr;
  return std::make_unique<PagedOp>(L);
}

// -- the operators' meaning on the CPU ------------------------------------------------

namespace {

double value(const void *p, int64_t i, int type) {
  if (type == KH_TYPE_F32) return static_cast<const float *>(p)[i];
  if (type == KH_TYPE_BF16) return (double)(float)static_cast<const __bf16 *>(p)[i];
  return (double)(float)static_cast<const _Float16 *>(p)[i];
}

double rounded(double x, int type) {
  if (type == KH_TYPE_F32) return x;
  if (type == KH_TYPE_BF16) return (double)(float)(__bf16)(float)x;
  return (double)(float)(_Float16)(float)x;
}

int64_t length_of(const kh_paged &p, int s) {
  return std::min<int64_t>(std::max<int64_t>(p.lengths[s], 0), (int64_t)p.width * p.page_size);
}

void host_select(const kh_paged &p) {
  const int group = p.heads / p.kv_heads;
  std::vector<double> score;
  std::vector<int> order;
  for (int s = 0; s < p.batch; ++s) {
    const int held = (int)((length_of(p, s) + p.page_size - 1) / p.page_size);
    for (int n = 0; n < p.draft; ++n)
      for (int c = 0; c < p.kv_heads; ++c) {
        score.assign((size_t)held, 0.0);
        order.resize((size_t)held);
        for (int b = 0; b < held; ++b) {
          order[(size_t)b] = b;
          const int page = p.table[s * p.table_s + b];
          if (page < 0 || page >= p.pages) continue;
          for (int d = 0; d < p.dim; ++d) {
            double q = 0.0;
            for (int h = 0; h < group; ++h)
              q += value(p.q, s * p.q_s + n * p.q_n + (int64_t)(c * group + h) * p.q_h + d, p.act_type);
            score[(size_t)b] += q * (double)p.k_means[page * p.m_p + c * p.m_h + d];
          }
        }
        auto better = [&](int x, int y) {
          if ((x == held - 1) != (y == held - 1)) return x == held - 1;
          const double a = score[(size_t)x], b = score[(size_t)y];
          if (std::isnan(a) != std::isnan(b)) return std::isnan(b);
          if (!std::isnan(a) && a != b) return a > b;
          return x < y;
        };
        std::sort(order.begin(), order.end(), better);
        const int take = std::min(held, p.top);
        std::sort(order.begin(), order.begin() + take);
        int32_t *out = p.selected + s * p.sel_s + n * p.sel_n + c * p.sel_h;
        for (int i = 0; i < p.top; ++i) out[i] = i < take ? order[(size_t)i] : -1;
      }
  }
}

void host_attention(const kh_paged &p) {
  const int group = p.heads / p.kv_heads;
  std::vector<double> q((size_t)p.dim), out((size_t)p.dim), score;
  std::vector<std::vector<double>> keys, values;
  for (int s = 0; s < p.batch; ++s) {
    const int64_t len = length_of(p, s);
    for (int n = 0; n < p.draft; ++n) {
      // the token's own path, or none where it is unused
      std::vector<int> path;
      bool used = true;
      for (int i = n; i >= 0;) {
        path.push_back(i);
        const int from = p.parents ? p.parents[s * p.parents_s + i] : i - 1;
        if (from < -1 || from >= i) {
          used = false;
          break;
        }
        i = from;
      }
      std::sort(path.begin(), path.end());
      for (int c = 0; c < p.kv_heads; ++c) {
        keys.clear();
        values.clear();
        auto cached = [&](int64_t col) {
          const int page = p.table[s * p.table_s + col];
          if (page < 0 || page >= p.pages) return;
          for (int64_t pos = col * p.page_size; pos < std::min(len, (col + 1) * p.page_size); ++pos) {
            keys.emplace_back();
            values.emplace_back();
            for (int d = 0; d < p.dim; ++d) {
              const int64_t slot = pos - col * p.page_size;
              keys.back().push_back(value(p.k_pages, page * p.kp_p + c * p.kp_h + slot * p.kp_t + d, p.cache_type));
              values.back().push_back(value(p.v_pages, page * p.vp_p + c * p.vp_h + slot * p.vp_t + d, p.cache_type));
            }
          }
        };
        if (p.top) {
          const int32_t *list = p.selected + s * p.sel_s + n * p.sel_n + c * p.sel_h;
          for (int i = 0; i < p.top; ++i)
            if (list[i] > (i ? list[i - 1] : -1) && list[i] >= 0 && list[i] < p.width) cached(list[i]);
        } else {
          for (int64_t col = 0; col * p.page_size < len; ++col) cached(col);
        }
        for (int i : path) {
          keys.emplace_back();
          values.emplace_back();
          for (int d = 0; d < p.dim; ++d) {
            keys.back().push_back(rounded(value(p.k, s * p.k_s + i * p.k_n + c * p.k_h + d, p.act_type), p.cache_type));
            values.back().push_back(rounded(value(p.v, s * p.v_s + i * p.v_n + c * p.v_h + d, p.act_type), p.cache_type));
          }
        }
        for (int h = c * group; h < (c + 1) * group; ++h) {
          std::fill(out.begin(), out.end(), 0.0);
          if (used) {
            for (int d = 0; d < p.dim; ++d) {
              q[(size_t)d] = value(p.q, s * p.q_s + n * p.q_n + h * p.q_h + d, p.act_type);
              if (p.one_pass) q[(size_t)d] = rounded(q[(size_t)d], p.cache_type);
            }
            double most = -INFINITY, total = 0.0;
            score.assign(keys.size(), 0.0);
            for (size_t j = 0; j < keys.size(); ++j) {
              for (int d = 0; d < p.dim; ++d) score[j] += q[(size_t)d] * keys[j][(size_t)d];
              score[j] *= p.scale;
              most = std::fmax(most, score[j]);
            }
            for (size_t j = 0; j < keys.size(); ++j) {
              const double e = std::exp(score[j] - most);
              total += e;
              for (int d = 0; d < p.dim; ++d) out[(size_t)d] += e * values[j][(size_t)d];
            }
            for (int d = 0; d < p.dim; ++d) out[(size_t)d] /= total;
          }
          for (int d = 0; d < p.dim; ++d) {
            const int64_t at = s * p.o_s + n * p.o_n + h * p.o_h + d;
            if (p.act_type == KH_TYPE_F32) static_cast<float *>(p.out)[at] = (float)out[(size_t)d];
            else if (p.act_type == KH_TYPE_BF16) static_cast<__bf16 *>(p.out)[at] = (__bf16)(float)out[(size_t)d];
            else static_cast<_Float16 *>(p.out)[at] = (_Float16)(float)out[(size_t)d];
          }
        }
      }
    }
  }
}

}  // namespace

void host_paged(const kh_paged &p) {
  if (p.variant == KH_PAGED_SELECT) host_select(p);
  else host_attention(p);
}

void host_paged_launch(const kh_launch &L, float *const *ptrs) {
  kh_paged p = paged_of_launch(L);
  patch_paged(p, L, ptrs);
  host_paged(p);
}

// -- checks of append and copy ----------------------------------------------------------

namespace {

int check_append(const kh_cache_append_op *a) {
  if (!a) return abi_fail(KH_ERR_INVALID, "null argument");
  if (a->layers < 0 || a->batch < 0 || a->draft < 0 || a->accept < 0 || a->kv_heads < 1 || a->dim < 1 || a->pages < 1 ||
      a->width < 0 || !type_ok(a->cache_type) || !type_ok(a->act_type))
    return abi_fail(KH_ERR_INVALID, "bad sizes or types");
  if (!a->rows && a->accept > a->draft) return abi_fail(KH_ERR_INVALID, "more tokens to append than there are");
  if (a->dim % 8 || a->dim > 256)
    return abi_fail(KH_ERR_UNSUPPORTED, "head dimension " + std::to_string(a->dim) + " (multiples of 8 up to 256 have kernels)");
  if (!page_size_ok(a->page_size))
    return abi_fail(KH_ERR_UNSUPPORTED, "page size " + std::to_string(a->page_size) + " (powers of two from 16 to 1024 have kernels)");
  if ((int64_t)a->batch * a->kv_heads > 65535 || a->layers > 65535)
    return abi_fail(KH_ERR_UNSUPPORTED, "more than 65535 (sequence, kv head) pairs or layers");
  const int ab = type_bytes(a->act_type), cb = type_bytes(a->cache_type);
  if (!aligned_strides({a->k_l, a->k_s, a->k_n, a->k_h, a->v_l, a->v_s, a->v_n, a->v_h}, ab) ||
      !aligned_strides({a->kp_l, a->kp_p, a->kp_h, a->kp_t, a->vp_l, a->vp_p, a->vp_h, a->vp_t}, cb))
    return abi_fail(KH_ERR_INVALID, "rows must start at multiples of 16 bytes");
  if (!a->layers || !a->batch || !a->accept) return KH_OK;
  auto odd = [](const void *x, int n) { return x == nullptr || (uintptr_t)x % n; };
  if (odd(a->k, 16) || odd(a->v, 16) || odd(a->k_pages, 16) || odd(a->v_pages, 16) || odd(a->lengths, 4) ||
      (a->width > 0 && odd(a->table, 4)) || (a->rows && odd(a->rows, 4)) || (a->k_means && odd(a->k_means, 4)))
    return abi_fail(KH_ERR_INVALID, "a null or unaligned pointer");
  return KH_OK;
}

int check_copy(const kh_pool *pools, int n_pools, int32_t pages, const int32_t *source, const int32_t *target, int n) {
  if (n < 0 || pages < 0 || n_pools < 0 || (n_pools > 0 && !pools) || (n > 0 && (!source || !target)))
    return abi_fail(KH_ERR_INVALID, "bad arguments");
  if (n_pools > KH_MAX_POOLS) return abi_fail(KH_ERR_UNSUPPORTED, "more than " + std::to_string(KH_MAX_POOLS) + " pools");
  int64_t layers = 0;
  for (int i = 0; i < n_pools; ++i) {
    const kh_pool &p = pools[i];
    if (p.layers < 0 || p.page_bytes < 0 || p.page_bytes % 4 || p.layer_bytes % 4 || (uintptr_t)p.base % 4 || (!p.base && n > 0))
      return abi_fail(KH_ERR_INVALID, "a pool's address or sizes");
    layers += p.layers;
  }
  if (layers > 65535) return abi_fail(KH_ERR_UNSUPPORTED, "more than 65535 layers");
  std::vector<uint8_t> role((size_t)pages, 0);   // 1: a source, 2: a target
  for (int i = 0; i < n; ++i) {
    if (source[i] < 0 || source[i] >= pages || target[i] < 0 || target[i] >= pages)
      return abi_fail(KH_ERR_INVALID, "page " + std::to_string(i) + " of the lists is outside the pool");
    role[(size_t)source[i]] |= 1;
  }
  for (int i = 0; i < n; ++i) {
    if (role[(size_t)target[i]])
      return abi_fail(KH_ERR_INVALID, "page " + std::to_string(target[i]) + " is a target twice, or a source too");
    role[(size_t)target[i]] = 2;
  }
  return KH_OK;
}

// No C++ exception leaves a C entry.
template <class F>
int guarded(F &&f) {
  try {
    return f();
  } catch (const std::bad_alloc &) {
    return abi_fail(KH_ERR_CAPACITY, "out of host memory");
  } catch (const std::exception &e) {
    return abi_fail(KH_ERR_INVALID, e.what());
  }
}

int check_run(const kh_paged *op) {
  if (!op) return abi_fail(KH_ERR_INVALID, "null argument");
  std::string err;
  bool unsupported = false;
  if (!check_paged(*op, err, unsupported)) return abi_fail(unsupported ? KH_ERR_UNSUPPORTED : KH_ERR_INVALID, err);
  if (!check_paged_pointers(*op, err)) return abi_fail(KH_ERR_INVALID, err);
  return KH_OK;
}

int hip_status(hipError_t e, const char *what) {
  return e == hipSuccess ? KH_OK : abi_fail(KH_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

}  // namespace
}  // namespace kh

extern "C" {

int kh_paged_sizes(size_t *sizes3) {
  if (!sizes3) return kh::abi_fail(KH_ERR_INVALID, "null argument");
  sizes3[0] = sizeof(kh_paged);
  sizes3[1] = sizeof(kh_cache_append_op);
  sizes3[2] = sizeof(kh_pool);
  return KH_OK;
}

int kh_paged_workspace_bytes(const kh_paged *op, size_t *bytes) {
  return kh::guarded([&] {
    if (!op || !bytes) return kh::abi_fail(KH_ERR_INVALID, "null argument");
    std::string err;
    bool unsupported = false;
    if (!kh::check_paged(*op, err, unsupported)) return kh::abi_fail(unsupported ? KH_ERR_UNSUPPORTED : KH_ERR_INVALID, err);
    *bytes = 4 * kh::workspace_floats(*op);
    return (int)KH_OK;
  });
}

int kh_paged_run(const kh_paged *op, void *workspace, size_t workspace_bytes, void *stream) {
  return kh::guarded([&] {
    const int rc = kh::check_run(op);
    if (rc != KH_OK) return rc;
    const size_t need = 4 * kh::workspace_floats(*op);
    if (workspace_bytes < need || (need && !workspace))
      return kh::abi_fail(KH_ERR_CAPACITY, "workspace of " + std::to_string(workspace_bytes) + " bytes, the operator needs " +
                                               std::to_string(need));
    if ((uintptr_t)workspace % 16) return kh::abi_fail(KH_ERR_INVALID, "workspace: not 16-byte aligned");
    float *ws = static_cast<float *>(workspace);
    const hipStream_t s = static_cast<hipStream_t>(stream);
    return kh::hip_status(op->variant == KH_PAGED_SELECT ? kh::launch_select(*op, ws, s) : kh::launch_paged(*op, ws, s),
                          "kh_paged_run");
  });
}

int kh_paged_host(const kh_paged *op) {
  return kh::guarded([&] {
    const int rc = kh::check_run(op);
    if (rc == KH_OK) kh::host_paged(*op);
    return rc;
  });
}

int kh_cache_append(const kh_cache_append_op *op, void *stream) {
  return kh::guarded([&] {
    const int rc = kh::check_append(op);
    if (rc != KH_OK) return rc;
    return kh::hip_status(kh::launch_append(*op, static_cast<hipStream_t>(stream)), "kh_cache_append");
  });
}

int kh_cache_append_host(const kh_cache_append_op *op) {
  return kh::guarded([&] {
    const int rc = kh::check_append(op);
    if (rc == KH_OK) kh::host_append(*op);
    return rc;
  });
}

int kh_cache_copy(const kh_pool *pools, int n_pools, int32_t pages, const int32_t *source, const int32_t *target,
                  int n, void *stream) {
  return kh::guarded([&] {
    const int rc = kh::check_copy(pools, n_pools, pages, source, target, n);
    if (rc != KH_OK) return rc;
    return kh::hip_status(kh::launch_copy(pools, n_pools, source, target, n, static_cast<hipStream_t>(stream)),
                          "kh_cache_copy");
  });
}

int kh_cache_copy_host(const kh_pool *pools, int n_pools, int32_t pages, const int32_t *source,
                       const int32_t *target, int n) {
  return kh::guarded([&] {
    const int rc = kh::check_copy(pools, n_pools, pages, source, target, n);
    if (rc != KH_OK) return rc;
    for (int i = 0; i < n_pools; ++i)
      for (int64_t layer = 0; layer < pools[i].layers; ++layer)
        for (int j = 0; j < n; ++j) {
          char *base = static_cast<char *>(pools[i].base) + layer * pools[i].layer_bytes;
          std::copy_n(base + source[j] * pools[i].page_bytes, pools[i].page_bytes, base + target[j] * pools[i].page_bytes);
        }
    return rc;
  });
}

}  // extern "C"
