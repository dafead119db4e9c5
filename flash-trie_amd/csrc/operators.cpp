// operators.cpp -- argument checks and launches of the model head's C ABI
// (include/flashtrie_amd.h).  Everything that the host can see is checked
// before the first launch; values on the device are checked by the kernels.
#include "operators.h"

#include <cmath>
#include <cstdio>
#include <cstring>

namespace {

using ftk::set_error;

int refuse(int code, const char* call, const char* what) {
  char msg[192];
  std::snprintf(msg, sizeof(msg), "%s: %s", call, what);
  return set_error(code, msg);
}

int hip_error(hipError_t e, const char* call) {
  return refuse(e == hipErrorOutOfMemory ? FT_E_NOMEM : FT_E_HIP, call, hipGetErrorString(e));
}

constexpr int kMaxDevices = 64;
constexpr uint64_t kMaxGrid = 0x7FFFFFFFull;  // workgroups of a launch
constexpr uint64_t kMaxThreads = 0xFFFFFFFFull;

constexpr uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// The caller's device is current during the call, and what was before after
// it.
struct OnDevice {
  int before = -1, device;
  hipError_t error;
  explicit OnDevice(int d) : device(d) {
    error = hipGetDevice(&before);
    if (error == hipSuccess && before != device) error = hipSetDevice(device);
  }
  ~OnDevice() {
    if (before >= 0 && before != device) (void)hipSetDevice(before);
  }
};

int check_device(int device, const char* call) {
  static bool known[kMaxDevices];  // gfx950 (a race would write the same)
  if (device < 0 || device >= kMaxDevices)
    return refuse(FT_E_DEVICE, call, "no such device");
  if (__atomic_load_n(&known[device], __ATOMIC_RELAXED)) return FT_OK;
  int n = 0;
  if (hipGetDeviceCount(&n) != hipSuccess || device >= n)
    return refuse(FT_E_DEVICE, call, "no such device");
  hipDeviceProp_t prop;
  const hipError_t e = hipGetDeviceProperties(&prop, device);
  if (e != hipSuccess) return hip_error(e, call);
  if (std::strncmp(prop.gcnArchName, "gfx950", 6) != 0)
    return refuse(FT_E_DEVICE, call, "the device is no gfx950");
  __atomic_store_n(&known[device], true, __ATOMIC_RELAXED);
  return FT_OK;
}

// Arguments of each call: a text of what is wrong, or null.
const char* wrong(const ft_adapter_logits_args& a, int* code) {
  *code = FT_E_ARG;
  if (a.dtype != FT_F16 && a.dtype != FT_BF16) return "x must be float16 or bfloat16";
  if (a.out_dtype != FT_F32 && a.out_dtype != a.dtype)
    return "the logits must be float32 or of the inputs' type";
  if (!a.hidden || !a.vocab) return "hidden and vocab must be at least 1";
  if (a.adapters && !a.rank) return "rank must be at least 1";
  *code = FT_E_LIMIT;
  if (a.rank > FT_MAX_RANK) return "rank must be at most 256";
  if (a.adapters > 0x7FFFFFFEu) return "too many adapters";
  if (a.vocab > FT_MAX_HEAD_VOCAB) return "vocab must be at most 2^24";
  if (a.hidden > (1u << 24)) return "hidden must be at most 2^24";
  // (the launches: 1024 threads for 16 rows; tiles of 128 tokens by 64 rows
  // with 256, by 256 rows with 1024)
  if (a.rows > kMaxGrid || ceil_div(a.rows, 16) * 1024 > kMaxThreads ||
      ceil_div(a.vocab, 128) * ceil_div(a.rows, 64) * 256 > kMaxThreads ||
      ceil_div(a.vocab, 128) * ceil_div(a.rows, 256) * 1024 > kMaxThreads)
    return "too many rows";
  *code = FT_E_ARG;
  if (a.rows) {
    if (!a.x || !a.weight || !a.adapter || !a.out) return "null pointer";
    if (a.adapters && (!a.down || !a.up || !a.scale)) return "null pointer";
    if (a.out_stride < (int64_t)a.vocab && a.rows > 1) return "rows of the logits overlap";
  }
  return nullptr;
}

const char* wrong(const ft_propose_args& a, int* code) {
  *code = FT_E_ARG;
  if (a.dtype != FT_F32 && a.dtype != FT_F16 && a.dtype != FT_BF16)
    return "logits must be float32, float16 or bfloat16";
  if (!a.topk || a.topk > a.vocab) return "topk must be from 1 to vocab";
  *code = FT_E_LIMIT;
  if (a.topk > FT_MAX_PROPOSALS) return "topk must be at most 4096";
  if (a.vocab > FT_MAX_HEAD_VOCAB) return "vocab must be at most 2^24";
  if (a.batch > kMaxGrid || a.steps > kMaxGrid || a.batch * a.steps > kMaxGrid / 16384)
    return "too many rows";
  *code = FT_E_ARG;
  if (a.batch && a.steps && (!a.logits || !a.ids || !a.logp)) return "null pointer";
  return nullptr;
}

const char* wrong(const ft_keys& k, int* code) {
  *code = FT_E_ARG;
  if (k.dtype != FT_F32 && k.dtype != FT_F16 && k.dtype != FT_BF16)
    return "logits must be float32, float16 or bfloat16";
  if (!k.vocab || !k.steps || !k.keys) return "vocab, steps and keys must be at least 1";
  *code = FT_E_LIMIT;
  if (k.keys > FT_MAX_KEYS) return "keys must be at most 4096";
  if (k.vocab > FT_MAX_HEAD_VOCAB) return "vocab must be at most 2^24";
  if (k.batch > kMaxGrid || k.steps > kMaxGrid || k.batch * k.steps > kMaxGrid / 16384 ||
      k.batch * k.keys > kMaxGrid / 4)
    return "too many rows";
  // (the gradient: 256 threads for 1024 vectors of a row)
  if (k.dlogits && k.batch * k.steps * ceil_div(k.vocab, k.dtype == FT_F32 ? 4096 : 8192) * 256 >
                       kMaxThreads)
    return "too many rows";
  *code = FT_E_ARG;
  if (!k.loss) return "null pointer";
  if (k.batch) {
    if (!k.logits || !k.tokens || !k.lengths || !k.logp) return "null pointer";
    // (a request's rows may share the gradient's memory with no other)
    if (k.dlogits && k.steps > 1 && k.dstride[1] < (int64_t)k.vocab)
      return "rows of the gradient overlap";
    if (k.dlogits && k.batch > 1 &&
        k.dstride[0] < (int64_t)(k.steps - 1) * k.dstride[1] + (int64_t)k.vocab)
      return "rows of the gradient overlap";
  }
  return nullptr;
}

const char* wrong(const ft_policy_loss_args& a, int* code) {
  if (const char* w = wrong(a.k, code)) return w;
  if (!(a.clip_low >= 0.0f && a.clip_low <= 1.0f) ||
      !(a.clip_high >= 0.0f && std::isfinite(a.clip_high)))
    return "clip_low must be in [0, 1] and clip_high at least 0";
  if (!std::isfinite(a.kl_coef)) return "kl_coef must be finite";
  if (a.kl_coef != 0.0f && !a.ref_logp && a.k.batch) return "kl_coef needs ref_logp";
  if (a.k.batch && (!a.old_logp || !a.advantage || !a.weight)) return "null pointer";
  return nullptr;
}

const char* wrong(const ft_preference_loss_args& a, int* code) {
  if (const char* w = wrong(a.k, code)) return w;
  if (!std::isfinite(a.beta)) return "beta must be finite";
  if (!(a.smoothing >= 0.0f && a.smoothing <= 1.0f)) return "smoothing must be in [0, 1]";
  if (a.pairs && !a.k.batch) return "pairs of no keys";
  if (a.pairs > kMaxGrid) {
    *code = FT_E_LIMIT;
    return "too many pairs";
  }
  if (ceil_div(a.k.batch * a.k.keys, 64) * 1024 > kMaxThreads) {  // 1024 threads for 64 keys
    *code = FT_E_LIMIT;
    return "too many keys";
  }
  if (a.pairs && (!a.pair || !a.weight)) return "null pointer";
  if (a.k.batch && !a.ref_logp) return "null pointer";
  return nullptr;
}

const char* wrong(const ft_cross_entropy_loss_args& a, int* code) {
  *code = FT_E_ARG;
  if (a.dtype != FT_F16 && a.dtype != FT_BF16) return "x must be float16 or bfloat16";
  if (!a.hidden || !a.vocab) return "hidden and vocab must be at least 1";
  if (!(a.smoothing >= 0.0f && a.smoothing <= 1.0f)) return "smoothing must be in [0, 1]";
  *code = FT_E_LIMIT;
  if (a.vocab > FT_MAX_HEAD_VOCAB) return "vocab must be at most 2^24";
  if (a.hidden > FT_MAX_TABLE_HIDDEN) return "hidden must be at most 2^16";
  // (the launches: 1024 threads for 16 rows; 256 for tiles of 128 tokens, or
  // hidden columns, by 64 rows, or tokens)
  if (a.rows > FT_MAX_TABLE_ROWS ||
      ceil_div(a.vocab, 128) * ceil_div(a.rows, 64) * 256 > kMaxThreads ||
      ceil_div(a.hidden, 128) * ceil_div(a.vocab + 256ull, 64) * 256 > kMaxThreads)
    return "too many rows";
  *code = FT_E_ARG;
  if (!a.loss) return "null pointer";
  if (a.rows && (!a.x || !a.weight || !a.target || !a.row_weight || !a.logp)) return "null pointer";
  if (a.dx && a.rows > 1 && a.dx_stride < (int64_t)a.hidden) return "rows of dx overlap";
  if (a.dweight && a.vocab > 1 && a.dweight_stride < (int64_t)a.hidden)
    return "rows of dweight overlap";
  return nullptr;
}

// The packed table's own sizes.
const char* wrong_table(uint32_t hidden, uint32_t vocab, uint32_t group, int* code) {
  *code = FT_E_ARG;
  if (!hidden || !vocab) return "hidden and vocab must be at least 1";
  if (group != 32 && group != 64 && group != 128) return "group must be 32, 64 or 128";
  *code = FT_E_LIMIT;
  if (vocab > FT_MAX_HEAD_VOCAB) return "vocab must be at most 2^24";
  if (hidden > FT_MAX_TABLE_HIDDEN) return "hidden must be at most 2^16";
  // (pack_weight: 64 threads for 16 tokens by 128 columns)
  if (ceil_div(vocab, 16) * ceil_div(hidden, 128) * 64 > kMaxThreads - 1024)
    return "the table is too large";
  return nullptr;
}

const char* wrong(const ft_pack_weight_args& a, int* code) {
  *code = FT_E_ARG;
  if (a.dtype != FT_F16 && a.dtype != FT_BF16) return "weight must be float16 or bfloat16";
  if (const char* w = wrong_table(a.hidden, a.vocab, a.group, code)) return w;
  *code = FT_E_ARG;
  if (!a.weight || !a.packed || !a.scales) return "null pointer";
  if ((uintptr_t)a.packed % 16 || (uintptr_t)a.scales % 8)
    return "packed must be 16-byte aligned, scales 8-byte";
  return nullptr;
}

const char* wrong(const ft_packed_logits_args& a, int* code) {
  *code = FT_E_ARG;
  if (a.dtype != FT_F16 && a.dtype != FT_BF16) return "x must be float16 or bfloat16";
  if (a.out_dtype != FT_F32 && a.out_dtype != a.dtype)
    return "the logits must be float32 or of x's type";
  if (const char* w = wrong_table(a.hidden, a.vocab, a.group, code)) return w;
  *code = FT_E_LIMIT;
  if (a.rows > FT_MAX_TABLE_ROWS) return "too many rows";
  *code = FT_E_ARG;
  if (a.rows) {
    if (!a.x || !a.packed || !a.scales || !a.out) return "null pointer";
    if ((uintptr_t)a.packed % 16 || (uintptr_t)a.scales % 8)
      return "packed must be 16-byte aligned, scales 8-byte";
    if (a.out_stride < (int64_t)a.vocab && a.rows > 1) return "rows of the logits overlap";
  }
  return nullptr;
}

// Tokens of keys and the table of ft_embed and ft_embed_grad; `threads` for
// 64 vectors of a token's row.
const char* wrong_tokens(int dtype, uint64_t groups, uint64_t steps, uint32_t hidden, uint32_t vocab,
                         uint64_t threads, int* code) {
  *code = FT_E_ARG;
  if (dtype != FT_F32 && dtype != FT_F16 && dtype != FT_BF16)
    return "the table must be float32, float16 or bfloat16";
  if (!hidden || !vocab) return "hidden and vocab must be at least 1";
  *code = FT_E_LIMIT;
  if (vocab > FT_MAX_HEAD_VOCAB) return "vocab must be at most 2^24";
  if (hidden > FT_MAX_TABLE_HIDDEN) return "hidden must be at most 2^16";
  if (groups > FT_MAX_TABLE_TOKENS || steps > FT_MAX_TABLE_TOKENS ||
      groups * steps > FT_MAX_TABLE_TOKENS ||
      (groups * steps + 32) * ceil_div(hidden, 64 * (dtype == FT_F32 ? 4 : 8)) * threads > kMaxThreads)
    return "too many tokens";
  return nullptr;
}

const char* wrong(const ft_embed_args& a, int* code) {
  if (const char* w = wrong_tokens(a.dtype, a.groups, a.steps, a.hidden, a.vocab, 16, code)) return w;
  *code = FT_E_ARG;
  if (a.groups && a.steps && (!a.tokens || !a.table || !a.out)) return "null pointer";
  return nullptr;
}

const char* wrong(const ft_embed_grad_args& a, int* code) {
  // (a workgroup of 256 joins 32 positions, or 8 of up to 16384)
  if (const char* w = wrong_tokens(a.dtype, a.groups, a.steps, a.hidden, a.vocab,
                                   a.groups * a.steps < 16384 ? 32 : 8, code))
    return w;
  *code = FT_E_ARG;
  if (!a.dtable || (a.groups && a.steps && (!a.tokens || !a.grad))) return "null pointer";
  if (a.vocab > 1 && a.dtable_stride < (int64_t)a.hidden) return "rows of the gradient overlap";
  return nullptr;
}

int device_of(const ft_adapter_logits_args& a) { return a.device; }
int device_of(const ft_propose_args& a) { return a.device; }
int device_of(const ft_policy_loss_args& a) { return a.k.device; }
int device_of(const ft_preference_loss_args& a) { return a.k.device; }
int device_of(const ft_cross_entropy_loss_args& a) { return a.device; }
int device_of(const ft_pack_weight_args& a) { return a.device; }
int device_of(const ft_packed_logits_args& a) { return a.device; }
int device_of(const ft_embed_args& a) { return a.device; }
int device_of(const ft_embed_grad_args& a) { return a.device; }

template <typename A>
size_t workspace(const A* a, uint64_t (*size)(const A&)) {
  int code;
  if (!a || wrong(*a, &code)) return 0;
  return (size_t)size(*a);
}

template <typename A>
int run(const A* a, void* ws, size_t ws_bytes, void* stream, const char* call,
        uint64_t (*size)(const A&), hipError_t (*launch)(const A&, uint8_t*, hipStream_t)) {
  if (!a) return refuse(FT_E_ARG, call, "null arguments");
  int code = FT_E_ARG;
  if (const char* w = wrong(*a, &code)) return refuse(code, call, w);
  const uint64_t need = size(*a);
  if (need && (!ws || (uintptr_t)ws % 256))
    return refuse(FT_E_ARG, call, "the workspace is null or not 256-byte aligned");
  if (ws_bytes < need) return refuse(FT_E_LIMIT, call, "the workspace is too small");
  if (int rc = check_device(device_of(*a), call)) return rc;
  OnDevice on(device_of(*a));
  if (on.error != hipSuccess) return hip_error(on.error, call);
  const hipError_t e = launch(*a, (uint8_t*)ws, (hipStream_t)stream);
  return e == hipSuccess ? FT_OK : hip_error(e, call);
}

}  // namespace

extern "C" {

const void* ft_hip_runtime(void) { return (const void*)&hipGetDevice; }

size_t ft_adapter_logits_workspace(const ft_adapter_logits_args* a) {
  return workspace(a, fto::adapter_logits_workspace);
}
int ft_adapter_logits(const ft_adapter_logits_args* a, void* ws, size_t n, void* stream) {
  return run(a, ws, n, stream, "ft_adapter_logits", fto::adapter_logits_workspace,
             fto::launch_adapter_logits);
}

size_t ft_propose_workspace(const ft_propose_args* a) {
  return workspace(a, fto::propose_workspace);
}
int ft_propose(const ft_propose_args* a, void* ws, size_t n, void* stream) {
  return run(a, ws, n, stream, "ft_propose", fto::propose_workspace, fto::launch_propose);
}

size_t ft_policy_loss_workspace(const ft_policy_loss_args* a) {
  return workspace(a, fto::policy_loss_workspace);
}
int ft_policy_loss(const ft_policy_loss_args* a, void* ws, size_t n, void* stream) {
  return run(a, ws, n, stream, "ft_policy_loss", fto::policy_loss_workspace,
             fto::launch_policy_loss);
}

size_t ft_preference_loss_workspace(const ft_preference_loss_args* a) {
  return workspace(a, fto::preference_loss_workspace);
}
int ft_preference_loss(const ft_preference_loss_args* a, void* ws, size_t n, void* stream) {
  return run(a, ws, n, stream, "ft_preference_loss", fto::preference_loss_workspace,
             fto::launch_preference_loss);
}

size_t ft_cross_entropy_loss_workspace(const ft_cross_entropy_loss_args* a) {
  return workspace(a, fto::cross_entropy_loss_workspace);
}
int ft_cross_entropy_loss(const ft_cross_entropy_loss_args* a, void* ws, size_t n, void* stream) {
  return run(a, ws, n, stream, "ft_cross_entropy_loss", fto::cross_entropy_loss_workspace,
             fto::launch_cross_entropy_loss);
}

size_t ft_pack_weight_workspace(const ft_pack_weight_args* a) {
  return workspace(a, fto::pack_weight_workspace);
}
int ft_pack_weight(const ft_pack_weight_args* a, void* ws, size_t n, void* stream) {
  return run(a, ws, n, stream, "ft_pack_weight", fto::pack_weight_workspace,
             fto::launch_pack_weight);
}

size_t ft_packed_logits_workspace(const ft_packed_logits_args* a) {
  return workspace(a, fto::packed_logits_workspace);
}
int ft_packed_logits(const ft_packed_logits_args* a, void* ws, size_t n, void* stream) {
  return run(a, ws, n, stream, "ft_packed_logits", fto::packed_logits_workspace,
             fto::launch_packed_logits);
}

size_t ft_embed_workspace(const ft_embed_args* a) {
  return workspace(a, fto::embed_workspace);
}
int ft_embed(const ft_embed_args* a, void* ws, size_t n, void* stream) {
  return run(a, ws, n, stream, "ft_embed", fto::embed_workspace,
             fto::launch_embed);
}

size_t ft_embed_grad_workspace(const ft_embed_grad_args* a) {
  return workspace(a, fto::embed_grad_workspace);
}
int ft_embed_grad(const ft_embed_grad_args* a, void* ws, size_t n, void* stream) {
  return run(a, ws, n, stream, "ft_embed_grad", fto::embed_grad_workspace,
             fto::launch_embed_grad);
}

}  // extern "C"
