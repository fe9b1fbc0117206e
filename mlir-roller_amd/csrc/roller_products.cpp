// C entry points of the products of a language model's feed-forward block: argument checks, workspaces,
// and the calls into the kernels' translation units (ffn.hip, orthogonalize.hip).  Declarations:
// include/roller_hip.h.
#include "roller_ffn.h"
#include "roller_hip.h"
#include "roller_internal.h"
#include "roller_ortho.h"

#include <cmath>
#include <cstdint>
#include <exception>
#include <map>

namespace {

struct Room {
  char* ptr = nullptr;
  size_t bytes = 0;
};
std::map<hipStream_t, Room> g_rooms;
std::mutex g_rooms_mutex;

int elem_size(int dtype) { return dtype == RL_F32 ? 4 : 2; }

// Nothing thrown inside a call leaves the library.
template <class F>
int guarded(F&& f) {
  try {
    return f();
  } catch (const std::exception& e) {
    return rl_fail(RL_ERR_INTERNAL, "internal error: %s", e.what());
  } catch (...) {
    return rl_fail(RL_ERR_INTERNAL, "internal error");
  }
}

// A row-major matrix argument: present, aligned to its elements, rows that do not overlap, and 256 of its
// rows within the 32-bit offsets that a tile addresses.
int check_matrix(const char* name, const void* p, int ld, int cols, int es) {
  if (!p) return rl_fail(RL_ERR_INVALID_ARG, "%s is NULL", name);
  if ((uintptr_t)p % es) return rl_fail(RL_ERR_INVALID_ARG, "%s is not aligned to its %d-byte elements", name, es);
  if (ld < cols) return rl_fail(RL_ERR_INVALID_ARG, "%s: leading dimension %d is less than its %d columns", name, ld, cols);
  if ((long)ld * es * 256 + 65536 > 0x7fffffffL) return rl_fail(RL_ERR_INVALID_ARG, "%s: leading dimension %d too large for 32-bit in-tile offsets", name, ld);
  return RL_OK;
}

// Extents: their dense rows, and the internal ones that are up to two lines longer, are within what check_matrix lets through.
constexpr int kMaxExtent = (1 << 20);

int check_stream(hipStream_t stream, int device) {
  if (!stream) return RL_OK;
  int on = device;
  if (hipStreamGetDevice(stream, &on) != hipSuccess) {
    (void)hipGetLastError();
    return RL_OK;
  }
  if (on != device) return rl_fail(RL_ERR_INVALID_ARG, "the stream belongs to device %d, rl_init chose device %d", on, device);
  return RL_OK;
}

int check_ffn(const rl_ffn_config* cfg) {
  if (!cfg) return rl_fail(RL_ERR_INVALID_ARG, "cfg is NULL");
  if (cfg->dtype < RL_F32 || cfg->dtype > RL_BF16) return rl_fail(RL_ERR_INVALID_ARG, "dtype is RL_F32, RL_F16 or RL_BF16, got %d", cfg->dtype);
  if (cfg->activation < RL_ACT_SILU || cfg->activation > RL_ACT_GELU_TANH) return rl_fail(RL_ERR_INVALID_ARG, "activation is RL_ACT_SILU, RL_ACT_GELU or RL_ACT_GELU_TANH, got %d", cfg->activation);
  if (cfg->d_model < 1 || cfg->d_ff < 1 || cfg->d_model > kMaxExtent || cfg->d_ff > kMaxExtent)
    return rl_fail(RL_ERR_INVALID_ARG, "d_model and d_ff are 1 to %d, got %d and %d", kMaxExtent, cfg->d_model, cfg->d_ff);
  return RL_OK;
}

int check_tokens(int T) {
  if (T < 0 || T > (1 << 24)) return rl_fail(RL_ERR_INVALID_ARG, "the number of tokens is 0 to %d, got %d", 1 << 24, T);
  return RL_OK;
}

FfnType type_of(int dtype) { return dtype == RL_F32 ? rl_ffn_f32() : dtype == RL_F16 ? rl_ffn_f16() : rl_ffn_bf16(); }

rl_product_tile tile_of(const product::Plan& p) { return {product::kTiles[p.tile].bm, product::kTiles[p.tile].bn, p.splits, p.whole}; }

#define TRY(expr)          \
  do {                     \
    const int rc_ = (expr); \
    if (rc_) return rc_;   \
  } while (0)

int check_ortho(const rl_ortho_config* cfg) {
  if (!cfg) return rl_fail(RL_ERR_INVALID_ARG, "cfg is NULL");
  if (cfg->dtype < RL_F32 || cfg->dtype > RL_BF16) return rl_fail(RL_ERR_INVALID_ARG, "dtype is RL_F32, RL_F16 or RL_BF16, got %d", cfg->dtype);
  if (cfg->rows < 1 || cfg->cols < 1 || cfg->rows > kMaxExtent || cfg->cols > kMaxExtent)
    return rl_fail(RL_ERR_INVALID_ARG, "rows and cols are 1 to %d, got %d and %d", kMaxExtent, cfg->rows, cfg->cols);
  if (cfg->batch < 0 || cfg->batch > 65535) return rl_fail(RL_ERR_INVALID_ARG, "batch is 0 to 65535, got %d", cfg->batch);
  if (cfg->steps < 0 || cfg->steps > 64) return rl_fail(RL_ERR_INVALID_ARG, "steps is 0 to 64, got %d", cfg->steps);
  if (!(cfg->eps >= 0.0f) || !std::isfinite(cfg->eps)) return rl_fail(RL_ERR_INVALID_ARG, "eps is finite and not negative");
  if (!std::isfinite(cfg->scale)) return rl_fail(RL_ERR_INVALID_ARG, "scale is finite");
  return RL_OK;
}

}  // namespace

int ProductRoom::take(hipStream_t stream, void* user, size_t user_bytes, size_t need, const char* what, char** out) {
  *out = nullptr;
  if (user) {
    if ((uintptr_t)user % 256) return rl_fail(RL_ERR_INVALID_ARG, "%s: the workspace must be 256-byte aligned", what);
    if (user_bytes < need) return rl_fail(RL_ERR_INVALID_ARG, "%s: this call needs a workspace of %zu bytes, got %zu (16-bit rows at odd elements, and backward gate and up weights with different leading dimensions, need room for a packed copy)", what, need, user_bytes);
    *out = (char*)user;
    return RL_OK;
  }
  if (need == 0) return RL_OK;
  // (one handle that means another stream in every thread: two of them would work in one buffer at once)
  if (stream == hipStreamPerThread)
    return rl_fail(RL_ERR_INVALID_ARG, "%s: a call on the per-thread stream needs the caller's workspace (%zu bytes): the library keeps one per stream handle, and this handle is another stream in every thread", what, need);
  hipStreamCaptureStatus capturing = hipStreamCaptureStatusNone;
  hipError_t e = hipStreamIsCapturing(stream, &capturing);
  if (e != hipSuccess) return rl_hip_fail(e, "hipStreamIsCapturing");
  if (capturing != hipStreamCaptureStatusNone)
    return rl_fail(RL_ERR_INVALID_ARG, "%s: a captured call needs the caller's workspace (%zu bytes): the library's may be freed or shared while the graph lives", what, need);
  lock_ = std::unique_lock<std::mutex>(g_rooms_mutex);
  Room& r = g_rooms[stream];
  if (r.bytes < need) {
    if (r.ptr) {
      e = hipStreamSynchronize(stream);   // calls queued earlier may still use it
      if (e == hipSuccess) e = hipFree(r.ptr);
      if (e != hipSuccess) return rl_hip_fail(e, "growing the stream's workspace");
      r = Room();
    }
    const size_t want = need + need / 4;
    e = hipMalloc((void**)&r.ptr, want);
    if (e != hipSuccess) {
      r = Room();
      return rl_hip_fail(e, "allocating the stream's workspace");
    }
    r.bytes = want;
  }
  *out = r.ptr;
  return RL_OK;
}

int rl_products_forget_stream(hipStream_t stream) {
  std::lock_guard<std::mutex> lock(g_rooms_mutex);
  auto it = g_rooms.find(stream);
  if (it == g_rooms.end()) return RL_OK;
  if (it->second.ptr) {
    hipError_t e = hipStreamSynchronize(stream);
    if (e == hipSuccess) e = hipFree(it->second.ptr);
    if (e != hipSuccess) return rl_hip_fail(e, "freeing the stream's workspace");
  }
  g_rooms.erase(it);
  return RL_OK;
}

extern "C" {

int rl_ffn_saved_bytes(const rl_ffn_config* cfg, int T, size_t* bytes) {
  return guarded([&]() -> int {
    TRY(check_ffn(cfg));
    TRY(check_tokens(T));
    if (!bytes) return rl_fail(RL_ERR_INVALID_ARG, "bytes is NULL");
    *bytes = ffn_saved(elem_size(cfg->dtype), T, cfg->d_ff).total;
    return RL_OK;
  });
}

int rl_ffn_workspace_bytes(const rl_ffn_config* cfg, int T, int backward, int unaligned, size_t* bytes) {
  return guarded([&]() -> int {
    TRY(check_ffn(cfg));
    TRY(check_tokens(T));
    if (!bytes) return rl_fail(RL_ERR_INVALID_ARG, "bytes is NULL");
    *bytes = 0;
    int device = 0;
    FfnCall c = {};
    TRY(rl_device(&device, &c.compute_units));
    c.T = T;
    c.D = cfg->d_model;
    c.F = cfg->d_ff;
    const FfnType t = type_of(cfg->dtype);
    if (T == 0) return RL_OK;
    // (no pointers here, and leading dimensions that are those of dense rows: packed copies are counted where
    // such rows start at odd elements, or for all with `unaligned`)
    c.x.ld = c.w_gate.ld = c.w_up.ld = c.dy.ld = c.D;
    c.w_down.ld = c.F;
    size_t need = t.forward_room(c, unaligned != 0);
    if (backward) {
      const size_t b = t.backward_room(c, unaligned != 0);
      if (b > need) need = b;
    }
    *bytes = need;
    return RL_OK;
  });
}

int rl_ffn_tiles(const rl_ffn_config* cfg, int T, int compute_units, rl_product_tile out[6]) {
  return guarded([&]() -> int {
    TRY(check_ffn(cfg));
    TRY(check_tokens(T));
    if (!out || T == 0 || compute_units < 1) return rl_fail(RL_ERR_INVALID_ARG, "rl_ffn_tiles: needs tokens, compute units and a place to write to");
    FfnCall c = {};
    c.T = T;
    c.D = cfg->d_model;
    c.F = cfg->d_ff;
    c.compute_units = compute_units;
    product::Plan plans[6];
    type_of(cfg->dtype).plans(c, plans);
    for (int i = 0; i < 6; ++i) out[i] = tile_of(plans[i]);
    return RL_OK;
  });
}

int rl_ffn_forward(const rl_ffn_config* cfg, const void* x, int ldx, const void* w_gate, int ld_gate, const void* w_up, int ld_up,
                   const void* w_down, int ld_down, void* y, int ldy, int T, void* saved, void* workspace,
                   size_t workspace_bytes, rl_stream stream) {
  return guarded([&]() -> int {
    TRY(check_ffn(cfg));
    TRY(check_tokens(T));
    if (T == 0) return RL_OK;
    DeviceScope device;
    TRY(device.status());
    TRY(check_stream((hipStream_t)stream, device.device()));
    const int es = elem_size(cfg->dtype);
    TRY(check_matrix("x", x, ldx, cfg->d_model, es));
    TRY(check_matrix("w_gate", w_gate, ld_gate, cfg->d_model, es));
    TRY(check_matrix("w_up", w_up, ld_up, cfg->d_model, es));
    TRY(check_matrix("w_down", w_down, ld_down, cfg->d_ff, es));
    TRY(check_matrix("y", y, ldy, cfg->d_model, es));
    if ((uintptr_t)saved % 256) return rl_fail(RL_ERR_INVALID_ARG, "saved must be 256-byte aligned");
    FfnCall c = {};
    c.activation = cfg->activation;
    c.T = T;
    c.D = cfg->d_model;
    c.F = cfg->d_ff;
    c.x = {x, ldx};
    c.w_gate = {w_gate, ld_gate};
    c.w_up = {w_up, ld_up};
    c.w_down = {w_down, ld_down};
    c.y = y;
    c.ldy = ldy;
    c.saved = saved;
    c.stream = (hipStream_t)stream;
    c.compute_units = device.compute_units();
    const FfnType t = type_of(cfg->dtype);
    ProductRoom room;
    TRY(room.take(c.stream, workspace, workspace_bytes, t.forward_room(c, false), "rl_ffn_forward", &c.room));
    return t.forward(c);
  });
}

int rl_ffn_backward(const rl_ffn_config* cfg, const void* dy, int lddy, const void* x, int ldx, const void* w_gate, int ld_gate,
                    const void* w_up, int ld_up, const void* w_down, int ld_down, const void* saved, void* dx, int lddx,
                    void* dw_gate, int ldd_gate, void* dw_up, int ldd_up, void* dw_down, int ldd_down, int T, void* workspace,
                    size_t workspace_bytes, rl_stream stream) {
  return guarded([&]() -> int {
    TRY(check_ffn(cfg));
    TRY(check_tokens(T));
    DeviceScope device;
    TRY(device.status());
    TRY(check_stream((hipStream_t)stream, device.device()));
    const int es = elem_size(cfg->dtype), D = cfg->d_model, F = cfg->d_ff;
    if (T > 0) {
      TRY(check_matrix("dy", dy, lddy, D, es));
      TRY(check_matrix("x", x, ldx, D, es));
      TRY(check_matrix("w_gate", w_gate, ld_gate, D, es));
      TRY(check_matrix("w_up", w_up, ld_up, D, es));
      TRY(check_matrix("w_down", w_down, ld_down, F, es));
      if (!saved) return rl_fail(RL_ERR_INVALID_ARG, "saved is NULL: the backward pass reads what rl_ffn_forward kept there");
      if ((uintptr_t)saved % 256) return rl_fail(RL_ERR_INVALID_ARG, "saved must be 256-byte aligned");
      if (dx) TRY(check_matrix("dx", dx, lddx, D, es));
    }
    if (!dw_gate != !dw_up) return rl_fail(RL_ERR_INVALID_ARG, "dw_gate and dw_up are asked for together");
    if (dw_gate) TRY(check_matrix("dw_gate", dw_gate, ldd_gate, D, es));
    if (dw_up) TRY(check_matrix("dw_up", dw_up, ldd_up, D, es));
    if (dw_down) TRY(check_matrix("dw_down", dw_down, ldd_down, F, es));
    FfnCall c = {};
    c.activation = cfg->activation;
    c.T = T;
    c.D = D;
    c.F = F;
    c.dy = {dy, lddy};
    c.x = {x, ldx};
    c.w_gate = {w_gate, ld_gate};
    c.w_up = {w_up, ld_up};
    c.w_down = {w_down, ld_down};
    c.saved = (void*)saved;
    c.dx = T > 0 ? dx : nullptr;
    c.ld_dx = lddx;
    c.dw_gate = dw_gate;
    c.ld_dw_gate = ldd_gate;
    c.dw_up = dw_up;
    c.ld_dw_up = ldd_up;
    c.dw_down = dw_down;
    c.ld_dw_down = ldd_down;
    c.stream = (hipStream_t)stream;
    c.compute_units = device.compute_units();
    const FfnType t = type_of(cfg->dtype);
    ProductRoom room;
    if (T > 0) TRY(room.take(c.stream, workspace, workspace_bytes, t.backward_room(c, false), "rl_ffn_backward", &c.room));
    return t.backward(c);
  });
}

int rl_ortho_workspace_bytes(const rl_ortho_config* cfg, size_t* bytes) {
  return guarded([&]() -> int {
    TRY(check_ortho(cfg));
    if (!bytes) return rl_fail(RL_ERR_INVALID_ARG, "bytes is NULL");
    *bytes = 0;
    int device = 0;
    OrthoCall c = {};
    TRY(rl_device(&device, &c.compute_units));
    if (cfg->batch == 0) return RL_OK;
    c.dtype = cfg->dtype;
    c.rows = cfg->rows;
    c.cols = cfg->cols;
    c.batch = cfg->batch;
    c.steps = cfg->steps;
    *bytes = rl_ortho_room(c);
    return RL_OK;
  });
}

int rl_ortho_tiles(const rl_ortho_config* cfg, int compute_units, rl_product_tile out[3]) {
  return guarded([&]() -> int {
    TRY(check_ortho(cfg));
    if (!out || cfg->batch == 0 || compute_units < 1) return rl_fail(RL_ERR_INVALID_ARG, "rl_ortho_tiles: needs matrices, compute units and a place to write to");
    OrthoCall c = {};
    c.dtype = cfg->dtype;
    c.rows = cfg->rows;
    c.cols = cfg->cols;
    c.batch = cfg->batch;
    c.compute_units = compute_units;
    product::Plan plans[3];
    rl_ortho_plans(c, plans);
    for (int i = 0; i < 3; ++i) out[i] = tile_of(plans[i]);
    return RL_OK;
  });
}

int rl_orthogonalize(const rl_ortho_config* cfg, const float* coefficients, const void* G, int ldg, long stride_g, void* O, int ldo,
                     long stride_o, void* workspace, size_t workspace_bytes, rl_stream stream) {
  return guarded([&]() -> int {
    TRY(check_ortho(cfg));
    if (cfg->batch == 0) return RL_OK;
    DeviceScope device;
    TRY(device.status());
    TRY(check_stream((hipStream_t)stream, device.device()));
    const int es = elem_size(cfg->dtype);
    TRY(check_matrix("G", G, ldg, cfg->cols, es));
    TRY(check_matrix("O", O, ldo, cfg->cols, es));
    const long least_g = (long)(cfg->rows - 1) * ldg + cfg->cols, least_o = (long)(cfg->rows - 1) * ldo + cfg->cols;
    if (cfg->batch > 1 && (stride_g < least_g || stride_o < least_o))
      return rl_fail(RL_ERR_INVALID_ARG, "matrices of the stack overlap (strides %ld and %ld, a matrix spans %ld and %ld elements)", stride_g, stride_o, least_g, least_o);
    float all[3 * 64];
    for (int k = 0; k < cfg->steps; ++k)
      for (int e = 0; e < 3; ++e) {
        static const float standard[3] = {3.4445f, -4.7750f, 2.0315f};
        const float v = coefficients ? coefficients[3 * k + e] : standard[e];
        if (!std::isfinite(v)) return rl_fail(RL_ERR_INVALID_ARG, "coefficient %d of step %d is not finite", e, k);
        all[3 * k + e] = v;
      }
    OrthoCall c = {};
    c.dtype = cfg->dtype;
    c.rows = cfg->rows;
    c.cols = cfg->cols;
    c.batch = cfg->batch;
    c.steps = cfg->steps;
    c.coefficients = all;
    c.eps = cfg->eps;
    c.scale = cfg->scale;
    c.g = G;
    c.ldg = ldg;
    c.stride_g = cfg->batch > 1 ? stride_g : 0;
    c.o = O;
    c.ldo = ldo;
    c.stride_o = cfg->batch > 1 ? stride_o : 0;
    c.stream = (hipStream_t)stream;
    c.compute_units = device.compute_units();
    ProductRoom room;
    TRY(room.take(c.stream, workspace, workspace_bytes, rl_ortho_room(c), "rl_orthogonalize", &c.room));
    return rl_ortho_run(c);
  });
}

}  // extern "C"
