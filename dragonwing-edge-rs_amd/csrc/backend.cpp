// HIP backend: the dragonwing_core::Backend contract
// (crates/dragonwing-core/src/backend.rs:127-199) on one gfx950 device,
// plus the op functions of dragonwing_vulkan::ops re-targeted to the HIP
// kernels.  Every op validates buffer sizes exactly and enqueues on the
// backend's single stream; nothing here computes on the CPU.
#include "backend.h"

#include <math.h>
#include <stddef.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <cmath>
#include <exception>
#include <thread>
#include <vector>

#include "../../include/dw_hip.h"

namespace dw {

static thread_local std::string g_last_error;

void set_last_error(const std::string& m) { g_last_error = m; }
void fail(int code, const std::string& msg) { throw Error{code, msg}; }
void hip_check(hipError_t e, const char* what) {
  if (e == hipSuccess) return;
  (void)hipGetLastError();  // reported here: the check behind a later call's launches must not find it
  fail(DW_ERR_BACKEND, std::string(what) + ": " + hipGetErrorString(e));
}

void* Backend::workspace(int slot, size_t bytes) {
  if (slot < 0 || slot >= kWsSlots) fail(DW_ERR_INVALID, "bad workspace slot");
  Ws& w = ws[slot];
  if (w.bytes < bytes) {
    if (w.ptr) {
      DW_HIP(hipStreamSynchronize(stream));
      DW_HIP(hipFree(w.ptr));
      w.ptr = nullptr;
      w.bytes = 0;
    }
    size_t want = std::max<size_t>(bytes, 4096);
    DW_HIP(hipMalloc(&w.ptr, want));
    w.bytes = want;
  }
  return w.ptr;
}

// Host -> device copy of small per-call parameter tables.  The source is a
// caller-owned (pageable) array, so the copy is completed before returning.
void Backend::upload_async(void* dst, const void* src, size_t bytes) {
  if (!bytes) return;
  DW_HIP(hipMemcpyAsync(dst, src, bytes, hipMemcpyHostToDevice, stream));
  DW_HIP(hipStreamSynchronize(stream));
}

// The first n slots; false if page-locked memory for them is refused.
bool Backend::slots_ready(int n) {
  for (int i = 0; i < n; ++i) {
    Slot& s = slots[i];
    if (!s.ev) DW_HIP(hipEventCreateWithFlags(&s.ev, hipEventDisableTiming));
    if (!s.p && hipHostMalloc((void**)&s.p, kSlotBytes, hipHostMallocDefault) != hipSuccess) {
      (void)hipGetLastError();
      s.p = nullptr;
      return false;
    }
  }
  return true;
}

// Chunks `thread`, thread + threads, ... of a download: the copy of one chunk
// out of its page-locked slot runs while the device fills the thread's other
// slot.  Every copy that was queued has ended when this returns.
hipError_t Backend::copy_chunks(uint8_t* dst, const uint8_t* src, size_t bytes, size_t chunk, int thread,
                                int threads) {
  hipError_t err = hipSetDevice(device);
  const size_t n = (bytes + chunk - 1) / chunk;
  auto queue = [&](size_t c, int slot) -> hipError_t {
    const size_t len = std::min(chunk, bytes - c * chunk);
    hipError_t e = hipMemcpyAsync(slots[slot].p, src + c * chunk, len, hipMemcpyDeviceToHost, stream);
    return e == hipSuccess ? hipEventRecord(slots[slot].ev, stream) : e;
  };
  size_t next = (size_t)thread, done = next;  // the next chunk to queue, to copy out
  int in = 0, out = 0;                        // their places among the thread's two slots
  const int first = 2 * thread;
  while (err == hipSuccess && done < n) {
    while (err == hipSuccess && next < n && next <= done + (size_t)threads) {
      err = queue(next, first + in);
      next += (size_t)threads;
      in ^= 1;
    }
    if (err == hipSuccess) err = hipEventSynchronize(slots[first + out].ev);
    if (err == hipSuccess) memcpy(dst + done * chunk, slots[first + out].p, std::min(chunk, bytes - done * chunk));
    done += (size_t)threads;
    out ^= 1;
  }
  if (err != hipSuccess) (void)hipStreamSynchronize(stream);
  return err;
}

// Through the page-locked slots: HIP's own copy to ordinary memory
// runs at 18 GB/s, and one to page-locked memory at 56 GB/s of which a thread
// moves 31 GB/s on (less into pages touched for the first time), so from 4 MiB
// on four threads copy.  Measured into warm memory: 1.8 MB 85 us, 59 MB 1.56
// ms (38 GB/s).  Up to 1 MiB a kernel fills the slot, whose end is the only
// thing waited for: 64 KiB 12.8 us, 1 MiB 58 us.  HIP's copies of more than 16
// KiB take 6 us longer there, or 110 us (seen after a 2 GB allocation was
// freed), and those to ordinary memory 12.5 and 60 us, or 130 and 145.
// Where no page-locked memory is to be had, HIP's copy to ordinary memory it is.
void Backend::download(void* dst, const void* src, size_t bytes) {
  const size_t mib = (size_t)1 << 20;
  const int threads = bytes >= 4 * mib ? kCopyThreads : 1;
  hipPointerAttribute_t at{};
  // memory the runtime knows (page-locked by the caller): the device copies there directly
  bool direct = bytes && hipPointerGetAttributes(&at, dst) == hipSuccess && at.type != hipMemoryTypeUnregistered;
  if (bytes && !direct) {
    (void)hipGetLastError();  // of an address that the runtime does not know
    direct = !slots_ready(bytes <= mib ? 1 : 2 * threads);
  }
  if (direct) DW_HIP(hipMemcpyAsync(dst, src, bytes, hipMemcpyDeviceToHost, stream));
  if (direct || !bytes) {
    DW_HIP(hipStreamSynchronize(stream));
    return;
  }
  uint8_t* d = (uint8_t*)dst;
  const uint8_t* s = (const uint8_t*)src;
  if (bytes <= mib) {
    launch_copy(stream, s, slots[0].p, (unsigned)bytes, slots[0].ev);
    DW_HIP(hipEventSynchronize(slots[0].ev));
    memcpy(d, slots[0].p, bytes);
    return;
  }
  // a chunk costs about 10 us beside its bytes, which half a MiB hides; large
  // downloads take whole slots
  const size_t chunk = bytes >= 16 * mib ? kSlotBytes : std::min(mib, (bytes / 2 + 4095) & ~(size_t)4095);
  hipError_t err[kCopyThreads] = {};
  std::thread helper[kCopyThreads];
  for (int t = 1; t < threads; ++t) try {
      helper[t] = std::thread([=, &err] { err[t] = copy_chunks(d, s, bytes, chunk, t, threads); });
    } catch (const std::exception&) {
      // no thread to be had: its share is copied below
    }
  err[0] = copy_chunks(d, s, bytes, chunk, 0, threads);
  for (int t = 1; t < threads; ++t) {
    if (helper[t].joinable())
      helper[t].join();
    else
      err[t] = copy_chunks(d, s, bytes, chunk, t, threads);
  }
  for (hipError_t e : err) hip_check(e, "download");
}

Backend::~Backend() {
  if (stream) {
    (void)hipStreamSynchronize(stream);
    for (auto& s : slots) {
      if (s.p) (void)hipHostFree(s.p);
      if (s.ev) (void)hipEventDestroy(s.ev);
    }
    for (auto& w : ws)
      if (w.ptr) (void)hipFree(w.ptr);
    (void)hipStreamDestroy(stream);
  }
}

}  // namespace dw

using dw::Backend;

struct dw_hip_buffer {
  Backend* be;
  void* ptr;
  size_t len;
};

#define API_BEGIN try {
#define API_END                                     \
  }                                                 \
  catch (const dw::Error& e) {                      \
    dw::set_last_error(e.msg);                      \
    return e.code;                                  \
  }                                                 \
  catch (const std::exception& e) {                 \
    dw::set_last_error(e.what());                   \
    return DW_ERR_BACKEND;                          \
  }                                                 \
  return DW_OK;

namespace {

Backend* B(dw_hip_backend* be) {
  if (!be) dw::fail(DW_ERR_INVALID, "null backend");
  Backend* b = reinterpret_cast<Backend*>(be);
  DW_HIP(hipSetDevice(b->device));
  return b;
}

void need(const dw_hip_buffer* b, size_t bytes, const char* what) {
  if (!b) dw::fail(DW_ERR_INVALID, std::string(what) + ": null buffer");
  if (b->len != bytes)
    dw::fail(DW_ERR_INVALID, std::string(what) + " mismatch: expected " + std::to_string(bytes) +
                                 ", got " + std::to_string(b->len));
}

void check_i32(size_t v, const char* what) {
  if (v >= (size_t)INT32_MAX) dw::fail(DW_ERR_UNSUPPORTED, std::string(what) + " exceeds 2^31");
}

struct Geo {
  size_t n, h, w, ci, co, kh, kw, sh, sw, ph, pw, ho, wo;
};

Geo geo(size_t n, size_t h, size_t w, size_t ci, size_t co, size_t kh, size_t kw, size_t sh,
        size_t sw, size_t ph, size_t pw) {
  if (!n || !h || !w || !ci || !co || !kh || !kw || !sh || !sw)
    dw::fail(DW_ERR_INVALID, "conv: zero-sized dimension");
  if (h + 2 * ph < kh || w + 2 * pw < kw) dw::fail(DW_ERR_INVALID, "conv: kernel larger than padded input");
  Geo g{n, h, w, ci, co, kh, kw, sh, sw, ph, pw, (h + 2 * ph - kh) / sh + 1, (w + 2 * pw - kw) / sw + 1};
  check_i32(n * h * w * ci * 4, "input bytes");
  check_i32(n * g.ho * g.wo * co * 4, "output bytes");
  return g;
}

dw::DirectArgs direct_args(const Geo& g, const void* x, const float* wf, void* y) {
  dw::DirectArgs a{};
  a.x = x;
  a.wf = wf;
  a.y = y;
  a.n = (int)g.n; a.h = (int)g.h; a.w = (int)g.w; a.cin = (int)g.ci; a.cout = (int)g.co;
  a.kh = (int)g.kh; a.kw = (int)g.kw; a.sh = (int)g.sh; a.sw = (int)g.sw;
  a.pt = (int)g.ph; a.pl = (int)g.pw; a.ho = (int)g.ho; a.wo = (int)g.wo;
  a.m = (int)(g.n * g.ho * g.wo);
  a.x_pix_stride = (int)g.ci; a.x_c_off = 0;
  a.y_pix_stride = (int)g.co; a.y_c_off = 0;
  return a;
}

dw::IgemmArgs igemm_args(const Geo& g, const void* x, const void* wpk, void* y, int esize) {
  dw::IgemmArgs a{};
  a.x = (const uint8_t*)x;
  a.wpk = (const uint8_t*)wpk;
  a.y = y;
  a.n = (int)g.n; a.h = (int)g.h; a.w = (int)g.w; a.cin = (int)g.ci; a.cout = (int)g.co;
  a.kh = (int)g.kh; a.kw = (int)g.kw; a.sh = (int)g.sh; a.sw = (int)g.sw;
  a.pt = (int)g.ph; a.pl = (int)g.pw; a.ho = (int)g.ho; a.wo = (int)g.wo;
  a.m = (int)(g.n * g.ho * g.wo);
  const size_t kbytes = g.kh * g.kw * g.ci * esize;
  a.ksteps = (int)((kbytes + 63) / 64);
  const int bc = dw::igemm_channel_tile((int)g.co);
  a.cout_pad = (int)((g.co + bc - 1) / bc * bc);
  a.x_pix_stride = (int)g.ci; a.x_c_off = 0;
  a.y_pix_stride = (int)g.co; a.y_c_off = 0;
  a.r_pix_stride = (int)g.co; a.r_c_off = 0;
  return a;
}

void require_igemm(const Geo& g, int esize) {
  if ((g.ci * esize) % 16 != 0)
    dw::fail(DW_ERR_UNSUPPORTED, "MFMA conv needs c_in*esize % 16 == 0 (got c_in=" +
                                     std::to_string(g.ci) + ")");
  if (g.co % 4 != 0) dw::fail(DW_ERR_UNSUPPORTED, "MFMA conv needs c_out % 4 == 0");
  if (g.kh * g.kw > 31) dw::fail(DW_ERR_UNSUPPORTED, "MFMA conv supports at most 31 filter taps");
}

// Packs HWIO weights into workspace slot 0 and returns the pointer.
void* pack_into_ws(Backend* b, const dw_hip_buffer* kernel, const dw::IgemmArgs& a, const Geo& g,
                   int esize) {
  const size_t bytes = (size_t)a.ksteps * a.cout_pad * 64;
  void* wpk = b->workspace(Backend::WS_WPACK, bytes);
  dw::launch_pack_weights(b->stream, kernel->ptr, wpk, (int)(g.kh * g.kw * g.ci), (int)g.co,
                          a.cout_pad, a.ksteps, esize);
  return wpk;
}

void ew(Backend* b, int op, int dtype, const dw_hip_buffer* x, const dw_hip_buffer* y2,
        dw_hip_buffer* y, size_t count, size_t in_es, size_t out_es, float s0 = 0, float s1 = 0,
        int z0 = 0, int z1 = 0, int z2 = 0, float s2 = 0, const uint8_t* lut = nullptr) {
  need(x, count * in_es, "input");
  if (y2) need(y2, count * in_es, "input b");
  need(y, count * out_es, "output");
  dw::EwArgs a{};
  a.op = op; a.dtype = dtype; a.a = x->ptr; a.b = y2 ? y2->ptr : nullptr; a.y = y->ptr;
  a.count = count; a.c = 1; a.s0 = s0; a.s1 = s1; a.s2 = s2; a.z0 = z0; a.z1 = z1; a.z2 = z2;
  a.lut = lut;
  dw::launch_elementwise(b->stream, a);
}

}  // namespace

extern "C" {

const char* dw_last_error(void) { return dw::g_last_error.c_str(); }

int dw_hip_backend_create(int device, dw_hip_backend** out) {
  API_BEGIN
  if (!out) dw::fail(DW_ERR_INVALID, "null out");
  int count = 0;
  DW_HIP(hipGetDeviceCount(&count));
  if (device < 0 || device >= count)
    dw::fail(DW_ERR_BACKEND, "no HIP device " + std::to_string(device) + " (found " +
                                 std::to_string(count) + ")");
  DW_HIP(hipSetDevice(device));
  hipDeviceProp_t prop;
  DW_HIP(hipGetDeviceProperties(&prop, device));
  if (strncmp(prop.gcnArchName, "gfx950", 6) != 0)
    dw::fail(DW_ERR_UNSUPPORTED, std::string("device is ") + prop.gcnArchName + ", need gfx950");
  void* scratch = dw::noalloc_scratch_setup(device);
  Backend* b = new Backend();
  b->device = device;
  b->num_cus = prop.multiProcessorCount;
  b->scratch = scratch;
  DW_HIP(hipStreamCreateWithFlags(&b->stream, hipStreamNonBlocking));
  *out = reinterpret_cast<dw_hip_backend*>(b);
  API_END
}

void dw_hip_backend_destroy(dw_hip_backend* be) {
  if (be) dw::release(reinterpret_cast<Backend*>(be));
}

const char* dw_hip_backend_name(const dw_hip_backend* be) {
  (void)be;
  return "hip-gfx950";
}

int dw_hip_alloc(dw_hip_backend* be, size_t len_bytes, int kind, dw_hip_buffer** out) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  if (kind != DW_BUFFER_STORAGE) dw::fail(DW_ERR_UNSUPPORTED, "unknown buffer kind");
  if (!out) dw::fail(DW_ERR_INVALID, "null out");
  void* p = nullptr;
  dw::hip_check(hipMalloc(&p, std::max<size_t>(len_bytes, 1)),
                ("alloc of " + std::to_string(len_bytes) + " bytes failed").c_str());
  *out = new dw_hip_buffer{b, p, len_bytes};
  dw::hold(b);
  API_END
}

void dw_hip_buffer_free(dw_hip_buffer* buf) {
  if (!buf) return;
  Backend* b = buf->be;
  (void)hipSetDevice(b->device);
  (void)hipStreamSynchronize(b->stream);
  (void)hipFree(buf->ptr);
  delete buf;
  dw::release(b);
}

size_t dw_hip_buffer_len_bytes(const dw_hip_buffer* buf) { return buf ? buf->len : 0; }
void* dw_hip_buffer_device_ptr(const dw_hip_buffer* buf) { return buf ? buf->ptr : nullptr; }

int dw_hip_upload(dw_hip_backend* be, dw_hip_buffer* dst, const void* src, size_t len) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  if (!dst) dw::fail(DW_ERR_INVALID, "null buffer");
  if (len != dst->len)
    dw::fail(DW_ERR_INVALID, "upload size mismatch: buffer " + std::to_string(dst->len) +
                                 " bytes, source " + std::to_string(len) + " bytes");
  if (len) {
    DW_HIP(hipMemcpyAsync(dst->ptr, src, len, hipMemcpyHostToDevice, b->stream));
    DW_HIP(hipStreamSynchronize(b->stream));
  }
  API_END
}

int dw_hip_download(dw_hip_backend* be, const dw_hip_buffer* src, void* dst, size_t len) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  if (!src) dw::fail(DW_ERR_INVALID, "null buffer");
  if (len != src->len)
    dw::fail(DW_ERR_INVALID, "download size mismatch: buffer " + std::to_string(src->len) +
                                 " bytes, destination " + std::to_string(len) + " bytes");
  if (len && !dst) dw::fail(DW_ERR_INVALID, "null destination");
  b->download(dst, src->ptr, len);
  API_END
}

int dw_hip_synchronize(dw_hip_backend* be) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  DW_HIP(hipStreamSynchronize(b->stream));
  API_END
}

// ---------------------------------------------------------------------------
// Convolutions
// ---------------------------------------------------------------------------

static int conv_f32_common(dw_hip_backend* be, const dw_hip_buffer* input, const dw_hip_buffer* kernel,
                           const dw_hip_buffer* bias, dw_hip_buffer* output, size_t n, size_t h_in,
                           size_t w_in, size_t c_in, size_t c_out, size_t k_h, size_t k_w,
                           size_t stride_h, size_t stride_w, size_t pad_h, size_t pad_w, int act) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  Geo g = geo(n, h_in, w_in, c_in, c_out, k_h, k_w, stride_h, stride_w, pad_h, pad_w);
  need(input, n * h_in * w_in * c_in * 4, "conv2d_f32: input");
  need(kernel, k_h * k_w * c_in * c_out * 4, "conv2d_f32: kernel");
  need(output, n * g.ho * g.wo * c_out * 4, "conv2d_f32: output");
  if (bias) need(bias, c_out * 4, "conv2d_f32: bias");
  dw::DirectArgs a = direct_args(g, input->ptr, (const float*)kernel->ptr, output->ptr);
  a.in_kind = 0;
  a.out_kind = 0;
  a.act = act;
  a.bias_f = bias ? (const float*)bias->ptr : nullptr;
  if (dw::conv_window_f32_ok(a)) {
    float* wq = (float*)b->workspace(Backend::WS_WPACK, k_h * k_w * c_in * c_out * 4);
    dw::launch_repack_oc4(b->stream, (const float*)kernel->ptr, wq, (int)(k_h * k_w * c_in), (int)c_out);
    a.wq = wq;
  }
  dw::launch_direct_conv(b->stream, a);
  API_END
}

int dw_hip_conv2d_f32_nhwc(dw_hip_backend* be, const dw_hip_buffer* input, const dw_hip_buffer* kernel,
                           dw_hip_buffer* output, size_t n, size_t h_in, size_t w_in, size_t c_in,
                           size_t c_out, size_t k_h, size_t k_w, size_t stride_h, size_t stride_w,
                           size_t pad_h, size_t pad_w) {
  return conv_f32_common(be, input, kernel, nullptr, output, n, h_in, w_in, c_in, c_out, k_h, k_w,
                         stride_h, stride_w, pad_h, pad_w, DW_ACT_NONE);
}

int dw_hip_conv2d_bias_act_f32_nhwc(dw_hip_backend* be, const dw_hip_buffer* input,
                                    const dw_hip_buffer* kernel, const dw_hip_buffer* bias,
                                    dw_hip_buffer* output, size_t n, size_t h_in, size_t w_in,
                                    size_t c_in, size_t c_out, size_t k_h, size_t k_w,
                                    size_t stride_h, size_t stride_w, size_t pad_h, size_t pad_w,
                                    int act) {
  return conv_f32_common(be, input, kernel, bias, output, n, h_in, w_in, c_in, c_out, k_h, k_w,
                         stride_h, stride_w, pad_h, pad_w, act);
}

int dw_hip_conv2d_bias_act_f16_nhwc(dw_hip_backend* be, const dw_hip_buffer* input,
                                    const dw_hip_buffer* kernel, const dw_hip_buffer* bias,
                                    dw_hip_buffer* output, size_t n, size_t h_in, size_t w_in,
                                    size_t c_in, size_t c_out, size_t k_h, size_t k_w,
                                    size_t stride_h, size_t stride_w, size_t pad_h, size_t pad_w,
                                    int act, int exact) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  Geo g = geo(n, h_in, w_in, c_in, c_out, k_h, k_w, stride_h, stride_w, pad_h, pad_w);
  need(input, n * h_in * w_in * c_in * 2, "conv2d_fp16: input");
  need(kernel, k_h * k_w * c_in * c_out * 2, "conv2d_fp16: kernel");
  need(output, n * g.ho * g.wo * c_out * 2, "conv2d_fp16: output");
  if (bias) need(bias, c_out * 2, "conv2d_fp16: bias");
  if (exact) {
    const size_t kcount = k_h * k_w * c_in * c_out;
    float* wf = (float*)b->workspace(Backend::WS_WPACK, kcount * 4);
    dw::EwArgs e{};
    e.op = dw::EW_F16_TO_F32; e.a = kernel->ptr; e.y = wf; e.count = kcount;
    dw::launch_elementwise(b->stream, e);
    dw::DirectArgs a = direct_args(g, input->ptr, wf, output->ptr);
    a.in_kind = 1;
    a.out_kind = 1;
    a.act = act;
    a.bias_h = bias ? (const uint16_t*)bias->ptr : nullptr;
    dw::launch_direct_conv(b->stream, a);
  } else {
    require_igemm(g, 2);
    dw::IgemmArgs a = igemm_args(g, input->ptr, nullptr, output->ptr, 2);
    a.wpk = (const uint8_t*)pack_into_ws(b, kernel, a, g, 2);
    a.epi = dw::EPI_F16;
    a.act = act;
    a.bias_h = bias ? (const uint16_t*)bias->ptr : nullptr;
    dw::launch_igemm(b->stream, a, 2);
  }
  API_END
}

static int dwconv_common(dw_hip_backend* be, int dtype, const dw_hip_buffer* input,
                         const dw_hip_buffer* kernel, const dw_hip_buffer* bias, dw_hip_buffer* output,
                         size_t n, size_t h_in, size_t w_in, size_t c, size_t k_h, size_t k_w,
                         size_t stride_h, size_t stride_w, size_t pad_h, size_t pad_w, int act) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  const size_t es = dtype == DW_DTYPE_F16 ? 2 : 4;
  Geo g = geo(n, h_in, w_in, c, c, k_h, k_w, stride_h, stride_w, pad_h, pad_w);
  // 3x3 with stride 1 or 2 runs on the row-marching kernel (in f16 with channel
  // groups of 4); every other shape on the generic one (groups of 8)
  const bool march = dtype == DW_DTYPE_F16 && k_h == 3 && k_w == 3 && (stride_w == 1 || stride_w == 2);
  if (c % (march ? 4 : 8) != 0)
    dw::fail(DW_ERR_UNSUPPORTED, march ? "depthwise: c must be a multiple of 4" : "depthwise: c must be a multiple of 8");
  need(input, n * h_in * w_in * c * es, "depthwise: input");
  need(kernel, k_h * k_w * c * es, "depthwise: kernel");
  need(output, n * g.ho * g.wo * c * es, "depthwise: output");
  if (bias) need(bias, c * es, "depthwise: bias");
  dw::DwArgs a{};
  a.x = input->ptr; a.wt = kernel->ptr; a.bias = bias ? bias->ptr : nullptr; a.y = output->ptr;
  a.n = (int)n; a.h = (int)h_in; a.w = (int)w_in; a.c = (int)c; a.kh = (int)k_h; a.kw = (int)k_w;
  a.sh = (int)stride_h; a.sw = (int)stride_w; a.pt = (int)pad_h; a.pl = (int)pad_w;
  a.ho = (int)g.ho; a.wo = (int)g.wo; a.act = act;
  a.x_pix_stride = (int)c; a.y_pix_stride = (int)c;
  dw::launch_dwconv(b->stream, a, dtype == DW_DTYPE_F16 ? dw::F16 : dw::F32);
  API_END
}

int dw_hip_depthwise_conv2d_f16_nhwc(dw_hip_backend* be, const dw_hip_buffer* input,
                                     const dw_hip_buffer* kernel, const dw_hip_buffer* bias,
                                     dw_hip_buffer* output, size_t n, size_t h_in, size_t w_in,
                                     size_t c, size_t k_h, size_t k_w, size_t stride_h,
                                     size_t stride_w, size_t pad_h, size_t pad_w, int act) {
  return dwconv_common(be, DW_DTYPE_F16, input, kernel, bias, output, n, h_in, w_in, c, k_h, k_w,
                       stride_h, stride_w, pad_h, pad_w, act);
}

int dw_hip_depthwise_conv2d_f32_nhwc(dw_hip_backend* be, const dw_hip_buffer* input,
                                     const dw_hip_buffer* kernel, const dw_hip_buffer* bias,
                                     dw_hip_buffer* output, size_t n, size_t h_in, size_t w_in,
                                     size_t c, size_t k_h, size_t k_w, size_t stride_h,
                                     size_t stride_w, size_t pad_h, size_t pad_w, int act) {
  return dwconv_common(be, DW_DTYPE_F32, input, kernel, bias, output, n, h_in, w_in, c, k_h, k_w,
                       stride_h, stride_w, pad_h, pad_w, act);
}

namespace {

// Where a QLinearConv's per-call device data goes: the backend's grow-only
// workspaces (wpk == nullptr), or caller-provided space of fixed capacity.
struct QconvSpace {
  void* wpk = nullptr;
  size_t wpk_cap = 0;
  float* ms = nullptr;
  int* bi = nullptr;
};

void qlinearconv_impl(Backend* b, const dw_hip_buffer* input, const dw_hip_buffer* kernel,
                      const dw_hip_buffer* bias, dw_hip_buffer* output, size_t n, size_t h_in, size_t w_in,
                      size_t c_in, size_t c_out, size_t k_h, size_t k_w, size_t stride_h, size_t stride_w,
                      size_t pad_h, size_t pad_w, float x_scale, int x_zp, const float* w_scales,
                      float y_scale, int y_zp, QconvSpace sp, float* m_host) {
  Geo g = geo(n, h_in, w_in, c_in, c_out, k_h, k_w, stride_h, stride_w, pad_h, pad_w);
  require_igemm(g, 1);
  need(input, n * h_in * w_in * c_in, "qlinearconv: input");
  need(kernel, k_h * k_w * c_in * c_out, "qlinearconv: kernel");
  need(output, n * g.ho * g.wo * c_out, "qlinearconv: output");
  if (bias) need(bias, c_out * 4, "qlinearconv: bias");
  if (!w_scales) dw::fail(DW_ERR_INVALID, "qlinearconv: null w_scales");
  if (x_zp < 0 || x_zp > 255 || y_zp < 0 || y_zp > 255)
    dw::fail(DW_ERR_INVALID, "qlinearconv: zero points must be in [0, 255]");
  if (!(x_scale > 0) || !(y_scale > 0)) dw::fail(DW_ERR_INVALID, "qlinearconv: scales must be > 0");
  for (size_t c = 0; c < c_out; ++c) {
    if (!(w_scales[c] > 0)) dw::fail(DW_ERR_INVALID, "qlinearconv: weight scales must be > 0");
    m_host[c] = (x_scale * w_scales[c]) / y_scale;
  }
  dw::IgemmArgs a = igemm_args(g, input->ptr, nullptr, output->ptr, 1);
  const size_t wpk_bytes = (size_t)a.ksteps * a.cout_pad * 64;
  if (sp.wpk) {
    if (wpk_bytes > sp.wpk_cap)
      dw::fail(DW_ERR_UNSUPPORTED, "qlinearconv: packed weights of " + std::to_string(wpk_bytes) +
                                       " bytes exceed the no-alloc scratch's " + std::to_string(sp.wpk_cap));
  } else {
    sp.wpk = b->workspace(Backend::WS_WPACK, wpk_bytes);
    sp.ms = (float*)b->workspace(Backend::WS_SCALE, c_out * 4);
    sp.bi = (int*)b->workspace(Backend::WS_BIAS, c_out * 4);
  }
  a.wpk = (const uint8_t*)sp.wpk;
  dw::launch_qconv_prep(b->stream, kernel->ptr, sp.wpk, bias ? (const int*)bias->ptr : nullptr, sp.bi, sp.ms, m_host,
                        (int)(k_h * k_w * c_in), (int)c_out, a.cout_pad, a.ksteps, 128 - x_zp);
  a.epi = dw::EPI_QU8;
  a.xxor = 0x80808080u;
  const uint32_t pb = (uint32_t)((x_zp ^ 0x80) & 0xff);
  a.xpad = pb * 0x01010101u;
  a.bias_i = sp.bi;
  a.mscale = sp.ms;
  a.y_zp = y_zp;
  dw::launch_igemm(b->stream, a, 1);
}

}  // namespace

int dw_hip_qlinearconv_u8s8(dw_hip_backend* be, const dw_hip_buffer* input, const dw_hip_buffer* kernel,
                            const dw_hip_buffer* bias, dw_hip_buffer* output, size_t n, size_t h_in,
                            size_t w_in, size_t c_in, size_t c_out, size_t k_h, size_t k_w,
                            size_t stride_h, size_t stride_w, size_t pad_h, size_t pad_w,
                            float x_scale, int x_zp, const float* w_scales, float y_scale, int y_zp) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  std::vector<float> m(c_out);
  qlinearconv_impl(b, input, kernel, bias, output, n, h_in, w_in, c_in, c_out, k_h, k_w, stride_h, stride_w,
                   pad_h, pad_w, x_scale, x_zp, w_scales, y_scale, y_zp, QconvSpace{}, m.data());
  API_END
}

int dw_hip_qlinearconv_u8s8_noalloc(dw_hip_backend* be, const dw_hip_buffer* input, const dw_hip_buffer* kernel,
                                    const dw_hip_buffer* bias, dw_hip_buffer* output, size_t n, size_t h_in,
                                    size_t w_in, size_t c_in, size_t c_out, size_t k_h, size_t k_w,
                                    size_t stride_h, size_t stride_w, size_t pad_h, size_t pad_w,
                                    float x_scale, int x_zp, const float* w_scales, float y_scale, int y_zp) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  if (!b->scratch) dw::fail(DW_ERR_BACKEND, "qlinearconv_noalloc: no scratch on this device");
  if (c_out > dw::kNoAllocMaxChannels)
    dw::fail(DW_ERR_UNSUPPORTED, "qlinearconv_noalloc: c_out above " + std::to_string(dw::kNoAllocMaxChannels));
  float m[dw::kNoAllocMaxChannels];
  dw::ScratchUse use(b->device, b->stream);
  QconvSpace sp;
  uint8_t* base = (uint8_t*)b->scratch;
  sp.ms = (float*)base;
  sp.bi = (int*)(base + dw::kNoAllocMaxChannels * 4);
  sp.wpk = base + dw::kNoAllocTableBytes;
  sp.wpk_cap = dw::kNoAllocScratchBytes - dw::kNoAllocTableBytes;
  qlinearconv_impl(b, input, kernel, bias, output, n, h_in, w_in, c_in, c_out, k_h, k_w, stride_h, stride_w,
                   pad_h, pad_w, x_scale, x_zp, w_scales, y_scale, y_zp, sp, m);
  API_END
}

int dw_hip_qgemm_u8s8(dw_hip_backend* be, const dw_hip_buffer* a, const dw_hip_buffer* b, const dw_hip_buffer* bias,
                      dw_hip_buffer* y, size_t m, size_t n, size_t k, int trans_b, float a_scale, int a_zp,
                      const float* b_scales, float y_scale, int y_zp) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  if (!m || !n || !k) dw::fail(DW_ERR_INVALID, "qgemm: zero size");
  check_i32(m * k, "qgemm: A");
  check_i32(k * n, "qgemm: B");
  need(b, k * n, "qgemm: B");
  // B as [k][n] (the 1x1 HWIO layout); a transposed B goes through a
  // workspace copy first
  dw_hip_buffer bt{bk, b->ptr, b->len};
  if (trans_b) {
    bt.ptr = bk->workspace(Backend::WS_POST, k * n);
    dw::launch_transpose_u8(bk->stream, b->ptr, bt.ptr, (int)n, (int)k);
  }
  std::vector<float> ms(n);
  // rows of A are the pixels of a 1x1 convolution over n = m images of 1 x 1
  qlinearconv_impl(bk, a, &bt, bias, y, m, 1, 1, k, n, 1, 1, 1, 1, 0, 0, a_scale, a_zp, b_scales, y_scale, y_zp,
                   QconvSpace{}, ms.data());
  API_END
}

int dw_hip_qlinear_global_avg_pool_u8(dw_hip_backend* be, const dw_hip_buffer* x, dw_hip_buffer* y, size_t n,
                                      size_t h, size_t w, size_t c, float x_scale, int x_zp, float y_scale,
                                      int y_zp) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  if (!n || !h || !w || !c) dw::fail(DW_ERR_INVALID, "qlinear_gap: zero size");
  check_i32(n * h * w * c, "qlinear_gap: input");
  if (h * w > (size_t)(1 << 23)) dw::fail(DW_ERR_UNSUPPORTED, "qlinear_gap: more than 2^23 pixels per image");
  if (!(x_scale > 0) || !(y_scale > 0)) dw::fail(DW_ERR_INVALID, "qlinear_gap: scales must be > 0");
  if (x_zp < 0 || x_zp > 255 || y_zp < 0 || y_zp > 255) dw::fail(DW_ERR_INVALID, "qlinear_gap: zero points");
  need(x, n * h * w * c, "qlinear_gap: input");
  need(y, n * c, "qlinear_gap: output");
  const float m = (x_scale / y_scale) / (float)(h * w);
  dw::launch_qlinear_gap(bk->stream, (const uint8_t*)x->ptr, (uint8_t*)y->ptr, (int)n, (int)(h * w), (int)c, x_zp, m,
                         y_zp);
  API_END
}

int dw_hip_conv2d_i8_nhwc(dw_hip_backend* be, const dw_hip_buffer* input, const dw_hip_buffer* kernel,
                          dw_hip_buffer* output_i32, size_t n, size_t h_in, size_t w_in, size_t c_in,
                          size_t c_out, size_t k_h, size_t k_w, size_t stride_h, size_t stride_w,
                          size_t pad_h, size_t pad_w) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  Geo g = geo(n, h_in, w_in, c_in, c_out, k_h, k_w, stride_h, stride_w, pad_h, pad_w);
  require_igemm(g, 1);
  need(input, n * h_in * w_in * c_in, "conv2d_i8: input");
  need(kernel, k_h * k_w * c_in * c_out, "conv2d_i8: kernel");
  need(output_i32, n * g.ho * g.wo * c_out * 4, "conv2d_i8: output");
  dw::IgemmArgs a = igemm_args(g, input->ptr, nullptr, output_i32->ptr, 1);
  a.wpk = (const uint8_t*)pack_into_ws(b, kernel, a, g, 1);
  a.epi = dw::EPI_I32;
  dw::launch_igemm(b->stream, a, 1);
  API_END
}

int dw_hip_conv2d_requant_relu_i8(dw_hip_backend* be, const dw_hip_buffer* input,
                                  const dw_hip_buffer* kernel, dw_hip_buffer* output, size_t n,
                                  size_t h_in, size_t w_in, size_t c_in, size_t c_out, size_t k_h,
                                  size_t k_w, size_t stride_h, size_t stride_w, size_t pad_h,
                                  size_t pad_w, float requant_scale, int do_relu) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  Geo g = geo(n, h_in, w_in, c_in, c_out, k_h, k_w, stride_h, stride_w, pad_h, pad_w);
  require_igemm(g, 1);
  need(input, n * h_in * w_in * c_in, "conv_fused: input");
  need(kernel, k_h * k_w * c_in * c_out, "conv_fused: kernel");
  need(output, n * g.ho * g.wo * c_out, "conv_fused: output");
  dw::IgemmArgs a = igemm_args(g, input->ptr, nullptr, output->ptr, 1);
  a.wpk = (const uint8_t*)pack_into_ws(b, kernel, a, g, 1);
  a.epi = dw::EPI_QS8_REF;
  a.tscale = requant_scale;
  a.act = do_relu ? dw::ACT_RELU : dw::ACT_NONE;
  dw::launch_igemm(b->stream, a, 1);
  API_END
}

// ---------------------------------------------------------------------------
// Elementwise
// ---------------------------------------------------------------------------
#define EW1(NAME, OP, DT, IES, OES)                                                              \
  int NAME(dw_hip_backend* be, const dw_hip_buffer* x, dw_hip_buffer* y, size_t count) {         \
    API_BEGIN Backend* b = B(be); std::lock_guard<std::mutex> lock(b->mu);                       \
    ew(b, OP, DT, x, nullptr, y, count, IES, OES);                                              \
    API_END                                                                                      \
  }
#define EW2(NAME, OP, DT, ES)                                                                    \
  int NAME(dw_hip_backend* be, const dw_hip_buffer* a, const dw_hip_buffer* bb, dw_hip_buffer* y, \
           size_t count) {                                                                       \
    API_BEGIN Backend* b = B(be); std::lock_guard<std::mutex> lock(b->mu);                       \
    ew(b, OP, DT, a, bb, y, count, ES, ES);                                                     \
    API_END                                                                                      \
  }

EW1(dw_hip_relu_f32, dw::EW_RELU, dw::F32, 4, 4)
EW1(dw_hip_relu_fp16, dw::EW_RELU, dw::F16, 2, 2)
EW1(dw_hip_sigmoid_f32, dw::EW_SIGMOID, dw::F32, 4, 4)
EW1(dw_hip_sigmoid_fp16, dw::EW_SIGMOID, dw::F16, 2, 2)
EW1(dw_hip_silu_f32, dw::EW_SILU, dw::F32, 4, 4)
EW1(dw_hip_silu_fp16, dw::EW_SILU, dw::F16, 2, 2)
EW1(dw_hip_relu_i8, dw::EW_RELU_I8, dw::I8, 1, 1)
EW2(dw_hip_add_f32, dw::EW_ADD, dw::F32, 4)
EW2(dw_hip_add_fp16, dw::EW_ADD, dw::F16, 2)
EW2(dw_hip_mul_f32, dw::EW_MUL, dw::F32, 4)
EW2(dw_hip_mul_fp16, dw::EW_MUL, dw::F16, 2)

int dw_hip_bias_add_f32_nhwc(dw_hip_backend* be, dw_hip_buffer* y, const dw_hip_buffer* bias,
                             size_t count, size_t c) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  need(y, count * 4, "bias_add: y");
  need(bias, c * 4, "bias_add: bias");
  if (c == 0 || count % c != 0) dw::fail(DW_ERR_INVALID, "bias_add: count must be a multiple of c");
  dw::EwArgs a{};
  a.op = dw::EW_BIAS_ADD; a.dtype = dw::F32; a.a = y->ptr; a.b = bias->ptr; a.y = y->ptr;
  a.count = count; a.c = (int)c;
  dw::launch_elementwise(b->stream, a);
  API_END
}

int dw_hip_requantize_i32_to_i8(dw_hip_backend* be, const dw_hip_buffer* x_i32, dw_hip_buffer* y_i8,
                                size_t count, float requant_scale) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  ew(b, dw::EW_REQUANT_I32_I8, dw::I32, x_i32, nullptr, y_i8, count, 4, 1, requant_scale);
  API_END
}

int dw_hip_quantize_f32_to_i8(dw_hip_backend* be, const dw_hip_buffer* x, dw_hip_buffer* y_i8,
                              size_t count, float scale) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  const float inv = 1.0f / scale;  // quantize_f32_to_i8 (ops.rs:3503-3516) multiplies by 1/scale
  ew(b, dw::EW_QUANT_F32_I8, dw::F32, x, nullptr, y_i8, count, 4, 1, inv);
  API_END
}

int dw_hip_dequantize_i8_to_f32(dw_hip_backend* be, const dw_hip_buffer* x_i8, dw_hip_buffer* y,
                                size_t count, float scale) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  ew(b, dw::EW_DEQUANT_I8_F32, dw::I8, x_i8, nullptr, y, count, 1, 4, scale);
  API_END
}

int dw_hip_add_i8(dw_hip_backend* be, const dw_hip_buffer* a, const dw_hip_buffer* bb, dw_hip_buffer* y,
                  size_t count, float scale_a_over_y, float scale_b_over_y) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  ew(b, dw::EW_ADD_I8, dw::I8, a, bb, y, count, 1, 1, scale_a_over_y, scale_b_over_y);
  API_END
}

int dw_hip_quantize_linear_f16_u8(dw_hip_backend* be, const dw_hip_buffer* x, dw_hip_buffer* y,
                                  size_t count, float scale, int zp) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  ew(b, dw::EW_QUANT_LINEAR_F16_U8, dw::F16, x, nullptr, y, count, 2, 1, scale, 0, zp);
  API_END
}

int dw_hip_dequantize_linear_u8_f16(dw_hip_backend* be, const dw_hip_buffer* x, dw_hip_buffer* y,
                                    size_t count, float scale, int zp) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  ew(b, dw::EW_DEQUANT_LINEAR_U8_F16, dw::U8, x, nullptr, y, count, 1, 2, scale, 0, zp);
  API_END
}

int dw_hip_qlinear_add_u8(dw_hip_backend* be, const dw_hip_buffer* a, const dw_hip_buffer* bb,
                          dw_hip_buffer* y, size_t count, float a_scale, int a_zp, float b_scale,
                          int b_zp, float y_scale, int y_zp) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  const float ra = a_scale / y_scale, rb = b_scale / y_scale;
  ew(b, dw::EW_QADD_U8, dw::U8, a, bb, y, count, 1, 1, ra, rb, a_zp, b_zp, y_zp);
  API_END
}

int dw_hip_lut_u8(dw_hip_backend* be, const dw_hip_buffer* x, dw_hip_buffer* y, size_t count,
                  const uint8_t* lut256) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  if (!lut256) dw::fail(DW_ERR_INVALID, "lut: null table");
  uint8_t* lut = (uint8_t*)b->workspace(Backend::WS_LUT, 256);
  b->upload_async(lut, lut256, 256);
  ew(b, dw::EW_LUT_U8, dw::U8, x, nullptr, y, count, 1, 1, 0, 0, 0, 0, 0, 0, lut);
  API_END
}

// ---------------------------------------------------------------------------
// Data movement
// ---------------------------------------------------------------------------

int dw_hip_maxpool2d_nhwc(dw_hip_backend* be, int dtype, const dw_hip_buffer* x, dw_hip_buffer* y,
                          size_t n, size_t h_in, size_t w_in, size_t c, size_t pool_h, size_t pool_w,
                          size_t stride_h, size_t stride_w, size_t pad_t, size_t pad_l, size_t pad_b,
                          size_t pad_r) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  if (dtype != DW_DTYPE_F32 && dtype != DW_DTYPE_F16 && dtype != DW_DTYPE_U8 && dtype != DW_DTYPE_I8)
    dw::fail(DW_ERR_UNSUPPORTED, "maxpool: dtype");
  if (!pool_h || !pool_w || !stride_h || !stride_w) dw::fail(DW_ERR_INVALID, "maxpool: zero size");
  if (pad_t >= pool_h || pad_b >= pool_h || pad_l >= pool_w || pad_r >= pool_w)
    dw::fail(DW_ERR_INVALID, "maxpool: pad must be smaller than the window");
  if (h_in + pad_t + pad_b < pool_h || w_in + pad_l + pad_r < pool_w)
    dw::fail(DW_ERR_INVALID, "maxpool: window larger than padded input");
  const size_t ho = (h_in + pad_t + pad_b - pool_h) / stride_h + 1;
  const size_t wo = (w_in + pad_l + pad_r - pool_w) / stride_w + 1;
  const size_t es = dw::dtype_size(dtype);
  need(x, n * h_in * w_in * c * es, "maxpool: input");
  need(y, n * ho * wo * c * es, "maxpool: output");
  dw::PoolArgs a{};
  a.x = {x->ptr, (int)c, 0};
  a.y = {y->ptr, (int)c, 0};
  a.n = (int)n; a.h = (int)h_in; a.w = (int)w_in; a.c = (int)c; a.kh = (int)pool_h; a.kw = (int)pool_w;
  a.sh = (int)stride_h; a.sw = (int)stride_w; a.pt = (int)pad_t; a.pl = (int)pad_l;
  a.ho = (int)ho; a.wo = (int)wo;
  dw::launch_maxpool(b->stream, a, dtype);
  API_END
}

int dw_hip_resize_nearest_nhwc(dw_hip_backend* be, int dtype, const dw_hip_buffer* x, dw_hip_buffer* y,
                               size_t n, size_t h_in, size_t w_in, size_t h_out, size_t w_out, size_t c) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  const size_t es = dw::dtype_size(dtype);
  if (!h_in || !w_in || !h_out || !w_out) dw::fail(DW_ERR_INVALID, "resize: zero size");
  need(x, n * h_in * w_in * c * es, "resize: input");
  need(y, n * h_out * w_out * c * es, "resize: output");
  dw::ResizeArgs a{};
  a.x = {x->ptr, (int)c, 0};
  a.y = {y->ptr, (int)c, 0};
  a.n = (int)n; a.h = (int)h_in; a.w = (int)w_in; a.c = (int)c; a.ho = (int)h_out; a.wo = (int)w_out;
  dw::launch_resize_nearest(b->stream, a, dtype);
  API_END
}

int dw_hip_concat_channels_nhwc(dw_hip_backend* be, int dtype, const dw_hip_buffer* const* inputs,
                                const size_t* channels, size_t num_inputs, dw_hip_buffer* y,
                                size_t pixels) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  const size_t es = dw::dtype_size(dtype);
  size_t total = 0;
  for (size_t i = 0; i < num_inputs; ++i) total += channels[i];
  need(y, pixels * total * es, "concat: output");
  size_t off = 0;
  for (size_t i = 0; i < num_inputs; ++i) {
    need(inputs[i], pixels * channels[i] * es, "concat: input");
    dw::launch_copy_channels(b->stream, {inputs[i]->ptr, (int)channels[i], 0},
                             {y->ptr, (int)total, (int)off}, (int)pixels, (int)channels[i], (int)es);
    off += channels[i];
  }
  API_END
}

int dw_hip_split_channels_nhwc(dw_hip_backend* be, int dtype, const dw_hip_buffer* x,
                               dw_hip_buffer* const* outputs, const size_t* channels,
                               size_t num_outputs, size_t pixels) {
  API_BEGIN
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  const size_t es = dw::dtype_size(dtype);
  size_t total = 0;
  for (size_t i = 0; i < num_outputs; ++i) total += channels[i];
  need(x, pixels * total * es, "split: input");
  size_t off = 0;
  for (size_t i = 0; i < num_outputs; ++i) {
    need(outputs[i], pixels * channels[i] * es, "split: output");
    dw::launch_copy_channels(b->stream, {x->ptr, (int)total, (int)off},
                             {outputs[i]->ptr, (int)channels[i], 0}, (int)pixels, (int)channels[i],
                             (int)es);
    off += channels[i];
  }
  API_END
}

// Classifier-head ops (see dw_hip.h for the reference functions each mirrors).
int dw_hip_gemm_f32(dw_hip_backend* be, const dw_hip_buffer* a, const dw_hip_buffer* b, dw_hip_buffer* c,
                    size_t m, size_t n, size_t k) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  if (!m || !n || !k) dw::fail(DW_ERR_INVALID, "gemm_f32: zero size");
  if (m > 65535 || n > INT32_MAX || k > INT32_MAX) dw::fail(DW_ERR_UNSUPPORTED, "gemm_f32: m > 65535 or n, k > 2^31 - 1");
  need(a, m * k * 4, "gemm_f32: A size");
  need(b, k * n * 4, "gemm_f32: B size");
  need(c, m * n * 4, "gemm_f32: C size");
  dw::launch_gemm(bk->stream, dw::F32, a->ptr, b->ptr, c->ptr, (int)m, (int)n, (int)k);
  API_END
}

int dw_hip_gemm_fp16(dw_hip_backend* be, const dw_hip_buffer* a, const dw_hip_buffer* b, dw_hip_buffer* c,
                     size_t m, size_t n, size_t k) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  if (!m || !n || !k) dw::fail(DW_ERR_INVALID, "gemm_fp16: zero size");
  if (m > 65535 || n > INT32_MAX || k > INT32_MAX) dw::fail(DW_ERR_UNSUPPORTED, "gemm_fp16: m > 65535 or n, k > 2^31 - 1");
  need(a, m * k * 2, "gemm_fp16: A size");
  need(b, k * n * 2, "gemm_fp16: B size");
  need(c, m * n * 2, "gemm_fp16: C size");
  dw::launch_gemm(bk->stream, dw::F16, a->ptr, b->ptr, c->ptr, (int)m, (int)n, (int)k);
  API_END
}

int dw_hip_gemm_i8(dw_hip_backend* be, const dw_hip_buffer* a, const dw_hip_buffer* b, dw_hip_buffer* c_i32,
                   size_t m, size_t n, size_t k) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  if (!m || !n || !k) dw::fail(DW_ERR_INVALID, "gemm_i8: zero size");
  if (m > 65535 || n > INT32_MAX || k > INT32_MAX) dw::fail(DW_ERR_UNSUPPORTED, "gemm_i8: m > 65535 or n, k > 2^31 - 1");
  need(a, m * k, "gemm_i8: A size");
  need(b, k * n, "gemm_i8: B size");
  need(c_i32, m * n * 4, "gemm_i8: C size");
  dw::launch_gemm(bk->stream, dw::I8, a->ptr, b->ptr, c_i32->ptr, (int)m, (int)n, (int)k);
  API_END
}

int dw_hip_global_avg_pool_nhwc(dw_hip_backend* be, int dtype, const dw_hip_buffer* x, dw_hip_buffer* y,
                                size_t n, size_t h, size_t w, size_t c) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  if (dtype != DW_DTYPE_F32 && dtype != DW_DTYPE_F16)
    dw::fail(DW_ERR_UNSUPPORTED, "global_avg_pool: unsupported dtype");
  if (!n || !h || !w || !c) dw::fail(DW_ERR_INVALID, "global_avg_pool: zero size");
  if (h * w > INT32_MAX || n > 65535 || c > INT32_MAX) dw::fail(DW_ERR_UNSUPPORTED, "global_avg_pool: size");
  const size_t es = dw::dtype_size(dtype);
  need(x, n * h * w * c * es, "global_avg_pool: input size");
  need(y, n * c * es, "global_avg_pool: output size");
  dw::launch_global_avg_pool(bk->stream, dtype, x->ptr, y->ptr, (int)n, (int)(h * w), (int)c);
  API_END
}

int dw_hip_softmax_f32(dw_hip_backend* be, const dw_hip_buffer* x, dw_hip_buffer* y, size_t rows, size_t n) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  if (!rows || !n) dw::fail(DW_ERR_INVALID, "softmax_f32: zero size");
  if (rows > INT32_MAX || n > INT32_MAX) dw::fail(DW_ERR_UNSUPPORTED, "softmax_f32: size");
  need(x, rows * n * 4, "softmax_f32: input size");
  need(y, rows * n * 4, "softmax_f32: output size");
  dw::launch_softmax_rows(bk->stream, (const float*)x->ptr, (float*)y->ptr, (int)rows, (int)n);
  API_END
}

static size_t dtype_bytes(int dtype) {
  if (dtype == DW_DTYPE_F32 || dtype == DW_DTYPE_I32) return 4;
  if (dtype == DW_DTYPE_F16) return 2;
  if (dtype == DW_DTYPE_I8 || dtype == DW_DTYPE_U8) return 1;
  dw::fail(DW_ERR_INVALID, "unknown dtype");
}

int dw_hip_transpose_nchw_to_nhwc(dw_hip_backend* be, const dw_hip_buffer* x, dw_hip_buffer* y, size_t n, size_t c,
                                  size_t h, size_t w, int dtype) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  const size_t es = dtype_bytes(dtype);
  if (!n || !c || !h || !w) dw::fail(DW_ERR_INVALID, "transpose: zero size");
  check_i32(c * h * w, "transpose: image");
  if (n > 65535) dw::fail(DW_ERR_UNSUPPORTED, "transpose: batch above 65535");
  need(x, n * c * h * w * es, "transpose: input");
  need(y, n * c * h * w * es, "transpose: output");
  dw::launch_transpose(bk->stream, x->ptr, y->ptr, (int)n, (int)c, (int)(h * w), (int)es);
  API_END
}

int dw_hip_transpose_nhwc_to_nchw(dw_hip_backend* be, const dw_hip_buffer* x, dw_hip_buffer* y, size_t n, size_t h,
                                  size_t w, size_t c, int dtype) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  const size_t es = dtype_bytes(dtype);
  if (!n || !c || !h || !w) dw::fail(DW_ERR_INVALID, "transpose: zero size");
  check_i32(c * h * w, "transpose: image");
  if (n > 65535) dw::fail(DW_ERR_UNSUPPORTED, "transpose: batch above 65535");
  need(x, n * c * h * w * es, "transpose: input");
  need(y, n * c * h * w * es, "transpose: output");
  dw::launch_transpose(bk->stream, x->ptr, y->ptr, (int)n, (int)(h * w), (int)c, (int)es);
  API_END
}

int dw_hip_fold_batchnorm(dw_hip_backend* be, const dw_hip_buffer* w, const dw_hip_buffer* bias_in,
                          const dw_hip_buffer* gamma, const dw_hip_buffer* beta, const dw_hip_buffer* mean,
                          const dw_hip_buffer* var, float epsilon, size_t c_out, size_t per_channel,
                          dw_hip_buffer* w_out, dw_hip_buffer* bias_out) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  if (!c_out || !per_channel) dw::fail(DW_ERR_INVALID, "fold_batchnorm: zero size");
  if (c_out > 65535) dw::fail(DW_ERR_UNSUPPORTED, "fold_batchnorm: more than 65535 channels");
  check_i32(c_out * per_channel, "fold_batchnorm: weights");
  need(w, c_out * per_channel * 4, "fold_batchnorm: weights");
  need(w_out, c_out * per_channel * 4, "fold_batchnorm: output weights");
  if (bias_in) need(bias_in, c_out * 4, "fold_batchnorm: bias");
  need(gamma, c_out * 4, "fold_batchnorm: gamma");
  need(beta, c_out * 4, "fold_batchnorm: beta");
  need(mean, c_out * 4, "fold_batchnorm: mean");
  need(var, c_out * 4, "fold_batchnorm: var");
  need(bias_out, c_out * 4, "fold_batchnorm: output bias");
  dw::launch_fold_batchnorm(bk->stream, (const float*)w->ptr, bias_in ? (const float*)bias_in->ptr : nullptr,
                            (const float*)gamma->ptr, (const float*)beta->ptr, (const float*)mean->ptr,
                            (const float*)var->ptr, epsilon, (int)c_out, (int)per_channel, (float*)w_out->ptr,
                            (float*)bias_out->ptr);
  API_END
}

int dw_hip_yolo_detect_tail(dw_hip_backend* be, int dtype, const dw_hip_buffer* const* levels, const int* h,
                            const int* w, const float* strides, int num_levels, size_t n, int nc, int reg_max,
                            dw_hip_buffer* out) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  if (!levels || !h || !w || !strides) dw::fail(DW_ERR_INVALID, "detect tail: null argument");
  if (num_levels < 1 || num_levels > 4) dw::fail(DW_ERR_UNSUPPORTED, "detect tail: 1 to 4 levels");
  if (dtype != DW_DTYPE_F16 && dtype != DW_DTYPE_F32) dw::fail(DW_ERR_UNSUPPORTED, "detect tail: f16 or f32");
  if (!n || nc < 1 || reg_max < 1) dw::fail(DW_ERR_INVALID, "detect tail: zero size");
  check_i32(n, "detect tail: batch");
  const size_t es = dtype == DW_DTYPE_F16 ? 2 : 4;
  const size_t pix = (size_t)4 * reg_max + (size_t)nc;
  dw::DetectTailArgs t{};
  size_t A = 0;
  for (int s = 0; s < num_levels; ++s) {
    if (h[s] < 1 || w[s] < 1) dw::fail(DW_ERR_INVALID, "detect tail: empty level");
    need(levels[s], n * (size_t)h[s] * w[s] * pix * es, "detect tail: level size");
    t.x[s] = levels[s]->ptr;
    t.h[s] = h[s];
    t.w[s] = w[s];
    t.pix[s] = (int)pix;
    t.stride[s] = strides[s];
    A += (size_t)h[s] * w[s];
  }
  check_i32(A * (4 + nc), "detect tail: output row");
  need(out, n * (4 + (size_t)nc) * A * 4, "detect tail: output size");
  t.levels = num_levels;
  t.nc = nc;
  t.reg_max = reg_max;
  dw::launch_detect_tail(bk->stream, dtype == DW_DTYPE_F16 ? dw::F16 : dw::F32, t, (float*)out->ptr, (int)n);
  API_END
}

int dw_hip_yolo_postprocess(dw_hip_backend* be, const dw_hip_buffer* raw, size_t n, int nc, size_t num_det,
                            uint32_t img_w, uint32_t img_h, float conf_threshold, float iou_threshold,
                            int agnostic, dw_detection* out, size_t cap, size_t* counts) {
  API_BEGIN
  Backend* bk = B(be);
  std::lock_guard<std::mutex> lock(bk->mu);
  static_assert(sizeof(dw_detection) == sizeof(dw::DwDetection), "detection layout");
  if (!counts || (cap && !out)) dw::fail(DW_ERR_INVALID, "postprocess: null output");
  if (!n || nc < 1 || !num_det) dw::fail(DW_ERR_INVALID, "postprocess: zero size");
  if (nc > 1024) dw::fail(DW_ERR_UNSUPPORTED, "postprocess: more than 1024 classes");
  if (num_det > 16384) dw::fail(DW_ERR_UNSUPPORTED, "postprocess: more than 16384 anchors per image");
  check_i32(n, "postprocess: batch");
  need(raw, n * (4 + (size_t)nc) * num_det * 4, "postprocess: raw output size");
  int dev_lds = 0;
  DW_HIP(hipDeviceGetAttribute(&dev_lds, hipDeviceAttributeMaxSharedMemoryPerBlock, bk->device));
  const int nmax = dw::kPPMaxCandidates;
  if ((size_t)dev_lds < dw::pp_nms_lds_bytes(nmax)) dw::fail(DW_ERR_UNSUPPORTED, "postprocess: LDS per workgroup");
  // workspace: keys, per-anchor detections, then per image nmax-sized arrays
  const size_t A = num_det;
  auto al = [](size_t v) { return (v + 255) & ~(size_t)255; };
  // the results (counts, then the kept detections of all images packed) lie
  // together at the end
  const size_t o_keys = 0, o_det = o_keys + al(n * A * 8), o_sa = o_det + al(n * A * 24);
  const size_t o_pp = o_sa + al(n * nmax * 4), o_cur = o_pp + al(n * nmax * 4), o_cnt = o_cur + 256;
  const size_t o_kept = o_cnt + n * 16, total = o_kept + n * nmax * sizeof(dw::DwKept);
  uint8_t* ws = (uint8_t*)bk->workspace(Backend::WS_POST, total);
  dw::PostprocessArgs a{};
  a.raw = (const float*)raw->ptr;
  a.n = (int)n;
  a.nc = nc;
  a.A = (int)A;
  const float model = 640.0f;  // the reference's fixed model size (postprocess.rs:98)
  a.sx = (float)img_w / model;
  a.sy = (float)img_h / model;
  a.img_w = (float)img_w;
  a.img_h = (float)img_h;
  a.conf = conf_threshold;
  a.iou = iou_threshold;
  a.agnostic = agnostic ? 1 : 0;
  a.nmax = nmax;
  a.keys = (unsigned long long*)(ws + o_keys);
  a.det = (dw::DwDetection*)(ws + o_det);
  a.sorted_anchor = (int*)(ws + o_sa);
  a.part_pos = (int*)(ws + o_pp);
  a.cursor = (int*)(ws + o_cur);
  a.counts = (int*)(ws + o_cnt);
  a.kept = (dw::DwKept*)(ws + o_kept);
  dw::launch_yolo_postprocess(bk->stream, a);
  // one download takes the counts and as many kept detections as frames
  // usually have; a second one the rest
  const size_t guess = n * (16 + 512 * sizeof(dw::DwKept)), most = total - o_cnt;
  std::vector<uint8_t> res(std::min(guess, most));
  bk->download(res.data(), ws + o_cnt, res.size());
  const int* cnt = (const int*)res.data();
  size_t kept = 0;
  for (size_t b = 0; b < n; ++b) {
    if (cnt[4 * b + 2])
      dw::fail(DW_ERR_UNSUPPORTED, "postprocess: image " + std::to_string(b) + " has " +
                                       std::to_string(cnt[4 * b]) + " candidates over the threshold (at most " +
                                       std::to_string(nmax) + ")");
    kept += (size_t)cnt[4 * b + 1];
  }
  const size_t have = res.size(), need_bytes = n * 16 + kept * sizeof(dw::DwKept);
  if (need_bytes > have) {
    res.resize(need_bytes);
    cnt = (const int*)res.data();
    bk->download(res.data() + have, ws + o_cnt + have, need_bytes - have);
  }
  const uint8_t* kd = res.data() + n * 16;
  // The reference removes suppressed entries from the back with swap_remove
  // (postprocess.rs:235-242): walking the sorted positions downwards, a
  // suppressed slot takes the current last element and the list shrinks.
  // Replayed on slots that name kept detections (-1: suppressed).
  bool over = false;
  std::vector<int> slot;
  for (size_t b = 0; b < n; ++b) {
    const int nc_b = cnt[4 * b], k = cnt[4 * b + 1];
    counts[b] = (size_t)k;
    if ((size_t)k > cap) {
      over = true;
      continue;
    }
    const uint8_t* mine = kd + (size_t)cnt[4 * b + 3] * sizeof(dw::DwKept);
    auto entry = [&](int i) { return mine + (size_t)i * sizeof(dw::DwKept); };
    slot.assign((size_t)nc_b, -1);
    for (int i = 0; i < k; ++i) {
      int pos;
      memcpy(&pos, entry(i) + offsetof(dw::DwKept, pos), sizeof pos);
      slot[(size_t)pos] = i;
    }
    int len = nc_b;
    for (int i = nc_b - 1; i >= 0; --i)
      if (slot[(size_t)i] < 0) {
        slot[(size_t)i] = slot[(size_t)len - 1];
        --len;
      }
    dw_detection* o = out + b * cap;
    for (int i = 0; i < len; ++i) memcpy(&o[i], entry(slot[(size_t)i]), sizeof(dw_detection));
  }
  if (over) dw::fail(DW_ERR_INVALID, "postprocess: more detections than cap in an image (see counts)");
  API_END
}

// Layers in 4 bits: MXFP4 rows, products with MXFP4 weights, rotary positions
// and attention over an MXFP4 cache.  What needs no device (sizes, types,
// options) is checked before the handles.
namespace {

constexpr size_t kMostMx = (size_t)1 << 24;  // of a product's rows and columns, and of a cache's tokens and pages

// A buffer of exactly `bytes` on the backend's device.
void need_on(const Backend* b, const dw_hip_buffer* x, size_t bytes, const char* what) {
  need(x, bytes, what);
  if (x->be->device != b->device)
    dw::fail(DW_ERR_INVALID, std::string(what) + ": on device " + std::to_string(x->be->device) + ", the backend is on " +
                                 std::to_string(b->device));
}

size_t float_bytes(int dtype, const char* what) {
  if (dtype != DW_DTYPE_F32 && dtype != DW_DTYPE_F16)
    dw::fail(DW_ERR_UNSUPPORTED, std::string(what) + ": dtype must be f32 or f16");
  return dw::dtype_size(dtype);
}

void check_mx_rows(size_t rows, size_t k, const char* what) {
  if (!rows || !k) dw::fail(DW_ERR_INVALID, std::string(what) + ": zero size");
  if (rows > INT32_MAX || k > INT32_MAX || rows * ((k + 31) / 32) > ((size_t)1 << 40))
    dw::fail(DW_ERR_UNSUPPORTED, std::string(what) + ": size");
}

void check_act(int act, const char* what) {
  if (act != DW_ACT_NONE && act != DW_ACT_RELU && act != DW_ACT_SILU)
    dw::fail(DW_ERR_INVALID, std::string(what) + ": unknown activation");
}

// `heads` heads of `dim` elements from column `off` of rows of `stride`.
void check_columns(size_t stride, size_t off, size_t heads, size_t dim, const char* what) {
  if (stride > kMostMx || off > stride || heads * dim > stride - off)
    dw::fail(DW_ERR_INVALID, std::string(what) + ": the heads do not fit the row");
}

// The sizes that append and attention share.
void check_kv(size_t tokens, size_t batch, size_t kv_heads, size_t d, size_t page, size_t num_pages, size_t max_pages,
              const char* what) {
  const std::string w(what);
  if (!tokens || !batch || !kv_heads || !num_pages || !max_pages) dw::fail(DW_ERR_INVALID, w + ": zero size");
  if (d != 64 && d != 128 && d != 256) dw::fail(DW_ERR_UNSUPPORTED, w + ": head_dim must be 64, 128 or 256");
  if (page < 16 || page > 65536 || (page & (page - 1)))
    dw::fail(DW_ERR_UNSUPPORTED, w + ": page_size must be a power of two from 16 to 65536");
  if (tokens >= kMostMx || batch > 65535 || kv_heads > 1024 || num_pages > INT32_MAX || max_pages > kMostMx ||
      max_pages * page > (size_t)1 << 30)
    dw::fail(DW_ERR_UNSUPPORTED, w + ": size");
}

dw::KvArgs kv_args(const Backend* b, dw_hip_buffer* kc, dw_hip_buffer* ks, dw_hip_buffer* vc, dw_hip_buffer* vs,
                   const dw_hip_buffer* table, const dw_hip_buffer* start, const dw_hip_buffer* len, size_t tokens,
                   size_t batch, size_t kv_heads, size_t d, size_t page, size_t num_pages, size_t max_pages) {
  const size_t rows = num_pages * kv_heads * page;
  need_on(b, kc, rows * d / 2, "key cache");
  need_on(b, ks, rows * d / 32, "key scales");
  need_on(b, vc, rows * d / 2, "value cache");
  need_on(b, vs, rows * d / 32, "value scales");
  need_on(b, table, batch * max_pages * 4, "block table");
  need_on(b, start, (batch + 1) * 4, "q_start");
  need_on(b, len, batch * 4, "kv_len");
  dw::KvArgs a{};
  a.kc = (uint32_t*)kc->ptr;
  a.ks = (uint8_t*)ks->ptr;
  a.vc = (uint32_t*)vc->ptr;
  a.vs = (uint8_t*)vs->ptr;
  a.table = (const int32_t*)table->ptr;
  a.start = (const int32_t*)start->ptr;
  a.len = (const int32_t*)len->ptr;
  a.tokens = (int)tokens;
  a.batch = (int)batch;
  a.kv_heads = (int)kv_heads;
  a.d = (int)d;
  a.page_shift = __builtin_ctzll(page);
  a.num_pages = (int)num_pages;
  a.max_pages = (int)max_pages;
  return a;
}

}  // namespace

int dw_hip_quantize_mxfp4(dw_hip_backend* be, int dtype, const dw_hip_buffer* x, dw_hip_buffer* q,
                          dw_hip_buffer* scales, size_t rows, size_t k) {
  API_BEGIN
  const size_t es = float_bytes(dtype, "quantize_mxfp4");
  check_mx_rows(rows, k, "quantize_mxfp4");
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  const size_t blocks = (k + 31) / 32;
  need_on(b, x, rows * k * es, "quantize_mxfp4: input");
  need_on(b, q, rows * blocks * 16, "quantize_mxfp4: packed rows");
  need_on(b, scales, rows * blocks, "quantize_mxfp4: scales");
  if (x == q || x == scales || q == scales) dw::fail(DW_ERR_INVALID, "quantize_mxfp4: buffers overlap");
  dw::launch_quantize_mxfp4(b->stream, dtype, x->ptr, q->ptr, scales->ptr, rows, k);
  API_END
}

int dw_hip_dequantize_mxfp4(dw_hip_backend* be, int dtype, const dw_hip_buffer* q, const dw_hip_buffer* scales,
                            dw_hip_buffer* y, size_t rows, size_t k) {
  API_BEGIN
  const size_t es = float_bytes(dtype, "dequantize_mxfp4");
  check_mx_rows(rows, k, "dequantize_mxfp4");
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  const size_t blocks = (k + 31) / 32;
  need_on(b, q, rows * blocks * 16, "dequantize_mxfp4: packed rows");
  need_on(b, scales, rows * blocks, "dequantize_mxfp4: scales");
  need_on(b, y, rows * k * es, "dequantize_mxfp4: output");
  if (y == q || y == scales) dw::fail(DW_ERR_INVALID, "dequantize_mxfp4: buffers overlap");
  dw::launch_dequantize_mxfp4(b->stream, dtype, q->ptr, scales->ptr, y->ptr, rows, k);
  API_END
}

int dw_hip_gemm_mxfp4(dw_hip_backend* be, int a_dtype, const dw_hip_buffer* a, const dw_hip_buffer* a_scales,
                      const dw_hip_buffer* w, const dw_hip_buffer* w_scales, const dw_hip_buffer* bias, int c_dtype,
                      dw_hip_buffer* c, size_t m, size_t n, size_t k, int act) {
  API_BEGIN
  if (a_dtype != DW_DTYPE_F16 && a_dtype != DW_DTYPE_MXFP4)
    dw::fail(DW_ERR_UNSUPPORTED, "gemm_mxfp4: A must be f16 or MXFP4");
  const size_t es = float_bytes(c_dtype, "gemm_mxfp4: C");
  check_act(act, "gemm_mxfp4");
  if (!m || !n || !k) dw::fail(DW_ERR_INVALID, "gemm_mxfp4: zero size");
  if (m > kMostMx || n > kMostMx || k > kMostMx / 4)
    dw::fail(DW_ERR_UNSUPPORTED, "gemm_mxfp4: m or n above 2^24, or k above 2^22");
  const bool mx = a_dtype == DW_DTYPE_MXFP4;
  if (mx != (a_scales != nullptr)) dw::fail(DW_ERR_INVALID, "gemm_mxfp4: scales of A for MXFP4 rows, and only for them");
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  const size_t blocks = (k + 31) / 32;
  need_on(b, a, mx ? m * blocks * 16 : m * k * 2, "gemm_mxfp4: A");
  if (mx) need_on(b, a_scales, m * blocks, "gemm_mxfp4: scales of A");
  need_on(b, w, n * blocks * 16, "gemm_mxfp4: W");
  need_on(b, w_scales, n * blocks, "gemm_mxfp4: scales of W");
  if (bias) need_on(b, bias, n * es, "gemm_mxfp4: bias");
  need_on(b, c, m * n * es, "gemm_mxfp4: C");
  if (c == a || c == a_scales || c == w || c == w_scales || c == bias)
    dw::fail(DW_ERR_INVALID, "gemm_mxfp4: C is an operand");
  dw::GemmMxArgs g{};
  g.a = a->ptr;
  g.as = mx ? (const uint8_t*)a_scales->ptr : nullptr;
  g.w = (const uint8_t*)w->ptr;
  g.ws = (const uint8_t*)w_scales->ptr;
  g.bias = bias ? bias->ptr : nullptr;
  g.c = c->ptr;
  g.m = (int)m;
  g.n = (int)n;
  g.k = (int)k;
  g.act = act;
  g.c_half = c_dtype == DW_DTYPE_F16;
  const size_t bytes = dw::gemm_mx_space(g);
  dw::launch_gemm_mx(b->stream, g, bytes ? b->workspace(Backend::WS_GEMM4, bytes) : nullptr);
  API_END
}

int dw_hip_rope_axes(dw_hip_backend* be, int dtype, const dw_hip_buffer* x, size_t x_stride, size_t x_off,
                     dw_hip_buffer* y, size_t y_stride, size_t y_off, const dw_hip_buffer* positions, size_t tokens,
                     size_t heads, size_t head_dim, size_t rotary_dim, const size_t* sections, size_t axes, int order,
                     int pairs, int freq, double base) {
  API_BEGIN
  const size_t es = float_bytes(dtype, "rope_axes");
  if (!tokens || !heads || !head_dim || !rotary_dim || !axes || !sections) dw::fail(DW_ERR_INVALID, "rope_axes: zero size");
  if (rotary_dim % 2 || rotary_dim > head_dim)
    dw::fail(DW_ERR_INVALID, "rope_axes: rotary_dim must be even and at most head_dim");
  if (rotary_dim > 256 || head_dim > 4096 || heads > 4096 || axes > 8 || tokens >= kMostMx)
    dw::fail(DW_ERR_UNSUPPORTED, "rope_axes: size");
  if ((order != 0 && order != 1) || (pairs != 0 && pairs != 1) || (freq != 0 && freq != 1))
    dw::fail(DW_ERR_INVALID, "rope_axes: unknown option");
  if (!(base > 0) || !std::isfinite(base)) dw::fail(DW_ERR_INVALID, "rope_axes: base must be positive");
  const size_t half = rotary_dim / 2;
  size_t sum = 0;
  for (size_t i = 0; i < axes; ++i) {
    if (sections[i] > half) dw::fail(DW_ERR_INVALID, "rope_axes: sections must add up to rotary_dim / 2");
    sum += sections[i];
  }
  if (sum != half) dw::fail(DW_ERR_INVALID, "rope_axes: sections must add up to rotary_dim / 2");
  check_columns(x_stride, x_off, heads, head_dim, "rope_axes: input");
  check_columns(y_stride, y_off, heads, head_dim, "rope_axes: output");
  if (x && x == y) {
    const size_t w = heads * head_dim;
    if (x_stride != y_stride || (x_off != y_off && x_off < y_off + w && y_off < x_off + w))
      dw::fail(DW_ERR_INVALID, "rope_axes: input and output overlap");
  }
  dw::RopeArgs a{};
  // the axis of each pair, and its frequency base^(-2 i / rotary_dim), i the
  // pair's index in the head (freq 0) or base^(-j / n), j its index among the
  // n pairs of its axis (freq 1): powers by repeated products in 80 bits
  size_t used[8] = {};
  long double power[9], step[9];
  for (size_t i = 0; i <= axes; ++i) {
    const size_t n = i < axes ? sections[i] : half;
    step[i] = n ? expl(-logl((long double)base) / (long double)n) : 1.0L;
    power[i] = 1.0L;
  }
  constexpr long double kTurn = 6.283185307179586476925286766559005768L;
  for (size_t i = 0, next = 0; i < half; ++i) {
    while (used[next] == sections[next]) next = (next + 1) % axes;  // some axis has pairs left
    a.table.axis[i] = (uint8_t)next;
    const size_t f = freq ? next : axes;
    a.table.freq[i] = (double)(power[f] / kTurn);
    if (!std::isfinite(a.table.freq[i] * 0x1p31))
      dw::fail(DW_ERR_INVALID, "rope_axes: base is so small that angles are no f64 numbers");
    power[f] *= step[f];
    ++used[next];
    if (order) next = (next + 1) % axes;
  }
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  need_on(b, x, tokens * x_stride * es, "rope_axes: input");
  need_on(b, y, tokens * y_stride * es, "rope_axes: output");
  need_on(b, positions, axes * tokens * 4, "rope_axes: positions");
  if (positions == y) dw::fail(DW_ERR_INVALID, "rope_axes: the positions are the output");
  a.x = x->ptr;
  a.y = y->ptr;
  a.pos = (const int32_t*)positions->ptr;
  a.x_stride = x_stride;
  a.x_off = x_off;
  a.y_stride = y_stride;
  a.y_off = y_off;
  a.tokens = tokens;
  a.heads = (int)heads;
  a.head_dim = (int)head_dim;
  a.half = (int)half;
  a.copy = !(x == y && x_off == y_off);
  dw::launch_rope(b->stream, dtype, a, pairs);
  API_END
}

int dw_hip_kv_append_mxfp4(dw_hip_backend* be, const dw_hip_buffer* k, size_t k_stride, size_t k_off,
                           const dw_hip_buffer* v, size_t v_stride, size_t v_off, dw_hip_buffer* k_cache,
                           dw_hip_buffer* k_scales, dw_hip_buffer* v_cache, dw_hip_buffer* v_scales,
                           const dw_hip_buffer* block_table, const dw_hip_buffer* q_start, const dw_hip_buffer* kv_len,
                           size_t tokens, size_t batch, size_t kv_heads, size_t head_dim, size_t page_size,
                           size_t num_pages, size_t max_pages) {
  API_BEGIN
  check_kv(tokens, batch, kv_heads, head_dim, page_size, num_pages, max_pages, "kv_append_mxfp4");
  check_columns(k_stride, k_off, kv_heads, head_dim, "kv_append_mxfp4: keys");
  check_columns(v_stride, v_off, kv_heads, head_dim, "kv_append_mxfp4: values");
  if (k_cache && (k_cache == v_cache || k_scales == v_scales))
    dw::fail(DW_ERR_INVALID, "kv_append_mxfp4: keys and values share a cache");
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  need_on(b, k, tokens * k_stride * 2, "kv_append_mxfp4: keys");
  need_on(b, v, tokens * v_stride * 2, "kv_append_mxfp4: values");
  const dw::KvArgs a = kv_args(b, k_cache, k_scales, v_cache, v_scales, block_table, q_start, kv_len, tokens, batch,
                               kv_heads, head_dim, page_size, num_pages, max_pages);
  for (const dw_hip_buffer* w : {k_cache, k_scales, v_cache, v_scales})
    if (w == k || w == v || w == block_table || w == q_start || w == kv_len)
      dw::fail(DW_ERR_INVALID, "kv_append_mxfp4: the cache is an input");
  dw::launch_kv_append(b->stream, a, k->ptr, k_stride, k_off, v->ptr, v_stride, v_off);
  API_END
}

int dw_hip_attention_mxfp4(dw_hip_backend* be, const dw_hip_buffer* q, size_t q_stride, size_t q_off,
                           const dw_hip_buffer* k_cache, const dw_hip_buffer* k_scales, const dw_hip_buffer* v_cache,
                           const dw_hip_buffer* v_scales, const dw_hip_buffer* block_table,
                           const dw_hip_buffer* q_start, const dw_hip_buffer* kv_len, dw_hip_buffer* y, size_t tokens,
                           size_t batch, size_t heads, size_t kv_heads, size_t head_dim, size_t page_size,
                           size_t num_pages, size_t max_pages, float scale, int causal, size_t window) {
  API_BEGIN
  check_kv(tokens, batch, kv_heads, head_dim, page_size, num_pages, max_pages, "attention_mxfp4");
  if (!heads || heads % kv_heads) dw::fail(DW_ERR_INVALID, "attention_mxfp4: heads must be a multiple of kv_heads");
  if (heads > 4096) dw::fail(DW_ERR_UNSUPPORTED, "attention_mxfp4: more than 4096 heads");
  if (tokens * heads > kMostMx || batch * heads > kMostMx / 4)
    dw::fail(DW_ERR_UNSUPPORTED, "attention_mxfp4: more than 2^24 rows, or 2^22 heads of all sequences");
  if (!std::isfinite(scale * 1.44269504f)) dw::fail(DW_ERR_INVALID, "attention_mxfp4: scale must be finite");
  if (causal != 0 && causal != 1) dw::fail(DW_ERR_INVALID, "attention_mxfp4: causal must be 0 or 1");
  if (window && !causal) dw::fail(DW_ERR_UNSUPPORTED, "attention_mxfp4: a window needs causal attention");
  check_columns(q_stride, q_off, heads, head_dim, "attention_mxfp4: queries");
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  need_on(b, q, tokens * q_stride * 2, "attention_mxfp4: queries");
  need_on(b, y, tokens * heads * head_dim * 2, "attention_mxfp4: output");
  const dw::KvArgs a = kv_args(b, const_cast<dw_hip_buffer*>(k_cache), const_cast<dw_hip_buffer*>(k_scales),
                               const_cast<dw_hip_buffer*>(v_cache), const_cast<dw_hip_buffer*>(v_scales), block_table,
                               q_start, kv_len, tokens, batch, kv_heads, head_dim, page_size, num_pages, max_pages);
  for (const dw_hip_buffer* r : {q, k_cache, k_scales, v_cache, v_scales, block_table, q_start, kv_len})
    if (r == y) dw::fail(DW_ERR_INVALID, "attention_mxfp4: the output is an input");
  dw::AttnArgs g{};
  g.q = (const uint16_t*)q->ptr;
  g.q_stride = q_stride;
  g.q_off = q_off;
  g.y = (uint16_t*)y->ptr;
  g.tokens = (int)tokens;
  g.heads = (int)heads;
  g.causal = causal;
  g.window = window > (size_t)INT32_MAX ? 0 : (long long)window;
  g.scale = std::max(fabsf(scale) * 1.44269504f, 1e-37f);  // above 0, where -inf stays so; as 0, to a score
  g.negate = scale < 0;
  dw::AttnPlan p{};
  const size_t bytes = dw::attention_space(a, g, &p);
  dw::launch_attention(b->stream, a, g, p, bytes ? b->workspace(Backend::WS_ATTN, bytes) : nullptr);
  API_END
}

// A mixture of experts: the sizes that its calls share.
static void check_experts(size_t slots, size_t experts, const char* what) {
  if (!slots || !experts) dw::fail(DW_ERR_INVALID, std::string(what) + ": zero size");
  if (slots > kMostMx || experts > 1024)
    dw::fail(DW_ERR_UNSUPPORTED, std::string(what) + ": more than 2^24 slots or 1024 experts");
}
static void check_choices(size_t tokens, size_t top_k, size_t experts, const char* what) {
  if (!tokens || !top_k) dw::fail(DW_ERR_INVALID, std::string(what) + ": zero size");
  if (top_k > 32) dw::fail(DW_ERR_UNSUPPORTED, std::string(what) + ": top_k above 32");
  if (tokens > kMostMx) dw::fail(DW_ERR_UNSUPPORTED, std::string(what) + ": more than 2^24 slots or 1024 experts");
  check_experts(tokens * top_k, experts, what);
}

int dw_hip_route_experts(dw_hip_backend* be, int dtype, const dw_hip_buffer* logits, size_t stride, size_t off,
                         const dw_hip_buffer* bias, dw_hip_buffer* ids, dw_hip_buffer* weights, size_t tokens,
                         size_t experts, size_t top_k, int score, size_t groups, size_t top_groups, int group_best,
                         int renorm, float scale) {
  API_BEGIN
  const size_t es = float_bytes(dtype, "route_experts");
  check_choices(tokens, top_k, experts, "route_experts");
  if (score != DW_SCORE_SOFTMAX && score != DW_SCORE_SIGMOID) dw::fail(DW_ERR_INVALID, "route_experts: unknown score");
  if (!groups || !top_groups || top_groups > groups || groups > experts || experts % groups)
    dw::fail(DW_ERR_INVALID, "route_experts: groups must divide the experts, top_groups be 1 to groups");
  if (top_k > top_groups * (experts / groups))
    dw::fail(DW_ERR_INVALID, "route_experts: top_k is more than the experts that take part");
  if (group_best != 1 && group_best != 2) dw::fail(DW_ERR_INVALID, "route_experts: group_best must be 1 or 2");
  if (renorm != 0 && renorm != 1) dw::fail(DW_ERR_INVALID, "route_experts: renorm must be 0 or 1");
  if (!std::isfinite(scale)) dw::fail(DW_ERR_INVALID, "route_experts: scale must be finite");
  check_columns(stride, off, 1, experts, "route_experts: logits");
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  need_on(b, logits, tokens * stride * es, "route_experts: logits");
  if (bias) need_on(b, bias, experts * 4, "route_experts: bias");
  need_on(b, ids, tokens * top_k * 4, "route_experts: ids");
  need_on(b, weights, tokens * top_k * 4, "route_experts: weights");
  if (ids == weights || ids == logits || ids == bias || weights == logits || weights == bias)
    dw::fail(DW_ERR_INVALID, "route_experts: buffers overlap");
  dw::RouteArgs a{};
  a.x = (const char*)logits->ptr + off * es;
  a.bias = bias ? (const float*)bias->ptr : nullptr;
  a.ids = (int32_t*)ids->ptr;
  a.weights = (float*)weights->ptr;
  a.stride = stride;
  a.tokens = tokens;
  a.half = dtype == DW_DTYPE_F16;
  a.experts = (int)experts;
  a.top_k = (int)top_k;
  a.sigmoid = score == DW_SCORE_SIGMOID;
  a.groups = (int)groups;
  a.top_groups = (int)top_groups;
  a.group_best = group_best;
  a.renorm = renorm;
  a.scale = scale;
  dw::launch_route(b->stream, a);
  API_END
}

int dw_hip_order_experts(dw_hip_backend* be, const dw_hip_buffer* ids, dw_hip_buffer* offsets, dw_hip_buffer* order,
                         size_t slots, size_t experts) {
  API_BEGIN
  check_experts(slots, experts, "order_experts");
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  need_on(b, ids, slots * 4, "order_experts: ids");
  need_on(b, offsets, (experts + 1) * 4, "order_experts: offsets");
  need_on(b, order, slots * 4, "order_experts: order");
  if (ids == offsets || ids == order || offsets == order) dw::fail(DW_ERR_INVALID, "order_experts: buffers overlap");
  dw::OrderArgs a{};
  a.ids = (const int32_t*)ids->ptr;
  a.offsets = (int32_t*)offsets->ptr;
  a.order = (int32_t*)order->ptr;
  a.slots = (int)slots;
  a.experts = (int)experts;
  const size_t bytes = dw::order_space(a);
  dw::launch_order(b->stream, a, bytes ? b->workspace(Backend::WS_ORDER, bytes) : nullptr);
  API_END
}

int dw_hip_gemm_mxfp4_experts(dw_hip_backend* be, int a_dtype, const dw_hip_buffer* a, const dw_hip_buffer* a_scales,
                              const dw_hip_buffer* w, const dw_hip_buffer* w_scales, const dw_hip_buffer* bias,
                              int c_dtype, dw_hip_buffer* c, const dw_hip_buffer* offsets, const dw_hip_buffer* order,
                              size_t slots, size_t experts, size_t n, size_t k, int act, size_t gather, int scatter) {
  API_BEGIN
  if (a_dtype != DW_DTYPE_F16 && a_dtype != DW_DTYPE_MXFP4)
    dw::fail(DW_ERR_UNSUPPORTED, "gemm_mxfp4_experts: A must be f16 or MXFP4");
  const size_t es = float_bytes(c_dtype, "gemm_mxfp4_experts: C");
  if (act != DW_ACT_SWIGLU) check_act(act, "gemm_mxfp4_experts");
  check_experts(slots, experts, "gemm_mxfp4_experts");
  if (!n || !k) dw::fail(DW_ERR_INVALID, "gemm_mxfp4_experts: zero size");
  if (n > kMostMx || k > kMostMx / 4) dw::fail(DW_ERR_UNSUPPORTED, "gemm_mxfp4_experts: n above 2^24 or k above 2^22");
  if (act == DW_ACT_SWIGLU && n % 2) dw::fail(DW_ERR_INVALID, "gemm_mxfp4_experts: gated columns come in pairs");
  if (gather && slots % gather) dw::fail(DW_ERR_INVALID, "gemm_mxfp4_experts: gather must divide the slots");
  if (scatter != 0 && scatter != 1) dw::fail(DW_ERR_INVALID, "gemm_mxfp4_experts: scatter must be 0 or 1");
  const bool mx = a_dtype == DW_DTYPE_MXFP4;
  if (mx != (a_scales != nullptr))
    dw::fail(DW_ERR_INVALID, "gemm_mxfp4_experts: scales of A for MXFP4 rows, and only for them");
  if ((gather || scatter) && !order) dw::fail(DW_ERR_INVALID, "gemm_mxfp4_experts: rows by order need the order");
  const size_t blocks = (k + 31) / 32, rows = gather ? slots / gather : slots;
  if (rows * (mx ? blocks * 16 : (k + 7) / 8 * 16) > (size_t)1 << 36)
    dw::fail(DW_ERR_UNSUPPORTED, "gemm_mxfp4_experts: A above 64 GiB");
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  need_on(b, a, mx ? rows * blocks * 16 : rows * k * 2, "gemm_mxfp4_experts: A");
  if (mx) need_on(b, a_scales, rows * blocks, "gemm_mxfp4_experts: scales of A");
  need_on(b, w, experts * n * blocks * 16, "gemm_mxfp4_experts: W");
  need_on(b, w_scales, experts * n * blocks, "gemm_mxfp4_experts: scales of W");
  if (bias) need_on(b, bias, experts * n * es, "gemm_mxfp4_experts: bias");
  need_on(b, c, slots * (act == DW_ACT_SWIGLU ? n / 2 : n) * es, "gemm_mxfp4_experts: C");
  need_on(b, offsets, (experts + 1) * 4, "gemm_mxfp4_experts: offsets");
  if (order) need_on(b, order, slots * 4, "gemm_mxfp4_experts: order");
  if (c == a || c == a_scales || c == w || c == w_scales || c == bias || c == offsets || c == order)
    dw::fail(DW_ERR_INVALID, "gemm_mxfp4_experts: C is an operand");
  dw::GemmExpertsArgs x{};
  x.g.a = a->ptr;
  x.g.as = mx ? (const uint8_t*)a_scales->ptr : nullptr;
  x.g.w = (const uint8_t*)w->ptr;
  x.g.ws = (const uint8_t*)w_scales->ptr;
  x.g.bias = bias ? bias->ptr : nullptr;
  x.g.c = c->ptr;
  x.g.m = (int)slots;
  x.g.n = (int)n;
  x.g.k = (int)k;
  x.g.act = act;
  x.g.c_half = c_dtype == DW_DTYPE_F16;
  x.offsets = (const int32_t*)offsets->ptr;
  x.order = order ? (const int32_t*)order->ptr : nullptr;
  x.experts = (int)experts;
  x.gather = (int)gather;
  x.scatter = scatter;
  const size_t bytes = dw::gemm_experts_space(x);
  dw::launch_gemm_experts(b->stream, x, bytes ? b->workspace(Backend::WS_GEMM4, bytes) : nullptr);
  API_END
}

int dw_hip_combine_experts(dw_hip_backend* be, int dtype, const dw_hip_buffer* x, const dw_hip_buffer* ids,
                           const dw_hip_buffer* weights, const dw_hip_buffer* base, dw_hip_buffer* y, size_t tokens,
                           size_t top_k, size_t experts, size_t n) {
  API_BEGIN
  const size_t es = float_bytes(dtype, "combine_experts");
  check_choices(tokens, top_k, experts, "combine_experts");
  if (!n) dw::fail(DW_ERR_INVALID, "combine_experts: zero size");
  if (n > kMostMx) dw::fail(DW_ERR_UNSUPPORTED, "combine_experts: n above 2^24");
  Backend* b = B(be);
  std::lock_guard<std::mutex> lock(b->mu);
  need_on(b, x, tokens * top_k * n * es, "combine_experts: rows");
  need_on(b, ids, tokens * top_k * 4, "combine_experts: ids");
  need_on(b, weights, tokens * top_k * 4, "combine_experts: weights");
  if (base) need_on(b, base, tokens * n * es, "combine_experts: base");
  need_on(b, y, tokens * n * es, "combine_experts: output");
  if (y == x || y == ids || y == weights) dw::fail(DW_ERR_INVALID, "combine_experts: the output is an input");
  dw::CombineArgs a{};
  a.x = x->ptr;
  a.ids = (const int32_t*)ids->ptr;
  a.weights = (const float*)weights->ptr;
  a.base = base ? base->ptr : nullptr;
  a.y = y->ptr;
  a.tokens = tokens;
  a.n = (int)n;
  a.top_k = (int)top_k;
  a.experts = (int)experts;
  dw::launch_combine(b->stream, dtype, a);
  API_END
}

}  // extern "C"
