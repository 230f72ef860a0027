// launch.h — the host side that the operators' libraries share: refusals with a
// message, what is known of the device, launches, and the factors of attention scores.
// Included inside namespace mi355fa's unnamed namespace; codes are those of the C ABIs,
// whose numbers agree.

constexpr int kOk = 0, kEinval = 1, kEworkspace = 2, kElaunch = 3, kEdevice = 4;
constexpr int kFp16 = 0, kBf16 = 1;   // element types

struct Err {
  char* text;
  size_t len;
  __attribute__((format(printf, 3, 4))) int fail(int rc, const char* fmt, ...) const {
    if (text && len) {
      va_list ap;
      va_start(ap, fmt);
      vsnprintf(text, len, fmt, ap);
      va_end(ap);
    }
    return rc;
  }
};

struct Device {
  int cus = 0;
  bool gfx950 = false;
};

Device device_info() {
  static Device known[64];
  static std::mutex mu;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) {
    (void)hipGetLastError();
    return Device{256, false};
  }
  std::lock_guard<std::mutex> lk(mu);
  Device& d = known[dev];
  if (!d.cus) {
    int n = 0;
    d.cus = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) == hipSuccess && n > 0 ? n : 256;
    hipDeviceProp_t prop;
    d.gfx950 = hipGetDeviceProperties(&prop, dev) == hipSuccess && strncmp(prop.gcnArchName, "gfx950", 6) == 0;
    (void)hipGetLastError();
  }
  return d;
}

// Launches; the error is the launch's own, whatever an earlier call left behind.
template <class A>
int run(const Err& err, const char* what, void (*kernel)(const A), int64_t grid, int threads, size_t lds, hipStream_t st, A& a) {
  // (a launch counts its threads in 32 bits)
  if (grid * threads >= (1LL << 32)) return err.fail(kEinval, "%s: problem too large: %lld workgroups", what, (long long)grid);
  void* args[] = {&a};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), dim3((unsigned)grid), dim3((unsigned)threads), args, lds, st);
  if (e == hipSuccess) return kOk;
  (void)hipGetLastError();
  return err.fail(kElaunch, "%s: launch failed: %s", what, hipGetErrorString(e));
}

bool rows_ok(const void* p, std::initializer_list<int64_t> strides) {
  int64_t x = (int64_t)(uintptr_t)p & 15;
  for (int64_t s : strides) x |= s & 7;
  return x == 0;
}

bool window_ok(int w) { return w >= 0; }
int window_of(int w) { return w == 0 ? kNoWindow : std::min(w, kNoWindow); }

// The factors of a call's scores (PackedArgs, DecodeArgs); false where scale or
// softcap is none the kernels can work with.
constexpr float kMaxSoftcap = 1000.f;   // above, 2·softcap·2^-24 of a score is lost to the tanh's rounding
template <class A> bool score_factors(A& a, float scale, float softcap) {
  if (!(scale > 0.f) || isinf(scale) || !(softcap >= 0.f) || softcap > kMaxSoftcap) return false;
  const bool cap = softcap > 0.f;
  a.u_scale = cap ? 2.f * kLog2e * scale / softcap : 0.f;
  a.c2 = cap ? 2.f * softcap * kLog2e : scale * kLog2e;
  a.bias = cap ? -0.5f / softcap : -1.f / scale;
  return std::isfinite(a.u_scale) && std::isfinite(a.c2) && a.c2 > 0.f && std::isfinite(a.bias) &&
         std::isfinite(kSlackLog2 / a.c2);
}

const char* kScoresText = "scale must be positive and finite, softcap 0 (none) or in (0, 1000]";

// f(integral_constant...) for the runtime values of (d, bf16)
template <class F> void by_type(int d, bool bf16, F f) {
  typedef std::integral_constant<int, 64> D64;
  typedef std::integral_constant<int, 128> D128;
  if (d == 64) bf16 ? f(D64{}, std::true_type{}) : f(D64{}, std::false_type{});
  else bf16 ? f(D128{}, std::true_type{}) : f(D128{}, std::false_type{});
}

int check_heads(const Err& err, int h, int hk, int d, int dtype) {
  if (dtype != kFp16 && dtype != kBf16)
    return err.fail(kEinval, "q must be float16 or bfloat16");
  if (d != 64 && d != 128) return err.fail(kEinval, "Only head_dim=64 or head_dim=128 is supported");
  if (hk <= 0 || h < 0 || h % hk) return err.fail(kEinval, "n_heads must be divisible by n_kv_heads (GQA)");
  return kOk;
}
