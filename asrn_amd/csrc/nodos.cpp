// Autograd nodes, in C++, of the fine-tuning losses and of the activations in 8 bits: they allocate, launch the library's
// entry points on torch's current stream and keep what the backward needs. These operators' kernels take a few
// microseconds, and a node written in Python costs more than they do: its backward runs Python on the autograd thread
// (a log-probability's forward and backward over 200 rows: 95 us a pass, 48 with these).
//
// The Python wrappers check every argument and hand over checked tensors. The entry points come as addresses from the
// library that Python has opened, so there is one library however it was chosen. The module is initialised once, by
// iniciar(); a failed call throws Fallo, which Python sees as ASRNHipError (in a backward, as a RuntimeError).
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <optional>
#include <stdexcept>
#include <string>
#include <utility>
#include <vector>

#include "asrn_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Function;
using torch::autograd::variable_list;
using Opcional = std::optional<Tensor>;

namespace {

struct Fallo : std::runtime_error {
  using std::runtime_error::runtime_error;
};

// the library's entry points, by the types its header declares
struct Biblioteca {
  decltype(&asrn_hip_last_error) error;
  decltype(&asrn_token_logp_fwd) logp_fwd;
  decltype(&asrn_token_logp_bwd) logp_bwd;
  decltype(&asrn_preference_workspace) pref_ws;
  decltype(&asrn_preference_fwd) pref_fwd;
  decltype(&asrn_preference_bwd) pref_bwd;
  decltype(&asrn_policy_workspace) pol_ws;
  decltype(&asrn_policy_fwd) pol_fwd;
  decltype(&asrn_policy_bwd) pol_bwd;
  decltype(&asrn_gelu8_fwd) gelu8_fwd;
  decltype(&asrn_gelu8_bwd) gelu8_bwd;
  decltype(&asrn_norm8_fwd) norm8_fwd;
  decltype(&asrn_norm8_bwd) norm8_bwd;
  decltype(&asrn_norm8_bwd_workspace) norm8_ws;
} lib;

void vale(int rc, const char* que) {
  if (rc != 0) throw Fallo(std::string(que) + ": " + lib.error());
}

// the tensor's device as the current one, and its current stream
struct En {
  c10::DeviceGuard guarda;
  void* st;
  explicit En(const Tensor& t) : guarda(t.device()), st((void*)c10::hip::getCurrentHIPStream(t.device().index()).stream()) {}
};

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const Opcional& t) { return t ? t->data_ptr() : nullptr; }
float* f32(const Tensor& t) { return static_cast<float*>(ptr(t)); }
float* f32(const Opcional& t) { return static_cast<float*>(ptr(t)); }
uint8_t* u8(const Opcional& t) { return static_cast<uint8_t*>(ptr(t)); }
Tensor vacio(at::IntArrayRef forma, const Tensor& como, at::ScalarType tipo = at::kFloat) {
  return at::empty(forma, como.options().dtype(tipo));
}
Tensor denso(const Tensor& g) { return g.scalar_type() == at::kFloat && g.is_contiguous() ? g : g.to(at::kFloat).contiguous(); }
bool es16(const Tensor& t) { return t.scalar_type() == at::kBFloat16; }
// the row and token strides of (B, L) tensors, 0 for an absent one
void pasos(const Opcional& t, int64_t* s) {
  s[0] = t ? t->stride(0) : 0;
  s[1] = t ? t->stride(1) : 0;
}
// The kernels have no second derivative: a backward that is itself recorded is refused, whatever the recording is for (a
// delayed error would be passed over where the second gradient also has another path).
void una_vez(const char* que) {
  if (at::GradMode::is_enabled())
    throw Fallo(std::string(que) + ": its gradient cannot be recorded (create_graph=True), the kernels have no second derivative");
}

// ---- log-probabilities of given tokens -----------------------------------------------------------------------------------
struct Filas {
  int32_t tipo;
  int64_t filas, L, V, sb, st, ignorar;
  double inv_t;
  bool entropia;
};

struct LogProbabilidades : Function<LogProbabilidades> {
  static variable_list forward(AutogradContext* ctx, const Tensor& logits, const Tensor& y, const Filas& f) {
    En en(logits);
    Tensor lp = vacio(y.sizes(), logits), stats = vacio({f.filas, 2}, logits), H;
    if (f.entropia) H = vacio(y.sizes(), logits);
    if (f.filas)
      vale(lib.logp_fwd(ptr(logits), f.tipo, f.filas, f.L, f.V, f.sb, f.st, y.data_ptr<int64_t>(), f.ignorar, (float)f.inv_t,
                        f32(lp), f32(H), f32(stats), en.st), "asrn_token_logp_fwd");
    variable_list guarda{logits, y, stats};
    if (f.entropia) guarda.push_back(H);
    ctx->save_for_backward(guarda);
    ctx->saved_data["n"] = std::vector<int64_t>{f.tipo, f.filas, f.L, f.V, f.sb, f.st, f.ignorar};
    ctx->saved_data["t"] = f.inv_t;
    ctx->set_materialize_grads(false);
    variable_list r{lp};
    if (f.entropia) r.push_back(H);
    return r;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    una_vez("log_probabilidades");
    Tensor gl = g[0], gh = g.size() > 1 ? g[1] : Tensor();
    if (!gl.defined() && !gh.defined()) return {Tensor(), Tensor(), Tensor()};
    const variable_list s = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    const Tensor &x = s[0], dx = at::empty(x.sizes(), x.options());
    En en(x);
    if (gl.defined()) gl = denso(gl);
    if (gh.defined()) gh = denso(gh);
    if (n[1])
      vale(lib.logp_bwd(ptr(x), (int32_t)n[0], n[1], n[2], n[3], n[4], n[5], s[1].data_ptr<int64_t>(), n[6],
                        (float)ctx->saved_data["t"].toDouble(), f32(s[2]), s.size() > 3 ? f32(s[3]) : nullptr, f32(gl), f32(gh),
                        ptr(dx), en.st), "asrn_token_logp_bwd");
    return {dx, Tensor(), Tensor()};
  }
};

// logits (B, L, V), (rows, V) or (V) with adjacent values, read through their strides; y int64, contiguous
py::tuple logp(const Tensor& x, const Tensor& y, int32_t tipo, int64_t ignorar, double inv_t, bool entropia) {
  variable_list r;
  {
    py::gil_scoped_release sin_gil;
    const int64_t V = x.size(-1);
    Filas f{tipo, 1, 1, V, 0, 0, ignorar, inv_t, entropia};
    if (x.dim() == 2) {
      f.filas = f.L = x.size(0);
      f.st = x.stride(0);
    } else if (x.dim() == 3) {
      f.filas = x.size(0) * x.size(1);
      f.L = x.size(1);
      f.sb = x.stride(0);
      f.st = x.stride(1);
    }
    r = LogProbabilidades::apply(x, y, f);
  }
  return entropia ? py::make_tuple(r[0], r[1]) : py::make_tuple(r[0], py::none());
}

// ---- the preference loss -------------------------------------------------------------------------------------------------
struct Pares {
  Opcional m, ref;
  int32_t forma, media;
  double beta, suavizado, margen;
};

struct Preferencia : Function<Preferencia> {
  static variable_list forward(AutogradContext* ctx, const Tensor& lp, const Pares& f) {
    En en(lp);
    const int64_t P = lp.size(0) / 2, L = lp.size(1), wsb = lib.pref_ws(P, L), fin = wsb < 0 ? 0 : wsb;
    // one buffer: the workspace, then the rows' coefficients, which the backward needs
    Tensor perdida = vacio({}, lp), rec = vacio({2 * P}, lp), ws = vacio({fin + 8 * P}, lp, at::kByte);
    char* w = static_cast<char*>(ws.data_ptr());
    const int32_t por_fila = !f.ref || f.ref->dim() != 1 ? 0 : f.ref->scalar_type() == at::kDouble ? 2 : 1;
    int64_t sl[2], sr[2] = {0, 0}, sm[2];
    pasos(lp, sl);
    pasos(f.m, sm);
    if (por_fila) sr[0] = f.ref->stride(0);
    else pasos(f.ref, sr);
    vale(lib.pref_fwd(f32(lp), sl, ptr(f.ref), sr, por_fila, u8(f.m), sm, P, L, f.forma, f.beta, f.suavizado, f.margen, f.media,
                      f32(perdida), f32(rec), reinterpret_cast<float*>(w + fin), w, wsb, en.st), "asrn_preference_fwd");
    ctx->save_for_backward(f.m ? variable_list{ws, *f.m} : variable_list{ws});
    ctx->saved_data["n"] = std::vector<int64_t>{P, L, fin};
    ctx->mark_non_differentiable({rec});
    ctx->set_materialize_grads(false);
    return {perdida, rec};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    una_vez("perdida_preferencia");
    if (!g[0].defined()) return {Tensor(), Tensor()};
    const variable_list s = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    const Opcional m = s.size() > 1 ? Opcional(s[1]) : std::nullopt;
    En en(s[0]);
    const Tensor dlp = vacio({2 * n[0], n[1]}, s[0]), gd = denso(g[0]);
    int64_t sm[2];
    pasos(m, sm);
    vale(lib.pref_bwd(reinterpret_cast<float*>(static_cast<char*>(s[0].data_ptr()) + n[2]), f32(gd), u8(m), sm, n[0], n[1], f32(dlp),
                      en.st), "asrn_preference_bwd");
    return {dlp, Tensor()};
  }
};

std::pair<Tensor, Tensor> preferencia(const Tensor& lp, Opcional m, Opcional ref, int32_t forma, double beta, double suavizado,
                                      double margen, bool media) {
  const variable_list r = Preferencia::apply(lp, Pares{std::move(m), std::move(ref), forma, media, beta, suavizado, margen});
  return {r[0], r[1]};
}

// ---- the policy loss -----------------------------------------------------------------------------------------------------
struct Ajustes {
  Tensor A;
  Opcional vieja, ref, m;
  double lo, hi, tope, beta, peso;
  bool por_texto, quiere;                     // quiere: lp's gradient will be asked for
};

struct Politica : Function<Politica> {
  static variable_list forward(AutogradContext* ctx, const Tensor& lp, const Opcional& H, const Ajustes& f) {
    En en(lp);
    const int64_t B = lp.size(0), L = lp.size(1), wsb = lib.pol_ws(B, L), fin = wsb < 0 ? 0 : wsb;
    // one buffer: the workspace, then what the backward needs: the texts' divisors and the tokens' gradients
    Tensor perdida = vacio({}, lp), datos = vacio({4}, lp),
           ws = vacio({fin + 4 * B + (f.quiere ? 4 * B * L : 0)}, lp, at::kByte);
    char* w = static_cast<char*>(ws.data_ptr());
    float* div = reinterpret_cast<float*>(w + fin);
    int64_t s[12];
    pasos(lp, s);
    pasos(f.A, s + 2);
    pasos(f.vieja, s + 4);
    pasos(f.ref, s + 6);
    pasos(H, s + 8);
    pasos(f.m, s + 10);
    vale(lib.pol_fwd(f32(lp), f32(f.A), f32(f.vieja), f32(f.ref), f32(H), u8(f.m), s, B, L, f.lo, f.hi, f.tope, f.beta, f.peso,
                     f.por_texto, f.quiere ? div + B : nullptr, f32(perdida), f32(datos), div, w, wsb, en.st), "asrn_policy_fwd");
    ctx->save_for_backward(f.m ? variable_list{ws, *f.m} : variable_list{ws});
    ctx->saved_data["n"] = std::vector<int64_t>{B, L, fin, H.has_value()};
    ctx->saved_data["w"] = f.peso;
    ctx->mark_non_differentiable({datos});
    ctx->set_materialize_grads(false);
    return {perdida, datos};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    una_vez("perdida_politica");
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor()};
    const variable_list s = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    const Opcional m = s.size() > 1 ? Opcional(s[1]) : std::nullopt;
    En en(s[0]);
    const int64_t B = n[0], L = n[1];
    const Tensor gd = denso(g[0]);
    Tensor dlp, dH;
    if (ctx->needs_input_grad(0)) dlp = vacio({B, L}, s[0]);
    if (n[3] && ctx->needs_input_grad(1)) dH = vacio({B, L}, s[0]);
    float* div = reinterpret_cast<float*>(static_cast<char*>(s[0].data_ptr()) + n[2]);
    int64_t sm[2];
    pasos(m, sm);
    vale(lib.pol_bwd(div + B, div, f32(gd), u8(m), sm, B, L, ctx->saved_data["w"].toDouble(), f32(dlp), f32(dH), en.st),
         "asrn_policy_bwd");
    return {dlp, dH, Tensor()};
  }
};

std::pair<Tensor, Tensor> politica(const Tensor& lp, Opcional H, Tensor A, Opcional vieja, Opcional ref, Opcional m, double lo,
                                   double hi, double tope, double beta, double peso, bool por_texto) {
  const bool quiere = at::GradMode::is_enabled() && lp.requires_grad();
  const variable_list r = Politica::apply(lp, H, Ajustes{std::move(A), std::move(vieja), std::move(ref), std::move(m), lo, hi, tope,
                                                         beta, peso, por_texto, quiere});
  return {r[0], r[1]};
}

// ---- activations in 8 bits -----------------------------------------------------------------------------------------------
// One buffer for rows (N, d): the codes, `datos` fp32 values a row (16-byte aligned), the groups' scale bytes
// (ops._partes8 gives the same places to its readers).
struct Sitio {
  int64_t N, d, m, s;
  Sitio(const Tensor& x, int64_t datos) : N(x.numel() / x.size(-1)), d(x.size(-1)) {
    m = (N * d + 15) / 16 * 16;
    s = m + (4 * datos * N + 15) / 16 * 16;
  }
  Tensor nuevo(const Tensor& x) const { return vacio({s + N * ((d + 31) / 32)}, x, at::kByte); }
};
int8_t* q_de(const Tensor& t) { return static_cast<int8_t*>(t.data_ptr()); }
uint8_t* e_de(const Tensor& t, int64_t s) { return static_cast<uint8_t*>(t.data_ptr()) + s; }

struct Gelu8 : Function<Gelu8> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Opcional& h) {
    En en(u);
    const Tensor uc = u.contiguous();
    const Opcional hc = h ? Opcional(h->contiguous()) : std::nullopt;
    const Sitio p(uc, 0);
    Tensor sitio = p.nuevo(uc), y = vacio(u.sizes(), u, h ? at::kFloat : u.scalar_type());
    vale(lib.gelu8_fwd(ptr(uc), es16(uc), f32(hc), p.N, p.d, ptr(y), q_de(sitio), e_de(sitio, p.s), en.st), "asrn_gelu8_fwd");
    ctx->save_for_backward({sitio});
    ctx->saved_data["n"] = std::vector<int64_t>{p.N, p.d, p.s, es16(u), h.has_value()};
    ctx->saved_data["f"] = u.sizes().vec();
    ctx->mark_non_differentiable({sitio});
    ctx->set_materialize_grads(false);
    return {y, sitio};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    una_vez("gelu8");
    if (!g[0].defined()) return {Tensor(), Tensor()};
    const variable_list s = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    En en(s[0]);
    Tensor du;
    if (ctx->needs_input_grad(0)) {
      const Tensor dy = es16(g[0]) ? g[0].contiguous() : denso(g[0]);
      du = vacio(ctx->saved_data["f"].toIntVector(), s[0], n[3] ? at::kBFloat16 : at::kFloat);
      vale(lib.gelu8_bwd(q_de(s[0]), e_de(s[0], n[2]), ptr(dy), es16(dy), n[0], n[1], (int32_t)n[3], ptr(du), en.st), "asrn_gelu8_bwd");
    }
    return {du, n[4] && ctx->needs_input_grad(1) ? g[0] : Tensor()};
  }
};

std::pair<Tensor, Tensor> gelu8(const Tensor& u, Opcional h) {
  const variable_list r = Gelu8::apply(u, h);
  return {r[0], r[1]};
}

// rows on the 16-byte boundary that the kernels read from
Tensor alineado(const Tensor& t) { return (uintptr_t)t.data_ptr() % 16 == 0 ? t : t.clone(); }

struct Norma8 : Function<Norma8> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gamma, const Tensor& beta, double eps,
                               bool sale16) {
    En en(x);
    const Tensor xc = alineado(x.contiguous()), g = alineado(denso(gamma)), b = alineado(denso(beta));
    const Sitio p(xc, 2);
    Tensor sitio = p.nuevo(xc), y = vacio(x.sizes(), x, sale16 ? at::kBFloat16 : at::kFloat);
    vale(lib.norm8_fwd(f32(xc), f32(g), f32(b), p.N, (int32_t)p.d, (float)eps, sale16, ptr(y),
                       reinterpret_cast<float*>(e_de(sitio, p.m)), q_de(sitio), e_de(sitio, p.s), en.st), "asrn_norm8_fwd");
    ctx->save_for_backward({sitio, g});
    ctx->saved_data["n"] = std::vector<int64_t>{p.N, p.d, p.m, p.s};
    ctx->saved_data["f"] = x.sizes().vec();
    ctx->mark_non_differentiable({sitio});
    ctx->set_materialize_grads(false);
    return {y, xc.view(x.sizes()), sitio};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    una_vez("norma8");
    const variable_list s = ctx->get_saved_variables();
    const auto n = ctx->saved_data["n"].toIntVector();
    const auto forma = ctx->saved_data["f"].toIntVector();
    if (!g[0].defined()) return {g[1], Tensor(), Tensor(), Tensor(), Tensor()};       // the residual path alone
    En en(s[0]);
    const Tensor dy = alineado(es16(g[0]) ? g[0].contiguous() : denso(g[0]));
    const Tensor dr = g[1].defined() ? alineado(denso(g[1])) : Tensor();
    const int64_t wsb = lib.norm8_ws(n[0], (int32_t)n[1]);
    Tensor dx = vacio(forma, s[0]), dp = vacio({2, n[1]}, s[0]), ws = vacio({wsb < 0 ? 0 : wsb}, s[0], at::kByte);
    vale(lib.norm8_bwd(q_de(s[0]), e_de(s[0], n[3]), f32(s[1]), reinterpret_cast<float*>(e_de(s[0], n[2])), n[0], (int32_t)n[1],
                       ptr(dy), es16(dy), f32(dr), f32(dx), f32(dp), ptr(ws), wsb, en.st), "asrn_norm8_bwd");
    return {dx, dp.select(0, 0), dp.select(0, 1), Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor, Tensor> norma8(const Tensor& x, const Tensor& gamma, const Tensor& beta, double eps, bool sale16) {
  const variable_list r = Norma8::apply(x, gamma, beta, eps, sale16);
  return {r[0], r[1], r[2]};
}

// Whether a graph recorded on the default stream still holds one of these leaves' accumulators. A backward inside a
// capture would run it on that stream, which no capture may wait for.
bool hojas_en_uso(const std::vector<Tensor>& hojas) {
  for (const Tensor& t : hojas) {
    const auto nodo = torch::autograd::impl::try_get_grad_accumulator(t);
    const auto corriente = nodo ? nodo->stream() : std::nullopt;
    if (corriente && corriente->id() == 0) return true;
  }
  return false;
}

// direccion(name): the address of an entry point of the opened library; error: the class of its failures
void iniciar(const py::function& direccion, py::object error) {
  const auto de = [&](auto& f, const char* nombre) {
    f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(direccion(nombre).cast<uintptr_t>());
  };
  de(lib.error, "asrn_hip_last_error");
  de(lib.logp_fwd, "asrn_token_logp_fwd");
  de(lib.logp_bwd, "asrn_token_logp_bwd");
  de(lib.pref_ws, "asrn_preference_workspace");
  de(lib.pref_fwd, "asrn_preference_fwd");
  de(lib.pref_bwd, "asrn_preference_bwd");
  de(lib.pol_ws, "asrn_policy_workspace");
  de(lib.pol_fwd, "asrn_policy_fwd");
  de(lib.pol_bwd, "asrn_policy_bwd");
  de(lib.gelu8_fwd, "asrn_gelu8_fwd");
  de(lib.gelu8_bwd, "asrn_gelu8_bwd");
  de(lib.norm8_fwd, "asrn_norm8_fwd");
  de(lib.norm8_bwd, "asrn_norm8_bwd");
  de(lib.norm8_ws, "asrn_norm8_bwd_workspace");
  static PyObject* clase;                     // held to the process's end
  clase = error.release().ptr();
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Fallo& f) {
      PyErr_SetString(clase, f.what());
    }
  });
}

}  // namespace

PYBIND11_MODULE(_nodos, m) {
  using Libre = py::call_guard<py::gil_scoped_release>;
  m.def("iniciar", &iniciar);
  m.def("hojas_en_uso", &hojas_en_uso);
  m.def("logp", &logp);
  m.def("preferencia", &preferencia, Libre());
  m.def("politica", &politica, Libre());
  m.def("gelu8", &gelu8, Libre());
  m.def("norma8", &norma8, Libre());
}
