// Autograd nodes, in C++, of the fine-tuning losses, of the activations in 8 bits and of a local block's operators with a
// state a channel: they allocate, launch the library's
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
#include <torch/csrc/autograd/autograd.h>
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
  decltype(&asrn_channel_conv_fwd) conv_fwd;
  decltype(&asrn_channel_conv_bwd_workspace) conv_ws;
  decltype(&asrn_channel_conv_bwd) conv_bwd;
  decltype(&asrn_channel_conv_step) conv_paso;
  decltype(&asrn_selective_checks) sel_marcas;
  decltype(&asrn_selective_fwd_workspace) sel_ws;
  decltype(&asrn_selective_fwd) sel_fwd;
  decltype(&asrn_selective_bwd_workspace) sel_bwd_ws;
  decltype(&asrn_selective_bwd) sel_bwd;
  decltype(&asrn_selective_step) sel_paso;
  decltype(&asrn_linear_act_workspace) act_ws;
  decltype(&asrn_linear_act_fwd) act_fwd;
  decltype(&asrn_act_grad_workspace) actg_ws;
  decltype(&asrn_act_grad) act_grad;
  decltype(&asrn_weight_grad_workspace) wg_ws;
  decltype(&asrn_weight_grad) wg;
  decltype(&asrn_gemm_workspace) gemm_ws;
  decltype(&asrn_gemm) gemm;
  decltype(&asrn_column_sums_workspace) cols_ws;
  decltype(&asrn_column_sums) cols;
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

// ---- a local block's operators with a state a channel ---------------------------------------------------------------------
int32_t tipo_de(const Tensor& t) { return t.scalar_type() == at::kFloat ? 0 : t.scalar_type() == at::kBFloat16 ? 1 : 2; }
// the channels next to each other: the kernels read the other axes through their strides
Tensor por_canal(const Tensor& t) { return !t.defined() || t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
// a scan's (B, L, .): its tokens within the kernels' 32-bit offsets too. The stride of a single token, or of none, may be
// anything (such a tensor is contiguous with it) and is not used: 0 stands for it.
int64_t paso_token(const Tensor& t) { return t.numel() && t.size(1) > 1 ? t.stride(1) : 0; }
Tensor cercanas(const Tensor& t) { return t.defined() && paso_token(t) >= (1 << 24) ? t.contiguous() : por_canal(t); }
void pasos_texto(const Tensor& t, int64_t* s) {
  s[0] = t.defined() ? t.stride(0) : 0;
  s[1] = t.defined() ? paso_token(t) : 0;
}
Tensor como(const Tensor& g, const Tensor& x) {       // a gradient in x's type, dense
  return g.scalar_type() == x.scalar_type() && g.is_contiguous() ? g : g.to(x.scalar_type()).contiguous();
}
Tensor f32_o_nada(const Tensor& t) { return t.defined() ? denso(t) : t; }
Tensor o_nada(const Opcional& t) { return t ? *t : Tensor(); }
Tensor espacio(int64_t n, const Tensor& x) { return vacio({n < 0 ? 0 : n}, x, at::kByte); }
bool con_gradiente(std::initializer_list<const Tensor*> ts) {
  if (at::GradMode::is_enabled())
    for (const Tensor* t : ts)
      if (t->defined() && t->requires_grad()) return true;
  return false;
}
// whether one carries a tangent of forward mode, which only the nodes refuse
bool con_tangente(std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    if (t->defined() && t->_fw_grad(0).defined()) return true;
  return false;
}
void sin_gradiente(const char* que, std::initializer_list<const Tensor*> ts) {
  if (con_gradiente(ts)) throw Fallo(std::string(que) + ": a token's step has no gradient: call it under torch.no_grad()");
  if (con_tangente(ts)) throw Fallo(std::string(que) + ": a token's step has no derivative in forward mode");
}

// t was written in place: a graph that kept it for its backward finds out
void escrito(const Tensor& t) {
  if (!t.is_inference()) torch::autograd::impl::bump_version(t);
}

// The gradients of a convolution of each channel in torch's operators, which record them: of z, w, b where they ask for one.
// Taken of aliases: the tensors' own hooks see the gradient once, when this backward has returned it.
variable_list conv_registrada(const Tensor& z0, const Tensor& w0, const Tensor& b0, const Tensor& gy, int64_t act) {
  const Tensor z = z0.alias(), w = w0.alias(), b = b0.defined() ? b0.alias() : b0;
  const int64_t L = z.size(1), d = z.size(2), k = w.size(-1);
  const Tensor zp = at::constant_pad_nd(z.to(at::kFloat), {0, 0, k - 1, 0}), wf = w.reshape({d, k}).to(at::kFloat);
  Tensor s = zp.narrow(1, 0, L) * wf.select(1, 0);
  for (int64_t j = 1; j < k; ++j) s = s + zp.narrow(1, j, L) * wf.select(1, j);
  if (b.defined()) s = s + b.to(at::kFloat);
  variable_list r(4), de;
  std::vector<int> sitio;
  for (int i = 0; i < 3; ++i) {
    const Tensor& t = i == 0 ? z : i == 1 ? w : b;
    if (!t.defined() || !t.requires_grad()) continue;
    de.push_back(t);
    sitio.push_back(i);
  }
  const variable_list g = torch::autograd::grad({act == 1 ? at::gelu(s) : act == 2 ? at::silu(s) : s}, de, {gy.to(at::kFloat)},
                                                /*retain_graph=*/true, /*create_graph=*/true);
  for (size_t i = 0; i < g.size(); ++i) r[sitio[i]] = g[i];
  return r;
}

// z (B, L, d), w (d, k) or (d, 1, k), b (d) or undefined
struct ConvCanal : Function<ConvCanal> {
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const Tensor& w, const Opcional& sesgo, int64_t act,
                               bool registrable) {
    En en(z);
    const Tensor b = o_nada(sesgo);
    const Tensor zc = por_canal(z), wc = denso(w), bc = f32_o_nada(b);
    Tensor y = vacio(z.sizes(), z, z.scalar_type());
    vale(lib.conv_fwd(ptr(zc), tipo_de(z), zc.stride(0), zc.stride(1), f32(wc), f32(bc), z.size(0), z.size(1), (int32_t)z.size(2),
                      (int32_t)w.size(-1), (int32_t)act, ptr(y), en.st), "asrn_channel_conv_fwd");
    // a recorded backward needs z itself, not a copy
    ctx->save_for_backward({registrable ? z : zc, w, b});
    ctx->saved_data["a"] = act;
    ctx->saved_data["r"] = registrable;
    return {y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    const bool registrada = at::GradMode::is_enabled() && ctx->saved_data["r"].toBool();
    if (!registrada) una_vez("conv_canal");
    const variable_list s = ctx->get_saved_variables();
    const Tensor &w = s[1], &b = s[2];
    const int64_t act = ctx->saved_data["a"].toInt();
    En en(s[0]);
    if (registrada) {
      variable_list r = conv_registrada(s[0], w, b, g[0], act);
      r.emplace_back();
      return r;
    }
    const Tensor z = por_canal(s[0]);
    const int64_t B = z.size(0), L = z.size(1), d = z.size(2), k = w.size(-1), wsb = lib.conv_ws(B, L, (int32_t)d, (int32_t)k);
    const Tensor gy = como(g[0], z), wc = denso(w), bc = f32_o_nada(b);
    Tensor dz = vacio(z.sizes(), z, z.scalar_type()), ws = espacio(wsb, z);
    Tensor dp = B * L ? vacio({k + 1, d}, z) : at::zeros({k + 1, d}, z.options().dtype(at::kFloat));
    vale(lib.conv_bwd(ptr(z), tipo_de(z), z.stride(0), z.stride(1), f32(wc), f32(bc), ptr(gy), B, L, (int32_t)d, (int32_t)k,
                      (int32_t)act, ptr(dz), f32(dp), ptr(ws), wsb, en.st), "asrn_channel_conv_bwd");
    return {dz, dp.narrow(0, 0, k).t().view_as(w).to(w.scalar_type()),
            b.defined() ? dp.select(0, k).to(b.scalar_type()) : Tensor(), Tensor(), Tensor()};
  }
};

Tensor conv_canal(const Tensor& z, const Tensor& w, const Opcional& b, int64_t act, bool registrable) {
  return ConvCanal::apply(z, w, b, act, registrable)[0];
}

// z (B, d), ventana (B, d, k - 1) dense -> y and the next window, the same tensor or a new one
std::pair<Tensor, Tensor> paso_conv_canal(const Tensor& z, const Tensor& ventana, const Tensor& w, const Opcional& b, int64_t act,
                                          bool en_sitio) {
  const Tensor bt = o_nada(b);
  sin_gradiente("paso_conv_canal", {&z, &ventana, &w, &bt});
  En en(z);
  const Tensor zc = por_canal(z), wc = denso(w), bc = f32_o_nada(bt);
  Tensor y = vacio(z.sizes(), z, z.scalar_type()), sig = en_sitio ? ventana : at::empty_like(ventana);
  vale(lib.conv_paso(ptr(zc), tipo_de(z), zc.stride(0), ptr(ventana), ptr(sig), f32(wc), f32(bc), z.size(0), (int32_t)z.size(1),
                     (int32_t)w.size(-1), (int32_t)act, ptr(y), en.st), "asrn_channel_conv_step");
  if (en_sitio) escrito(ventana);
  return {y, sig};
}

// u, dl, z (B, L, d), Bm, C (B, L, N) of one type; A (d, N), D, sesgo (d), h0 (B, d, N); D, z, sesgo, h0 may be undefined
struct Selectivo : Function<Selectivo> {
  static variable_list forward(AutogradContext* ctx, const Tensor& u, const Tensor& dl, const Tensor& A, const Tensor& Bm,
                               const Tensor& C, const Opcional& D_, const Opcional& z_, const Opcional& sesgo_,
                               const Opcional& h0_, bool softplus, bool guarda, bool estado) {
    En en(u);
    const Tensor D = o_nada(D_), z = o_nada(z_), sesgo = o_nada(sesgo_), h0 = o_nada(h0_);
    const int64_t B = u.size(0), L = u.size(1), d = u.size(2), N = A.size(1), wsb = lib.sel_ws(B, L, (int32_t)d, (int32_t)N);
    const Tensor uc = cercanas(u), dc = cercanas(dl), Bc = cercanas(Bm), Cc = cercanas(C), zc = cercanas(z);
    const Tensor Ac = denso(A), Dc = f32_o_nada(D), sc = f32_o_nada(sesgo), hc = f32_o_nada(h0);
    Tensor y = vacio(u.sizes(), u, u.scalar_type()), ws = espacio(wsb, u), fin, marcas;
    if (estado)      // no tokens: the state that came
      fin = B * L ? vacio({B, d, N}, u) : hc.defined() ? hc.clone() : at::zeros({B, d, N}, u.options().dtype(at::kFloat));
    if (guarda) marcas = vacio({lib.sel_marcas(B, L, (int32_t)d, (int32_t)N)}, u);
    int64_t st[10];
    pasos_texto(uc, st);
    pasos_texto(dc, st + 2);
    pasos_texto(Bc, st + 4);
    pasos_texto(Cc, st + 6);
    pasos_texto(zc, st + 8);
    vale(lib.sel_fwd(ptr(uc), ptr(dc), ptr(Bc), ptr(Cc), ptr(zc), tipo_de(u), st, f32(Ac), f32(Dc), f32(sc), f32(hc), B, L,
                     (int32_t)d, (int32_t)N, softplus, ptr(y), f32(fin), f32(marcas), ptr(ws), wsb, en.st), "asrn_selective_fwd");
    ctx->save_for_backward({uc, dc, A, Bc, Cc, D, zc, sesgo, marcas});
    ctx->saved_data["n"] = std::vector<int64_t>{softplus, h0.defined() ? (int64_t)h0.scalar_type() : -1};
    ctx->set_materialize_grads(false);
    return estado ? variable_list{y, fin} : variable_list{y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    una_vez("escaneo_selectivo");
    const variable_list s = ctx->get_saved_variables();
    const Tensor &u = s[0], &dl = s[1], &A = s[2], &Bm = s[3], &C = s[4], &D = s[5], &z = s[6], &sesgo = s[7], &marcas = s[8];
    const Tensor gfin = g.size() > 1 ? f32_o_nada(g[1]) : Tensor();
    variable_list r(12);
    if (!g[0].defined() && !gfin.defined()) return r;
    const auto n = ctx->saved_data["n"].toIntVector();
    En en(u);
    const auto tipo = u.scalar_type();
    const Tensor gy = g[0].defined() ? como(g[0], u) : at::zeros(u.sizes(), u.options());
    const int64_t B = u.size(0), L = u.size(1), d = u.size(2), N = A.size(1), wsb = lib.sel_bwd_ws(B, L, (int32_t)d, (int32_t)N);
    const Tensor Ac = denso(A), Dc = f32_o_nada(D), sc = f32_o_nada(sesgo);
    Tensor du = vacio(u.sizes(), u, tipo), ddl = vacio(u.sizes(), u, tipo), dB = vacio(Bm.sizes(), u, tipo),
           dC = vacio(C.sizes(), u, tipo), dz = z.defined() ? vacio(u.sizes(), u, tipo) : Tensor(), dh, ws = espacio(wsb, u);
    Tensor dp = B * L ? vacio({d * N + 2 * d}, u) : at::zeros({d * N + 2 * d}, u.options().dtype(at::kFloat));
    if (n[1] >= 0)
      dh = B * L ? vacio({B, d, N}, u) : gfin.defined() ? gfin.clone() : at::zeros({B, d, N}, u.options().dtype(at::kFloat));
    int64_t st[12];
    pasos_texto(u, st);
    pasos_texto(dl, st + 2);
    pasos_texto(Bm, st + 4);
    pasos_texto(C, st + 6);
    pasos_texto(z, st + 8);
    pasos_texto(gy, st + 10);
    vale(lib.sel_bwd(ptr(u), ptr(dl), ptr(Bm), ptr(C), ptr(z), ptr(gy), tipo_de(u), st, f32(Ac), f32(Dc), f32(sc), f32(marcas),
                     f32(gfin), B, L, (int32_t)d, (int32_t)N, (int32_t)n[0], ptr(du), ptr(ddl), ptr(dB), ptr(dC), ptr(dz), f32(dp),
                     f32(dh), ptr(ws), wsb, en.st), "asrn_selective_bwd");
    r[0] = du;
    r[1] = ddl;
    r[2] = dp.narrow(0, 0, d * N).view({d, N}).to(A.scalar_type());
    r[3] = dB;
    r[4] = dC;
    if (D.defined()) r[5] = dp.narrow(0, d * N, d).to(D.scalar_type());
    r[6] = dz;
    if (sesgo.defined()) r[7] = dp.narrow(0, d * N + d, d).to(sesgo.scalar_type());
    if (dh.defined()) r[8] = dh.to((at::ScalarType)n[1]);
    return r;
  }
};

std::pair<Tensor, Opcional> selectivo(const Tensor& u, const Tensor& dl, const Tensor& A, const Tensor& Bm, const Tensor& C,
                                      const Opcional& D, const Opcional& z, const Opcional& sesgo, const Opcional& h0,
                                      bool softplus, bool estado) {
  const Tensor Dt = o_nada(D), zt = o_nada(z), st = o_nada(sesgo), ht = o_nada(h0);
  const variable_list r = Selectivo::apply(u, dl, A, Bm, C, D, z, sesgo, h0, softplus,
                                           con_gradiente({&u, &dl, &A, &Bm, &C, &Dt, &zt, &st, &ht}), estado);
  return {r[0], estado ? Opcional(r[1]) : std::nullopt};
}

// u, dl, z (B, d), Bm, C (B, N), h (B, d, N) fp32 dense -> y and the next state, the same tensor or a new one
std::pair<Tensor, Tensor> paso_selectivo(const Tensor& u, const Tensor& dl, const Tensor& A, const Tensor& Bm, const Tensor& C,
                                         const Tensor& h, const Opcional& D, const Opcional& z, const Opcional& sesgo,
                                         bool softplus, bool en_sitio) {
  const Tensor zt = o_nada(z), Dt = o_nada(D), st_ = o_nada(sesgo);
  sin_gradiente("paso_selectivo", {&u, &dl, &A, &Bm, &C, &h, &zt, &Dt, &st_});
  En en(u);
  const Tensor uc = por_canal(u), dc = por_canal(dl), Bc = por_canal(Bm), Cc = por_canal(C), zc = por_canal(zt);
  const Tensor Ac = denso(A), Dc = f32_o_nada(Dt), sc = f32_o_nada(st_);
  Tensor y = vacio(u.sizes(), u, u.scalar_type()), sig = en_sitio ? h : at::empty_like(h);
  const int64_t st[5] = {uc.stride(0), dc.stride(0), Bc.stride(0), Cc.stride(0), zc.defined() ? zc.stride(0) : 0};
  vale(lib.sel_paso(ptr(uc), ptr(dc), ptr(Bc), ptr(Cc), ptr(zc), tipo_de(u), st, f32(Ac), f32(Dc), f32(sc), f32(h), f32(sig),
                    u.size(0), (int32_t)u.size(1), (int32_t)A.size(1), softplus, ptr(y), en.st), "asrn_selective_step");
  if (en_sitio) escrito(h);
  return {y, sig};
}

// ---- the product with its epilogue ----------------------------------------------------------------------------------------
// (M, k) rows of (..., k): adjacent values, a row stride that holds a row (an expanded tensor's does not) and fits the
// kernels' 32-bit offsets
Tensor filas(const Tensor& t) {
  const int64_t k = t.size(-1);
  Tensor r = (t.dim() == 2 ? t : t.reshape({k ? t.numel() / k : 0, k}));
  return r.size(0) > 1 && (r.stride(0) < k || r.stride(0) >= (1 << 21)) ? r.contiguous()
         : k > 1 && r.stride(1) != 1 ? r.contiguous() : r;
}
bool en_unidades(const Tensor& t) {    // 16-bit rows in whole units of 16 bytes
  return t.scalar_type() != at::kFloat && t.size(1) % 8 == 0 && (t.size(0) < 2 || t.stride(0) % 8 == 0) &&
         reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
}
// a single row's stride may be anything
int64_t paso_fila(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }

// How the gradients' products run, by the rules in lineal.py: x's and w's on asrn_gemm, or the weight gradient as one product
// (slabs 1) or a batch of slabs of the rows; w's from 16-bit rows on 16-byte boundaries on asrn_weight_grad instead
struct PlanLineal {
  int64_t gx_gemm, gw_gemm, slabs;
};

// x's rows (M, K) -> y in its own shape (..., N): no view, which a caller under autograd could not change in place
Tensor producto_act(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& res, int64_t act, at::ScalarType tipo_y,
                    const Tensor& pre, at::IntArrayRef forma, const En& en) {
  const int64_t M = x.size(0), K = x.size(1), N = w.size(0), wsb = lib.act_ws(M, N, K, tipo_de(x));
  Tensor y = vacio(forma, x, tipo_y), ws = wsb > 0 ? espacio(wsb, x) : Tensor();
  vale(lib.act_fwd(ptr(x), paso_fila(x), ptr(w), paso_fila(w), tipo_de(x), ptr(b), M, N, K, (int32_t)act, ptr(res),
                   res.defined() ? paso_fila(res) : N, res.defined() && res.scalar_type() == at::kFloat, ptr(pre), N, ptr(y), N,
                   tipo_y == at::kFloat, 0, ptr(ws), wsb, en.st), "asrn_linear_act_fwd");
  return y;
}

// the operands are cast here, and only here
struct SinAutocast {
  c10::impl::ExcludeDispatchKeyGuard guarda{c10::autocast_dispatch_keyset};
};

struct LinealActiva : Function<LinealActiva> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const Opcional& b_, const Opcional& res_,
                               int64_t act, int64_t dt_, const PlanLineal& plan) {
    En en(x);
    const SinAutocast sin;
    const auto dt = (at::ScalarType)dt_;
    const Tensor b = o_nada(b_), res = o_nada(res_);
    const Tensor x2 = filas(x.to(dt)), wc = filas(w.to(dt)), bc = b.defined() ? b.to(dt).contiguous() : b;
    Tensor pre = act ? vacio({x2.size(0), wc.size(0)}, x2, dt) : Tensor();
    auto forma = x.sizes().vec();
    forma.back() = wc.size(0);
    Tensor y = producto_act(x2, wc, bc, res.defined() ? filas(res) : res, act, res.defined() ? res.scalar_type() : dt, pre, forma, en);
    ctx->save_for_backward({x2, wc, pre});
    ctx->saved_data["n"] = std::vector<int64_t>{act, dt_, (int64_t)x.scalar_type(), (int64_t)w.scalar_type(),
                                                b.defined() ? (int64_t)b.scalar_type() : -1, res.defined(), plan.gx_gemm, plan.gw_gemm,
                                                plan.slabs};
    ctx->saved_data["f"] = x.sizes().vec();
    return {y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list g) {
    una_vez("lineal_activa");
    const variable_list s = ctx->get_saved_variables();
    const Tensor &x = s[0], &w = s[1], &pre = s[2];
    const auto n = ctx->saved_data["n"].toIntVector();
    const auto dt = (at::ScalarType)n[1];
    const bool con_b = n[4] >= 0, con_res = n[5] != 0;
    En en(x);
    const SinAutocast sin;
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    const bool qx = ctx->needs_input_grad(0), qw = ctx->needs_input_grad(1), qb = con_b && ctx->needs_input_grad(2);
    Tensor gx, gw, gb, cols;
    if (M == 0 || N == 0) {
      if (qx) gx = at::zeros(ctx->saved_data["f"].toIntVector(), x.options().dtype((at::ScalarType)n[2]));
      if (qw) gw = at::zeros({N, K}, x.options().dtype((at::ScalarType)n[3]));
      if (qb) gb = at::zeros({N}, x.options().dtype((at::ScalarType)n[4]));
    } else if (qx || qw || qb) {
      Tensor g2 = filas(g[0]), gp = g2;
      const bool propio = n[0] != 0 || g2.scalar_type() != dt;
      const bool unidades = en_unidades(x) && N % 8 == 0 && N < (1 << 21);
      const bool suma = qb && (propio || !(qw && n[7] && !unidades));          // else the weight gradient's product sums the columns too
      if (propio || suma) {
        const int64_t wsb = suma ? lib.actg_ws(M, N) : 0;
        Tensor ws = suma ? espacio(wsb, x) : Tensor();
        if (propio) gp = vacio({M, N}, x, dt);
        if (suma) cols = vacio({N}, x);
        vale(lib.act_grad(ptr(g2), paso_fila(g2), g2.scalar_type() == at::kFloat, ptr(pre), N, tipo_de(x), M, N, (int32_t)n[0],
                          propio ? ptr(gp) : nullptr, f32(cols), ptr(ws), wsb, en.st), "asrn_act_grad");
      }
      if (qx) {
        if (n[6]) {
          const Tensor gc = alineado(gp.contiguous());
          gx = vacio({M, K}, x);
          const int64_t wsb = lib.gemm_ws(M, K, N, 0, 0, 0, 0);
          Tensor ws = espacio(wsb, x);
          vale(lib.gemm(ptr(gc), N, 0, ptr(w), paso_fila(w), 0, 0, f32(gx), K, M, K, N, nullptr, 0, nullptr, 0, 0, ptr(ws), wsb, en.st),
               "asrn_gemm");
        } else {
          gx = at::mm(gp, w);
        }
        gx = gx.to((at::ScalarType)n[2]).view(ctx->saved_data["f"].toIntVector());
      }
      if (qw) {
        if (unidades) {
          const Tensor gc = en_unidades(gp) ? gp : alineado(gp.contiguous());
          gw = vacio({N, K}, x, (at::ScalarType)n[3] == dt ? dt : at::kFloat);
          const int64_t wsb = lib.wg_ws(M, N, K, 0, 0);
          Tensor ws = wsb > 0 ? espacio(wsb, x) : Tensor();
          vale(lib.wg(ptr(gc), paso_fila(gc), ptr(x), paso_fila(x), tipo_de(x), M, N, K, ptr(gw), gw.scalar_type() == at::kFloat, 0, 0,
                      ptr(ws), wsb, en.st), "asrn_weight_grad");
        } else if (n[7]) {
          const Tensor gc = alineado(gp.contiguous());
          gw = vacio({N, K}, x);
          const bool columnas = qb && !cols.defined();
          if (columnas) cols = vacio({N}, x);
          const int32_t bf = es16(x);
          const int64_t wsb = lib.gemm_ws(N, K, M, bf, columnas, 0, 0);
          Tensor ws = espacio(wsb, x);
          vale(lib.gemm(ptr(gc), N, 1, ptr(x), paso_fila(x), 0, bf, f32(gw), K, N, K, M, nullptr, 0, columnas ? f32(cols) : nullptr, 0, 0,
                        ptr(ws), wsb, en.st), "asrn_gemm");
        } else if (n[8] <= 1) {
          gw = at::mm(gp.t(), x);
        } else {
          // left operand: the transposed slab of gp; right operand: x's slab as stored (never a transposed view). The slabs'
          // products stay in fp32: rounded to 16 bits, sums that cancel would keep their roundings (16 slabs of 1,024 rows of
          // ones and minus ones: 56 for a sum of 44), and the time is the same (1001 x 775 over 16384 rows 56 us)
          const int64_t S = n[8];
          const Tensor gs = gp.contiguous().view({S, M / S, N}).transpose(1, 2), xs = x.contiguous().view({S, M / S, K});
          const Tensor partes = dt == at::kFloat ? at::bmm(gs, xs) : at::bmm(gs, xs, at::kFloat);
          gw = vacio({N, K}, x);
          const int64_t wsb = lib.cols_ws(S, N * K);
          Tensor ws = espacio(wsb, x);
          vale(lib.cols(ptr(partes), 0, S, N * K, N * K, f32(gw), ptr(ws), wsb, en.st), "asrn_column_sums");
        }
        gw = gw.to((at::ScalarType)n[3]);
      }
      if (qb) gb = cols.to((at::ScalarType)n[4]);
    }
    return {gx, gw, gb, con_res && ctx->needs_input_grad(con_b ? 3 : 2) ? g[0] : Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor lineal_activa(const Tensor& x, const Tensor& w, const Opcional& b, const Opcional& res, int64_t act, at::ScalarType dt,
                     int64_t gx_gemm, int64_t gw_gemm, int64_t slabs) {
  const Tensor bt = o_nada(b), rt = o_nada(res);
  if (con_gradiente({&x, &w, &bt, &rt}) || con_tangente({&x, &w, &bt, &rt}))
    return LinealActiva::apply(x, w, b, res, act, (int64_t)dt, PlanLineal{gx_gemm, gw_gemm, slabs})[0];
  En en(x);
  const SinAutocast sin;
  auto forma = x.sizes().vec();
  forma.back() = w.size(0);
  return producto_act(filas(x.to(dt)), filas(w.to(dt)), bt.defined() ? bt.to(dt).contiguous() : bt,
                      rt.defined() ? filas(rt) : rt, act, rt.defined() ? rt.scalar_type() : dt, Tensor(), forma, en);
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
  de(lib.conv_fwd, "asrn_channel_conv_fwd");
  de(lib.conv_ws, "asrn_channel_conv_bwd_workspace");
  de(lib.conv_bwd, "asrn_channel_conv_bwd");
  de(lib.conv_paso, "asrn_channel_conv_step");
  de(lib.sel_marcas, "asrn_selective_checks");
  de(lib.sel_ws, "asrn_selective_fwd_workspace");
  de(lib.sel_fwd, "asrn_selective_fwd");
  de(lib.sel_bwd_ws, "asrn_selective_bwd_workspace");
  de(lib.sel_bwd, "asrn_selective_bwd");
  de(lib.sel_paso, "asrn_selective_step");
  de(lib.act_ws, "asrn_linear_act_workspace");
  de(lib.act_fwd, "asrn_linear_act_fwd");
  de(lib.actg_ws, "asrn_act_grad_workspace");
  de(lib.act_grad, "asrn_act_grad");
  de(lib.wg_ws, "asrn_weight_grad_workspace");
  de(lib.wg, "asrn_weight_grad");
  de(lib.gemm_ws, "asrn_gemm_workspace");
  de(lib.gemm, "asrn_gemm");
  de(lib.cols_ws, "asrn_column_sums_workspace");
  de(lib.cols, "asrn_column_sums");
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
  m.def("conv_canal", &conv_canal, Libre());
  m.def("paso_conv_canal", &paso_conv_canal, Libre());
  m.def("selectivo", &selectivo, Libre());
  m.def("paso_selectivo", &paso_selectivo, Libre());
  m.def("lineal_activa", &lineal_activa, Libre());
}
