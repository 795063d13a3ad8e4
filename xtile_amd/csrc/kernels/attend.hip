// Masked attention, softmax(scores) v with the scores' cap, distance bias and masks
// (xtile_amd.dsl.attend states them), in one pass over the keys: a running maximum
// m and total l of a row, and its sum of weighted values, rescaled where m grows:
//   s = q . k;  m' = max(m, s);  l = l e^(m - m') + sum e^(s - m');  o likewise
// Scores and sums are held in 32 bits in units of log2; weights are rounded to the
// values' type for the second product.
//
// The products run transposed, scores^T = K Q^T and result^T = V^T P^T, on 32 x 32
// MFMA tiles: a lane then holds one query row, so the running maximum and total are
// one register each, reduced within the lane and with one swap of lane halves, and
// the weights leave the first product in the registers in which the second takes
// them (keys in the order of the accumulator's registers; the values are read in
// that order by transposing LDS reads).
//
// All heads that share a key head are one list of rows, token by token, so they
// read the keys once.  128 rows a workgroup, the keys shared through LDS by its four
// waves; up to 32 rows (single tokens), every wave takes tiles of keys of its own.
// The cap: cap tanh(z), z = score / cap, as cap (1 - 2 / (e^2z + 1)), off by a few
// 2^-24 cap, or, for a tile of scores with |z| <= 1/2 throughout (caps are set far
// above ordinary scores), as z times a polynomial in z^2 fitted to tanh(z) / z there
// (relative error 5.4e-7 by fit, 6.2e-7 in 32 bits): five operations a score in place
// of five of which two take twice the time.  A few 2^-24 of a large cap are more than a
// score may be off by, so above 256 (and where the polynomial's coefficients are no normal
// numbers) kernels of their own take, in tiles with larger |z|, the form that each score
// asks for.
//
// Tiles that no row sees are not read: the visible ones are two runs, the prefix
// and the band between window and diagonal, cut to the keys whose documents may be
// the rows'.  Few rows over many keys are split over workgroups that leave their
// m, l and sums in the workspace, and a second kernel joins them.
//
// Drafted trees (parents): a token's ancestors are 64 bits, made in each wave by lanes that
// double how far up they have seen, and are turned into the tiles' masks where a tile has
// drafted tokens; the rest of the cache is seen whole.  The kernels are those of other rows,
// in instantiations of their own, and one more for 33 to 64 rows.  What only needs to know the
// Block (parents, slopes, q) is on its way first, and where no other workgroup reads the same
// keys a Block's are on all XCDs (16 sequences of different lengths: 107 -> 101 us).
// 4 x 16 rows on 8 key heads of 128 over 4096 keys take 15 us, most of it a chain of waits:
// two launches 4, what the first loads wait for 4, four tiles 4, the join 3.  4 x 32 rows in
// 16 sequences of up to 8192 keys take 101 us, 0.5 PFLOP/s and 3.6 TB/s; 8 x 64 rows over
// 131072 keys, capped, 356 to 376, 0.73 to 0.78 PFLOP/s.  Weights are rounded to the values' type,
// as other rows' are: against 64 bits these three are off by 0.0020, 0.0022 and (f16) 0.00028,
// with weights of 32 bits by 0.0017, 0.0017 and 0.00021, most of it the result's own rounding.
//
// Many rows are bound by the arithmetic of the softmax (4096 tokens, 32 heads of 128
// columns on 8 key heads, causal, capped: 166 to 181 us, 0.76 to 0.83 PFLOP/s; 158 without
// the cap), single tokens by HBM (64 heads of 128 on 8, 131072 keys: 102 to 107 us, 5.0 to
// 5.2 TB/s).
#include "attend_kernels.h"

#include <cmath>

#include "launch.h"

namespace xtk {

extern template hipError_t run_attend<32>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
extern template hipError_t run_attend<64>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
extern template hipError_t run_attend<96>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
extern template hipError_t run_attend<128>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
extern template hipError_t run_attend<160>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
extern template hipError_t run_attend<192>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
extern template hipError_t run_attend<224>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);
extern template hipError_t run_attend<256>(bool, bool, const AttendArgs&, const FineCap*, hipStream_t);

extern template hipError_t run_attend_tree<32>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
extern template hipError_t run_attend_tree<64>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
extern template hipError_t run_attend_tree<96>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
extern template hipError_t run_attend_tree<128>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
extern template hipError_t run_attend_tree<160>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
extern template hipError_t run_attend_tree<192>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
extern template hipError_t run_attend_tree<224>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);
extern template hipError_t run_attend_tree<256>(bool, bool, const AttendArgs&, const TreeCap&, bool, hipStream_t);

hipError_t launch_attend(const xt::Plan& p, void* const* bufs, void* work, hipStream_t s, std::string& why) {
  const xt::AttendPlan& t = p.attend;
  // a workgroup reads its own query rows before it stores them, so the result may
  // lie over q, element for element, where no two Blocks have the same; over nothing else
  auto apart = [&](int in) {
    if (in < 0 || (in != t.o.arg && !buffers_meet(p, bufs, t.o.arg, in))) return true;
    const xt::TileAddr &a = t.q.addr, &b = t.o.addr;
    if (in == t.q.arg && bufs[in] == bufs[t.o.arg] && t.q.head == t.o.head && t.q.row == t.o.row && a.c0 == b.c0 &&
        a.sx == b.sx && a.sy == b.sy && a.sz == b.sz && own_tiles(p, b))
      return true;
    why = "buffer " + std::to_string(t.o.arg) + " is stored and meets buffer " + std::to_string(in) +
          ", which the program reads elsewhere";
    return false;
  };
  for (const xt::AttendAccess* a : {&t.q, &t.k, &t.v, &t.extra[0], &t.extra[1], &t.extra[2], &t.extra[3], &t.extra[4],
                                    &t.extra[5], &t.extra[6]})
    if (!apart(a->arg)) return hipErrorInvalidValue;
  auto off = [](const xt::AttendAccess& a) {  // tile steps are not negative
    return Walk{static_cast<unsigned long long>(a.addr.sx), static_cast<unsigned long long>(a.addr.sy),
                static_cast<unsigned long long>(a.addr.sz)};
  };
  auto bytes = [&](const xt::AttendAccess& a) {
    return static_cast<unsigned char*>(bufs[a.arg]) + a.addr.c0 * xt::elem_bytes(a.elem);
  };
  AttendArgs a{};
  a.q = bytes(t.q);
  a.k = bytes(t.k);
  a.v = bytes(t.v);
  a.o = bytes(t.o);
  a.tq = off(t.q);
  a.tk = off(t.k);
  a.tv = off(t.v);
  a.to = off(t.o);
  a.q_head = t.q.head;
  a.q_row = t.q.row;
  a.o_head = t.o.head;
  a.o_row = t.o.row;
  a.ldk = t.k.row;
  a.ldv = t.v.row;
  if (t.extra[0].arg >= 0) {
    a.slopes = reinterpret_cast<const float*>(bytes(t.extra[0]));
    a.tslopes = off(t.extra[0]);
    a.slope_step = t.extra[0].row;
  }
  auto ints = [&](int e, const int*& at, Walk& o) {
    if (t.extra[e].arg < 0) return;
    at = reinterpret_cast<const int*>(bytes(t.extra[e]));
    o = off(t.extra[e]);
  };
  ints(1, a.start, a.tstart);
  ints(2, a.length, a.tlength);
  ints(3, a.prefix, a.tprefix);
  ints(4, a.qdocs, a.tqdocs);
  ints(5, a.kdocs, a.tkdocs);
  a.qdoc_step = t.extra[4].row;
  a.heads = static_cast<int>(t.heads);
  a.rows = static_cast<int>(t.heads * t.rows);
  a.keys = static_cast<int>(t.keys);
  const bool few = a.rows <= xt::kAttendFewRows;
  const int per = static_cast<int>(few ? xt::kAttendFewRows : xt::kAttendRows);
  a.tiles = (a.rows + per - 1) / per;
  a.splits = work ? t.splits : 1;
  a.work = static_cast<float*>(work);
  const long long blocks = grid_blocks(p), nwg = blocks * a.tiles * a.splits;
  if (!grid_fits(nwg, 256) || (a.splits > 1 && !grid_fits(blocks * a.rows, 256))) {
    why = "attend: " + std::to_string(nwg) + " workgroups exceed one launch";
    return hipErrorInvalidValue;
  }
  a.nwg = static_cast<int>(nwg);
  a.blocks = block_decode(p.grid[0], p.grid[1], false);
  a.d_heads = div31(a.heads);
  a.d_work = div31(a.tiles * a.splits);
  a.d_splits = div31(a.splits);
  a.scale_log2 = t.scale * 1.44269504088896340736f;
  FineCap fine{};
  const FineCap* look = nullptr;
  if (t.cap > 0) {
    // z = s scale / cap of a product s.  The polynomial's powers of scale / cap go into its
    // coefficients where they are normal numbers, else z is worked out (mul).  What passes
    // half of float's range is held there: such caps leave scores alone, or near 0.
    static constexpr double most = 1.7e38;
    auto held = [](double v) { return static_cast<float>(v < most ? v : most); };
    const double scale = t.scale, z = scale / t.cap, log2e = 1.4426950408889634;
    const bool ordinary = z > 1e-4 && z < 1e4;
    a.cap_in = held(2.0 * z * log2e);
    a.cap_log2 = held(std::max<double>(t.cap * log2e, 1.17549435e-38));
    fine.mul = ordinary ? 1.0f : held(z);
    a.cap_near = held(0.5 / z);
    static const double poly[4] = {0.999999456, -0.33326318, 0.131902967, -0.0444022264};
    for (int i = 0; i < 4; ++i) a.cap_poly[i] = held(poly[i] * scale * log2e * (ordinary ? std::pow(z, 2 * i) : 1.0));
    // a few 2^-24 of 256 are less than half precision's rounding of a weight
    if (!ordinary || t.cap > 256) look = &fine;
  }
  a.causal = t.causal;
  a.window = static_cast<int>(t.window);
  // DMA takes 16-byte aligned rows, of which 64 lie within a descriptor's 4 GiB;
  // other rows go through registers
  auto chunks = [&](const xt::AttendAccess& x) {
    const xt::TileAddr& d = x.addr;
    return reinterpret_cast<uintptr_t>(bufs[x.arg]) % 16 == 0 && x.row % 8 == 0 && d.c0 % 8 == 0 && d.sx % 8 == 0 &&
           d.sy % 8 == 0 && d.sz % 8 == 0;
  };
  a.dma = chunks(t.k) && chunks(t.v);
  const bool b = t.elem == xt::Elem::BF16;
  if (t.extra[6].arg >= 0) {
    TreeCap tree{};
    tree.mul = fine.mul;
    ints(6, tree.parents, tree.tparents);
    tree.step = t.extra[6].row;
    tree.tokens = static_cast<int>(t.rows);
    const bool l = look != nullptr;
    switch (t.d) {
      case 32: return run_attend_tree<32>(b, few, a, tree, l, s);
      case 64: return run_attend_tree<64>(b, few, a, tree, l, s);
      case 96: return run_attend_tree<96>(b, few, a, tree, l, s);
      case 128: return run_attend_tree<128>(b, few, a, tree, l, s);
      case 160: return run_attend_tree<160>(b, few, a, tree, l, s);
      case 192: return run_attend_tree<192>(b, few, a, tree, l, s);
      case 224: return run_attend_tree<224>(b, few, a, tree, l, s);
      default: return run_attend_tree<256>(b, few, a, tree, l, s);
    }
  }
  switch (t.d) {
    case 32: return run_attend<32>(b, few, a, look, s);
    case 64: return run_attend<64>(b, few, a, look, s);
    case 96: return run_attend<96>(b, few, a, look, s);
    case 128: return run_attend<128>(b, few, a, look, s);
    case 160: return run_attend<160>(b, few, a, look, s);
    case 192: return run_attend<192>(b, few, a, look, s);
    case 224: return run_attend<224>(b, few, a, look, s);
    default: return run_attend<256>(b, few, a, look, s);
  }
}

}  // namespace xtk
