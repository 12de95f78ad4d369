// The attention block between the q|k|v product and the output projection: rotary positions, the 8-bit cache, attention over it.
// A part of class Engine (included in it).

  // ---- rotary positions.  freq: radians a position step, one for each pair; kept as 64-bit fractions of a turn (kernels/rope.hip).
  struct Rope {
    int pairs = 0, axes = 1;
    bool neighbours = false;
    float mscale = 1.0f;
    cl_mem tab = nullptr;
  };
  Rope make_rope(int pairs, const double* freq, const uint8_t* axis, int axes, bool neighbours, float mscale) {
    if (pairs < 1 || pairs > 512 || !freq || axes < 1 || axes > 255)
      throw std::runtime_error("make_rope: 1 to 512 pairs on 1 to 255 axes");
    std::vector<uint64_t> tab(pairs + (pairs + 1) / 2, 0);
    for (int i = 0; i < pairs; ++i) {
      if (!std::isfinite(freq[i])) throw std::runtime_error("make_rope: frequency " + std::to_string(i) + " is no number");
      if (axis && axis[i] >= axes) throw std::runtime_error("make_rope: pair " + std::to_string(i) + " on axis " + std::to_string(axis[i]) + " of " + std::to_string(axes));
      const long double turns = (long double)freq[i] / 6.283185307179586476925286766559L, part = turns - floorl(turns);
      const long double f = floorl(part * 18446744073709551616.0L + 0.5L);
      tab[i] = f >= 18446744073709551616.0L ? 0 : (uint64_t)f;   // (a whole turn)
      ((int*)&tab[pairs])[i] = axis ? axis[i] : 0;
    }
    Rope r;
    r.pairs = pairs;
    r.axes = axes;
    r.neighbours = neighbours;
    r.mscale = mscale;
    r.tab = buf(tab.size() * 8, tab.data());
    return r;
  }

  // The bytes of a buffer that a call takes (none: empty).  Each buffer's place is looked up once a call.
  struct Place {
    uintptr_t b = 0, e = 0;
  };
  static bool overlap(Place a, Place b) { return a.b < b.e && b.b < a.e; }
  // Rows that a call of this part reads or writes: T rows of `width` values from column `off` on, a row every ld.
  struct Rows {
    uintptr_t begin, end;
    int ld, width;
    bool vec() const { return begin % 16 == 0 && ld % 4 == 0; }
    Place place() const { return {begin, end}; }   // (the columns between the rows too)
  };
  static Rows rows_of(const char* what, cl_mem m, int ld, int off, int width, int T) {
    if (off < 0 || width <= 0 || ld < 0 || (int64_t)off + width > ld)
      throw std::runtime_error(std::string(what) + ": columns " + std::to_string(off) + " ... of " + std::to_string(width) + " in rows of " + std::to_string(ld));
    const uintptr_t p = (uintptr_t)arcz_mem_ptr(m);
    const size_t last = ((size_t)(T - 1) * ld + (size_t)off + width) * 4;
    if (!m || p % 4 || arcz_mem_size(m) < last)
      throw std::runtime_error(std::string(what) + ": the buffer is too small for " + std::to_string(T) + " rows of " + std::to_string(ld));
    return {p + (size_t)off * 4, p + last, ld, width};
  }
  // Whether two such sets of rows have a value in common (or may have: rows of different strides in one place).
  static bool overlap(const Rows& a, const Rows& b) {
    if (!overlap(a.place(), b.place())) return false;
    if (a.ld != b.ld || (a.begin > b.begin ? a.begin - b.begin : b.begin - a.begin) % 4) return true;
    const size_t ld = (size_t)a.ld;
    const size_t d = a.begin <= b.begin ? (b.begin - a.begin) / 4 % ld : (ld - (a.begin - b.begin) / 4 % ld) % ld;
    return d < (size_t)a.width || d + (size_t)b.width > ld;
  }
  static Place ints(const char* what, const char* part, cl_mem m, size_t n) {
    const uintptr_t p = (uintptr_t)arcz_mem_ptr(m);
    if (!m || p % 4 || arcz_mem_size(m) < n * 4) throw std::runtime_error(std::string(what) + ": " + part + " holds less than " + std::to_string(n) + " values");
    return {p, p + n * 4};
  }

  void rope(const Rope& r, cl_mem x, int ldx, int x_off, cl_mem y, int ldy, int y_off, int T, int heads, int hd, cl_mem pos, int ld_pos) {
    if (!r.tab) throw std::runtime_error("rope: no rotation");
    if (T == 0) return;
    if (T < 0 || heads < 1 || hd < 1 || (int64_t)heads * hd > 0x7FFFFFFF || 2 * r.pairs > hd)
      throw std::runtime_error("rope: " + std::to_string(heads) + " heads of " + std::to_string(hd) + " values, " + std::to_string(r.pairs) + " pairs");
    const Rows a = rows_of("rope: x", x, ldx, x_off, heads * hd, T), b = rows_of("rope: y", y, ldy, y_off, heads * hd, T);
    if (!(a.begin == b.begin && ldx == ldy) && overlap(a, b)) throw std::runtime_error("rope: x and y overlap (in place: the same columns of the same rows)");
    if (ld_pos < T) throw std::runtime_error("rope: positions of " + std::to_string(T) + " rows on axes " + std::to_string(ld_pos) + " apart");
    if (overlap(b.place(), ints("rope", "pos", pos, (size_t)(r.axes - 1) * ld_pos + T))) throw std::runtime_error("rope: y overlaps pos");
    int vec = a.vec() && b.vec() && hd % 4 == 0, nb = r.neighbours, ax = r.axes, pairs = r.pairs;
    float ms = r.mscale;
    // (few tokens: a token's heads over several work-groups)
    int per = T >= 256 ? heads : std::min(heads, 8);
    cl_kernel k = variant("attn", {}, "rope");
    set_args(k, 0, x, ldx, x_off, y, ldy, y_off, pos, ld_pos, r.tab, pairs, ax, nb, ms, heads, hd, per, vec);
    size_t g[2] = {(size_t)T * 256, (size_t)((heads + per - 1) / per)}, l[2] = {256, 1};
    run("rope", k, 2, g, l);
  }

  // Norm and rotation of `nq` heads of queries and nk of keys behind them (kernels/norm_rope.hip).
  void norm_rope(const Rope& r, cl_mem x, int ldx, int x_off, cl_mem y, int ldy, int y_off, int T, int nq, int nk, int hd, cl_mem wq, cl_mem wk, float eps, cl_mem pos,
                 int ld_pos) {
    if (!r.tab) throw std::runtime_error("norm_rope: no rotation");
    if (T < 0 || nq < 0 || nk < 0 || (int64_t)nq + nk < 1 || hd < 1 || ((int64_t)nq + nk) * hd > 0x7FFFFFFF || 2 * r.pairs > hd)
      throw std::runtime_error("norm_rope: " + std::to_string(nq) + " and " + std::to_string(nk) + " heads of " + std::to_string(hd) + " values, " + std::to_string(r.pairs) + " pairs");
    if (!std::isfinite(eps) || eps < 0.0f) throw std::runtime_error("norm_rope: eps");
    if (T == 0) return;
    int heads = nq + nk;
    const Rows a = rows_of("norm_rope: x", x, ldx, x_off, heads * hd, T), b = rows_of("norm_rope: y", y, ldy, y_off, heads * hd, T);
    if (!(a.begin == b.begin && ldx == ldy) && overlap(a, b)) throw std::runtime_error("norm_rope: x and y overlap (in place: the same columns of the same rows)");
    if (ld_pos < T) throw std::runtime_error("norm_rope: positions of " + std::to_string(T) + " rows on axes " + std::to_string(ld_pos) + " apart");
    Place weights[2];
    if (wq) weights[0] = ints("norm_rope", "the queries' weight", wq, (size_t)hd);
    if (wk) weights[1] = ints("norm_rope", "the keys' weight", wk, (size_t)hd);
    if (overlap(b.place(), ints("norm_rope", "pos", pos, (size_t)(r.axes - 1) * ld_pos + T)) || overlap(b.place(), weights[0]) || overlap(b.place(), weights[1]))
      throw std::runtime_error("norm_rope: y overlaps pos or a weight");
    int nb = r.neighbours, ax = r.axes, pairs = r.pairs, rest = hd - 2 * pairs, L = 0;
    float ms = r.mscale;
    // lanes a head: eight values each, four behind the pairs
    const int need = nb ? (hd + 7) / 8 : std::max(pairs, rest) / 4;
    if (a.vec() && b.vec() && hd % 4 == 0 && pairs % (nb ? 2 : 4) == 0 && need <= 64) L = 1 << log2_of(need);
    // Few tokens: a token's heads over several work-groups, as long as these are one round of the chip (40 heads of 128 values, us, one work-group a
    // token / three: 64 tokens 4.8 / 3.6, 256 tokens 5.7 / 4.8; 777 11.2 / 12.5 (24 of 256), 2500 24.0 / 28.3, 8192 63 / 78).  Few heads: several tokens a
    // work-group, as far as their sines fit.
    const int lanes = L ? L : 64, round = 256 / lanes;
    int per = (int64_t)T * ((heads + round - 1) / round) > 8 * arcz_device_cus() ? heads : std::min(heads, round), tpw = 1;
    if (per == heads) tpw = std::max(1, std::min({T, round / heads, 512 / pairs}));
    cl_kernel k = variant("attn", {{"FORM", L ? nb : 2}}, "norm_rope");
    set_args(k, 0, x, ldx, x_off, y, ldy, y_off, wq, wk, eps, pos, ld_pos, r.tab, pairs, ax, nb, ms, T, nq, heads, hd, tpw, per, L);
    size_t g[2] = {(size_t)((T + tpw - 1) / tpw) * 256, (size_t)((heads + per - 1) / per)}, l[2] = {256, 1};
    run("norm_rope", k, 2, g, l);
  }

  // ---- the cache
  struct Kv {
    int pages = 0, page = 0, block = 0, heads = 0, hd = 0, ps = 0, bs = 0;
    cl_mem b[4] = {nullptr, nullptr, nullptr, nullptr};   // keys, values (int8), their scales (f32)
    size_t bytes[4] = {0, 0, 0, 0};                       // ... what the cache takes of each
    bool mine[4] = {false, false, false, false};
  };
  static int log2_of(int v) {
    int n = 0;
    while ((1 << n) < v) ++n;
    return n;
  }
  Kv make_kv(int pages, int page, int block, int heads, int hd, const cl_mem* given) {
    if (pages < 1 || heads < 1 || heads > 32767 || (hd != 64 && hd != 128 && hd != 256) || page < 16 || page > 256 || (page & (page - 1)) || block < 1 || block > page || (block & (block - 1)))
      throw std::runtime_error("make_kv: " + std::to_string(pages) + " pages of " + std::to_string(page) + " tokens in blocks of " + std::to_string(block) + ", " +
                               std::to_string(heads) + " heads of " + std::to_string(hd) +
                               " (pages of 16, 32, 64, 128 or 256 tokens, blocks of a power of two up to the page, heads of 64, 128 or 256)");
    Kv c;
    c.pages = pages; c.page = page; c.block = block; c.heads = heads; c.hd = hd;
    c.ps = log2_of(page);
    c.bs = log2_of(block);
    const size_t rows = (size_t)pages * heads * page, size[4] = {rows * hd, rows * hd, rows / block * 4, rows / block * 4};
    Place given_at[4];
    for (int i = 0; i < 4; ++i) {
      cl_mem m = given ? given[i] : nullptr;
      c.bytes[i] = size[i];
      if (!m) continue;
      const uintptr_t at = (uintptr_t)arcz_mem_ptr(m);
      if (arcz_mem_size(m) < size[i] || at % (i < 2 ? 16 : 4))
        throw std::runtime_error("make_kv: buffer " + std::to_string(i) + " holds " + std::to_string(arcz_mem_size(m)) + " bytes, the cache takes " + std::to_string(size[i]) +
                                 " (the values' at an address of 16)");
      given_at[i] = {at, at + size[i]};
      for (int j = 0; j < i; ++j)
        if (overlap(given_at[i], given_at[j])) throw std::runtime_error("make_kv: two of the buffers overlap");
      c.b[i] = m;
    }
    try {
      for (int i = 0; i < 4; ++i)
        if (!c.b[i]) {
          c.b[i] = buf(size[i]);
          c.mine[i] = true;
        }
    } catch (...) {
      for (int i = 0; i < 4; ++i)
        if (c.mine[i]) release(c.b[i]);
      throw;
    }
    return c;
  }
  void free_kv(Kv& c) {
    for (int i = 0; i < 4; ++i)
      if (c.mine[i]) not_listed(c.b[i], "free_kv");
    for (int i = 0; i < 4; ++i)
      if (c.mine[i] && c.b[i]) {
        release(c.b[i]);
        c.b[i] = nullptr;
      }
  }

  struct Batch {
    cl_mem rows, len, table;
    int seqs, ld_table, T, max_rows, max_len;
  };
  // What a launch reads of a batch is not what it writes: work-groups that begin later would see it changed.
  struct Places {
    Place cache[4], rows, len, table;
    bool in_cache(const Rows& r) const { return in_cache(r.place()); }
    bool in_cache(Place p) const {
      for (const Place& c : cache)
        if (overlap(p, c)) return true;
      return false;
    }
    bool in_batch(Place p) const { return overlap(p, rows) || overlap(p, len) || overlap(p, table); }
  };
  // false: nothing to do
  bool check_batch(const char* what, const Kv& c, const Batch& b, Places& at) {
    if (!c.b[0]) throw std::runtime_error(std::string(what) + ": no cache");
    for (int i = 0; i < 4; ++i) {   // (a buffer that was freed under the cache, or another one in its handle's place)
      const uintptr_t p = (uintptr_t)arcz_mem_ptr(c.b[i]);
      if (arcz_mem_size(c.b[i]) < c.bytes[i] || p % (i < 2 ? 16 : 4)) throw std::runtime_error(std::string(what) + ": a buffer of the cache is gone");
      at.cache[i] = {p, p + c.bytes[i]};
    }
    if (b.seqs < 0 || b.T < 0 || b.max_rows < 0 || b.ld_table < 0 || b.seqs > 65535)
      throw std::runtime_error(std::string(what) + ": a batch of " + std::to_string(b.seqs) + " sequences, " + std::to_string(b.T) + " rows");
    if (b.seqs == 0 || b.T == 0 || b.max_rows == 0) return false;
    if (b.ld_table < 1 || (int64_t)b.ld_table * c.page > 0x7FFFF000)
      throw std::runtime_error(std::string(what) + ": " + std::to_string(b.ld_table) + " pages of " + std::to_string(c.page) + " a sequence");
    at.rows = ints(what, "rows", b.rows, (size_t)b.seqs + 1);
    at.len = ints(what, "len", b.len, (size_t)b.seqs);
    at.table = ints(what, "table", b.table, (size_t)b.seqs * b.ld_table);
    return true;
  }
  // ---- a pass's batch made on the GPU (kernels/plan.hip)
  struct Plan {
    cl_mem add, before, ring, state, after, shared, pos, slot;
    int pages, page;
  };
  void kv_plan(const Batch& b, const Plan& p) {
    const std::string what = "kv_plan";
    if (b.seqs < 0 || b.seqs > 65535 || b.T < 0 || b.max_rows < 0 || b.ld_table < 0)
      throw std::runtime_error(what + ": a batch of " + std::to_string(b.seqs) + " sequences, " + std::to_string(b.T) + " rows");
    if (p.pages < 1 || p.page < 16 || p.page > 256 || (p.page & (p.page - 1)))
      throw std::runtime_error(what + ": " + std::to_string(p.pages) + " pages of " + std::to_string(p.page) + " tokens (16, 32, 64, 128 or 256)");
    if (p.slot && (int64_t)p.pages * p.page > 0x7FFFFFFF) throw std::runtime_error(what + ": places of " + std::to_string(p.pages) + " pages of " + std::to_string(p.page) + " tokens do not fit 32 bits");
    if (b.seqs == 0) return;
    if (b.ld_table < 1 || (int64_t)b.ld_table * p.page > 0x7FFFF000) throw std::runtime_error(what + ": " + std::to_string(b.ld_table) + " pages of " + std::to_string(p.page) + " a sequence");
    const size_t n = (size_t)b.seqs;
    const char* const name = "kv_plan";
    // what is written, then what is read
    Place out[7] = {ints(name, "rows", b.rows, n + 1), ints(name, "len", b.len, n), ints(name, "table", b.table, n * b.ld_table), ints(name, "ring", p.ring, (size_t)p.pages),
                    ints(name, "after", p.after, 4)};
    if (p.pos) out[5] = ints(name, "pos", p.pos, (size_t)b.T);
    if (p.slot) out[6] = ints(name, "slot", p.slot, (size_t)b.T);
    Place in[4] = {ints(name, "add", p.add, n), ints(name, "before", p.before, n), ints(name, "state", p.state, 4)};
    if (p.shared) in[3] = ints(name, "shared", p.shared, n);
    for (int i = 0; i < 7; ++i) {
      for (int j = 0; j < i; ++j)
        if (overlap(out[i], out[j])) throw std::runtime_error(what + ": two of rows, len, table, ring, after, pos and slot overlap");
      for (int j = 0; j < 4; ++j)   // (lengths and the ring's state may be brought on where they are)
        if (overlap(out[i], in[j]) && !((i == 1 && j == 1) || (i == 4 && j == 2)) ) throw std::runtime_error(what + ": what is written overlaps add, before, state or shared");
    }
    if ((overlap(out[1], in[1]) && out[1].b != in[1].b) || (overlap(out[4], in[2]) && out[4].b != in[2].b))
      throw std::runtime_error(what + ": before and len, or state and after, overlap (in place: the same values)");
    // Few rows: the work-group that makes the batch writes their places too; more are a second launch.  (us, one launch / two: 256 sequences of a token
    // 3.8 / 6.5, of four 4.4 / 6.6, of eight 5.6 / 6.3; 512 of eight 8.6 / 7.5; 64 of 32 8.3 / 6.4; one of 4096 13.4 / 6.9.)
    int seqs = b.seqs, ldt = b.ld_table, T = b.T, mr = b.max_rows, pages = p.pages, ps = log2_of(p.page);
    const bool places = (p.pos || p.slot) && T > 0 && mr > 0;
    int with = places && std::min<int64_t>(T, (int64_t)seqs * mr) <= (mr <= 8 ? 2048 : 1024) ? 1 : 0;
    cl_kernel k = variant("attn", {}, "kv_plan");
    set_args(k, 0, p.add, p.before, b.len, b.rows, b.table, ldt, p.ring, p.state, p.after, p.shared, p.pos, p.slot, seqs, T, mr, pages, ps, with);
    // (us, 256 threads / 1024: 256 sequences of a token 3.8 / 5.2, 512 12.6 / 5.3)
    size_t g1 = seqs <= 256 ? 256 : 1024, l1 = g1;
    run("kv_plan", k, 1, &g1, &l1);
    if (!places || with) return;
    cl_kernel k2 = variant("attn", {}, "kv_places");
    set_args(k2, 0, b.rows, b.len, b.table, ldt, p.pos, p.slot, T, mr, pages, ps);
    size_t g[2] = {(size_t)((std::min(mr, T) - 1) / 1024 + 1) * 256, n}, l[2] = {256, 1};
    run("kv_places", k2, 2, g, l);
  }
  void kv_write(const Kv& c, const Batch& b, cl_mem k, int ldk, int k_off, cl_mem v, int ldv, int v_off) {
    Places at;
    if (!check_batch("kv_write", c, b, at)) return;
    const int w = c.heads * c.hd, most = std::min(b.max_rows, b.T);
    const Rows rk = rows_of("kv_write: k", k, ldk, k_off, w, b.T), rv = rows_of("kv_write: v", v, ldv, v_off, w, b.T);
    if (at.in_cache(rk) || at.in_cache(rv)) throw std::runtime_error("kv_write: the rows overlap the cache");
    if (at.in_cache(at.rows) || at.in_cache(at.len) || at.in_cache(at.table)) throw std::runtime_error("kv_write: the cache overlaps the batch's rows, len or table");
    int vec = rk.vec() && rv.vec(), pages = c.pages, heads = c.heads, ps = c.ps, bs = c.bs, ldt = b.ld_table, T = b.T, mr = b.max_rows;
    // A work-group's tokens: whole blocks, and up to the eight rows a thread that it holds in registers (read once instead of twice:
    // 8192 rows x 8 heads x 128 values, blocks of 32 tokens, 25 -> 19.6 us; ragged prompts, 4 x 256, a scale a token, 26 -> 14.8; the rows in
    // the 256 MB behind the L2s).
    const int full = 8 * 1024 / c.hd;
    int tile = std::max(c.block, most == 1 ? 1 : std::min(full, 1 << log2_of(most)));
    cl_kernel kn = variant("attn", {{"HD", c.hd}}, "kv_write");
    set_args(kn, 0, k, ldk, k_off, v, ldv, v_off, c.b[0], c.b[1], c.b[2], c.b[3], pages, heads, ps, bs, b.rows, b.len, b.table, ldt, T, mr, tile, vec);
    size_t g[3] = {((size_t)(most - 1) / tile + 2) * 256, (size_t)b.seqs, (size_t)heads * 2}, l[3] = {256, 1, 1};
    if (most == 1) g[0] = 256;
    run("kv_write", kn, 3, g, l);
  }
  void kv_read(const Kv& c, const Batch& b, cl_mem k, int ldk, int k_off, cl_mem v, int ldv, int v_off) {
    Places at;
    if (!check_batch("kv_read", c, b, at)) return;
    const int w = c.heads * c.hd, most = std::min(b.max_rows, b.T);
    const Rows rk = rows_of("kv_read: k", k, ldk, k_off, w, b.T), rv = rows_of("kv_read: v", v, ldv, v_off, w, b.T);
    if (overlap(rk, rv)) throw std::runtime_error("kv_read: k and v overlap");
    if (at.in_cache(rk) || at.in_cache(rv)) throw std::runtime_error("kv_read: the rows overlap the cache");
    if (at.in_batch(rk.place()) || at.in_batch(rv.place())) throw std::runtime_error("kv_read: k or v overlaps the batch's rows, len or table");
    int vec = rk.vec() && rv.vec(), pages = c.pages, heads = c.heads, hd = c.hd, ps = c.ps, bs = c.bs, ldt = b.ld_table, T = b.T, mr = b.max_rows;
    int per = std::max(1, 4096 / w);   // (four values a thread, four times)
    cl_kernel kn = variant("attn", {}, "kv_read");
    set_args(kn, 0, k, ldk, k_off, v, ldv, v_off, c.b[0], c.b[1], c.b[2], c.b[3], pages, heads, hd, ps, bs, b.rows, b.len, b.table, ldt, T, mr, per, vec);
    size_t g[3] = {(size_t)((most + per - 1) / per) * 256, (size_t)b.seqs, 2}, l[3] = {256, 1, 1};
    run("kv_read", kn, 3, g, l);
  }

  // ---- attention
  struct Attn {
    float scale, cap;
    int window;
    cl_mem slopes, prefix, first;
  };
  // Room for the pieces that keys are shared out in, and attn_few's counts of those that are written (zeros between launches).  Made by
  // the first call that needs it, for the most that any call does, so that no longer sequence and no larger batch allocates or
  // waits behind it: where keys are shared out, attn_many has at most 256 rows of pieces a compute unit, attn_few less than four
  // pieces of at most 32 rows a compute unit, for less than two (sequence, head) pairs a compute unit (the rules in attention()); a
  // piece has hd + 2 values a row (256 compute units: 68 MB).  Launch lists name it too: all launches are in one stream's order, so
  // lists and calls that use it do not meet there.
  cl_mem at_ws_ = nullptr, at_counts_ = nullptr;
  void at_room() {
    const size_t cus = arcz_device_cus();
    if (!at_ws_) at_ws_ = buf(256 * cus * (256 + 2) * 4);
    if (at_counts_) return;
    cl_mem m = buf(2 * cus * 4);
    const uint32_t zero = 0;
    if (arcz_fill(m, &zero, 4, 0, 2 * cus * 4) != 0) {
      release(m);
      throw std::runtime_error("attention: the counts are not cleared");
    }
    at_counts_ = m;
  }
  // How attention() takes a batch, by what the host knows of it: rows in tiles of 32 to a wave (few: all of a sequence's in one), its keys in nsplit pieces.
  struct Pieces {
    bool few;
    int waves, tiles, least, nsplit;
  };
  static Pieces pieces_of(const Kv& c, const Batch& b, int heads, const Attn& a) {
    Pieces p = {};
    const int most = std::min(b.max_rows, b.T), window = std::min(a.window, 1 << 30);
    const int64_t M = (int64_t)most * (heads / c.heads);
    const size_t pairs = (size_t)b.seqs * c.heads;
    const int keys = std::max(1, std::min(b.max_len > 0 ? b.max_len : b.ld_table * c.page, window ? (int)std::min<int64_t>((int64_t)most + window, 0x7FFFF000) : 0x7FFFF000));
    p.few = M <= (c.hd == 256 ? 16 : 32);
    if (p.few) {
      // Pieces of one length for all sequences, so that long ones are more work-groups, not longer ones: two work-groups a
      // compute unit if every sequence has the most keys, of at least 256 keys each.
      const size_t want = ((size_t)2 * arcz_device_cus() + pairs - 1) / pairs;
      p.least = (int)std::max<size_t>(8, ((size_t)(keys + 31) / 32 + want - 1) / want);
      p.nsplit = (int)(((int64_t)keys + (int64_t)32 * p.least - 1) / ((int64_t)32 * p.least));
      return p;
    }
    // Heads of 128 values, blocks of 32 tokens and more: work-groups of eight waves and 256 rows, one a compute unit, where rows are many
    // and see thousands of keys; else of four and 128 rows, two of them, which fill the chip sooner and read and write rows while the
    // other computes.  (us, 32 heads over 8, eight waves / four: 1024 rows over 9000 keys 266 / 287, 4096 over 4096 257 / 279, 512 over
    // 8192 139 / 145, 2048 over 16000 854 / 905, 8192 over 9000 1103 / 1158; 512 over 3000 71.2 / 70.8, 3000 over 3000 163 / 154, 2048 over
    // 2048 107 / 99, 512 over 512 43 / 34, ragged documents 74.5 / 62.3.  Two that the rule misses: 1024 over 1024 54 / 55.5, 100 over 4000
    // 44.7 / 46.2.)
    const int seen = std::max(0, (b.max_len > 0 ? b.max_len : b.ld_table * c.page) - most / 2);
    p.waves = c.hd == 128 && c.block >= 32 && M >= 1024 && !a.first && (window ? std::min(window, seen) : seen) >= 2000 ? 8 : 4;
    p.tiles = (int)((M + 32 * p.waves - 1) / (32 * p.waves));
    // rows that fill less than the chip: their keys shared out, at least 256 to a piece
    p.nsplit = (int)std::max<size_t>(1, std::min<size_t>((size_t)8 / p.waves * arcz_device_cus() / (pairs * p.tiles), (size_t)(keys + 255) / 256));
    return p;
  }
  void attention(const Kv& c, const Batch& b, cl_mem q, int ldq, int q_off, int heads, cl_mem out, int ldo, int o_off, const Attn& a) {
    Places at;
    if (!check_batch("attention", c, b, at)) return;
    if (heads < 1 || heads % c.heads || (int64_t)heads * c.hd > 0x7FFFFFFF) throw std::runtime_error("attention: " + std::to_string(heads) + " heads over " + std::to_string(c.heads) + " of the cache");
    if (!std::isfinite(a.scale) || !(a.cap >= 0.0f) || a.cap > 0x1p100f || (a.cap > 0.0f && a.cap < 0x1p-100f) || a.window < 0 || b.max_len < 0)
      throw std::runtime_error("attention: scale, cap, window or max_len");
    const Rows rq = rows_of("attention: q", q, ldq, q_off, heads * c.hd, b.T), ro = rows_of("attention: out", out, ldo, o_off, heads * c.hd, b.T);
    if (overlap(rq, ro)) throw std::runtime_error("attention: q and out overlap");
    if (at.in_cache(ro)) throw std::runtime_error("attention: out overlaps the cache");
    Place slopes, prefix, first;
    if (a.slopes) slopes = ints("attention", "slopes", a.slopes, (size_t)heads);
    if (a.prefix) prefix = ints("attention", "prefix", a.prefix, (size_t)b.seqs);
    if (a.first) first = ints("attention", "first", a.first, (size_t)b.T);
    if (at.in_batch(ro.place()) || overlap(ro.place(), slopes) || overlap(ro.place(), prefix) || overlap(ro.place(), first))
      throw std::runtime_error("attention: out overlaps rows, len, table, slopes, prefix or first");
    const int G = heads / c.heads, most = std::min(b.max_rows, b.T);
    const int64_t M = (int64_t)most * G;
    if (M > 0x7FFFFF00) throw std::runtime_error("attention: too many rows");
    const size_t pairs = (size_t)b.seqs * c.heads;
    int pages = c.pages, ps = c.ps, bs = c.bs, ldt = b.ld_table, T = b.T, mr = most, kvh = c.heads, window = std::min(a.window, 1 << 30);
    float scale = a.scale, cap2 = a.cap * 1.4426950408889634f;
    const int form = (a.cap > 0.0f ? 1 : 0) | (a.slopes ? 2 : 0);
    const Pieces p = pieces_of(c, b, heads, a);
    int nsplit = p.nsplit;
    int vec = rq.vec() ? 1 : 0;
    if (ro.vec()) vec |= 2;
    if (p.few) {
      const int rt = M > 16 ? 2 : 1, pack = M <= 8 ? 1 : 0;
      int least = p.least;
      if (nsplit > 1) at_room();
      cl_mem w = nsplit > 1 ? at_ws_ : nullptr, counts = nsplit > 1 ? at_counts_ : nullptr;
      if (pairs > 0xFFFFFFFFull / 256) throw std::runtime_error("attention: too many sequences");
      vec &= 1;
      cl_kernel k = variant("attn", {{"HD", c.hd}, {"RT", rt}, {"PACK", pack}, {"FINE", c.block < 4 ? 1 : 0}, {"FORM", form}}, "attn_few");
      set_args(k, 0, q, ldq, q_off, c.b[0], c.b[1], c.b[2], c.b[3], pages, ps, bs, b.rows, b.len, b.table, ldt, T, mr, heads, kvh, out, ldo, o_off, scale, cap2, window,
               a.slopes, a.prefix, a.first, w, counts, nsplit, least, vec);
      size_t g[2] = {pairs * 256, (size_t)nsplit}, l[2] = {256, 1};
      run("attention", k, 2, g, l);
      return;
    }
    const int waves = p.waves, bm = 32 * waves;
    int tiles = p.tiles;
    if (pairs * tiles > 0xFFFFFFFFull / (64 * waves)) throw std::runtime_error("attention: too many rows");
    if (nsplit > 1) at_room();
    cl_mem w = nsplit > 1 ? at_ws_ : nullptr;
    cl_kernel k = variant("attn", {{"HD", c.hd}, {"FINE", c.block < 32 ? 1 : 0}, {"FORM", form}, {waves == 8 ? "W8" : nullptr, 1}}, "attn_many");
    set_args(k, 0, q, ldq, q_off, c.b[0], c.b[1], c.b[2], c.b[3], pages, ps, bs, b.rows, b.len, b.table, ldt, T, mr, heads, kvh, out, ldo, o_off, scale, cap2, window,
             a.slopes, a.prefix, a.first, w, nsplit, tiles, vec);
    size_t g[2] = {pairs * tiles * 64 * waves, (size_t)nsplit}, l[2] = {(size_t)64 * waves, 1};
    run("attention", k, 2, g, l);
    if (nsplit > 1) join(c, b, w, nsplit, bm, tiles, mr, heads, out, ldo, o_off);
  }
  // ---- attention for sequences that share a prefix (kernels/attn_shared.hip)
  struct Shared {
    cl_mem groups, len;
    int n, max_rows, max_len;
  };
  // The launches of a call, by what the host knows of it, and where its workspace has what they leave.
  struct SharedShape {
    int G, form, M, M1, waves1, bm1, tiles1, n1, few, rt, pack, tiles2, n2, least, places, per;
    size_t ws1, ws2, bytes;
    bool one;
  };
  SharedShape shared_shape(const Kv& c, const Batch& b, const Shared& sh, int heads, const Attn& a) {
    if (heads < 1 || heads % c.heads || (int64_t)heads * c.hd > 0x7FFFFFFF) throw std::runtime_error("attention_shared: " + std::to_string(heads) + " heads over " + std::to_string(c.heads) + " of the cache");
    if (sh.n < 0 || sh.n > 65535 || sh.max_rows < 0 || sh.max_len < 0 || b.max_len < 0) throw std::runtime_error("attention_shared: " + std::to_string(sh.n) + " groups of " + std::to_string(sh.max_rows) + " rows");
    SharedShape p = {};
    p.G = heads / c.heads;
    p.form = (a.cap > 0.0f ? 1 : 0) | (a.slopes ? 2 : 0);
    const int64_t M = (int64_t)std::min(b.max_rows, b.T) * p.G, M1 = (int64_t)std::min(sh.max_rows, b.T) * p.G;
    if (M > 0x7FFFFF00 || M1 > 0x7FFFFF00) throw std::runtime_error("attention_shared: too many rows");
    p.M = (int)M;
    p.M1 = (int)M1;
    const double rows = (double)std::min<int64_t>(b.T, (int64_t)b.seqs * std::min(b.max_rows, b.T));   // (that the batch may have: its buffers may be for more)
    const size_t cus = (size_t)arcz_device_cus(), pairs = (size_t)b.seqs * c.heads, pairs1 = (size_t)sh.n * c.heads;
    const int all = b.max_len > 0 ? b.max_len : b.ld_table * c.page, shared = sh.max_len > 0 ? std::min(sh.max_len, all) : all, own = std::max(1, sh.max_len > 0 ? all - shared : all);
    // Work-groups of eight waves from 512 rows on (us, with eight / four: 512 rows behind 16384 keys 80 / 83, 4000 behind 6000 150 / 170; 256 rows behind 1024
    // 22 / 18, behind 8192 38 / 37).
    p.waves1 = c.hd == 128 && c.block >= 32 && M1 >= 512 ? 8 : 4;
    p.bm1 = 32 * p.waves1;
    p.tiles1 = (int)((M1 + p.bm1 - 1) / p.bm1);
    const double rate = c.hd == 64 ? 0.8e9 : c.hd == 128 ? 1.0e9 : 0.7e9, key = 2.0 * c.heads * c.hd, mean = rows / std::max(1, b.seqs) * p.G;
    // The group's keys in pieces of at least 128 (us, 4 to 16 sequences of a token behind 512 - 4096 keys, at least 256 / 128 / 64: 28 - 30 / 24 - 28 / 21 - 34): one
    // or the most that one to four work-groups for every compute unit make, whichever takes the least -- rounds of a piece's keys and what a work-group takes
    // beside them (as 128 keys would), and each piece written and read.  (us, pieces 1, 2, 3 ...: 24 of 16 heads of 256 values and up to 90 rows behind 4000
    // 370 354 333 323 335 344; eight of 32 of 128 and up to 120 rows behind 8000 366 229 179 162 215 194.)
    double front = 0.0;
    if (p.tiles1 && pairs1) {
      const double sets = c.heads * std::min((double)sh.n * p.tiles1, std::ceil(rows * p.G / p.bm1) + 0.5 * (sh.n - 1));
      // (max_rows may say more than the groups have: the grid is for what it says)
      const int most = (int)std::max<size_t>(1, std::min<size_t>((size_t)(shared + 127) / 128, 8 * cus / (pairs1 * p.tiles1)));
      for (int r = 0; r <= 4; ++r) {
        const int n = r ? std::min(most, (int)(r * cus / sets)) : 1;
        if (n < 1) continue;
        const double t = std::ceil(sets * n / cus) * p.bm1 * ((double)shared / n + 128.0) * 8.0 * c.hd / rate * cus + rows * heads * n * (c.hd + 2) * 8.0 / 5.0e6;
        if (r && t >= front) continue;
        front = t;
        p.n1 = n;
      }
    }
    // its own: as attention() does
    p.few = M <= (c.hd == 256 ? 16 : 32);
    if (p.few) {
      p.rt = M > 16 ? 2 : 1;
      p.pack = M <= 8 ? 1 : 0;
      p.tiles2 = 1;
      const size_t want = (2 * cus + pairs - 1) / std::max<size_t>(1, pairs);
      p.least = (int)std::max<size_t>(8, ((size_t)(own + 31) / 32 + want - 1) / std::max<size_t>(1, want));
      p.n2 = (int)(((int64_t)own + (int64_t)32 * p.least - 1) / ((int64_t)32 * p.least));
    } else {
      p.tiles2 = (int)((M + 127) / 128);
      p.n2 = (int)std::max<size_t>(1, std::min<size_t>(2 * cus / std::max<size_t>(1, pairs * p.tiles2), (size_t)(own + 255) / 256));
    }
    // What both ways would take (us): attention as it is -- its launch, each sequence's keys of all, of which what they share comes from the caches, or
    // its rows in whole tiles (a third of a round lost to their ends) -- and three launches, the groups' rows in whole tiles, their own keys and the pieces.  Rates as
    // measured: keys 9.5 TB/s shared (sequences of a token behind 1324 - 16984 keys 10 - 445 us), 5 of their own, products in tiles by the head's
    // length.  (us, one launch / three: 16 sequences behind 4096 keys 23 / 28, 32 behind 2048 23 / 28, 64 behind 1024 22 / 31, 64 behind 8192 124 / 51, 128 behind
    // 16384 426 / 105; eight of up to 120 rows behind 8000 250 / 165, 24 of up to 90 behind 4000 225 / 250; of 16 heads of 256 values, 24 of up to 90
    // behind 4000 425 / 351.  Two that the rule misses: eight of up to 200 of those heads behind 2000 187 / 147, four of 250 rows of 32 heads behind 6000 196 / 204.)
    const double last = std::max(1.0, (mean + 64.0) / 128.0);   // (tiles of a sequence, half of the last one empty)
    auto tiles = [&](double keys, int pieces) {   // (heads of 256 values: one work-group a compute unit, so whole rounds)
      const double sets = b.seqs * c.heads * last * pieces / cus, rounds = c.hd == 256 ? std::ceil(sets) : std::max(1.0, sets + 0.3);
      return rounds * cus * 128.0 * (keys / pieces + 128.0) * 8.0 * c.hd / rate;
    };
    const int pieces = (int)std::max<size_t>(1, std::min<size_t>(2 * cus / std::max<size_t>(1, pairs * ((M + 127) / 128)), (size_t)(all + 255) / 256));
    const double one = 8.0 + (p.few ? b.seqs * (double)all * key / 9.5e6 : tiles(all, pieces));
    const double three = 24.0 + front + (p.few ? b.seqs * (double)own * key / 5.0e6 : tiles(own, p.n2)) + rows * heads * p.n2 * (c.hd + 2) * 8.0 / 5.0e6;
    p.one = attn_shared_ < 0 ? one <= three : attn_shared_ == 0;
    if (p.one) {
      p.bytes = 256;
      return p;
    }
    // A piece has a place for each row of the buffers or, where that is less (buffers for more rows than the batch may have), for each of the most
    // rows of every sequence.  (The last launch has a thread for each four values of it.)
    const int mr = std::min(b.max_rows, b.T);
    p.per = (int64_t)b.seqs * mr <= b.T ? mr : 0;
    p.places = p.per ? b.seqs * mr : b.T;
    const size_t each = (size_t)p.places * heads;
    if (pairs * p.tiles2 > 0xFFFFFFFFull / 256 || pairs1 * p.tiles1 > 0xFFFFFFFFull / 512 || each > 0x7FFFFFFF || each * c.hd / 4 > 0xFFFFFF00ull) throw std::runtime_error("attention_shared: too many rows");
    auto place = [&](size_t bytes) {
      const size_t at = p.bytes;
      p.bytes += (bytes + 255) / 256 * 256;
      return at;
    };
    p.ws1 = place(each * p.n1 * (c.hd + 2) * 4);
    p.ws2 = place(each * p.n2 * (c.hd + 2) * 4);
    p.bytes = std::max<size_t>(p.bytes, 256);
    return p;
  }
  int attn_shared_ = -1;   // ARCZ_ATTN_SHARED
  size_t attention_shared_room(const Kv& c, const Batch& b, const Shared& sh, int heads, const Attn& a) {
    Places at;
    if (!check_batch("attention_shared", c, b, at)) return 256;
    const SharedShape p = shared_shape(c, b, sh, heads, a);
    if (p.one && pieces_of(c, b, heads, a).nsplit > 1) at_room();   // (so that no call does)
    return p.bytes;
  }
  void attention_shared(const Kv& c, const Batch& b, const Shared& sh, cl_mem q, int ldq, int q_off, int heads, cl_mem out, int ldo, int o_off, const Attn& a, cl_mem room) {
    Places at;
    if (!check_batch("attention_shared", c, b, at)) return;
    const SharedShape p = shared_shape(c, b, sh, heads, a);
    if (!std::isfinite(a.scale) || !(a.cap >= 0.0f) || a.cap > 0x1p100f || (a.cap > 0.0f && a.cap < 0x1p-100f) || a.window < 0) throw std::runtime_error("attention_shared: scale, cap or window");
    const Rows rq = rows_of("attention_shared: q", q, ldq, q_off, heads * c.hd, b.T), ro = rows_of("attention_shared: out", out, ldo, o_off, heads * c.hd, b.T);
    const char* const name = "attention_shared";
    Place in[5] = {};
    if (a.slopes) in[0] = ints(name, "slopes", a.slopes, (size_t)heads);
    if (a.prefix) in[1] = ints(name, "prefix", a.prefix, (size_t)b.seqs);
    if (a.first) in[2] = ints(name, "first", a.first, (size_t)b.T);
    if (sh.n) {
      in[3] = ints(name, "groups", sh.groups, (size_t)sh.n + 1);
      in[4] = ints(name, "the groups' len", sh.len, (size_t)sh.n);
    }
    const uintptr_t w = (uintptr_t)arcz_mem_ptr(room);
    if (!room || w % 16 || arcz_mem_size(room) < p.bytes)
      throw std::runtime_error("attention_shared: the room holds " + std::to_string(arcz_mem_size(room)) + " bytes, the call takes " + std::to_string(p.bytes) + " (at an address of 16)");
    const Place work = {w, w + p.bytes};
    if (overlap(rq, ro)) throw std::runtime_error("attention_shared: q and out overlap");
    if (at.in_cache(ro) || at.in_batch(ro.place())) throw std::runtime_error("attention_shared: out overlaps the cache or the batch");
    if (at.in_cache(work) || at.in_batch(work) || overlap(work, rq.place()) || overlap(work, ro.place())) throw std::runtime_error("attention_shared: the room overlaps the cache, the batch, q or out");
    for (const Place& i : in)
      if (overlap(ro.place(), i) || overlap(work, i)) throw std::runtime_error("attention_shared: out or the room overlaps slopes, prefix, first or the groups");
    if (p.one) return attention(c, b, q, ldq, q_off, heads, out, ldo, o_off, a);
    int pages = c.pages, ps = c.ps, bs = c.bs, ldt = b.ld_table, T = b.T, mr = std::min(b.max_rows, b.T), kvh = c.heads, window = std::min(a.window, 1 << 30), hd = c.hd, seqs = b.seqs, n = sh.n;
    int mr1 = std::min(sh.max_rows, b.T), vec = rq.vec() ? 1 : 0, n1 = p.n1, n2 = p.n2, t1 = p.tiles1, t2 = p.tiles2, least = p.least, places = p.places, per = p.per;
    float scale = a.scale, cap2 = a.cap * 1.4426950408889634f;
    auto part = [&](const char* name, int front, size_t sets, int rows, int waves, int tiles, int nsplit, size_t ws) {
      cl_kernel k = variant("attn", {{"HD", c.hd}, {"FINE", c.block < 32 ? 1 : 0}, {"FORM", p.form}, {waves == 8 ? "W8" : nullptr, 1}}, "attn_part");
      set_args(k, 0, q, ldq, q_off, c.b[0], c.b[1], c.b[2], c.b[3], pages, ps, bs, b.rows, b.len, b.table, ldt, T, rows, heads, kvh, scale, cap2, window, a.slopes, a.prefix, a.first,
               sh.groups, sh.len, n, seqs, mr, front, places, per, room, ws, nsplit, tiles, vec);
      size_t g[2] = {sets * c.heads * tiles * 64 * waves, (size_t)nsplit}, l[2] = {(size_t)64 * waves, 1};
      run(name, k, 2, g, l);
    };
    if (n1) part("attention_shared", 1, (size_t)n, mr1, p.waves1, t1, n1, p.ws1);
    if (p.few) {
      cl_kernel k = variant("attn", {{"HD", c.hd}, {"RT", p.rt}, {"PACK", p.pack}, {"FINE", c.block < 4 ? 1 : 0}, {"FORM", p.form}}, "attn_part_few");
      set_args(k, 0, q, ldq, q_off, c.b[0], c.b[1], c.b[2], c.b[3], pages, ps, bs, b.rows, b.len, b.table, ldt, T, mr, heads, kvh, scale, cap2, window, a.slopes, a.prefix, a.first,
               sh.groups, sh.len, n, places, per, room, p.ws2, n2, least, vec);
      size_t g[2] = {(size_t)seqs * c.heads * 256, (size_t)n2}, l[2] = {256, 1};
      run("attention_own", k, 2, g, l);
    } else {
      part("attention_own", 0, (size_t)seqs, mr, 4, t2, n2, p.ws2);
    }
    cl_kernel k = variant("attn", {}, "attn_meet");
    set_args(k, 0, room, p.ws1, n1, p.ws2, n2, hd, b.rows, T, mr, heads, sh.groups, sh.len, n, seqs, mr1, places, per, out, ldo, o_off);
    const size_t each = 1024 / c.hd;
    size_t g = ((size_t)places * heads + each - 1) / each * 256, l = 256;
    run("attention_meet", k, 1, &g, &l);
  }
  void join(const Kv& c, const Batch& b, cl_mem w, int nsplit, int rows, int blocks, int mr, int heads, cl_mem out, int ldo, int o_off) {
    int hd = c.hd, most_len = b.ld_table * c.page, T = b.T, kvh = c.heads, per = 1024 / c.hd;
    cl_kernel k = variant("attn", {}, "attn_join");
    set_args(k, 0, w, nsplit, rows, blocks, hd, b.rows, b.len, most_len, T, mr, heads, kvh, out, ldo, o_off);
    size_t g[2] = {(size_t)b.seqs * c.heads * blocks * 256, (size_t)((rows + per - 1) / per)}, l[2] = {256, 1};
    run("attention_join", k, 2, g, l);
  }
