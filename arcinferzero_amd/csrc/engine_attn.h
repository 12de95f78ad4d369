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
    int pages = c.pages, ps = c.ps, bs = c.bs, ldt = b.ld_table, T = b.T, mr = most, kvh = c.heads, window = std::min(a.window, 1 << 30), nsplit = 1;
    float scale = a.scale, cap2 = a.cap * 1.4426950408889634f;
    const int form = (a.cap > 0.0f ? 1 : 0) | (a.slopes ? 2 : 0);
    const int keys = std::max(1, std::min(b.max_len > 0 ? b.max_len : ldt * c.page, window ? (int)std::min<int64_t>((int64_t)most + window, 0x7FFFF000) : 0x7FFFF000));
    int vec = rq.vec() ? 1 : 0;
    if (ro.vec()) vec |= 2;
    if (M <= (c.hd == 256 ? 16 : 32)) {
      const int rt = M > 16 ? 2 : 1, pack = M <= 8 ? 1 : 0;
      // Pieces of one length for all sequences, so that long ones are more work-groups, not longer ones: two work-groups a
      // compute unit if every sequence has the most keys, of at least 256 keys each.
      const size_t want = ((size_t)2 * arcz_device_cus() + pairs - 1) / pairs;
      int least = (int)std::max<size_t>(8, ((size_t)(keys + 31) / 32 + want - 1) / want);
      nsplit = (int)(((int64_t)keys + (int64_t)32 * least - 1) / ((int64_t)32 * least));
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
    // Heads of 128 values, blocks of 32 tokens and more: work-groups of eight waves and 256 rows, one a compute unit, where rows are many
    // and see thousands of keys; else of four and 128 rows, two of them, which fill the chip sooner and read and write rows while the
    // other computes.  (us, 32 heads over 8, eight waves / four: 1024 rows over 9000 keys 266 / 287, 4096 over 4096 257 / 279, 512 over
    // 8192 139 / 145, 2048 over 16000 854 / 905, 8192 over 9000 1103 / 1158; 512 over 3000 71.2 / 70.8, 3000 over 3000 163 / 154, 2048 over
    // 2048 107 / 99, 512 over 512 43 / 34, ragged documents 74.5 / 62.3.  Two that the rule misses: 1024 over 1024 54 / 55.5, 100 over 4000
    // 44.7 / 46.2.)
    const int seen = std::max(0, (b.max_len > 0 ? b.max_len : ldt * c.page) - most / 2);
    const int waves = c.hd == 128 && c.block >= 32 && M >= 1024 && !a.first && (window ? std::min(window, seen) : seen) >= 2000 ? 8 : 4, bm = 32 * waves;
    int tiles = (int)((M + bm - 1) / bm);
    if (pairs * tiles > 0xFFFFFFFFull / (64 * waves)) throw std::runtime_error("attention: too many rows");
    // rows that fill less than the chip: their keys shared out, at least 256 to a piece
    nsplit = (int)std::max<size_t>(1, std::min<size_t>((size_t)8 / waves * arcz_device_cus() / (pairs * tiles), (size_t)(keys + 255) / 256));
    if (nsplit > 1) at_room();
    cl_mem w = nsplit > 1 ? at_ws_ : nullptr;
    cl_kernel k = variant("attn", {{"HD", c.hd}, {"FINE", c.block < 32 ? 1 : 0}, {"FORM", form}, {waves == 8 ? "W8" : nullptr, 1}}, "attn_many");
    set_args(k, 0, q, ldq, q_off, c.b[0], c.b[1], c.b[2], c.b[3], pages, ps, bs, b.rows, b.len, b.table, ldt, T, mr, heads, kvh, out, ldo, o_off, scale, cap2, window,
             a.slopes, a.prefix, a.first, w, nsplit, tiles, vec);
    size_t g[2] = {pairs * tiles * 64 * waves, (size_t)nsplit}, l[2] = {(size_t)64 * waves, 1};
    run("attention", k, 2, g, l);
    if (nsplit > 1) join(c, b, w, nsplit, bm, tiles, mr, heads, out, ldo, o_off);
  }
  void join(const Kv& c, const Batch& b, cl_mem w, int nsplit, int rows, int blocks, int mr, int heads, cl_mem out, int ldo, int o_off) {
    int hd = c.hd, most_len = b.ld_table * c.page, T = b.T, kvh = c.heads, per = 1024 / c.hd;
    cl_kernel k = variant("attn", {}, "attn_join");
    set_args(k, 0, w, nsplit, rows, blocks, hd, b.rows, b.len, most_len, T, mr, heads, kvh, out, ldo, o_off);
    size_t g[2] = {(size_t)b.seqs * c.heads * blocks * 256, (size_t)((rows + per - 1) / per)}, l[2] = {256, 1};
    run("attention_join", k, 2, g, l);
  }
