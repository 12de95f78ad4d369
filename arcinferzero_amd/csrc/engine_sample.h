// A token from each row of logits (kernels/sample.hip).  A part of class Engine (included in it, behind engine_attn.h).

  // Sixteen work-groups a row, in four launches, for few long rows (sample.hip's Place, 108760 bytes of the attention's room, for each).  Measured, us, one
  // work-group a row / sixteen, with a temperature, k = 50 and p, p alone, and rows of all kinds: 16 x 16384 15 21 28 27 / 18 30 35 36;
  // 16 x 32001 20 23 39 36 / 19 29 36 36; 16 x 65536 29 27 59 55 / 19 29 39 37; 32 x 65536 29 28 59 55 / 23 35 54 43; 1 x 151936 54 32 106 54 / 19 27 34 21;
  // 48 x 151936 57 36 119 109 / 37 43 88 56; 96 x 151936 61 40 122 118 / 60 65 152 90.  (Rows whose largest logit is all that is asked for: 13 / 15 and, 48 of
  // them, 14 / 24; a cut by p behind one of 2000 tokens, which one work-group does behind the others' launches: 104 / 116.  What a row asks for is
  // known on the device only; which buffers a call does not give is known here, and the rule does not go by it.)
  int sample_split_ = -1;   // ARCZ_SAMPLE_SPLIT
  static int split_rows() { return std::min(96, 2 * arcz_device_cus()); }   // (the room has 264192 bytes a compute unit)
  bool split_pays(int V, int T) const { return V >= 3000 * std::max(T, 16); }
  struct Sampling {
    cl_mem temperature, top_k, top_p, min_p;
  };
  void sample(cl_mem logits, int ld, int off, int V, int T, const Sampling& f, cl_mem u, cl_mem token, cl_mem prob) {
    // (the sums of weights hold 2^21 of the largest)
    if (V < 1 || V > (1 << 20) || T < 0) throw std::runtime_error("sample: " + std::to_string(T) + " rows of " + std::to_string(V) + " logits (1 to 2^20)");
    if (T == 0) return;
    const char* const name = "sample";
    const Rows x = rows_of("sample: logits", logits, ld, off, V, T);
    const size_t n = (size_t)T;
    const Place out[2] = {ints(name, "token", token, n), prob ? ints(name, "prob", prob, n) : Place()};
    Place in[6] = {x.place(), ints(name, "u", u, n)};
    if (f.temperature) in[2] = ints(name, "temperature", f.temperature, n);
    if (f.top_k) in[3] = ints(name, "top_k", f.top_k, n);
    if (f.top_p) in[4] = ints(name, "top_p", f.top_p, n);
    if (f.min_p) in[5] = ints(name, "min_p", f.min_p, n);
    if (overlap(out[0], out[1])) throw std::runtime_error("sample: token and prob overlap");
    for (const Place& o : out)
      for (const Place& i : in)
        if (overlap(o, i)) throw std::runtime_error("sample: token or prob overlaps what is read");
    if (T <= split_rows() && (sample_split_ < 0 ? split_pays(V, T) : sample_split_)) {
      at_room();
      for (const char* step : {"sample_top", "sample_scan", "sample_cut", "sample_draw"}) {
        cl_kernel k = variant("ops", {}, step);
        set_args(k, 0, logits, ld, off, V, f.temperature, f.top_k, f.top_p, f.min_p, u, token, prob, at_ws_);
        const bool last = step[7] == 'd';
        size_t g[2] = {last ? n * 1024 : 16 * 1024, last ? 1 : n}, l[2] = {1024, 1};
        run(step, k, 2, g, l);
      }
      return;
    }
    cl_kernel k = variant("ops", {}, "sample");
    set_args(k, 0, logits, ld, off, V, f.temperature, f.top_k, f.top_p, f.min_p, u, token, prob);
    size_t g = n * 1024, l = 1024;
    if (n > 0xFFFFFFFFull / 1024) throw std::runtime_error("sample: too many rows");
    run("sample", k, 1, &g, &l);
  }
