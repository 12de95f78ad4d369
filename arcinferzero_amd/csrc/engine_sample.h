// A token from each row of logits (kernels/sample.hip).  A part of class Engine (included in it, behind engine_attn.h).

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
    cl_kernel k = variant("ops", {}, "sample");
    set_args(k, 0, logits, ld, off, V, f.temperature, f.top_k, f.top_p, f.min_p, u, token, prob);
    size_t g = n * 1024, l = 1024;
    if (n > 0xFFFFFFFFull / 1024) throw std::runtime_error("sample: too many rows");
    run("sample", k, 1, &g, &l);
  }
