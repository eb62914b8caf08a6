// beam_test.cpp — a beam search over made-up logits through the C++ layer (include/radx/radx_beam.hpp), checked
// against the same search on the host with whole hypotheses copied from step to step.
//
//   beam_test [--batch B] [--beams N] [--vocab V] [--steps T] [--width W] [--seed S] [--device D]
//
// A step's logits are whole numbers / 8 drawn from the seed, so that the scores (log probabilities are taken as
// given) are exact and every token, score and state has to be equal.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <string>
#include <vector>

#include <radx/radx.hpp>

namespace {

struct Options {
    uint32_t batch = 3, beams = 5, vocab = 20011, steps = 9, width = 77;
    uint64_t seed = 1;
    int device = 0;
};

template <class T>
T* upload(const std::vector<T>& v) {
    void* p = nullptr;
    radx::check_hip(hipMalloc(&p, v.size() * sizeof(T)), "hipMalloc");
    radx::check_hip(hipMemcpy(p, v.data(), v.size() * sizeof(T), hipMemcpyHostToDevice), "hipMemcpy");
    return static_cast<T*>(p);
}
template <class T>
std::vector<T> download(const T* p, size_t n) {
    std::vector<T> v(n);
    radx::check_hip(hipMemcpy(v.data(), p, n * sizeof(T), hipMemcpyDeviceToHost), "hipMemcpy");
    return v;
}

struct Hypothesis {
    float score;
    std::vector<int32_t> tokens;
    std::vector<float> state;
};

int run(const Options& o) {
    const uint32_t rows = o.batch * o.beams;
    auto helper = std::make_shared<radx::PhysicalDeviceHelper>(radx::PhysicalDevice(o.device));
    auto device = std::make_shared<radx::Device>()->initialize(radx::LogicalDevice(o.device), helper);
    auto search = std::make_shared<radx::BeamSearch>();
    search->initialize(device, o.batch, o.beams, o.vocab, o.beams);
    hipStream_t stream = nullptr;
    radx::check_hip(hipStreamCreate(&stream), "hipStreamCreate");

    std::mt19937_64 rng(o.seed);
    std::vector<float> state(static_cast<size_t>(rows) * o.width), cum(rows, -INFINITY);
    for (auto& s : state) s = static_cast<float>(static_cast<int>(rng() % 64)) / 8;
    for (uint32_t b = 0; b < o.batch; ++b) cum[b * o.beams] = 0.f;
    std::vector<std::vector<Hypothesis>> hyps(o.batch);
    for (uint32_t b = 0; b < o.batch; ++b)
        hyps[b].push_back({0.f, {}, std::vector<float>(state.begin() + static_cast<size_t>(b) * o.beams * o.width, state.begin() + (static_cast<size_t>(b) * o.beams + 1) * o.width)});

    float* d_state = upload(state);
    float* d_cum[2] = {upload(cum), upload(cum)};
    int32_t* d_tokens = upload(std::vector<int32_t>(static_cast<size_t>(o.steps) * rows));
    int32_t* d_parents = upload(std::vector<int32_t>(static_cast<size_t>(o.steps) * rows));
    int32_t* d_out = upload(std::vector<int32_t>(static_cast<size_t>(o.steps) * rows));

    for (uint32_t t = 0; t < o.steps; ++t) {
        std::vector<float> logits(static_cast<size_t>(rows) * o.vocab);
        for (auto& x : logits) x = -static_cast<float>(rng() % 4096) / 8;
        float* d_logits = upload(logits);

        radx_hip_beam_select_args args{};
        args.logits = d_logits;
        args.row_stride = o.vocab;
        args.cum = d_cum[t & 1];
        args.scores = d_cum[1 - (t & 1)];
        args.parents = d_parents + static_cast<size_t>(t) * rows;
        args.tokens = d_tokens + static_cast<size_t>(t) * rows;
        args.batch = o.batch;
        args.beams = o.beams;
        args.vocab = o.vocab;
        args.k = o.beams;
        args.dtype = RADX_HIP_F32;
        args.normalize = 0;
        radx_hip_beam_state moved{};
        moved.src = moved.dst = d_state;
        moved.src_row = moved.dst_row = o.width * sizeof(float);
        moved.outer[0] = moved.outer[1] = 1;
        moved.unit_bytes = o.width * sizeof(float);
        moved.units = 1;
        search->select(radx::CommandBuffer(stream), args)
            .reorder(radx::CommandBuffer(stream), {moved}, radx::DescriptorBufferInfo(d_parents, static_cast<size_t>(t) * rows * 4, rows * 4), {}, o.batch,
                     o.beams, o.beams, o.beams);
        radx::check_hip(hipStreamSynchronize(stream), "hipStreamSynchronize");
        radx::check_hip(hipFree(d_logits), "hipFree");

        for (uint32_t b = 0; b < o.batch; ++b) {
            struct Candidate { float score; uint32_t beam, token; };
            std::vector<Candidate> all;
            for (uint32_t i = 0; i < hyps[b].size(); ++i)
                for (uint32_t v = 0; v < o.vocab; ++v)
                    all.push_back({hyps[b][i].score + logits[(static_cast<size_t>(b) * o.beams + i) * o.vocab + v], i, v});
            // equal scores: the lower beam, in it the larger logit (they are equal too), the lower token
            std::stable_sort(all.begin(), all.end(), [](const Candidate& p, const Candidate& q) { return p.score > q.score; });
            std::vector<Hypothesis> next;
            for (uint32_t j = 0; j < o.beams; ++j) {
                Hypothesis h = hyps[b][all[j].beam];
                h.score = all[j].score;
                h.tokens.push_back(static_cast<int32_t>(all[j].token));
                next.push_back(h);
            }
            hyps[b] = next;
        }
    }
    search->backtrace(radx::CommandBuffer(stream), radx::DescriptorBufferInfo(d_tokens, 0, static_cast<size_t>(o.steps) * rows * 4),
                      radx::DescriptorBufferInfo(d_parents, 0, static_cast<size_t>(o.steps) * rows * 4), {}, o.steps, o.batch, o.beams,
                      radx::DescriptorBufferInfo(d_out, 0, static_cast<size_t>(o.steps) * rows * 4), o.steps);
    radx::check_hip(hipStreamSynchronize(stream), "hipStreamSynchronize");

    const auto sequences = download(d_out, static_cast<size_t>(o.steps) * rows);
    const auto scores = download(d_cum[o.steps & 1], rows);
    const auto states = download(d_state, static_cast<size_t>(rows) * o.width);
    uint64_t wrong = 0;
    for (uint32_t b = 0; b < o.batch; ++b)
        for (uint32_t j = 0; j < o.beams; ++j) {
            const Hypothesis& h = hyps[b][j];
            const size_t r = static_cast<size_t>(b) * o.beams + j;
            wrong += scores[r] != h.score;
            wrong += !std::equal(h.tokens.begin(), h.tokens.end(), sequences.begin() + r * o.steps);
            wrong += !std::equal(h.state.begin(), h.state.end(), states.begin() + r * o.width);
        }
    for (void* p : {static_cast<void*>(d_state), static_cast<void*>(d_cum[0]), static_cast<void*>(d_cum[1]), static_cast<void*>(d_tokens),
                    static_cast<void*>(d_parents), static_cast<void*>(d_out)})
        (void)hipFree(p);
    (void)hipStreamDestroy(stream);
    std::printf("Beam search of %u steps, %u x %u beams, %u tokens: %s\n", o.steps, o.batch, o.beams, o.vocab, wrong ? "FAIL" : "PASS");
    return wrong ? 1 : 0;
}

}  // namespace

int main(int argc, char** argv) {
    Options o;
    for (int i = 1; i + 1 < argc; i += 2) {
        const std::string name = argv[i];
        const unsigned long long value = std::strtoull(argv[i + 1], nullptr, 10);
        if (name == "--batch") o.batch = static_cast<uint32_t>(value);
        else if (name == "--beams") o.beams = static_cast<uint32_t>(value);
        else if (name == "--vocab") o.vocab = static_cast<uint32_t>(value);
        else if (name == "--steps") o.steps = static_cast<uint32_t>(value);
        else if (name == "--width") o.width = static_cast<uint32_t>(value);
        else if (name == "--seed") o.seed = value;
        else if (name == "--device") o.device = static_cast<int>(value);
        else { std::fprintf(stderr, "unknown option %s\n", name.c_str()); return 2; }
    }
    if (o.beams > o.vocab) { std::fprintf(stderr, "the first step needs at least as many tokens as beams\n"); return 2; }
    try {
        return run(o);
    } catch (const radx::Error& e) {
        std::fprintf(stderr, "beam_test: %s\n", e.what());
        return 3;
    }
}
