#pragma once
// radx_beam.hpp — beam search beside the sort for C++ hosts: selection over beams and vocabulary, the survivors'
// states moved to their places, the sequences out of the recorded choices.  The reference has no counterpart;
// the class follows its manner (initialize with a device and limits, commands that enqueue on the caller's
// stream) over the radx_hip_beam_* calls of include/radx_hip.h.
//
//   auto beams = std::make_shared<radx::BeamSearch>();
//   beams->initialize(device, batch, beamCount, vocabulary, k);
//   beams->select(cmdBuf, args).reorder(cmdBuf, states, parents, {}, batch, beamCount, beamCount, k);
//   beams->backtrace(cmdBuf, tokens, parents, {}, steps, batch, k, out, steps);
#include <vector>

#include "radx_device.hpp"

namespace radx {

    class BeamSearch : public std::enable_shared_from_this<BeamSearch> {
    protected:
        std::shared_ptr<Device> device{};
        radx_hip_beam* beam = nullptr;

    public:
        BeamSearch() {}
        BeamSearch(const BeamSearch&) = delete;
        BeamSearch& operator=(const BeamSearch&) = delete;
        virtual ~BeamSearch() { (void)radx_hip_beam_destroy(beam); }

        // Limits of the selections to come; the scratch of one of them in flight: calls on several command buffers' streams
        // are put in order by the caller, or get an object each.
        virtual BeamSearch& initialize(const std::shared_ptr<Device>& device, uint32_t maxBatch, uint32_t maxBeams, uint32_t maxVocabulary,
                                       uint32_t maxPlaces) {
            radx_hip_beam* made = nullptr;
            check_abi(radx_hip_beam_create(device->ordinal(), maxBatch, maxBeams, maxVocabulary, maxPlaces, &made));
            (void)radx_hip_beam_destroy(beam);
            beam = made;
            this->device = device;
            return *this;
        }

        virtual BeamSearch& select(const CommandBuffer& cmdBuf, const radx_hip_beam_select_args& args) {
            check_abi(radx_hip_beam_select(beam, &args, cmdBuf.stream));
            return *this;
        }

        // lengths: empty (all positions move) or one per batch item.
        virtual BeamSearch& reorder(const CommandBuffer& cmdBuf, const std::vector<radx_hip_beam_state>& states, const DescriptorBufferInfo& parents,
                                    const DescriptorBufferInfo& lengths, uint32_t batch, uint32_t sourceBeams, uint32_t targetBeams, uint32_t places) {
            require(parents, static_cast<std::size_t>(batch) * places * 4, "BeamSearch::reorder: parents range smaller than batch * places");
            if (lengths.buffer) require(lengths, static_cast<std::size_t>(batch) * 4, "BeamSearch::reorder: lengths range smaller than batch");
            check_abi(radx_hip_beam_reorder(states.data(), static_cast<uint32_t>(states.size()), static_cast<const int32_t*>(parents.address()),
                                            static_cast<const int32_t*>(lengths.address()), batch, sourceBeams, targetBeams, places, cmdBuf.stream));
            return *this;
        }

        // steps: empty (all of them) or one per batch item.
        virtual BeamSearch& backtrace(const CommandBuffer& cmdBuf, const DescriptorBufferInfo& tokens, const DescriptorBufferInfo& parents,
                                      const DescriptorBufferInfo& steps, uint32_t totalSteps, uint32_t batch, uint32_t places,
                                      const DescriptorBufferInfo& out, uint64_t outStride) {
            const std::size_t recorded = static_cast<std::size_t>(totalSteps) * batch * places * 4;
            require(tokens, recorded, "BeamSearch::backtrace: tokens range smaller than steps * batch * places");
            require(parents, recorded, "BeamSearch::backtrace: parents range smaller than steps * batch * places");
            if (steps.buffer) require(steps, static_cast<std::size_t>(batch) * 4, "BeamSearch::backtrace: steps range smaller than batch");
            if (recorded) require(out, ((static_cast<std::size_t>(batch) * places - 1) * outStride + totalSteps) * 4, "BeamSearch::backtrace: out range too small");
            check_abi(radx_hip_beam_backtrace(static_cast<const int32_t*>(tokens.address()), static_cast<const int32_t*>(parents.address()),
                                              static_cast<const int32_t*>(steps.address()), totalSteps, batch, places,
                                              static_cast<int32_t*>(out.address()), outStride, cmdBuf.stream));
            return *this;
        }

    private:
        static void require(const DescriptorBufferInfo& info, std::size_t bytes, const char* what) {
            if (bytes && info.range < bytes) throw Error(static_cast<int>(hipErrorInvalidValue), what);
        }
    };
}
