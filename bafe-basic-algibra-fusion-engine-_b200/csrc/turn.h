// turn.h -- one run after the other on a device, whatever streams they are on.
#pragma once

namespace bafe_cuda {

// A run that needs the turn begins by waiting, on its stream, for the end of
// the last one and ends by recording its own.  Inside a graph capture nothing
// is ordered (a captured run's order is its graph's).
//   Api: Stream; Event (null: none); int capturing(Stream, bool&), wait(Stream, Event),
//        make(Event&), record(Event, Stream): 0, or an error code that they reported.
template <class Api>
class Turn {
public:
    Turn(Api api, typename Api::Event& last, typename Api::Stream stream) : api_(api), last_(last), stream_(stream) {}

    // Nothing may be enqueued where this fails: its order would be lost.
    int begin(bool needed) {
        bool captured = false;
        if (!needed) return 0;
        if (int rc = api_.capturing(stream_, captured)) return rc;
        if (captured) return 0;
        if (!last_)
            if (int rc = api_.make(last_)) return rc;
        if (int rc = api_.wait(stream_, last_)) return rc;       // one that nothing recorded yet is no wait
        mine_ = true;
        return 0;
    }
    // rc: what the run itself came to.  What it enqueued before it failed has to
    // be waited for as well.
    int end(int rc) {
        if (!mine_) return rc;
        mine_ = false;
        const int recorded = api_.record(last_, stream_);
        return rc ? rc : recorded;
    }

private:
    Api api_;
    typename Api::Event& last_;
    typename Api::Stream stream_;
    bool mine_ = false;
};

}  // namespace bafe_cuda
