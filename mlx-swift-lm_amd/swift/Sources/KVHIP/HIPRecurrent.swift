// A gated delta layer's state, and beam search over caches.
import CKVHIP
import Foundation

/// What hybrid models keep in a `MambaCache` (KVCache.swift:1307-1726) beside the KV caches of their attention layers: the short
/// convolution's window [B, W - 1, C] and the delta rule's state [B, Hv, Dv, Dk] in float32.  Not trimmable: keep the old arrays.
public final class HIPGatedDeltaCache<A: HIPArray> {
    public var window: A?, deltaState: A?
    public private(set) var offset = 0
    public var stream: UnsafeMutableRawPointer? = nil  // hipStream_t of the owning generation loop

    public init() {}
    public var isTrimmable: Bool { false }
    @discardableResult public func trim(_ n: Int) -> Int { 0 }

    /// The short convolution of x [B, L, C] with weight [C, W] behind the window, which moves on.
    public func convolve(_ x: A, weight: A, bias: A? = nil, silu: Bool = true, leftPad: UnsafePointer<Int32>? = nil,
                         lengths: UnsafePointer<Int32>? = nil) -> A {
        let s = x.shape, t = x.kvhipDType
        must(s.count == 3 && weight.shape.count == 2 && weight.shape[0] == s[2] && weight.shape[1] > 0 && weight.kvhipDType == t,
             "weight \(weight.shape) does not go with x \(s)")
        let w = weight.shape[1]
        if let bias = bias { must(bias.shape == [s[2]] && bias.kvhipDType == t, "bias \(bias.shape) does not go with x \(s)") }
        if let window = window { must(window.shape == [s[0], w - 1, s[2]] && window.kvhipDType == t, "x \(s) does not go with the window \(window.shape)") }
        let out = A.empty(s, dtype: t)
        let new = window ?? A.empty([s[0], w - 1, s[2]], dtype: t)
        must(kvhip_short_convolution(x.devicePointer, Int64(s[1] * s[2]), Int64(s[2]), weight.devicePointer, bias?.devicePointer, Int32(s[0]),
                                     Int32(s[1]), Int32(s[2]), Int32(w), t, silu ? 1 : 0, leftPad, lengths,
                                     window?.devicePointer, new.devicePointer, out.devicePointer, stream))
        window = new
        return out
    }

    /// Heads that lie in an array [B, L, ...] of `row` elements a token, from element `first` of a token on.
    private struct Part {
        var array: A, first: Int, row: Int
        var pointer: UnsafeRawPointer {
            UnsafeRawPointer(array.devicePointer).advanced(by: first * (array.kvhipDType == Int32(KVHIP_F32.rawValue) ? 4 : 2))
        }
    }

    /// `gatedDeltaUpdate` (GatedDelta.swift:112): q, k [B, L, Hk, Dk], v [B, L, Hv, Dv], a, b [B, L, Hv]; aLog and dtBias [Hv] in float32.
    public func update(q: A, k: A, v: A, a: A, b: A, aLog: A, dtBias: A, scale: Float? = nil, normEps: Float = 1e-6,
                       leftPad: UnsafePointer<Int32>? = nil, lengths: UnsafePointer<Int32>? = nil) -> A {
        let sk = k.shape, sv = v.shape
        must(q.shape.count == 4 && q.shape == sk && sv.count == 4 && Array(sk[0 ..< 2]) == Array(sv[0 ..< 2]),
             "queries \(q.shape), keys \(sk) and values \(sv) do not go together")
        must(q.kvhipDType == v.kvhipDType && k.kvhipDType == v.kvhipDType, "queries, keys and values are of different types")
        return update(q: Part(array: q, first: 0, row: sk[2] * sk[3]), k: Part(array: k, first: 0, row: sk[2] * sk[3]),
                      v: Part(array: v, first: 0, row: sv[2] * sv[3]), size: [sv[0], sv[1], sk[2], sv[2], sk[3], sv[3]], a: a, b: b, aLog: aLog,
                      dtBias: dtBias, scale: scale, normEps: normEps, leftPad: leftPad, lengths: lengths)
    }

    /// The same for what the convolution hands on, mixed [B, L, 2 Hk Dk + Hv Dv]: queries, keys and values side by side, taken from there.
    public func update(mixed: A, keyHeads: Int, keyDim: Int, valueHeads: Int, valueDim: Int, a: A, b: A, aLog: A, dtBias: A, scale: Float? = nil,
                       normEps: Float = 1e-6, leftPad: UnsafePointer<Int32>? = nil, lengths: UnsafePointer<Int32>? = nil) -> A {
        let s = mixed.shape, keys = keyHeads * keyDim, row = 2 * keys + valueHeads * valueDim
        must(s.count == 3 && s[2] == row, "\(s) does not hold \(keyHeads) x \(keyDim) queries and keys and \(valueHeads) x \(valueDim) values")
        return update(q: Part(array: mixed, first: 0, row: row), k: Part(array: mixed, first: keys, row: row),
                      v: Part(array: mixed, first: 2 * keys, row: row), size: [s[0], s[1], keyHeads, valueHeads, keyDim, valueDim], a: a, b: b,
                      aLog: aLog, dtBias: dtBias, scale: scale, normEps: normEps, leftPad: leftPad, lengths: lengths)
    }

    private func update(q: Part, k: Part, v: Part, size: [Int], a: A, b: A, aLog: A, dtBias: A, scale: Float?, normEps: Float,
                        leftPad: UnsafePointer<Int32>?, lengths: UnsafePointer<Int32>?) -> A {
        let f32 = Int32(KVHIP_F32.rawValue)
        let (B, L, Hk, Hv, Dk, Dv) = (size[0], size[1], size[2], size[3], size[4], size[5])
        must(a.shape == [B, L, Hv] && b.shape == [B, L, Hv] && a.kvhipDType == b.kvhipDType, "a \(a.shape) and b \(b.shape) are [B, L, Hv] of one type")
        must(aLog.shape == [Hv] && dtBias.shape == [Hv] && aLog.kvhipDType == f32 && dtBias.kvhipDType == f32, "aLog and dtBias are float32 [Hv]")
        if let deltaState = deltaState {
            must(deltaState.shape == [B, Hv, Dv, Dk] && deltaState.kvhipDType == f32, "the state \(deltaState.shape) is not float32 \([B, Hv, Dv, Dk])")
        }
        let out = A.empty([B, L, Hv, Dv], dtype: v.array.kvhipDType)
        let new = deltaState ?? A.empty([B, Hv, Dv, Dk], dtype: f32)
        var x = kvhip_gated_delta_args()
        (x.q, x.k, x.v) = (q.pointer, k.pointer, v.pointer)
        (x.a, x.b) = (UnsafeRawPointer(a.devicePointer), UnsafeRawPointer(b.devicePointer))
        (x.q_stride_b, x.q_stride_l) = (Int64(L * q.row), Int64(q.row))
        (x.k_stride_b, x.k_stride_l) = (Int64(L * k.row), Int64(k.row))
        (x.v_stride_b, x.v_stride_l) = (Int64(L * v.row), Int64(v.row))
        (x.a_stride_b, x.a_stride_l) = (Int64(L * Hv), Int64(Hv))
        (x.b_stride_b, x.b_stride_l) = (x.a_stride_b, x.a_stride_l)
        x.a_log = UnsafePointer(aLog.devicePointer.assumingMemoryBound(to: Float.self))
        x.dt_bias = UnsafePointer(dtBias.devicePointer.assumingMemoryBound(to: Float.self))
        (x.left_pad, x.lengths) = (leftPad, lengths)
        x.state_in = deltaState.map { UnsafePointer($0.devicePointer.assumingMemoryBound(to: Float.self)) }
        x.state_out = new.devicePointer.assumingMemoryBound(to: Float.self)
        x.out = out.devicePointer
        (x.B, x.L, x.Hk, x.Hv, x.Dk, x.Dv) = (Int32(B), Int32(L), Int32(Hk), Int32(Hv), Int32(Dk), Int32(Dv))
        (x.dtype, x.gate_dtype) = (v.array.kvhipDType, a.kvhipDType)
        (x.scale, x.norm_eps) = (scale ?? pow(Float(Dk), -0.5), normEps)
        let need = kvhip_gated_delta_workspace(&x)
        let scratch = need > 0 ? A.empty([(need + 3) / 4], dtype: f32) : nil
        must(kvhip_gated_delta(&x, scratch?.devicePointer, need, stream))
        deltaState = new
        offset += L
        return out
    }

    /// Sequence b becomes what sequence order[b] was.  `order`: one row number to each sequence, on the device.
    public func reorder(order: UnsafePointer<Int32>) {
        let held = [window, deltaState].compactMap { $0 }.filter { $0.shape.allSatisfy { $0 > 0 } }
        guard let rows = held.first?.shape[0] else { return }
        must(held.allSatisfy { $0.shape[0] == rows }, "window and state hold different numbers of sequences")
        var at: [UnsafeMutableRawPointer?] = held.map { $0.devicePointer }
        var bytes = held.map { a in a.shape.dropFirst().reduce(1, *) * (a.kvhipDType == Int32(KVHIP_F32.rawValue) ? 4 : 2) }
        must(kvhip_reorder_rows(Int32(held.count), &at, &bytes, Int32(rows), order, stream))
    }
}

/// Arrays that do not go together: a programmer's error, as `must` of a status is.
@inline(__always) private func must(_ fits: Bool, _ message: @autoclosure () -> String) {
    if !fits { fatalError(message()) }
}

extension HIPKVCache {
    /// Sequence b of the batch becomes what sequence order[b] was (`beamSelect`'s rows, on the device); the first `shared` positions
    /// are known to be the same.
    public func reorder(order: UnsafePointer<Int32>, shared: Int = 0) {
        must(kvhip_cache_reorder(handle, order, Int64(shared), stream))
    }
}

/// The `count` best continuations of each batch row's beams, logits [B, K, V] and scores [B, K] (float32): best first, into device arrays
/// [B, count]; `done` holds B K bytes; `rows` is an order for every cache's `reorder` when count is K.
public func beamSelect<A: HIPArray>(logits: A, scores: A?, count: Int, rows: UnsafeMutablePointer<Int32>, tokens: UnsafeMutablePointer<Int32>,
                                    best: UnsafeMutablePointer<Float>, done: UnsafePointer<UInt8>? = nil, padToken: Int = 0,
                                    stream: UnsafeMutableRawPointer? = nil) throws {
    let s = logits.shape
    let fits = s.count == 3 && (scores.map { $0.shape == [s[0], s[1]] && $0.kvhipDType == Int32(KVHIP_F32.rawValue) } ?? true)
    if !fits {
        throw KVHIPError(status: -2, description: "logits \(s) are not [B, K, V] or scores not float32 [B, K]")  // (KVHIP_ERR_INVALID_ARG)
    }
    let need = kvhip_beam_select_workspace(Int32(s[0]), Int32(s[1]), Int32(s[2]), logits.kvhipDType, Int32(count))
    let scratch = A.empty([max((need + 3) / 4, 1)], dtype: Int32(KVHIP_F32.rawValue))
    try check(kvhip_beam_select(logits.devicePointer, Int64(s[2]), Int32(s[0]), Int32(s[1]), Int32(s[2]), logits.kvhipDType,
                                scores.map { UnsafePointer($0.devicePointer.assumingMemoryBound(to: Float.self)) }, done, Int32(count),
                                Int32(padToken), rows, tokens, best, scratch.devicePointer, need, stream))
}
